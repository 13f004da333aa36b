"""4-bit operators without a GPU: weight quantisation, allocation, and the calls that are refused
(by the Python entry points and by the C entry points, which check sizes before they touch CUDA)."""
import pytest
import torch

from hexgen2_b200 import _lib, ops
from hexgen2_b200.checkpoint import dequantize_weight_q4, quantize_weight_q4


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (5, 192, 64), (16, 256, 128)])
def test_quantize_weight(dtype, n, k, group):
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(n + k)).to(dtype)
    w[0, :group] = 0  # an empty group
    codes, scales = quantize_weight_q4(w, group)
    assert codes.shape == (n, k // 2) and codes.dtype == torch.uint8 and codes.is_contiguous()
    assert scales.shape == (n, k // group) and scales.dtype == dtype
    back = dequantize_weight_q4(codes, scales)
    # Half a step from the value, plus what rounding the scale to dtype moves seven steps by.
    step = scales.double().repeat_interleave(group, 1)
    slack = step * (0.5 + 7 * torch.finfo(dtype).eps / 2 + 1e-6)
    assert ((back.double() - w.double()).abs() <= slack).all()
    assert not back[0, :group].any()
    # The low nibble of byte j is element 2j.
    assert back[-1, 2].item() == pytest.approx(((codes[-1, 1] & 15).item() - 8) * scales[-1, 0].item())


@pytest.mark.parametrize("shape,group", [((4, 100), 32), ((4, 128), 16), ((128,), 32)])
def test_quantize_weight_refuses(shape, group):
    with pytest.raises(ValueError):
        quantize_weight_q4(torch.zeros(shape), group)


def q4(b=2, hk=2, s=8, d=32):
    return ops.allocate_cache_q4(b, hk, s, d, device="cpu")


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_allocate():
    assert q4(3, 2, 8, 64).shape == (3, 2, 8, 80) and q4().dtype == torch.uint8


@pytest.mark.parametrize("call", [
    lambda c: ops.quantize_cache_q4(c, i32(1, 1), q4()),
    lambda c: ops.dequantize_cache_q4(q4(), i32(1, 1), c),
    lambda c: ops.rotary_cache_write_q4(torch.zeros(2, 6 * 32), 2, 1, 2, 2, 32, i32(0, 0),
                                        torch.zeros(8, 16), torch.zeros(8, 16), q4()),
    lambda c: ops.decode_attention_q4(torch.zeros(2, 4, 32), q4(), i32(1, 1), 2, 8, 1.0),
    lambda c: ops.gemm_q4(torch.zeros(2, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2)),
    lambda c: ops.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.long)),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(ValueError, match="CUDA"):
        call(torch.zeros(2, 8, 2, 2, 32))


@pytest.mark.parametrize("call,match", [
    (lambda c: ops.quantize_cache_q4(c[:, :, :1], i32(1, 1), q4()), "cache must be"),
    (lambda c: ops.quantize_cache_q4(c.transpose(3, 4), i32(1, 1), q4()), "contiguous"),
    (lambda c: ops.quantize_cache_q4(c, i32(1), q4()), "counts"),
    (lambda c: ops.quantize_cache_q4(c, i32(1, 1).long(), q4()), "counts"),
    (lambda c: ops.quantize_cache_q4(c, i32(1, 1), q4(), starts=i32(0)), "starts"),
    (lambda c: ops.quantize_cache_q4(c, i32(1, 1), q4(hk=4)), "KV heads"),
    (lambda c: ops.quantize_cache_q4(c, i32(1, 1), q4(d=64)), "KV heads"),
    (lambda c: ops.quantize_cache_q4(c, i32(1, 1), q4().float()), "uint8"),
    (lambda c: ops.quantize_cache_q4(c, i32(1, 1), q4(), batch_offset=1), "sequences"),
    (lambda c: ops.quantize_cache_q4(c, i32(1, 1), q4(s=16)[:, :, ::2]), "contiguous"),
    (lambda c: ops.quantize_cache_q4(c, i32(1, 1), q4(b=1).expand(2, -1, -1, -1)), "share"),
    (lambda c: ops.dequantize_cache_q4(q4(), i32(1, 1), c[:1].expand(2, -1, -1, -1, -1)), "share"),
    (lambda c: ops.dequantize_cache_q4(q4(), i32(1, 1), c, batch_offset=-1), "sequences"),
    (lambda c: ops.rotary_cache_write_q4(torch.zeros(2, 5 * 32), 2, 1, 2, 2, 32, i32(0, 0),
                                         torch.zeros(8, 16), torch.zeros(8, 16), q4()), "qkv"),
    (lambda c: ops.rotary_cache_write_q4(torch.zeros(2, 6 * 32), 2, 1, 2, 2, 32, i32(0, 0),
                                         torch.zeros(8, 32), torch.zeros(8, 32), q4()), "cos and sin"),
    (lambda c: ops.rotary_cache_write_q4(torch.zeros(2, 6 * 32), 2, 1, 2, 2, 32, i32(0, 0),
                                         torch.zeros(8, 16).half(), torch.zeros(8, 16).half(), q4()), "cos and sin"),
    (lambda c: ops.decode_attention_q4(torch.zeros(2, 4, 64)[:, :, ::2], q4(), i32(1, 1), 2, 8, 1.0), "contiguous"),
    (lambda c: ops.decode_attention_q4(torch.zeros(2, 4, 32), q4(), i32(1, 1), 2, 9, 1.0), "max_seqlen"),
    (lambda c: ops.decode_attention_q4(torch.zeros(3, 4, 32), q4(), i32(1, 1, 1), 2, 8, 1.0), "sequences"),
    (lambda c: ops.gemm_q4(torch.zeros(2, 64), torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1)), "w_q4"),
    (lambda c: ops.gemm_q4(torch.zeros(2, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2).half()), "scales"),
    (lambda c: ops.gemm_q4(torch.zeros(2, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 3)), "scales"),
    (lambda c: ops.gemm_q4(torch.zeros(2, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2),
                           ops.HX_EPI_RESIDUAL), "residual"),
    (lambda c: ops.gemm_q4(torch.zeros(2, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2),
                           residual=torch.zeros(2, 4)), "residual"),
    (lambda c: ops.gemm_q4(torch.zeros(2, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2),
                           out=torch.zeros(4).expand(2, 4)), "share"),
    (lambda c: ops.token_logprobs(torch.zeros(2, 8), torch.zeros(3, dtype=torch.long)), "tokens"),
    (lambda c: ops.token_logprobs(torch.zeros(8, 2).t(), torch.zeros(2, dtype=torch.long)), "contiguous"),
    (lambda c: ops.token_logprobs(torch.zeros(2, 8)), "nothing"),
])
def test_bad_arguments_are_refused(call, match):
    with pytest.raises(ValueError, match=match):
        call(torch.zeros(2, 8, 2, 2, 32))


@pytest.mark.parametrize("shape", [(16,), (1, 16), (1, 8, 16), (8, 1, 16), (8, 2, 8)])
def test_rotary_tables_have_a_row_for_each_position(shape):
    """Tables of another rank are refused: the kernel takes the first size for the number of rows (16 rows of 16 in a
    table of 16 values would be read past its end). One row is a table of one position."""
    def call():
        t = torch.zeros(shape)
        ops.rotary_cache_write_q4(torch.zeros(2, 6 * 32), 2, 1, 2, 2, 32, i32(0, 0), t, t, q4())
    with pytest.raises(ValueError, match="CUDA" if shape == (1, 16) else "cos and sin"):
        call()


P = 1 << 20  # an aligned address that is never followed: every call below fails its checks first


@pytest.mark.parametrize("name,args", [
    ("hx_quantize_cache_q4", [P, 64, 64, 8, None, None, 1, 1, 32, P, 384, 384, 0, 8, 0, None]),  # no counts
    ("hx_quantize_cache_q4", [P, 64, 64, 8, None, P, 1, 1, 48, P, 512, 512, 0, 8, 0, None]),  # head_dim
    ("hx_quantize_cache_q4", [P, 64, 64, 8, None, P, 1, 1, 32, P + 8, 384, 384, 0, 8, 0, None]),  # alignment
    ("hx_quantize_cache_q4", [P, 64, 64, 8, None, P, 1, 1, 32, P, 384, 368, 0, 8, 0, None]),  # head stride
    ("hx_quantize_cache_q4", [P + 4, 64, 64, 8, None, P, 1, 1, 32, P, 384, 384, 0, 8, 0, None]),  # row alignment
    ("hx_quantize_cache_q4", [P, 64, 32, 8, None, P, 1, 1, 32, P, 384, 384, 0, 8, 0, None]),  # row stride
    ("hx_quantize_cache_q4", [P, 64, 64, 8, None, P, 65536, 1, 32, P, 384, 384, 0, 8, 0, None]),  # batch
    ("hx_dequantize_cache_q4", [P, 384, 384, 0, 8, None, P, 1, 1, 32, P, 64, 40, 8, 0, None]),
    ("hx_dequantize_cache_q4", [P, 380, 384, 0, 8, None, P, 1, 1, 32, P, 64, 64, 8, 0, None]),
    ("hx_rotary_cache_write_q4", [P, 1, 1, 3, 2, 32, P, P, P, 8, 1, P, P, 768, 384, 0, 8, 0, None]),  # grouping
    ("hx_rotary_cache_write_q4", [P + 2, 1, 1, 2, 2, 32, P, P, P, 8, 1, P, P, 768, 384, 0, 8, 1, None]),
    ("hx_rotary_cache_write_q4", [P, 1, 1, 2, 2, 32, P, P, P, 8, 1, P, P, 768, 384, 0, 0, 1, None]),  # empty cache
    ("hx_decode_attention_q4", [P, 64, P, 384, 384, P, 1, 3, 2, 32, 8, 1.0, P, None, 0, 0, None]),
    ("hx_decode_attention_q4", [P, 64, P, 384, 384, P, 1, 2, 1, 40, 8, 1.0, P, None, 0, 0, None]),
    ("hx_decode_attention_q4", [P, 64, P, 384, 384, P, 1, 2, 1, 32, 9, 1.0, P, None, 0, 0, None]),  # beyond
    ("hx_decode_attention_q4", [P, 64, P, 1 << 24, 1 << 24, P, 1, 2, 1, 32, 100000, 1.0, P, P, 16, 0, None]),
    ("hx_gemm_q4", [P, P, P, P, 65, 32, 64, 32, 64, 32, 0, None, 0, P, 1 << 30, 0, None]),  # rows
    ("hx_gemm_q4", [P, P, P, P, 1, 32, 96, 64, 96, 32, 0, None, 0, P, 1 << 30, 0, None]),  # k % group
    ("hx_gemm_q4", [P, P, P, P, 1, 32, 64, 16, 64, 32, 0, None, 0, P, 1 << 30, 0, None]),  # group
    ("hx_gemm_q4", [P, P, P, P, 1, 48, 64, 32, 64, 48, 2, None, 0, P, 1 << 30, 0, None]),  # SwiGLU n
    ("hx_gemm_q4", [P, P, P, P, 1, 32, 64, 32, 64, 32, 1, None, 0, P, 1 << 30, 0, None]),  # no residual
    ("hx_gemm_q4", [P, P, P, P, 1, 32, 64, 32, 64, 32, 3, P, 32, P, 1 << 30, 0, None]),  # epilogue
    ("hx_gemm_q4", [P, P, P, P, 2, 32, 64, 32, 66, 32, 0, None, 0, P, 1 << 30, 1, None]),  # lda
    ("hx_gemm_q4", [P, P, P, P, 2, 32, 64, 32, 64, 31, 0, None, 0, P, 1 << 30, 1, None]),  # ldc
    ("hx_gemm_q4", [P + 4, P, P, P, 1, 32, 64, 32, 64, 32, 0, None, 0, P, 1 << 30, 0, None]),
    ("hx_gemm_q4", [P, P, P, P, 9, 32, 4224, 32, 4224, 32, 0, None, 0, P, 16, 1, None]),  # workspace
    ("hx_gemm_q4", [P, P, P, P, 9, 32, 4224, 32, 4224, 32, 0, None, 0, P + 8, 1 << 30, 1, None]),
    ("hx_token_logprobs", [P, 2, 8, 7, P, 0, P, None, None, None, 0, None]),  # ld
    ("hx_token_logprobs", [P, 2, 8, 8, P, 9, P, None, P, P, 0, None]),  # top_k > cols
    ("hx_token_logprobs", [P, 2, 80, 80, P, 33, P, None, P, P, 0, None]),  # top_k > 32
    ("hx_token_logprobs", [P, 2, 8, 8, P, 2, P, None, None, P, 0, None]),
    ("hx_token_logprobs", [P, 2, 8, 8, None, 0, P, None, None, None, 0, None]),  # no tokens
])
def test_c_entry_points_refuse(name, args):
    lib = _lib.lib()
    assert getattr(lib, name)(*args) == _lib.HX_ERR_INVALID
    assert name in lib.hx_last_error().decode()


def test_unsupported_dtype_and_empty_calls():
    lib = _lib.lib()
    assert lib.hx_gemm_q4(P, P, P, P, 1, 32, 64, 32, 64, 32, 0, None, 0, P, 1 << 30, 7, None) == _lib.HX_ERR_UNSUPPORTED
    assert lib.hx_gemm_q4(P, P, P, P, 0, 32, 64, 32, 64, 32, 0, None, 0, P, 1 << 30, 0, None) == _lib.HX_OK
    assert lib.hx_token_logprobs(P, 0, 8, 8, P, 0, P, None, None, None, 0, None) == _lib.HX_OK
    assert lib.hx_quantize_cache_q4(P, 64, 64, 8, None, P, 0, 1, 32, P, 384, 384, 0, 8, 0, None) == _lib.HX_OK


def test_attention_workspace_covers_the_partials():
    """The query needs no GPU; one short sequence per KV head needs no more than its own splits."""
    w = ops.decode_q4_workspace_bytes
    assert w(0, 8, 2, 128, 100) == 0 and w(1, 8, 2, 128, 0) == 0
    assert w(1, 8, 1, 128, 100000) > 0
    assert w(1, 8, 1, 128, 100000) % 4 == 0


@pytest.mark.parametrize("m,n,k,dtype,launches", [
    (1, 32000, 4096, _lib.HX_BF16, 1), (16, 32000, 4096, _lib.HX_BF16, 1), (17, 32000, 4096, _lib.HX_BF16, 3),
    (32, 4096, 4096, _lib.HX_F16, 3), (32, 4095, 4096, _lib.HX_F16, 1), (40, 40, 8448, _lib.HX_BF16, 1),
    (64, 32000, 4096, _lib.HX_F32, 1), (0, 32000, 4096, _lib.HX_BF16, 0)])
def test_gemm_q4_launches(m, n, k, dtype, launches):
    """One kernel, or three on tcgen05 (2^29 products of more than 16 rows); running sums alone, which need a
    workspace too, do not make it three."""
    assert _lib.lib().hx_gemm_q4_launches(m, n, k, dtype) == launches
