"""Torch-facing wrappers over the C ABI: one function per kernel entry point.

Tensors are passed as raw device pointers plus sizes/strides; every launch goes on torch's
current CUDA stream. Scratch space (split-K partials, decode split partials) comes from a
per-device buffer that grows on demand and is reused across calls on the same stream; the
4-bit operators take a buffer of their own for every call, so that calls on several streams and
captured graphs never share one.
"""
from __future__ import annotations

from collections import namedtuple

import torch

from . import _lib
from ._lib import HX_EPI_NONE, HX_EPI_RESIDUAL, HX_EPI_SWIGLU, check  # noqa: F401

DTYPE_CODE = {torch.float32: _lib.HX_F32, torch.float16: _lib.HX_F16, torch.bfloat16: _lib.HX_BF16}


def _L():
    return _lib.lib()


def _code(t: torch.Tensor) -> int:
    try:
        return DTYPE_CODE[t.dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {t.dtype}") from None


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _p(t):
    return None if t is None else t.data_ptr()


def _require_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("hexgen2_b200 kernels take CUDA tensors (there is no CPU path)")


_workspaces: dict[int, torch.Tensor] = {}

# Number of kernels launched through this module (bench.py reports it as gpu_launches; a CUDA
# graph replay adds the launches it captured).
LAUNCHES = 0
# Bumped whenever a scratch buffer is reallocated: CUDA graphs that captured the old address
# must not be replayed.
WORKSPACE_GEN = 0


def _count(launches=1):
    global LAUNCHES
    LAUNCHES += launches


def workspace(nbytes: int, device=None, kind: str = "attn") -> torch.Tensor | None:
    """Per-device scratch buffer of at least nbytes (None for 0), one per kind, reused across
    calls on the same stream (GEMM split-K partials, decode-attention split partials)."""
    if nbytes == 0:
        return None
    dev = torch.cuda.current_device() if device is None else torch.device(device).index
    key = (dev, kind)
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        global WORKSPACE_GEN
        size = max(nbytes, 0 if buf is None else buf.numel() * 2)
        buf = torch.empty(size, dtype=torch.uint8, device=f"cuda:{dev}")
        _workspaces[key] = buf
        WORKSPACE_GEN += 1
    return buf


def _device_of(first, *others) -> int:
    """The one CUDA device that all of the given tensors are on."""
    dev = first.get_device()  # -1 on the CPU
    for t in others:
        if t is not None and t.get_device() != dev:
            if dev >= 0 and t.is_cuda:
                raise ValueError("all tensors of a call must be on the same device")
            dev = -1
    if dev < 0:
        raise ValueError("hexgen2_b200 kernels take CUDA tensors (there is no CPU path)")
    return dev


# The current stream of a device as an address, without making a Stream object (3 us of a call that takes
# 10); and the device made current for a call whose tensors are elsewhere.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _call(dev: int, fn, *args):
    """Calls a C entry point with the current stream of device `dev`, whichever device is current."""
    if dev == torch.cuda.current_device():
        st = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, _raw_stream(dev))
    if st:
        check(st, fn.__name__)


# ----------------------------------------------------------------------------- norms
def rmsnorm(x, weight, eps, add=None, residual_out=None, out=None, rows=None, in_stride=None):
    """out = RMSNorm(x (+ add)) * weight, residual_out = x (+ add); rows of x at in_stride."""
    _require_cuda(x, weight, add)
    hidden = weight.shape[0]
    if rows is None:
        rows = x.numel() // hidden
    if in_stride is None:
        in_stride = x.stride(-2) if x.dim() >= 2 else hidden
    if out is None:
        out = torch.empty(rows, hidden, dtype=x.dtype, device=x.device)
    check(_L().hx_rmsnorm(_p(x), _p(add), _p(residual_out), _p(out), _p(weight), rows, hidden,
                          in_stride, out.stride(-2) if out.dim() >= 2 else hidden, float(eps),
                          _code(x), _stream()), "hx_rmsnorm")
    _count(1)
    return out


def embed_rmsnorm(ids, table, weight, eps, residual_out, normed_out):
    _require_cuda(ids, table)
    check(_L().hx_embed_rmsnorm(_p(ids), ids.numel(), _p(table), table.shape[1], _p(weight),
                                float(eps), _p(residual_out), _p(normed_out), _code(table),
                                _stream()), "hx_embed_rmsnorm")
    _count(1)


def embedding(ids, table, vocab_start=0, out=None):
    _require_cuda(ids, table)
    hidden = table.shape[1]
    if out is None:
        out = torch.empty(ids.numel(), hidden, dtype=table.dtype, device=table.device)
    check(_L().hx_embedding(_p(ids), ids.numel(), _p(table), vocab_start, table.shape[0], hidden,
                            _p(out), _code(table), _stream()), "hx_embedding")
    _count(1)
    return out


# ----------------------------------------------------------------------------- rotary
def rotary_cache_write(qkv, batch, seqlen, n_heads, n_heads_kv, head_dim, pos_start, cos, sin,
                       cache, q_out=None, batch_offset=0, interleaved=True):
    """Rotates q/k of the packed qkv and writes k/v into cache [B, S_max, 2, hkv, d]."""
    _require_cuda(qkv, cache, pos_start)
    if q_out is None:
        q_out = torch.empty(batch, seqlen, n_heads, head_dim, dtype=qkv.dtype, device=qkv.device)
    assert cache.stride(-1) == 1 and cache.stride(-2) == head_dim and cache.stride(-3) == n_heads_kv * head_dim
    check(_L().hx_rotary_cache_write(_p(qkv), batch, seqlen, n_heads, n_heads_kv, head_dim,
                                     _p(pos_start), _p(cos), _p(sin), cos.shape[0],
                                     1 if interleaved else 0, _p(q_out), _p(cache),
                                     cache.stride(0), cache.stride(1), batch_offset,
                                     cache.shape[1], _code(qkv), _stream()),
          "hx_rotary_cache_write")
    _count(1)
    return q_out


# ----------------------------------------------------------------------------- gemm
def gemm(a, w, epilogue=HX_EPI_NONE, residual=None, out=None):
    """out = a @ w.T with an epilogue; a [M, K] (row-strided), w [N, K]."""
    _require_cuda(a, w, residual)
    M, K = a.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"gemm: shape mismatch {tuple(a.shape)} x {tuple(w.shape)}^T")
    n_out = N // 2 if epilogue == HX_EPI_SWIGLU else N
    if out is None:
        out = torch.empty(M, n_out, dtype=a.dtype, device=a.device)
    code = _code(a)
    nbytes = _L().hx_gemm_workspace(M, N, K, epilogue, code)
    ws = workspace(nbytes, kind="gemm" if code != _lib.HX_F32 else "attn")
    check(_L().hx_gemm(_p(a), _p(w), _p(out), M, N, K, a.stride(0), w.stride(0), out.stride(0),
                       epilogue, _p(residual), residual.stride(0) if residual is not None else 0,
                       _p(ws), nbytes, code, _stream()), "hx_gemm")
    _count(2 if nbytes else 1)
    return out


def gemm_qkv_rotary(x, w_qkv, seqlen, n_heads, n_heads_kv, head_dim, pos_start, cos, sin,
                    cache, q_out=None, batch_offset=0):
    """Wqkv GEMM with rotary + KV-cache write fused into its epilogue (f16/bf16): returns q
    [rows, n_heads, head_dim]; k, v land in cache[batch_offset + b, pos_start[b] + s]."""
    _require_cuda(x, w_qkv, cache, pos_start)
    M, K = x.shape
    N = w_qkv.shape[0]
    if q_out is None:
        q_out = torch.empty(M, n_heads, head_dim, dtype=x.dtype, device=x.device)
    code = _code(x)
    nbytes = _L().hx_gemm_workspace(M, N, K, _lib.HX_EPI_QKV_ROTARY, code)
    ws = workspace(nbytes, kind="gemm")
    check(_L().hx_gemm_qkv_rotary(_p(x), _p(w_qkv), M, K, x.stride(0), seqlen, n_heads,
                                  n_heads_kv, head_dim, _p(pos_start), _p(cos), _p(sin),
                                  cos.shape[0], _p(q_out), _p(cache), cache.stride(0),
                                  cache.stride(1), batch_offset, cache.shape[1], _p(ws), nbytes,
                                  code, _stream()), "hx_gemm_qkv_rotary")
    _count(2 if (nbytes and M > 64) else 1)
    return q_out


def gemm_qkv_rotary_varlen(x, w_qkv, lengths, slots, n_heads, n_heads_kv, head_dim, cos, sin,
                           cache, q_out, meta=None):
    """gemm_qkv_rotary over prompts packed row after row in x [T, K] (prompt b: lengths[b]
    rows, cache row slots[b], positions from 0): q into q_out [T, n_heads, head_dim], k and v
    into cache[slots[b], s]. meta: a varlen_meta table (the same one prefill_attention_varlen
    reads; built here when omitted)."""
    _require_cuda(x, w_qkv, cache, q_out)
    M, K = x.shape
    N = w_qkv.shape[0]
    n = len(lengths)
    table, _, _ = meta if meta is not None else varlen_meta(lengths, slots, x.device)
    base = table.data_ptr()
    code = _code(x)
    nbytes = _L().hx_gemm_workspace(M, N, K, _lib.HX_EPI_QKV_ROTARY, code)
    ws = workspace(nbytes, kind="gemm")
    check(_L().hx_gemm_qkv_rotary_varlen(
        _p(x), _p(w_qkv), M, K, x.stride(0), base, base + 4 * (n + 1), base + 4 * (2 * n + 1), n,
        n_heads, n_heads_kv, head_dim, _p(cos), _p(sin), cos.shape[0], _p(q_out), _p(cache),
        cache.stride(0), cache.stride(1), cache.shape[0], cache.shape[1], _p(ws), nbytes, code,
        _stream()), "hx_gemm_qkv_rotary_varlen")
    _count(2 if (nbytes and M > 64) else 1)
    return q_out


def gemm_workspace_bytes(M, N, K, epilogue, dtype) -> int:
    return _L().hx_gemm_workspace(M, N, K, epilogue, DTYPE_CODE[dtype])


# ----------------------------------------------------------------------------- attention
def prefill_attention(q, cache, pos_start, n_heads_kv, softmax_scale, causal=True, out=None,
                      batch_offset=0):
    """q [B, S, hq, d] against cache[batch_offset + b, :pos_start[b] + S]."""
    _require_cuda(q, cache, pos_start)
    B, S, hq, d = q.shape
    if out is None:
        out = torch.empty_like(q)
    check(_L().hx_prefill_attention(_p(q), _p(cache), cache.stride(0), cache.stride(1),
                                    batch_offset, _p(pos_start), B, S, hq, n_heads_kv, d,
                                    1 if causal else 0, float(softmax_scale), _p(out), _code(q),
                                    _stream()), "hx_prefill_attention")
    _count(1)
    return out


def varlen_table(lengths, slots):
    """Host layout of a packed pass's metadata, as int32 values: row offsets [n + 1], cache
    slots [n], start positions [n] (0: prefill from an empty cache), a pad to an even count, then
    the (prompt, 128-query block) work items, heaviest causal work (latest block) first.
    Returns (values, n_items, index of the first item)."""
    n = len(lengths)
    if n == 0 or len(slots) != n or any(L <= 0 for L in lengths):
        raise ValueError("varlen_table needs one slot and a positive length per prompt")
    offs = [0]
    for L in lengths:
        offs.append(offs[-1] + L)
    items = sorted(((b, qb) for b, L in enumerate(lengths) for qb in range(-(-L // 128))),
                   key=lambda it: (-it[1], it[0]))
    head = offs + list(slots) + [0] * n
    if len(head) % 2:
        head.append(0)  # the (prompt, block) pairs are read as 8-byte int2
    return head + [v for it in items for v in it], len(items), len(head)


def varlen_meta(lengths, slots, device):
    """varlen_table on the device (pinned host copy, asynchronous H2D on the current stream):
    the table prefill_attention_varlen and gemm_qkv_rotary_varlen read. Returns (table,
    n_items, items start index)."""
    values, n_items, items_at = varlen_table(lengths, slots)
    meta = torch.tensor(values, dtype=torch.int32).pin_memory()
    return meta.to(device, non_blocking=True), n_items, items_at


def prefill_attention_varlen(q, cache, lengths, slots, n_heads_kv, softmax_scale, out,
                             meta=None) -> bool:
    """Causal prefill attention of several prompts packed row after row in q [T, hq, d] (prompt
    b: lengths[b] rows, cache row slots[b], positions from 0) in ONE launch, into out. meta: a
    varlen_meta table (built here when omitted; build it beforehand for a CUDA-graph capture).
    Returns False, launching nothing, for shapes the tensor-core kernel does not cover (f32,
    head_dim 32); the caller then attends prompt by prompt."""
    _require_cuda(q, cache, out)
    T, hq, d = q.shape
    n = len(lengths)
    table, n_items, items_at = meta if meta is not None else varlen_meta(lengths, slots, q.device)
    base = table.data_ptr()
    st = _L().hx_prefill_attention_varlen(
        _p(q), _p(cache), cache.stride(0), cache.stride(1), cache.shape[0], base,
        base + 4 * (n + 1), base + 4 * (2 * n + 1), base + 4 * items_at, n, n_items, T, hq,
        n_heads_kv, d, 1, float(softmax_scale), _p(out), _code(q), _stream())
    if st == _lib.HX_ERR_UNSUPPORTED:
        return False
    check(st, "hx_prefill_attention_varlen")
    _count(1)
    return True


def decode_attention(q, cache, seqlens, n_heads_kv, max_seqlen, softmax_scale, out=None):
    """q [B, hq, d] against cache[b, :seqlens[b]] (seqlens int32 on device)."""
    _require_cuda(q, cache, seqlens)
    B, hq, d = q.shape[0], q.shape[-2], q.shape[-1]
    if out is None:
        out = torch.empty(B, hq, d, dtype=q.dtype, device=q.device)
    nbytes = _L().hx_decode_attention_workspace(B, hq, d, max_seqlen)
    ws = workspace(nbytes)
    check(_L().hx_decode_attention(_p(q), _p(cache), cache.stride(0), cache.stride(1),
                                   _p(seqlens), B, hq, n_heads_kv, d, max_seqlen,
                                   float(softmax_scale), _p(out), _p(ws), nbytes, _code(q),
                                   _stream()), "hx_decode_attention")
    _count(2 if nbytes else 1)
    return out


def decode_workspace_bytes(batch, n_heads, head_dim, max_seqlen) -> int:
    return _L().hx_decode_attention_workspace(batch, n_heads, head_dim, max_seqlen)


# ----------------------------------------------------------------------------- 4-bit KV cache
Q4_META_BYTES = 16  # k_scale, k_min, v_scale, v_min (f32) behind the codes of a record


def allocate_cache_q4(batch, n_heads_kv, max_seqlen, head_dim, device=None) -> torch.Tensor:
    """A KV cache of one layer held in 4 bits: uint8 [batch, n_heads_kv, max_seqlen, head_dim + 16],
    one record (K codes, V codes, scales and minima) per position and KV head, 144 bytes where 16
    bits take 512 (head_dim 128). The format is described at hx_quantize_cache_q4."""
    return torch.empty(batch, n_heads_kv, max_seqlen, head_dim + Q4_META_BYTES, dtype=torch.uint8,
                       device="cuda" if device is None else device)


def _check_q4(what, cache_q4, n_heads_kv, head_dim, first=0, batch=0, written=False):
    if cache_q4.dtype != torch.uint8 or cache_q4.dim() != 4:
        raise ValueError(f"{what}: the 4-bit cache is uint8 [batch, kv heads, positions, head_dim + 16]")
    shape, stride = cache_q4.shape, cache_q4.stride()
    if shape[1] != n_heads_kv or shape[3] != head_dim + Q4_META_BYTES:
        raise ValueError(f"{what}: 4-bit cache of shape {tuple(shape)} for {n_heads_kv} KV heads of {head_dim}")
    if stride[3] != 1 or stride[2] != shape[3]:
        raise ValueError(f"{what}: the records of a head must be contiguous")
    if first < 0 or first + batch > shape[0]:
        raise ValueError(f"{what}: sequences {first}..{first + batch} of a 4-bit cache of {shape[0]}")
    if written and shape[0] > 1 and stride[0] == 0:
        raise ValueError(f"{what}: the 4-bit cache is written, its sequences must not share memory")


def _check_int32(what, name, t, n):
    if t.dtype != torch.int32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be {n} contiguous int32 values")


def _check_rows(what, cache):
    if cache.dim() != 5 or cache.shape[2] != 2:
        raise ValueError(f"{what}: cache must be [batch, rows, 2, kv heads, head_dim]")
    hk, d = cache.shape[3:]
    if cache.stride(2) != hk * d or (cache.stride(3) != d and hk > 1) or cache.stride(4) != 1:
        raise ValueError(f"{what}: the values of a cache row must be contiguous")
    return hk, d


def quantize_cache_q4(cache, counts, cache_q4, starts=None, batch_offset=0):
    """Rows [0, counts[b]) of cache[b] ([B, rows, 2, hkv, d]) become the records at positions
    starts[b] + i (0 + i when starts is None) of cache_q4[batch_offset + b]; counts and starts are
    int32 on the device. Returns cache_q4. Rows outside either buffer are skipped and reported in
    the device error word (2)."""
    hk, d = _check_rows("quantize_cache_q4", cache)
    B = cache.shape[0]
    _check_q4("quantize_cache_q4", cache_q4, hk, d, batch_offset, B, written=True)
    _check_int32("quantize_cache_q4", "counts", counts, B)
    if starts is not None:
        _check_int32("quantize_cache_q4", "starts", starts, B)
    dev = _device_of(cache, counts, cache_q4, starts)
    if cache.numel() == 0:
        return cache_q4
    _call(dev, _L().hx_quantize_cache_q4, cache.data_ptr(), cache.stride(0), cache.stride(1),
          cache.shape[1], _p(starts), counts.data_ptr(), B, hk, d, cache_q4.data_ptr(),
          cache_q4.stride(0), cache_q4.stride(1), batch_offset, cache_q4.shape[2], _code(cache))
    _count(1)
    return cache_q4


def dequantize_cache_q4(cache_q4, counts, cache, starts=None, batch_offset=0):
    """The way back: records [starts[b], starts[b] + counts[b]) of cache_q4[batch_offset + b] as
    rows [0, counts[b]) of cache[b] ([B, rows, 2, hkv, d]). Returns cache."""
    hk, d = _check_rows("dequantize_cache_q4", cache)
    B = cache.shape[0]
    if B > 1 and cache.stride(0) == 0 or cache.shape[1] > 1 and cache.stride(1) == 0:
        raise ValueError("dequantize_cache_q4: cache is written, its rows must not share memory")
    _check_q4("dequantize_cache_q4", cache_q4, hk, d, batch_offset, B)
    _check_int32("dequantize_cache_q4", "counts", counts, B)
    if starts is not None:
        _check_int32("dequantize_cache_q4", "starts", starts, B)
    dev = _device_of(cache, counts, cache_q4, starts)
    if cache.numel() == 0:
        return cache
    _call(dev, _L().hx_dequantize_cache_q4, cache_q4.data_ptr(), cache_q4.stride(0),
          cache_q4.stride(1), batch_offset, cache_q4.shape[2], _p(starts), counts.data_ptr(), B, hk,
          d, cache.data_ptr(), cache.stride(0), cache.stride(1), cache.shape[1], _code(cache))
    _count(1)
    return cache


def rotary_cache_write_q4(qkv, batch, seqlen, n_heads, n_heads_kv, head_dim, pos_start, cos, sin,
                          cache_q4, q_out=None, batch_offset=0, interleaved=True):
    """rotary_cache_write into a 4-bit cache: rotates q/k of the packed qkv and writes k/v as the
    records at positions pos_start[b] + s of cache_q4[batch_offset + b]. Returns q [batch, seqlen,
    n_heads, head_dim]."""
    what = "rotary_cache_write_q4"
    _check_q4(what, cache_q4, n_heads_kv, head_dim, batch_offset, batch, written=True)
    _check_int32(what, "pos_start", pos_start, batch)
    if qkv.numel() != batch * seqlen * (n_heads + 2 * n_heads_kv) * head_dim or not qkv.is_contiguous():
        raise ValueError(f"{what}: qkv must be contiguous [batch, seqlen, (n_heads + 2 n_heads_kv) * head_dim]")
    for t in (cos, sin):
        if (t.dim() != 2 or t.dtype != qkv.dtype or t.shape != cos.shape or t.shape[1] * 2 != head_dim
                or not t.is_contiguous()):
            raise ValueError(f"{what}: cos and sin must be contiguous [positions, head_dim / 2] in qkv's dtype")
    dev = _device_of(qkv, cache_q4, pos_start, cos, sin, q_out)
    if q_out is None:
        q_out = torch.empty(batch, seqlen, n_heads, head_dim, dtype=qkv.dtype, device=qkv.device)
    elif (q_out.numel() != batch * seqlen * n_heads * head_dim or q_out.dtype != qkv.dtype
          or not q_out.is_contiguous()):
        raise ValueError(f"{what}: q_out must be contiguous [batch, seqlen, n_heads, head_dim] in qkv's dtype")
    if qkv.numel() == 0:
        return q_out
    _call(dev, _L().hx_rotary_cache_write_q4, qkv.data_ptr(), batch, seqlen, n_heads, n_heads_kv,
          head_dim, pos_start.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0],
          1 if interleaved else 0, q_out.data_ptr(), cache_q4.data_ptr(), cache_q4.stride(0),
          cache_q4.stride(1), batch_offset, cache_q4.shape[2], _code(qkv))
    _count(1)
    return q_out


def decode_attention_q4(q, cache_q4, seqlens, n_heads_kv, max_seqlen, softmax_scale, out=None):
    """decode_attention over a 4-bit cache: q [B, hq, d] against the first seqlens[b] records of
    cache_q4[b] (seqlens int32 on device, each at most max_seqlen; 0 gives zeros)."""
    what = "decode_attention_q4"
    if q.dim() != 3 or q.stride(2) != 1 or (q.stride(1) != q.shape[2] and q.shape[1] > 1):
        raise ValueError(f"{what}: q must be [batch, n_heads, head_dim] with contiguous heads")
    B, hq, d = q.shape
    _check_q4(what, cache_q4, n_heads_kv, d, 0, B)
    _check_int32(what, "seqlens", seqlens, B)
    if not 0 <= max_seqlen <= cache_q4.shape[2]:
        raise ValueError(f"{what}: max_seqlen {max_seqlen} of a 4-bit cache of {cache_q4.shape[2]} positions")
    dev = _device_of(q, cache_q4, seqlens, out)
    if out is None:
        out = torch.empty(B, hq, d, dtype=q.dtype, device=q.device)
    elif out.numel() != q.numel() or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"{what}: out must be contiguous [batch, n_heads, head_dim] in q's dtype")
    if B == 0:
        return out
    nbytes = decode_q4_workspace_bytes(B, hq, n_heads_kv, d, max_seqlen)
    # A buffer of its own for every call: calls on several streams, and graphs, do not share it.
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _call(dev, _L().hx_decode_attention_q4, q.data_ptr(), q.stride(0) if B > 1 else hq * d, cache_q4.data_ptr(),
          cache_q4.stride(0), cache_q4.stride(1), seqlens.data_ptr(), B, hq, n_heads_kv, d,
          max_seqlen, float(softmax_scale), out.data_ptr(), _p(ws), nbytes, _code(q))
    _count(2 if nbytes else 1)
    return out


def decode_q4_workspace_bytes(batch, n_heads, n_heads_kv, head_dim, max_seqlen) -> int:
    return _L().hx_decode_attention_q4_workspace(batch, n_heads, n_heads_kv, head_dim, max_seqlen)


# ----------------------------------------------------------------------------- 4-bit weights
def gemm_q4(a, w_q4, scales, epilogue=HX_EPI_NONE, residual=None, out=None):
    """gemm with a 4-bit weight for decode batches: out = a @ w.T with an epilogue, a [M, K] (M <= 64),
    w_q4 uint8 [N, K / 2] and scales [N, K / group] in a's dtype as checkpoint.quantize_weight_q4
    makes them (w = scale * (code - 8), group 32, 64 or 128)."""
    what = "gemm_q4"
    if a.dim() != 2 or w_q4.dim() != 2 or scales.dim() != 2 or a.stride(1) != 1:
        raise ValueError(f"{what}: a, w_q4 and scales must be matrices, the rows of a contiguous")
    M, K = a.shape
    N = w_q4.shape[0]
    if w_q4.dtype != torch.uint8 or w_q4.shape[1] * 2 != K or not w_q4.is_contiguous():
        raise ValueError(f"{what}: w_q4 must be contiguous uint8 [N, K / 2]: got {tuple(w_q4.shape)} for K = {K}")
    if (scales.dtype != a.dtype or scales.shape[0] != N or not scales.is_contiguous()
            or scales.shape[1] == 0 or K % scales.shape[1]):
        raise ValueError(f"{what}: scales must be contiguous [N, K / group] in a's dtype")
    cols = N // 2 if epilogue == HX_EPI_SWIGLU else N
    if (residual is None) != (epilogue != HX_EPI_RESIDUAL):
        raise ValueError(f"{what}: a residual goes with HX_EPI_RESIDUAL and only with it")
    for t in (residual, out):
        if t is not None and (tuple(t.shape) != (M, cols) or t.dtype != a.dtype or t.stride(1) != 1):
            raise ValueError(f"{what}: residual and out must be [M, {cols}] in a's dtype with contiguous rows")
    if out is not None and M > 1 and out.stride(0) < cols:
        raise ValueError(f"{what}: the rows of out must not share memory")
    dev = _device_of(a, w_q4, scales, residual, out)
    if out is None:
        out = torch.empty(M, cols, dtype=a.dtype, device=a.device)
    if M == 0:
        return out
    group, code, nbytes, ws = K // scales.shape[1], _code(a), 0, None
    if M > 8 or K > 4096:  # a buffer of its own for every call, as in decode_attention_q4
        nbytes = _L().hx_gemm_q4_workspace(M, N, K, group, code)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=a.device) if nbytes else None
    _call(dev, _L().hx_gemm_q4, a.data_ptr(), w_q4.data_ptr(), scales.data_ptr(), out.data_ptr(), M, N,
          K, group, a.stride(0) if M > 1 else K,
          out.stride(0) if M > 1 else cols, epilogue, _p(residual),
          0 if residual is None else residual.stride(0) if M > 1 else cols, _p(ws), nbytes, code)
    _count(_L().hx_gemm_q4_launches(M, N, K, code) if nbytes else 1)
    return out


# ----------------------------------------------------------------------------- sampling
def argmax(logits, out=None):
    _require_cuda(logits)
    rows, cols = logits.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.long, device=logits.device)
    check(_L().hx_argmax(_p(logits), rows, cols, logits.stride(0), _p(out), _code(logits),
                         _stream()), "hx_argmax")
    _count(1)
    return out


TokenLogprobs = namedtuple("TokenLogprobs", ["logprobs", "entropy", "top_logprobs", "top_tokens"])


def token_logprobs(logits, tokens=None, top_k=0, entropy=False) -> TokenLogprobs:
    """What a row of logits [rows, vocab] says of its tokens, in f32: logprobs [rows] of the given
    tokens (int64 [rows]; None without them; NaN for a token outside the vocabulary), the
    distribution's entropy in nats [rows] (None unless asked for), and the top_k <= 32 most likely
    tokens with their log probabilities [rows, top_k] (None for 0), equal logits by the lower index.
    Masked (-inf) logits have probability 0; a row with a NaN or +inf, or of -inf alone, gives NaN."""
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("token_logprobs: logits must be [rows, vocab] with contiguous rows")
    rows, cols = logits.shape
    if tokens is not None and (tokens.dtype != torch.long or tokens.numel() != rows
                               or not tokens.is_contiguous()):
        raise ValueError(f"token_logprobs: tokens must be {rows} contiguous int64 values")
    if tokens is None and not entropy and top_k == 0:
        raise ValueError("token_logprobs: nothing is asked for")
    dev = _device_of(logits, tokens)
    f32 = dict(dtype=torch.float32, device=logits.device)
    logp = None if tokens is None else torch.empty(rows, **f32)
    ent = torch.empty(rows, **f32) if entropy else None
    top = ids = None
    if top_k > 0:
        top = torch.empty(rows, top_k, **f32)
        ids = torch.empty(rows, top_k, dtype=torch.long, device=logits.device)
    if rows == 0:
        return TokenLogprobs(logp, ent, top, ids)
    _call(dev, _L().hx_token_logprobs, logits.data_ptr(), rows, cols,
          logits.stride(0) if rows > 1 else max(cols, logits.stride(0)), _p(tokens), top_k, _p(logp),
          _p(ent), _p(top), _p(ids), _code(logits))
    _count(1)
    return TokenLogprobs(logp, ent, top, ids)


# ----------------------------------------------------------------------------- KV handoff
def kv_pack(src_ptrs, live_rows, dst_offsets, n_outer, outer_stride_bytes, row_stride_bytes,
            row_bytes, max_live_rows, dst):
    """Gather-pack of live rows (see hx_kv_pack). Pointer/length/offset arrays are int64 CUDA
    tensors; dst may be a peer GPU's buffer given as a raw address (int)."""
    dst_ptr = dst if isinstance(dst, int) else dst.data_ptr()
    check(_L().hx_kv_pack(_p(src_ptrs), _p(live_rows), _p(dst_offsets), src_ptrs.numel(),
                          n_outer, outer_stride_bytes, row_stride_bytes, row_bytes,
                          max_live_rows, dst_ptr, _stream()), "hx_kv_pack")
    _count(1)


def kv_unpack(src, src_offsets, live_rows, dst_ptrs, n_outer, outer_stride_bytes,
              row_stride_bytes, row_bytes, max_live_rows):
    src_ptr = src if isinstance(src, int) else src.data_ptr()
    check(_L().hx_kv_unpack(src_ptr, _p(src_offsets), _p(live_rows), _p(dst_ptrs),
                            dst_ptrs.numel(), n_outer, outer_stride_bytes, row_stride_bytes,
                            row_bytes, max_live_rows, _stream()), "hx_kv_unpack")
    _count(1)


def device_error(clear=True) -> int:
    return _L().hx_device_error(1 if clear else 0)
