"""The 4-bit operators on the GPU against plain 64-bit forms: records written and read back, decode
attention over them, products with 4-bit weights, and a decode layer that chains them."""
import pytest
import torch

from hexgen2_b200 import ops
from hexgen2_b200.checkpoint import dequantize_weight_q4, quantize_weight_q4
from oracle.llama_ref import Rotary

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------ plain records
def encode(x):
    """(codes, scale, lo) of rows by the format's definition, f32 operation by operation."""
    x = x.float()
    lo = x.amin(-1)
    span = x.amax(-1) - lo
    bad = ~torch.isfinite(x).all(-1) | ~torch.isfinite(span)
    flat = span < 2.0 ** -100
    fifteen = torch.full_like(span, 15.0)  # tensor by tensor: divisions by or of a number do not round once
    rate = fifteen / torch.where(flat, torch.ones_like(span), span)
    codes = torch.round((x - lo[..., None]) * rate[..., None]).clamp(max=15)
    codes = torch.where((bad | flat)[..., None], torch.zeros_like(codes), codes)
    nan = torch.full_like(span, float("nan"))
    scale = torch.where(bad, nan, torch.where(flat, torch.zeros_like(span), span / fifteen))
    return codes.to(torch.uint8), scale, torch.where(bad, nan, lo)


def records(k, v):
    kc, ks, kl = encode(k)
    vc, vs, vl = encode(v)
    meta = torch.stack((ks, kl, vs, vl), -1).contiguous().view(torch.uint8)
    return torch.cat((kc[..., 0::2] | kc[..., 1::2] << 4, vc[..., 0::2] | vc[..., 1::2] << 4, meta), -1)


def rows64(rec):
    d = rec.shape[-1] - 16
    meta = rec[..., d:].contiguous().view(torch.float32).double()
    c = torch.stack((rec[..., :d] & 15, rec[..., :d] >> 4), -1).flatten(-2).double()
    return (meta[..., 1, None] + meta[..., 0, None] * c[..., :d],
            meta[..., 3, None] + meta[..., 2, None] * c[..., d:])


def same_records(got, want):
    """Bytes equal, any NaN standing for any other."""
    d = got.shape[-1] - 16
    assert torch.equal(got[..., :d], want[..., :d])
    a, b = (r[..., d:].contiguous().view(torch.float32) for r in (got, want))
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


# ------------------------------------------------------------------------------ write and read back
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hk,d,counts,starts", [
    (1, 32, [0, 1, 5], None),
    (3, 64, [7, 40, 33], [1, 0, 7]),
    (8, 128, [40, 0, 17], [0, 40, 3]),
    (32, 128, [1], [39]),
])
def test_quantize_and_back(dtype, hk, d, counts, starts):
    dt, cap, b0 = DT[dtype], 40, 2
    B = len(counts)
    g = torch.Generator().manual_seed(hk * d + B)
    whole = torch.randn(B, cap + 5, 2, hk, d, generator=g).to(dt)
    cache = whole[:, 3:3 + cap]  # a strided view of longer rows
    q4 = ops.allocate_cache_q4(B + b0 + 1, hk, cap, d)
    q4.fill_(0xA5)
    ops.quantize_cache_q4(whole.cuda()[:, 3:3 + cap], i32(counts), q4, batch_offset=b0,
                          starts=None if starts is None else i32(starts))
    want = torch.full_like(q4, 0xA5).cpu()
    kv = cache.permute(0, 3, 2, 1, 4)  # [B, hk, 2, cap, d]
    for b, n in enumerate(counts):
        s = 0 if starts is None else starts[b]
        want[b0 + b, :, s:s + n] = records(kv[b, :, 0, :n], kv[b, :, 1, :n])
    assert ops.device_error() == 0
    same_records(q4.cpu(), want)
    back = torch.full((B, cap, 2, hk, d), 9.0, dtype=dt, device="cuda")
    ops.dequantize_cache_q4(q4, i32(counts), back, batch_offset=b0,
                            starts=None if starts is None else i32(starts))
    assert ops.device_error() == 0
    for b, n in enumerate(counts):
        s = 0 if starts is None else starts[b]
        k, v = rows64(want[b0 + b, :, s:s + n])
        exact = torch.stack((k, v), 1).permute(2, 1, 0, 3)
        off = (back[b, :n].cpu().double() - exact).abs()
        # f32 first (one fused operation), then the row's type: two half steps.
        assert (off <= exact.abs() * (half_step(dt) + 2.0 ** -23) + 1e-30).all()
        assert (back[b, n:] == 9).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_quantize_special_rows(dtype):
    """Flat rows, rows with NaN or infinities, a span that overflows f32, one below 2^-100, signed
    zeros, and values that land on code borders."""
    dt, d = DT[dtype], 64
    x = torch.zeros(1, 9, 2, 1, d, dtype=torch.float32)
    ramp = torch.arange(d, dtype=torch.float32)
    x[0, 0] = 3.0
    x[0, 1, 0, 0, 5] = float("nan")
    x[0, 2, 1, 0, 63] = float("inf")
    x[0, 3, 0, 0, 0] = float("-inf")
    big = torch.finfo(dt).max
    x[0, 4, 0, 0, 1], x[0, 4, 0, 0, 2] = big, -big
    x[0, 5, 0, 0, 7] = 2.0 ** -101 if dtype != "f16" else 2.0 ** -24
    x[0, 6, 0, 0, ::2] = -0.0
    x[0, 7] = (ramp % 31) / 2  # steps of 1: every odd multiple of 0.5 lies on a border
    x[0, 8] = -5.0 - ramp / 16
    x = x.to(dt)
    q4 = ops.allocate_cache_q4(1, 1, 9, d)
    ops.quantize_cache_q4(x.cuda(), i32([9]), q4)
    kv = x.permute(0, 3, 2, 1, 4)
    same_records(q4.cpu(), records(kv[:, :, 0], kv[:, :, 1]))
    back = ops.dequantize_cache_q4(q4, i32([9]), torch.zeros_like(x, device="cuda")).cpu()
    for t, half in ((1, 0), (2, 1), (3, 0)):
        assert back[0, t, half].isnan().all() and not back[0, t, 1 - half].isnan().any()
    assert (back[0, 0] == 3).all() and not back[0, 6].any()
    assert ops.device_error() == 0


def test_ranges_outside_the_buffers_are_skipped():
    """Counts or starts beyond either buffer: nothing outside is read or written, the part that
    fits is done, and the device error word says so."""
    d, hk, cap = 64, 2, 16
    x = torch.randn(1, 10, 2, hk, d, device="cuda")
    for count, start, fits in ((11, 0, 10), (10, 9, 7), (5, 16, 0), (5, 40, 0), (-1, 0, 0), (3, -1, 0)):
        guard = torch.full((3, hk, cap, d + 16), 0x5A, dtype=torch.uint8, device="cuda")
        ops.quantize_cache_q4(x, i32([count]), guard[1:2], starts=i32([start]))
        assert ops.device_error() == 2
        assert (guard[0] == 0x5A).all() and (guard[2] == 0x5A).all()
        live = torch.zeros(cap, dtype=torch.bool)
        live[max(start, 0):max(start, 0) + fits] = fits > 0
        assert (guard[1][:, ~live] == 0x5A).all()
        kv = x.cpu().permute(0, 3, 2, 1, 4)
        if fits:
            same_records(guard[1][:, live].cpu(), records(kv[0, :, 0, :fits], kv[0, :, 1, :fits]))
        rows = torch.full((3, 10, 2, hk, d), 7.0, device="cuda")
        full = torch.zeros(1, hk, cap, d + 16, dtype=torch.uint8, device="cuda")
        ops.dequantize_cache_q4(full, i32([count]), rows[1:2], starts=i32([start]))
        assert ops.device_error() == 2
        assert (rows[0] == 7).all() and (rows[2] == 7).all()
        assert not rows[1, :fits].any() and (rows[1, fits:] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("hq,hk,d,S", [(4, 2, 32, 3), (6, 6, 64, 1), (32, 4, 128, 5), (1, 1, 128, 1)])
def test_rotary_write_equals_rotary_then_quantize(dtype, interleaved, hq, hk, d, S):
    dt, cap, starts, b0 = DT[dtype], 24, [0, 19, 7], 1
    B = len(starts)
    g = torch.Generator().manual_seed(d + hq)
    qkv = torch.randn(B, S, (hq + 2 * hk) * d, generator=g).to(dt).cuda()
    cos, sin = (t.cuda() for t in Rotary(d, 10000.0).tables(cap, dt))
    cache = torch.zeros(B, cap, 2, hk, d, dtype=dt, device="cuda")
    q_ref = ops.rotary_cache_write(qkv, B, S, hq, hk, d, i32(starts), cos, sin, cache,
                                   interleaved=interleaved)
    q4 = torch.full((B + 2, hk, cap, d + 16), 0x33, dtype=torch.uint8, device="cuda")
    q = ops.rotary_cache_write_q4(qkv, B, S, hq, hk, d, i32(starts), cos, sin, q4, batch_offset=b0,
                                  interleaved=interleaved)
    assert ops.device_error() == 0
    want = torch.full_like(q4, 0x33).cpu()
    kv = cache.cpu().permute(0, 3, 2, 1, 4)
    for b, p in enumerate(starts):
        want[b0 + b, :, p:p + S] = records(kv[b, :, 0, p:p + S], kv[b, :, 1, p:p + S])
    if dt != torch.float32:  # products of 16-bit values are exact in f32: the same bits
        assert torch.equal(q, q_ref)
        same_records(q4.cpu(), want)
        return
    # f32: either kernel may fuse a product into the sum; a row's values then differ by an ulp or
    # two of its largest, which moves a code by at most one step.
    torch.testing.assert_close(q, q_ref, rtol=2.0 ** -22, atol=2.0 ** -21)
    got = q4.cpu()
    live = torch.zeros(got.shape[:3], dtype=torch.bool)
    for b, p in enumerate(starts):
        live[b0 + b, :, p:p + S] = True
    assert (got[~live] == 0x33).all()
    for b, p in enumerate(starts):
        for got_row, want_row in zip(rows64(got[b0 + b, :, p:p + S]), rows64(want[b0 + b, :, p:p + S])):
            step = (want_row.amax(-1) - want_row.amin(-1)) / 15
            assert ((got_row - want_row).abs() <= 1.001 * step[..., None]).all()
            assert ((got_row - want_row).abs() > 0.5 * step[..., None]).double().mean() < 1e-2


def test_rotary_write_outside_the_cache_is_skipped():
    hq, hk, d, cap = 4, 2, 64, 8
    qkv = torch.randn(3, 2, (hq + 2 * hk) * d, device="cuda")
    cos = torch.ones(32, d // 2, device="cuda")
    for table in (cos, cos[:6]):
        q4 = torch.full((5, hk, cap, d + 16), 0x11, dtype=torch.uint8, device="cuda")
        q = torch.full((3, 2, hq, d), 5.0, device="cuda")
        ops.rotary_cache_write_q4(qkv, 3, 2, hq, hk, d, i32([-1, 3, 7 if table is cos else 5]), table,
                                  table * 0, q4[1:4], q_out=q)
        assert ops.device_error() == 2
        assert (q4[0] == 0x11).all() and (q4[4] == 0x11).all()
        assert (q[0, 0] == 5).all() and (q[2, 1] == 5).all()  # positions -1 and one too far
        assert torch.equal(q[1], qkv[1].view(2, -1, d)[:, :hq])
        assert (q4[1, :, 1:] == 0x11).all() and (q4[2, :, 3:5] != 0x11).any()


# ------------------------------------------------------------------------------ attention
def make_cache(B, hk, cap, d, g, dt, spread=1.0):
    k = torch.randn(B, hk, cap, d, generator=g) * torch.exp(spread * torch.randn(hk, 1, d, generator=g))
    v = torch.randn(B, hk, cap, d, generator=g) * torch.exp(spread * torch.randn(B, hk, cap, 1, generator=g))
    return records(k.to(dt), v.to(dt))


def attention64(q, rec, lens, scale):
    """(out, bound on its error before the last rounding) in 64 bits; f32 work on codes 0..15 and a
    bias of up to 128 keeps a score within (d + 16) roundings of 2^-24 of scale * sum |q| (|k| and
    the bias' share, 16 steps of k), and a probability's relative error is at most twice that; values
    enter with 2^-16 relative to their own size and the bias' share."""
    B, hq, d = q.shape
    hk = rec.shape[1]
    out = torch.zeros(B, hq, d, dtype=torch.float64)
    bound = torch.zeros(B, hq, 1, dtype=torch.float64)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        k, v = rows64(rec[b, :, :n])
        k, v = (t.repeat_interleave(hq // hk, 0) for t in (k, v))
        x = q[b].double()
        out[b] = (torch.softmax(scale * (k @ x[:, :, None])[..., 0], -1)[:, None] @ v)[:, 0]
        wide = k.abs().amax(-1).amax(-1)  # [hq]
        delta = scale * x.abs().sum(-1) * wide * 17 * (d + 16) * 2.0 ** -24
        bound[b] = ((2 * delta + 2.0 ** -16 + n * 2.0 ** -24) * v.abs().amax(-1).amax(-1))[:, None]
    return out, bound


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hq,hk,d", [(2, 2, 32), (8, 8, 64), (4, 4, 128), (6, 2, 64), (8, 1, 128),
                                     (12, 1, 128), (32, 2, 64), (20, 1, 32), (40, 2, 128)])
@pytest.mark.parametrize("lens", [[0, 1, 2], [15, 16, 17], [33, 0, 127, 128, 129], [700, 5, 1025]])
def test_decode_attention(dtype, hq, hk, d, lens):
    dt, B, cap = DT[dtype], len(lens), max(lens) + 3
    g = torch.Generator().manual_seed(sum(lens) + d + hq)
    rec = make_cache(B, hk, cap, d, g, dt, 0.3)
    q = torch.randn(B, hq, d, generator=g).to(dt)
    dev = rec.clone()
    for b, n in enumerate(lens):
        dev[b, :, n:] = 0xFF  # NaN scales and full codes behind the live records
    out = ops.decode_attention_q4(q.cuda(), dev.cuda(), i32(lens), hk, cap, d ** -0.5)
    assert ops.device_error() == 0
    want, bound = attention64(q, rec, lens, d ** -0.5)
    off = (out.cpu().double() - want).abs()
    assert (off <= want.abs() * half_step(dt) * 1.01 + bound).all(), (off - bound).max()
    for b, n in enumerate(lens):
        if n == 0:
            assert not out[b].any()


@pytest.mark.parametrize("hq,hk,d,lens,cap", [(8, 1, 128, [40000, 3, 20011], 40000), (4, 4, 64, [9000], 9001),
                                              (32, 8, 128, [5000, 1, 0, 4097, 2048, 77], 6000)])
def test_decode_attention_long(hq, hk, d, lens, cap):
    """Keys over many splits and their merge, with scores that grow along the sequence."""
    dt = torch.bfloat16
    g = torch.Generator().manual_seed(cap)
    k = torch.randn(len(lens), hk, cap, d, generator=g) * (1 + 3 * torch.arange(cap) / cap)[:, None]
    v = torch.randn(len(lens), hk, cap, d, generator=g)
    rec = records(k.to(dt), v.to(dt))
    q = torch.randn(len(lens), hq, d, generator=g).to(dt)
    out = ops.decode_attention_q4(q.cuda(), rec.cuda(), i32(lens), hk, cap, d ** -0.5)
    want, bound = attention64(q, rec, lens, d ** -0.5)
    assert ((out.cpu().double() - want).abs() <= want.abs() * half_step(dt) * 1.01 + bound).all()
    again = ops.decode_attention_q4(q.cuda(), rec.cuda(), i32(lens), hk, cap, d ** -0.5)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_attention_values_of_very_different_size(dtype):
    """The likeliest key has values a million times smaller than the others' (an attention sink):
    its own digits must survive."""
    dt, d = DT[dtype], 64
    g = torch.Generator().manual_seed(5)
    k = torch.randn(1, 1, 50, d, generator=g)
    v = torch.randn(1, 1, 50, d, generator=g)
    q = torch.randn(1, 1, d, generator=g).to(dt)
    k[0, 0, 20] = 60 * q[0, 0].float() / q[0, 0].float().norm()
    v[0, 0, 20] *= 1e-6
    rec = records(k.to(dt), v.to(dt))
    out = ops.decode_attention_q4(q.cuda(), rec.cuda(), i32([50]), 1, 50, 1.0)
    want, _ = attention64(q, rec, [50], 1.0)
    sink = rows64(rec[0, 0, 20:21])[1].abs().max()
    assert want.abs().max() < 2 * sink  # the sink takes all of the probability
    assert ((out.cpu().double() - want).abs() <= half_step(dt) * want.abs() * 1.01 + 2.0 ** -15 * sink).all()


def test_decode_attention_nan_and_strides():
    """A NaN record gives NaN to its own sequence and KV head only; q may be a slice of a larger
    projection, the cache a slice of a larger batch or a shared prefix."""
    dt, hq, hk, d, cap = torch.bfloat16, 4, 2, 128, 300
    g = torch.Generator().manual_seed(1)
    rec = make_cache(3, hk, cap, d, g, dt, 0.3)
    lens = [300, 260, 17]
    proj = torch.randn(3, hq + 2 * hk, d, generator=g).to(dt)
    clean = ops.decode_attention_q4(proj[:, :hq].contiguous().cuda(), rec.cuda(), i32(lens), hk, cap, 0.1)
    bad = rec.clone()
    bad[1, 1, 255, d:] = 0xFF
    big = torch.zeros(5, hk + 1, cap, d + 16, dtype=torch.uint8, device="cuda")
    big[1:4, :hk] = bad.cuda()
    out = ops.decode_attention_q4(proj.cuda()[:, :hq], big[1:4, :hk], i32(lens), hk, cap, 0.1)
    assert out[1, 2:].isnan().all()
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2]) and torch.equal(out[1, :2], clean[1, :2])
    shared = ops.decode_attention_q4(proj.cuda()[:, :hq], rec[:1].cuda().expand(3, -1, -1, -1), i32(lens),
                                     hk, cap, 0.1)
    alone = ops.decode_attention_q4(proj.cuda()[:, :hq], rec[:1].repeat(3, 1, 1, 1).cuda(), i32(lens), hk, cap, 0.1)
    assert torch.equal(shared, alone) and ops.device_error() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_attention_sizes_of_one_have_any_stride(dtype):
    """One query, and one head per sequence, whose strides torch leaves open."""
    dt, d = DT[dtype], 64
    g = torch.Generator().manual_seed(12)
    rec = make_cache(3, 1, 40, d, g, dt, 0.3).cuda()
    wide = torch.randn(1, 4 * d + 3, generator=g).to(dt).cuda()
    q = wide[:, :4 * d].view(1, 4, d)  # 4 d + 3 elements from one sequence to the next
    run = lambda q, n: ops.decode_attention_q4(q, rec[:n], i32([40, 7, 33][:n]), 1, 40, 0.1)  # noqa: E731
    assert torch.equal(run(q, 1), run(q.contiguous(), 1))
    q = torch.randn(1, 3, d, generator=g).to(dt).cuda().transpose(0, 1)  # heads 3 d apart, contiguous all the same
    assert q.stride(1) != d and torch.equal(run(q, 3), run(q.clone(memory_format=torch.contiguous_format), 3))


def test_records_of_one_head_of_any_stride():
    """Rows [batch, rows, 2, 1, d] of a single KV head, 2 d apart as torch has it."""
    d, n = 64, i32([5, 3])
    rows = torch.randn(2, 5, 1, 2, d, device="cuda").transpose(2, 3)
    assert rows.is_contiguous() and rows.stride(3) != d
    q4 = ops.quantize_cache_q4(rows, n, ops.allocate_cache_q4(2, 1, 5, d).zero_())
    assert torch.equal(q4, ops.quantize_cache_q4(rows.clone(memory_format=torch.contiguous_format), n, torch.zeros_like(q4)))
    back = ops.dequantize_cache_q4(q4, n, torch.zeros_like(rows))
    assert torch.equal(back, ops.dequantize_cache_q4(q4, n, torch.zeros(2, 5, 2, 1, d, device="cuda")))
    assert ops.device_error() == 0


def test_decode_attention_lengths_beyond_the_promise():
    dt, d = torch.bfloat16, 128
    g = torch.Generator().manual_seed(3)
    rec = make_cache(3, 1, 600, d, g, dt, 0.3).cuda()
    q = torch.randn(3, 2, d, generator=g).to(dt).cuda()
    for most in (600, 100, 0):
        out = ops.decode_attention_q4(q, rec, i32([most + 1, -5, most]), 1, most, 0.1)
        assert ops.device_error() == 2
        cut = ops.decode_attention_q4(q, rec, i32([most, 0, most]), 1, most, 0.1)
        assert torch.equal(out, cut) and not out[1].any() and ops.device_error() == 0


def test_decode_attention_in_graphs_and_on_streams():
    """Two captured graphs and a side stream at once, each with scratch of its own, give the eager
    results whichever order they run in."""
    dt, hq, hk, d, cap = torch.bfloat16, 8, 2, 128, 5000
    g = torch.Generator().manual_seed(9)
    rec = make_cache(2, hk, cap, d, g, dt, 0.3).cuda()
    qs = [torch.randn(2, hq, d, generator=g).to(dt).cuda() for _ in range(3)]
    lens = i32([cap, 3001])
    want = [ops.decode_attention_q4(q, rec, lens, hk, cap, 0.1) for q in qs]
    graphs, outs = [], []
    for q in qs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.decode_attention_q4(q, rec, lens, hk, cap, 0.1))
        graphs.append(graph)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graphs[1].replay()
        with torch.cuda.stream(side):
            graphs[0].replay()
            third = ops.decode_attention_q4(qs[2], rec, lens, hk, cap, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(third, want[2])
    assert ops.device_error() == 0


def test_records_move_with_the_handoff_kernels():
    """kv_pack / kv_unpack move the live records of two requests of a layer byte for byte."""
    hk, d, cap, lens = 3, 128, 50, [17, 50]
    rb = d + 16
    src = torch.randint(0, 256, (2, hk, cap, rb), dtype=torch.uint8, device="cuda")
    dst = torch.zeros_like(src)
    offs = [0, hk * lens[0] * rb]
    packed = torch.zeros(hk * sum(lens) * rb, dtype=torch.uint8, device="cuda")
    i64 = lambda v: torch.tensor(v, dtype=torch.int64, device="cuda")  # noqa: E731
    ops.kv_pack(i64([src[0].data_ptr(), src[1].data_ptr()]), i64(lens), i64(offs), hk, cap * rb, rb, rb, 50, packed)
    ops.kv_unpack(packed, i64(offs), i64(lens), i64([dst[0].data_ptr(), dst[1].data_ptr()]), hk, cap * rb, rb, rb, 50)
    for b, n in enumerate(lens):
        assert torch.equal(dst[b, :, :n], src[b, :, :n]) and not dst[b, :, n:].any()


def test_empty_batches():
    q4, rows = ops.allocate_cache_q4(2, 1, 4, 32), torch.zeros(0, 3, 2, 1, 32, device="cuda")
    assert ops.quantize_cache_q4(rows, i32([]), q4) is q4 and ops.dequantize_cache_q4(q4, i32([]), rows) is rows
    assert ops.decode_attention_q4(torch.zeros(0, 2, 32, device="cuda"), q4, i32([]), 1, 4, 1.0).shape == (0, 2, 32)
    cos = torch.ones(4, 16, device="cuda")
    assert ops.rotary_cache_write_q4(torch.zeros(0, 128, device="cuda"), 0, 1, 2, 1, 32, i32([]), cos, cos,
                                     q4).shape == (0, 1, 2, 32)


# ------------------------------------------------------------------------------ 4-bit weights
def linear64(a, codes, scales, epilogue, residual):
    """(result, bound on its error before the last rounding): products of f32 accuracy over K terms
    of |a| * scale * (8 and a bias of up to 136)."""
    w = dequantize_weight_q4(codes, scales).double()
    x = a.double()
    y = x @ w.t()
    k, groups = a.shape[1], scales.shape[1]
    wide = (x.abs() @ scales.double().repeat_interleave(k // groups, 1).t()) * 144
    bound = wide * 24 * 2.0 ** -24
    if epilogue == 1:
        return y + residual.double(), bound + 2.0 ** -23 * (y.abs() + residual.double().abs())
    if epilogue == 2:
        n = y.shape[1]
        gate = torch.arange(n) // 16 % 2 == 1
        up, gt = y[:, ~gate], y[:, gate]
        act = torch.nn.functional.silu(gt)
        bound = bound[:, ~gate] * act.abs() + up.abs() * (1.1 * bound[:, gate] + 2.0 ** -20 * act.abs())
        return up * act, bound
    return y, bound


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,N,K,group,epilogue", [
    (1, 1, 32, 32, 0), (1, 7, 96, 32, 1), (2, 33, 128, 128, 0), (3, 64, 192, 64, 2), (1, 4096, 1024, 128, 1),
    (8, 100, 512, 128, 1), (9, 160, 640, 64, 2), (16, 257, 4096, 128, 0), (17, 96, 2208, 32, 2),
    (31, 130, 1152, 128, 1), (33, 64, 256, 64, 2), (64, 515, 1088, 64, 0), (64, 1024, 2048, 128, 1),
    (3, 96, 8320, 64, 2), (8, 50, 16512, 128, 1), (20, 64, 4128, 32, 2), (40, 40, 8448, 128, 0),
    # large enough for the tcgen05 kernel
    (17, 8005, 4096, 128, 1), (32, 4128, 4160, 64, 2), (33, 4000, 4224, 64, 0), (64, 2080, 4128, 32, 2),
    (50, 1100, 11008, 128, 1)])
def test_gemm_q4(dtype, M, N, K, group, epilogue):
    dt = DT[dtype]
    g = torch.Generator().manual_seed(M * N + K)
    a = torch.randn(M, K, generator=g).to(dt)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scales = (0.05 * torch.exp(torch.randn(N, K // group, generator=g))).to(dt)
    res = torch.randn(M, N, generator=g).to(dt) if epilogue == 1 else None
    out = ops.gemm_q4(a.cuda(), codes.cuda(), scales.cuda(), epilogue, residual=None if res is None else res.cuda())
    want, bound = linear64(a, codes, scales, epilogue, res)
    off = (out.cpu().double() - want).abs()
    assert (off <= want.abs() * half_step(dt) * 1.01 + bound + 1e-7).all(), (off - bound).max()
    again = ops.gemm_q4(a.cuda(), codes.cuda(), scales.cuda(), epilogue, residual=None if res is None else res.cuda())
    assert torch.equal(out, again) and ops.device_error() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gemm_q4_strides_and_in_place(dtype):
    """Rows of a inside a wider buffer, out inside a wider buffer with its neighbours left alone,
    the residual updated in place, and an empty batch."""
    dt, M, N, K = DT[dtype], 5, 72, 256
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(M, K + 64, generator=g).to(dt).cuda()
    a = wide[:, 32:32 + K]
    codes, scales = quantize_weight_q4(torch.randn(N, K, generator=g).to(dt), 64)
    codes, scales = codes.cuda(), scales.cuda()
    plain = ops.gemm_q4(a.contiguous(), codes, scales)
    room = torch.full((M, N + 9), 3.0, dtype=dt, device="cuda")
    ops.gemm_q4(a, codes, scales, out=room[:, 4:4 + N])
    assert torch.equal(room[:, 4:4 + N], plain)
    assert (room[:, :4] == 3).all() and (room[:, 4 + N:] == 3).all()
    res = torch.randn(M, N, generator=g).to(dt).cuda()
    want = ops.gemm_q4(a, codes, scales, ops.HX_EPI_RESIDUAL, residual=res)
    ops.gemm_q4(a, codes, scales, ops.HX_EPI_RESIDUAL, residual=res, out=res)
    assert torch.equal(res, want)
    assert ops.gemm_q4(a[:0], codes, scales).shape == (0, N)


def test_gemm_q4_rows_do_not_mix():
    """A row of infinities or NaN stays in its own output row; each row equals its batch-1 product's
    value within the f32 sums' bound (the same rounding to bf16 or its neighbour)."""
    dt, M, N, K = torch.bfloat16, 20, 96, 512
    g = torch.Generator().manual_seed(6)
    a = torch.randn(M, K, generator=g).to(dt).cuda()
    codes, scales = (t.cuda() for t in quantize_weight_q4(torch.randn(N, K, generator=g).to(dt), 128))
    clean = ops.gemm_q4(a, codes, scales)
    bad = a.clone()
    bad[3, 100], bad[11, 5] = float("inf"), float("nan")
    out = ops.gemm_q4(bad, codes, scales)
    keep = [i for i in range(M) if i not in (3, 11)]
    assert torch.equal(out[keep], clean[keep])
    assert not out[3].isfinite().any() or out[3].isnan().any()
    assert out[11].isnan().all()


# Small products, several passes of one kernel, running sums over k, and the tcgen05 kernels (2^29 products of 17 and more
# rows) with 32 and 64 rows to a block.
PATHS = [(5, 96, 256, 64), (20, 160, 512, 128), (12, 64, 8448, 128), (20, 8192, 4096, 128), (40, 4128, 4096, 64)]


@pytest.mark.parametrize("M,N,K,group", PATHS)
@pytest.mark.parametrize("epilogue", [0, 1, 2])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_gemm_q4_strides_and_in_place_on_every_path(dtype, epilogue, M, N, K, group):
    """a, residual and out inside wider buffers whose neighbours are left alone, and the residual updated in place:
    the bits of the contiguous call."""
    dt = DT[dtype]
    g = torch.Generator().manual_seed(M + N + epilogue)
    cols = N // 2 if epilogue == 2 else N
    wide = torch.full((M, K + 64), float("nan"))
    wide[:, 32:32 + K] = torch.randn(M, K, generator=g)
    wide = wide.to(dt).cuda()
    a = wide[:, 32:32 + K]
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8).cuda()
    scales = (0.02 * torch.exp(0.3 * torch.randn(N, K // group, generator=g))).to(dt).cuda()
    res = torch.randn(M, cols + 3, generator=g).to(dt).cuda()[:, 1:1 + cols] if epilogue == 1 else None
    want = ops.gemm_q4(a.contiguous(), codes, scales, epilogue, residual=None if res is None else res.contiguous())
    assert want.isfinite().all()
    room = torch.full((M, cols + 9), 3.0, dtype=dt, device="cuda")
    ops.gemm_q4(a, codes, scales, epilogue, residual=res, out=room[:, 5:5 + cols])
    assert torch.equal(room[:, 5:5 + cols], want)
    assert (room[:, :5] == 3).all() and (room[:, 5 + cols:] == 3).all()
    if epilogue == 1:
        room[:, 5:5 + cols] = res
        ops.gemm_q4(a, codes, scales, epilogue, residual=room[:, 5:5 + cols], out=room[:, 5:5 + cols])
        assert torch.equal(room[:, 5:5 + cols], want)
        assert (room[:, :5] == 3).all() and (room[:, 5 + cols:] == 3).all()
    assert ops.device_error() == 0


@pytest.mark.parametrize("M,N,K,group", PATHS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_gemm_q4_rows_with_infinities_and_nan_on_every_path(dtype, M, N, K, group):
    """A row of a with an infinity or NaN gives NaN in all of its own row, and nothing in another."""
    dt = DT[dtype]
    g = torch.Generator().manual_seed(N)
    a = torch.randn(M, K, generator=g).to(dt).cuda()
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8).cuda()
    scales = (0.02 * torch.exp(0.3 * torch.randn(N, K // group, generator=g))).to(dt).cuda()
    bad = a.clone()
    rows = {0: float("inf"), 2: float("-inf"), M - 1: float("nan")}
    for r, x in rows.items():
        bad[r, (r * 37 + 100) % K] = x
    keep = [i for i in range(M) if i not in rows]
    for epilogue in (0, 2):
        clean, out = (ops.gemm_q4(x, codes, scales, epilogue) for x in (a, bad))
        assert torch.equal(out[keep], clean[keep])
        assert out[list(rows)].isnan().all()


@pytest.mark.parametrize("M,N,K,group", PATHS)
def test_gemm_q4_in_graphs_and_on_streams(M, N, K, group):
    """Two captured graphs and eager calls on a side stream at once, each with scratch of its own, give the
    eager results whichever order they run in."""
    dt = torch.bfloat16
    g = torch.Generator().manual_seed(K)
    xs = [torch.randn(M, K, generator=g).to(dt).cuda() for _ in range(3)]
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8).cuda()
    scales = (0.02 * torch.exp(0.3 * torch.randn(N, K // group, generator=g))).to(dt).cuda()
    want = [ops.gemm_q4(x, codes, scales, ops.HX_EPI_SWIGLU) for x in xs]
    graphs, outs = [], []
    for x in xs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.gemm_q4(x, codes, scales, ops.HX_EPI_SWIGLU))
        graphs.append(graph)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graphs[1].replay()
        with torch.cuda.stream(side):
            graphs[0].replay()
            third = ops.gemm_q4(xs[2], codes, scales, ops.HX_EPI_SWIGLU)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(third, want[2])
    assert ops.device_error() == 0


@pytest.mark.parametrize("M,N,K,launches", [(1, 64, 256, 1), (12, 64, 8448, 1), (40, 40, 8448, 1), (20, 8192, 4096, 3)])
def test_gemm_q4_counts_its_launches(M, N, K, launches):
    """ops.LAUNCHES grows by the kernels that a call launches; a workspace does not say how many."""
    a = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(N, K // 2, dtype=torch.uint8, device="cuda")
    scales = torch.ones(N, K // 128, dtype=torch.bfloat16, device="cuda")
    before = ops.LAUNCHES
    ops.gemm_q4(a, w, scales)
    assert ops.LAUNCHES - before == launches


def test_one_row_of_any_stride():
    """A single row of a whose stride is not a multiple of 16 bytes."""
    g = torch.Generator().manual_seed(2)
    codes, scales = (t.cuda() for t in quantize_weight_q4(torch.randn(48, 64, generator=g).bfloat16(), 32))
    row = torch.randn(1, 67, generator=g).bfloat16().cuda()[:, :64]
    assert torch.equal(ops.gemm_q4(row, codes, scales), ops.gemm_q4(row.contiguous(), codes, scales))


def test_an_error_left_by_another_call_spoils_nothing():
    """The device error word is set (a count beyond the cache) and not yet read: products and
    attention still wait for their data."""
    g = torch.Generator().manual_seed(8)
    codes, scales = (t.cuda() for t in quantize_weight_q4(torch.randn(4096, 4096, generator=g).bfloat16(), 128))
    xs = [torch.randn(m, 4096, generator=g).bfloat16().cuda() for m in (1, 12, 40)]
    rec = make_cache(2, 4, 3000, 128, g, torch.bfloat16, 0.3).cuda()
    q = torch.randn(2, 4, 128, generator=g).bfloat16().cuda()
    lens = i32([3000, 1500])
    run = lambda: [ops.gemm_q4(x, codes, scales) for x in xs] + [ops.decode_attention_q4(q, rec, lens, 4, 3000, 0.1)]  # noqa: E731
    clean = run()
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    ops.quantize_cache_q4(torch.zeros(1, 2, 2, 1, 32, device="cuda"), i32([3]), ops.allocate_cache_q4(1, 1, 2, 32))
    for _ in range(3):
        flush.zero_()  # weights and records come from HBM again
        assert all(torch.equal(a, b) for a, b in zip(run(), clean))
    assert ops.device_error() == 2


# ------------------------------------------------------------------------------ far offsets
def test_offsets_beyond_32_bits():
    """Caches of more than 2^32 bytes and 2^31 elements: rows near the end of the last sequence become records near the
    end of the last sequence and head, are attended to and read back as in a small cache."""
    d, hk, n, S = 128, 2, 5, 1 << 23
    dt = torch.bfloat16
    g = torch.Generator().manual_seed(31)
    rows = torch.randn(1, n, 2, hk, d, generator=g).to(dt).cuda()
    far = torch.empty(3, 1 << 22, 2, hk, d, dtype=dt, device="cuda")  # 2^31 elements a sequence
    far[2, :n] = rows[0]
    far[2, -n:] = rows[0].flip(0)
    small, big = ops.allocate_cache_q4(1, hk, n, d), ops.allocate_cache_q4(4, hk, S, d)  # 2.4e9 bytes a sequence
    ops.quantize_cache_q4(rows, i32([n]), small)
    big[3, :, :n], big[3, :, -n:] = 0x77, 0x77
    ops.quantize_cache_q4(far, i32([0, 0, n]), big, starts=i32([0, 0, S - n]), batch_offset=1)
    assert torch.equal(big[3, :, S - n:], small[0]) and (big[3, :, :n] == 0x77).all()
    back = ops.dequantize_cache_q4(small, i32([n]), torch.zeros_like(rows))
    far[2, :n] = 0
    ops.dequantize_cache_q4(big, i32([0, 0, n]), far, starts=i32([0, 0, S - n]), batch_offset=1)
    assert torch.equal(far[2, :n], back[0])
    # All rows of a sequence: the last ones lie beyond 2^31 elements.
    ops.quantize_cache_q4(far[2:], i32([1 << 22]), big, batch_offset=3)
    assert torch.equal(big[3, :, (1 << 22) - n:1 << 22].flip(1), small[0])
    q = torch.randn(1, 4, d, generator=g).to(dt).cuda()
    ops.quantize_cache_q4(rows, i32([n]), big, batch_offset=3)
    assert torch.equal(ops.decode_attention_q4(q, big[3:], i32([n]), hk, n, 0.1),
                       ops.decode_attention_q4(q, small, i32([n]), hk, n, 0.1))
    # The last record of the longest sequence takes all of the probability.
    big[3].zero_()
    spike = torch.zeros(1, 1, 2, hk, d, dtype=dt, device="cuda")
    spike[:, :, 0] = 30 * q.view(1, 1, hk, 2, d).sum(3)
    spike[:, :, 1] = rows[:, :1, 1]
    ops.quantize_cache_q4(spike, i32([1]), big, starts=i32([S - 1]), batch_offset=3)
    last = ops.allocate_cache_q4(1, hk, 1, d)
    ops.quantize_cache_q4(spike, i32([1]), last)
    out = ops.decode_attention_q4(q, big[3:], i32([S]), hk, S, 1.0)
    assert torch.equal(out, ops.decode_attention_q4(q, last, i32([1]), hk, 1, 1.0)) and ops.device_error() == 0


@pytest.mark.parametrize("M", [3, 40])
def test_gemm_q4_weights_beyond_32_bits(M):
    """A weight of more than 2^32 bytes: its last rows against 64 bits."""
    N, K, n = (1 << 20) + 128, 8192, 256
    g = torch.Generator().manual_seed(M)
    w = torch.full((N, K // 2), 0x88, dtype=torch.uint8, device="cuda")
    w[-n:] = torch.randint(0, 256, (n, K // 2), generator=g, dtype=torch.uint8).cuda()
    scales = torch.ones(N, K // 128, dtype=torch.bfloat16, device="cuda")
    a = torch.randn(M, K, generator=g).bfloat16().cuda()
    out = ops.gemm_q4(a, w, scales)
    want, bound = linear64(a.cpu(), w[-n:].cpu(), scales[-n:].cpu(), 0, None)
    off = (out[:, -n:].cpu().double() - want).abs()
    assert (off <= want.abs() * half_step(torch.bfloat16) * 1.01 + bound).all()
    # Weights of 0 (code 8) and the scales of the rows above: f32 sums of a's share of the codes and of their offset,
    # which cancel up to the same bound.
    assert (out[:, :-n].abs().amax(1).cpu().double() <= bound[:, 0]).all() and ops.device_error() == 0


# ------------------------------------------------------------------------------ together
def layer(x, res, w, cos, sin, q4, pos, seqlens, hq, hk, d, cap, head):
    """One decode step of one layer and the LM head, in 4 bits."""
    B = x.shape[0]
    qkv = ops.gemm_q4(x, *w["qkv"])
    q = ops.rotary_cache_write_q4(qkv, B, 1, hq, hk, d, pos, cos, sin, q4)
    ctx = ops.decode_attention_q4(q.view(B, hq, d), q4, seqlens, hk, cap, d ** -0.5)
    res = ops.gemm_q4(ctx.view(B, hq * d), *w["out"], ops.HX_EPI_RESIDUAL, residual=res)
    act = ops.gemm_q4(res, *w["fc1"], ops.HX_EPI_SWIGLU)
    res = ops.gemm_q4(act, *w["fc2"], ops.HX_EPI_RESIDUAL, residual=res)
    logits = ops.gemm_q4(res, *w["head"])
    return logits, ops.token_logprobs(logits, head, top_k=4, entropy=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_decode_step_in_four_bits(dtype):
    """Prefill rows quantised into the cache, then a decode step through every operator: against the
    same step in 64 bits (f32), and captured in a graph (bf16, bit for bit the eager step)."""
    dt, B, hq, hk, d, cap, inner, vocab = DT[dtype], 3, 4, 2, 64, 70, 160, 96
    h = hq * d
    g = torch.Generator().manual_seed(11)
    lens = [64, 1, 33]
    w = {name: quantize_weight_q4((torch.randn(n, k, generator=g) * k ** -0.5).to(dt), 32)
         for name, (n, k) in {"qkv": ((hq + 2 * hk) * d, h), "out": (h, h), "fc1": (2 * inner, h),
                              "fc2": (h, inner), "head": (vocab, h)}.items()}
    dev = {n: tuple(t.cuda() for t in v) for n, v in w.items()}
    x, res = (torch.randn(B, h, generator=g).to(dt) for _ in range(2))
    past = torch.randn(B, cap, 2, hk, d, generator=g).to(dt)
    cos, sin = Rotary(d, 10000.0).tables(cap, dt)
    tokens = torch.tensor([5, 95, 0])
    q4 = ops.allocate_cache_q4(B, hk, cap, d)
    q4.fill_(0xFF)
    ops.quantize_cache_q4(past.cuda(), i32(lens), q4)
    args = (dev, cos.cuda(), sin.cuda(), q4, i32(lens), i32([n + 1 for n in lens]), hq, hk, d, cap, tokens.cuda())
    logits, probs = layer(x.cuda(), res.cuda(), *args)
    assert ops.device_error() == 0
    if dtype == "bf16":
        xs, rs = x.cuda(), res.cuda()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits2, probs2 = layer(xs, rs, *args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, logits2)
        assert all(torch.equal(a, b) for a, b in zip(probs, probs2))
        assert probs.logprobs.isfinite().all() and ops.device_error() == 0
        return
    W = {n: dequantize_weight_q4(*v).double() for n, v in w.items()}
    qkv = (x.double() @ W["qkv"].t()).view(B, hq + 2 * hk, d)
    z = torch.complex(cos.double(), sin.double())[lens][:, None]
    turned = torch.view_as_real(torch.view_as_complex(qkv[:, :hq + hk].reshape(B, hq + hk, d // 2, 2)) * z).flatten(2)
    kv = past.permute(0, 3, 2, 1, 4)
    ctx = torch.zeros(B, hq, d, dtype=torch.float64)
    for b, n in enumerate(lens):
        rec = torch.cat((records(kv[b, :, 0, :n], kv[b, :, 1, :n]),
                         records(turned[b, hq:, None].float(), qkv[b, hq + hk:, None].float())), 1)
        ctx[b] = attention64(turned[b:b + 1, :hq], rec[None], [n + 1], d ** -0.5)[0][0]
    r = res.double() + ctx.view(B, h) @ W["out"].t()
    u = r @ W["fc1"].t()
    gate = torch.arange(2 * inner) // 16 % 2 == 1
    r = r + (u[:, ~gate] * torch.nn.functional.silu(u[:, gate])) @ W["fc2"].t()
    want = r @ W["head"].t()
    # f32 through five products of at most 256 terms of size ~1 each: a few 1e-6 per stage. A code of
    # the new record may land on the other side of a border (then one value of one row moves by a
    # step); the seed's does not.
    torch.testing.assert_close(logits.cpu().double(), want, rtol=1e-4, atol=1e-4)
    logp = torch.log_softmax(want, -1)
    torch.testing.assert_close(probs.logprobs.cpu().double(), logp.gather(1, tokens[:, None])[:, 0], rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(probs.entropy.cpu().double(), -(logp.exp() * logp).sum(-1), rtol=1e-4, atol=1e-4)
    assert torch.equal(probs.top_tokens.cpu(), want.topk(4).indices)
