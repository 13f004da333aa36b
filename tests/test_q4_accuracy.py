"""How near decode attention over the 4-bit cache comes to 64 bits on long sequences, where outputs are small beside the
values that average out, by a bound in the 2-norm that a lost split, a wrong merge weight or coarser weights exceed."""
import pytest
import torch

from hexgen2_b200 import ops
from q4_forms import attention64, far, parts64, records

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# heads, KV heads, head_dim, lengths, scale
CASES = [(8, 1, 128, [1025, 700], 128 ** -0.5), (4, 4, 64, [9000], 0.02), (4, 2, 128, [5000, 4097], 0.02),
         (2, 1, 128, [40000, 1], 128 ** -0.5), (20, 1, 32, [2500, 129], 0.1), (32, 32, 64, [300 + 7 * i for i in range(20)], 0.05)]


def case(hq, hk, d, lens, wide, dt):
    """(q, records, outputs that count): plain values, or (wide) rows with a pair of channels of opposite sign that
    are far larger than the others, which are what counts then."""
    g = torch.Generator().manual_seed(sum(lens) + d)
    k, v = (torch.randn(len(lens), hk, max(lens), d, generator=g) for _ in range(2))
    keep = torch.ones(d, dtype=torch.bool)
    if wide:
        v[..., 3] = 20 + 20 * v[..., 3].abs()
        v[..., d // 2] = -v[..., 3]
        keep[3] = keep[d // 2] = False
    return torch.randn(len(lens), hq, d, generator=g).to(dt), records(k.to(dt), v.to(dt)), keep


def splits_of(B, hq, hk, d, cap):
    return max(1, ops.decode_q4_workspace_bytes(B, hq, hk, d, cap) // (B * hq * (d + 2) * 4))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("hq,hk,d,lens,scale", CASES)
def test_decode_attention_in_the_2_norm(dtype, wide, hq, hk, d, lens, scale):
    dt, cap = DT[dtype], max(lens)
    q, rec, keep = case(hq, hk, d, lens, wide, dt)
    out = ops.decode_attention_q4(q.cuda(), rec.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), hk, cap, scale)
    assert ops.device_error() == 0
    want, bound = attention64(q, rec, lens, scale, splits_of(len(lens), hq, hk, d, cap), keep)
    assert far(out.cpu()[..., keep], want, bound, dt) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("mix", ["alone", "zeros", "flat"])
@pytest.mark.parametrize("log_size", [-90, -60, -30, 30, 60, 100])
def test_values_of_any_size(dtype, mix, log_size):
    """Values from 2^-90 to 2^100 in size: alone, beside likelier positions whose values are all zero, and beside
    flat rows (one value throughout, no codes) of the same size or of size 1."""
    dt, hq, hk, d, n, scale = DT[dtype], 4, 2, 64, 400, 0.1
    g = torch.Generator().manual_seed(log_size + 200)
    k, v = (torch.randn(1, hk, n, d, generator=g) for _ in range(2))
    q = torch.randn(1, hq, d, generator=g).to(dt)
    v = v * 2.0 ** log_size
    some = torch.arange(n) % 5 == 0
    some[100:300] = True  # whole tiles and, in turn with them, single positions
    if mix == "zeros":
        v[:, :, some] = 0.0
        k[:, :, some] += 3 * q.float().view(1, hk, hq // hk, d).mean(2)[:, :, None] / 8 ** 0.5
    if mix == "flat":
        flat = torch.randn(1, hk, n, 1, generator=g) * torch.where(torch.arange(n) % 2 == 0, 2.0 ** log_size, 1.0)[:, None]
        v[:, :, some] = flat[:, :, some].expand(-1, -1, -1, d)
    rec = records(k.to(dt), v.to(dt))
    for promise, splits in ((n, 4), (130000, 1)):
        cache = torch.zeros(1, hk, promise, d + 16, dtype=torch.uint8)
        cache[:, :, :n] = rec
        assert splits_of(1, hq, hk, d, promise) >= splits
        out = ops.decode_attention_q4(q.cuda(), cache.cuda(), torch.tensor([n], dtype=torch.int32, device="cuda"), hk,
                                      promise, scale)
        # Weights fall below f16's 2^-14 where v_scale is below 2^-80: 2^-25 beside 2^-5 of the largest at 2^-92.
        want, bound = attention64(q, rec, [n], scale, splits, least=2.0 ** -32 if log_size > -70 else 2.0 ** -20)
        assert far(out.cpu(), want, bound, dt) <= 1, promise


def emulated(q, rec, lens, scale, dt, chunk, lose=None, weights=torch.float16, centred=True, merge=True):
    """The kernel's sums with its weights rounded to `weights` times the scale, and mistakes: a lost chunk, codes
    that are not centred, parts added up without their maxima."""
    B, hq, d = q.shape
    out = torch.zeros(B, hq, d, dtype=torch.float64)
    for b, n in enumerate(lens):
        for h in range(hq):
            kc, ks, km, vc, vs, vm = parts64(rec[b, h // (hq // rec.shape[1]), :n])
            s = (scale * ((km + ks * kc) @ q[b, h].double())).float().double()
            c = 7.5 * float(centred)
            O = L = 0
            for i, at in enumerate(range(0, n, chunk)):
                if i == lose:
                    continue
                t = slice(at, at + chunk)
                p = torch.exp(s[t, None] - (s.max() if merge else s[t].max()))
                rounded = (p * vs[t] * 128).to(weights).double() / 128
                O = O + (rounded * (vc[t] - c) + p * (vm[t] + c * vs[t])).sum(0)
                L = L + p.sum()
            out[b, h] = O / L
    return out.to(dt)


@pytest.mark.parametrize("hq,hk,d,lens,scale", [CASES[0], CASES[2]])
def test_the_bound_bites(hq, hk, d, lens, scale):
    """On the CPU: sums as they should be are inside the bound; a chunk left out, parts merged without their maxima,
    weights of eight bits and codes whose offset is added with other weights are outside."""
    dt = torch.bfloat16
    for wide in (False, True):
        q, rec, keep = case(hq, hk, d, lens, wide, dt)
        want, bound = attention64(q, rec, lens, scale, splits_of(len(lens), hq, hk, d, max(lens)), keep)
        is_far = lambda **kw: far(emulated(q, rec, lens, scale, dt, 128, **kw)[..., keep], want, bound, dt)  # noqa: E731
        assert is_far() <= 1
        assert far(torch.zeros_like(want), want, bound, dt) > 50
        assert is_far(lose=1) > 1 and is_far(merge=False) > 1
        if wide:
            assert is_far(weights=torch.bfloat16, centred=False) > 1 and is_far(centred=False) > 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hq,hk,d,n,scale", [(1, 1, 128, 200000, 128 ** -0.5), (8, 1, 64, 65536, 0.125), (32, 4, 128, 30000, 0.05),
                                            (4, 4, 32, 100001, 0.1), (64, 64, 128, 20000, 0.0)])
def test_long_sequences_keep_the_digits_of_their_type(dtype, hq, hk, d, n, scale):
    """Over many positions outputs are hundreds of times smaller than the codes that are summed: what the sums lose is at
    most half of what the output's rounding loses, 1.12 times that in all."""
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(n)
    rows = torch.randn(1, n, 2, hk, d, generator=g, device="cuda").to(dt)
    q = torch.randn(1, hq, d, generator=g, device="cuda").to(dt)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    rec = ops.quantize_cache_q4(rows, lens, ops.allocate_cache_q4(1, hk, n, d))
    out = ops.decode_attention_q4(q, rec, lens, hk, n, scale)
    want = torch.empty(hq, d, dtype=torch.float64, device="cuda")
    for h in range(hk):
        kc, ks, km, vc, vs, vm = parts64(rec[0, h])
        mine = slice(h * hq // hk, (h + 1) * hq // hk)
        want[mine] = torch.softmax(scale * (q[0, mine].double() @ (km + ks * kc).t()), -1) @ (vm + vs * vc)
    off, rounding = (out[0].double() - want).norm(), (want.to(dt).double() - want).norm()
    if dtype == "f32":  # scores and exponentials within 2^-21, sums of distances from the rows' middles
        assert off <= 2.0 ** -19 * want.norm(), (off / want.norm()).item()
    else:
        assert off <= 1.12 * rounding, (off / rounding).item()
