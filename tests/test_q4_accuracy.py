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
