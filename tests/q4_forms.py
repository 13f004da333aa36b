"""Plain 64-bit forms of the 4-bit cache for the tests: records, and decode attention with a bound on how far a kernel's
sums may be from it."""
import torch


def encode(x):
    """(codes, scale, lo) of rows of finite values, f32 operation by operation."""
    x = x.float()
    lo = x.amin(-1)
    span = x.amax(-1) - lo
    flat = span < 2.0 ** -100
    fifteen = torch.full_like(span, 15.0)  # tensor by tensor: divisions by or of a number do not round once
    rate = fifteen / torch.where(flat, torch.ones_like(span), span)
    codes = torch.round((x - lo[..., None]) * rate[..., None]).clamp(max=15)
    codes = torch.where(flat[..., None], torch.zeros_like(codes), codes)
    return codes.to(torch.uint8), torch.where(flat, torch.zeros_like(span), span / fifteen), lo


def records(k, v):
    kc, ks, kl = encode(k)
    vc, vs, vl = encode(v)
    meta = torch.stack((ks, kl, vs, vl), -1).contiguous().view(torch.uint8)
    return torch.cat((kc[..., 0::2] | kc[..., 1::2] << 4, vc[..., 0::2] | vc[..., 1::2] << 4, meta), -1)


def parts64(rec):
    """Of records [..., d + 16]: K codes, K scale, K minimum, V codes, V scale, V minimum."""
    d = rec.shape[-1] - 16
    meta = rec[..., d:].contiguous().view(torch.float32).double()
    c = torch.stack((rec[..., :d] & 15, rec[..., :d] >> 4), -1).flatten(-2).double()
    return c[..., :d], meta[..., :1], meta[..., 1:2], c[..., d:], meta[..., 2:3], meta[..., 3:]


def attention64(q, rec, lens, scale, splits, keep=slice(None), least=2.0 ** -32):
    """Attention of q [B, hq, d] over the first lens[b] records of rec [B, hkv, S, d + 16] in 64 bits, and a bound
    [B, hq] on the 2-norm, over the outputs `keep`, of the error of f32 sums in up to `splits` parts, before the output
    rounds to its type. All outputs that are not in `keep` are left out. With w the softmax weights, c a position's codes, vs and mid = vmin + 7.5 vs its scale and middle:
      - weights times vs enter as f16, each off by at most half a step, 2^-11, at random (so 2^-11 / sqrt(3) rms), and by
        `least` of the largest. As mid is added apart, that moves vs (c - 7.5): twice the rms of the sum's norm.
        (f16 outputs take two f16 a weight, 2^-22; the bound is that of one all the same.)
      - a score is off by delta = scale sum|q| (15 ks (d / 16 + 3) + 2 |kmin|) 2^-23 (a sum of d / 16 matrix products,
        the sum of q, scaling) and 2^-22 |s| (the product's rounding at the exponential's), and the exponential by
        2^-21; delta of a weight moves the output by w delta (v - out).
      - sums: the codes' sum of each warp is built up in 2 matrix products per 128 positions of its part, each off by
        2^-23 of it, the parts are added one by one at 2^-24."""
    B, hq, d = q.shape
    G = hq // rec.shape[1]
    out = torch.zeros(B, hq, d, dtype=torch.float64)[..., keep]
    bound = torch.zeros(B, hq, dtype=torch.float64)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        for h in range(hq):
            kc, ks, km, vc, vs, vm = parts64(rec[b, h // G, :n])
            vc = vc[:, keep]
            x, v = q[b, h].double(), vm + vs * vc
            s = scale * ((km + ks * kc) @ x)
            w = torch.softmax(s, -1)[:, None]
            o = (w * v).sum(0)
            out[b, h] = o
            off = vs * (vc - 7.5)
            rounding = 2 * 2.0 ** -11 / 3 ** 0.5 * (w * off).square().sum().sqrt()
            rounding = rounding + n * least * (w * vs).max() * 7.5 * vc.shape[1] ** 0.5
            delta = scale * x.abs().sum() * (15 * ks * (d / 16 + 3) + 2 * km.abs()) * 2.0 ** -23
            delta = delta + (s[:, None].abs() + 2) * 2.0 ** -22
            scores = (w * delta * (v - o).abs()).sum(0).norm()
            steps = 2 * -(-(-(-n // 128)) // splits) + 4
            sums = (steps * 2.0 ** -23 * (w * (vs * vc + (vm + 7.5 * vs).abs() + 7.5 * vs)).sum(0)
                    + (splits + 8) * 2.0 ** -24 * (w * v.abs()).sum(0)).norm()
            bound[b, h] = rounding + scores + sums
    return out, bound


def far(out, want, bound, dt):
    """How far out [B, hq, d] is from want, over what it may be: want's own rounding to dt (its mean square a fifth more
    for outputs that round the other way) and the bounds, in the 2-norm over all outputs."""
    rounding = (want.to(dt).double() - want).norm()
    return ((out.double() - want).norm() / (1.2 * rounding.square() + bound.square().sum()).sqrt()).item()
