"""Cases of the 4-bit decoding operators and of token scoring: the KV cache held in 4-bit records
(written by rotary_cache_write_q4 and quantize_cache_q4, read by decode_attention_q4 and
dequantize_cache_q4), products with 4-bit group-scaled weights (gemm_q4) and token_logprobs.

`run` computes a case in plain torch operations, or through hexgen2_b200.ops where `own` is true.

A record holds one position of one KV head in d + 16 bytes: d/2 bytes of K codes (element 2j in the
low nibble of byte j, 2j + 1 in the high one), d/2 bytes of V codes, then k_scale, k_min, v_scale,
v_min in f32. A row x of d values is stored as lo = min x, R = max x - lo, scale = R / 15 and codes
rint((x - lo) * (15 / R)), all in f32 (R < 2^-100: scale 0, codes 0), and stands for
lo + scale * code. A 4-bit weight [N, K] is bytes [N, K / 2] in the same nibble order plus
scales [N, K / group], and stands for scale * (code - 8).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TINY = 2.0 ** -100


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One decode step of one layer for a single short chat request, 32 heads of 128.
        {"name": "step one request", "kind": "step", "batch": 1, "heads": 32, "heads_kv": 32,
         "head_dim": 128, "longest": 300, "spare": 20, "dtype": "bf16"},
        # The same layer at the serving benchmark's ragged batch of 32.
        {"name": "step ragged batch", "kind": "step", "batch": 32, "heads": 32, "heads_kv": 32,
         "head_dim": 128, "longest": 2478, "spare": 256, "dtype": "bf16"},
        # Grouped heads over long documents: the cache is far larger than L2.
        {"name": "step long documents", "kind": "step", "batch": 4, "heads": 64, "heads_kv": 8,
         "head_dim": 128, "longest": 65536, "spare": 64, "dtype": "bf16"},
        # Narrow heads in f16, odd lengths and batch.
        {"name": "step narrow heads", "kind": "step", "batch": 7, "heads": 32, "heads_kv": 4,
         "head_dim": 64, "longest": 4095, "spare": 3, "dtype": "f16"},
        # Handoff of one prompt: its 16-bit rows become records, and rows again on arrival.
        {"name": "handoff one prompt", "kind": "handoff", "batch": 1, "heads_kv": 8,
         "head_dim": 128, "longest": 777, "spare": 5, "dtype": "f16"},
        # Handoff of a packed prefill pass of ragged prompts.
        {"name": "handoff packed pass", "kind": "handoff", "batch": 16, "heads_kv": 32,
         "head_dim": 128, "longest": 2048, "spare": 256, "dtype": "bf16"},
        # Attention output projection of a single request, added to the residual stream.
        {"name": "projection one request", "kind": "linear", "rows": 1, "n": 4096, "k": 4096,
         "group": 128, "epilogue": "residual", "dtype": "bf16"},
        # Gate and up projection of the serving batch.
        {"name": "gated projection batch", "kind": "linear", "rows": 32, "n": 22016, "k": 4096,
         "group": 128, "epilogue": "swiglu", "dtype": "bf16"},
        # LM head for a handful of requests, finer groups.
        {"name": "vocabulary projection", "kind": "linear", "rows": 5, "n": 32000, "k": 4096,
         "group": 64, "epilogue": "none", "dtype": "f16"},
        # The token just served, with five alternatives.
        {"name": "logprobs one token", "kind": "logprobs", "rows": 1, "vocab": 32000, "top": 5,
         "dtype": "bf16"},
        # Scoring every token of a prompt.
        {"name": "logprobs prompt", "kind": "logprobs", "rows": 4096, "vocab": 32000, "top": 1,
         "dtype": "bf16"},
        # A decode batch over a large odd vocabulary in f32 with twenty alternatives.
        {"name": "logprobs large vocabulary", "kind": "logprobs", "rows": 32, "vocab": 128007,
         "top": 20, "dtype": "f32"},
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["step", "step", "handoff", "linear", "linear", "logprobs"])
    if kind == "step":
        heads, heads_kv = rng.choice([(32, 32), (32, 8), (64, 8), (32, 4), (16, 2), (12, 1), (6, 2)])
        head_dim = rng.choice([64, 128, 128])
        batch = _spread(rng, 1, 64)
        most = min(65536, (300 << 20) // (batch * heads_kv * (head_dim + 16)))
        return {"kind": kind, "batch": batch, "heads": heads, "heads_kv": heads_kv,
                "head_dim": head_dim, "longest": _spread(rng, 1, most),
                "spare": rng.randint(0, 300), "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if kind == "handoff":
        heads_kv, head_dim = rng.choice([1, 2, 4, 8, 32]), rng.choice([64, 128, 128])
        batch = _spread(rng, 1, 32)
        most = min(8192, (256 << 20) // (batch * heads_kv * head_dim * 4))
        return {"kind": kind, "batch": batch, "heads_kv": heads_kv, "head_dim": head_dim,
                "longest": _spread(rng, 1, most), "spare": rng.randint(0, 64),
                "dtype": rng.choice(["bf16", "f16", "f32"])}
    if kind == "linear":
        group = rng.choice([32, 64, 128, 128])
        epilogue = rng.choice(["none", "residual", "swiglu"])
        n = _spread(rng, 64, 32000)
        return {"kind": kind, "rows": _spread(rng, 1, 64),
                "n": -(-n // 32) * 32 if epilogue == "swiglu" else n,
                "k": group * -(-_spread(rng, 256, 11008) // group), "group": group,
                "epilogue": epilogue, "dtype": rng.choice(["bf16", "bf16", "f16"])}
    vocab = _spread(rng, 1000, 150000)
    return {"kind": kind, "rows": _spread(rng, 1, max(1, min(8192, (1 << 27) // vocab))),
            "vocab": vocab, "top": rng.choice([0, 1, 5, 20]),
            "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}


def _lengths(case):
    """Live lengths after the pass: spread over (0, longest] by the golden ratio, the longest first."""
    b, longest = case["batch"], case["longest"]
    return [longest] + [1 + int((longest - 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(1, b)]


# ------------------------------------------------------------------------------------ inputs
def _encode(x):
    """Codes (uint8, one per value) and (scale, lo) in f32 of rows of f32 values."""
    lo, span = x.amin(-1), x.amax(-1) - x.amin(-1)
    flat = span < TINY
    fifteen = torch.full_like(span, 15.0)  # tensor by tensor: divisions by or of a number do not round once
    rate = fifteen / torch.where(flat, torch.ones_like(span), span)
    code = torch.round((x - lo[..., None]) * rate[..., None]).clamp(max=15.0)
    code = torch.where(flat[..., None], torch.zeros_like(code), code)
    return code.to(torch.uint8), torch.where(flat, torch.zeros_like(span), span / fifteen), lo


def _records(k, v):
    """Records [..., d + 16] (uint8) of f32 rows k and v [..., d]."""
    kc, ks, kl = _encode(k)
    vc, vs, vl = _encode(v)
    meta = torch.stack((ks, kl, vs, vl), -1).contiguous().view(torch.uint8)
    return torch.cat((kc[..., 0::2] | kc[..., 1::2] << 4, vc[..., 0::2] | vc[..., 1::2] << 4, meta), -1)


def _rows(records):
    """The f32 rows k and v [..., d] that records [..., d + 16] stand for."""
    d = records.shape[-1] - 16
    meta = records[..., d:].contiguous().view(torch.float32)
    codes = records[..., :d]
    codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    return (meta[..., 1, None] + meta[..., 0, None] * codes[..., :d],
            meta[..., 3, None] + meta[..., 2, None] * codes[..., d:])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case, dt=dt)
    if case["kind"] == "step":
        b, hq, hk, d = case["batch"], case["heads"], case["heads_kv"], case["head_dim"]
        lens = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        cap = case["longest"] + case["spare"]
        s["cache"] = torch.zeros(b, hk, cap, d + 16, dtype=torch.uint8, device="cuda")
        # Keys have channels of different size, as trained models' do; values are plain.
        wide = torch.exp(0.5 * normal(hk, 1, d))
        for i in range(b):
            k, v = normal(hk, case["longest"], d) * wide, normal(hk, case["longest"], d)
            s["cache"][i, :, :case["longest"]] = _records(k.to(dt).float(), v.to(dt).float())
        s["qkv"] = normal(b, (hq + 2 * hk) * d).to(dt)
        angle = torch.outer(torch.arange(cap, device="cuda", dtype=torch.float64),
                            10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d))
        s["cos"], s["sin"] = angle.cos().to(dt), angle.sin().to(dt)
        s["seqlens"], s["pos"] = lens, lens - 1
        s["scale"] = d ** -0.5
        s["ones"] = torch.ones(b, dtype=torch.int32, device="cuda")
        s["rows"] = torch.empty(b, 1, 2, hk, d, dtype=dt, device="cuda")
    elif case["kind"] == "handoff":
        b, hk, d = case["batch"], case["heads_kv"], case["head_dim"]
        cap = case["longest"] + case["spare"]
        s["counts"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        s["cache"] = normal(b, cap, 2, hk, d).to(dt)
        s["records"] = torch.zeros(b, hk, cap, d + 16, dtype=torch.uint8, device="cuda")
        s["arrived"] = torch.zeros(b, cap, 2, hk, d, dtype=dt, device="cuda")
    elif case["kind"] == "linear":
        m, n, k, group = case["rows"], case["n"], case["k"], case["group"]
        s["a"] = normal(m, k).to(dt)
        s["w"] = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        s["scales"] = (0.004 * torch.exp(0.3 * normal(n, k // group))).to(dt)
        s["residual"] = normal(m, n).to(dt) if case["epilogue"] == "residual" else None
    else:
        r, v = case["rows"], case["vocab"]
        s["logits"] = (3.0 * normal(r, v)).to(dt)
        s["tokens"] = torch.randint(0, v, (r,), generator=g, device="cuda")
    return s


# ------------------------------------------------------------------------------------ plain forms
def _rotated(x, cos, sin):
    """Interleaved rotary of f32 heads x [b, h, d] with tables [b, d / 2]."""
    c, sn = cos.float()[:, None], sin.float()[:, None]
    x0, x1 = x[..., 0::2], x[..., 1::2]
    return torch.stack((x0 * c - x1 * sn, x0 * sn + x1 * c), -1).flatten(-2)


def _step(s):
    b, hq, hk, d, dt = s["batch"], s["heads"], s["heads_kv"], s["head_dim"], s["dt"]
    pos = s["pos"].long()
    x = s["qkv"].float().view(b, hq + 2 * hk, d)
    turned = _rotated(x[:, :hq + hk], s["cos"][pos], s["sin"][pos]).to(dt)
    q = turned[:, :hq]
    fresh = _records(turned[:, hq:].float(), x[:, hq + hk:])
    s["cache"][torch.arange(b, device=pos.device), :, pos] = fresh
    k, v = _rows(s["cache"][:, :, :s["longest"]])
    score = s["scale"] * (q.float().view(b, hk, hq // hk, d) @ k.transpose(-1, -2))
    live = torch.arange(s["longest"], device=pos.device) < s["seqlens"][:, None]
    score = score.masked_fill(~live[:, None, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p @ v) / p.sum(-1, keepdim=True)
    return q, out.to(dt).view(b, hq, d), torch.stack(_rows(fresh), 1).to(dt)[:, None]


def _handoff(s):
    live = (torch.arange(s["cache"].shape[1], device="cuda") < s["counts"][:, None])[:, :, None, None, None]
    kv = s["cache"].float().transpose(1, 3)  # [b, hkv, 2, cap, d]
    fresh = _records(kv[:, :, 0], kv[:, :, 1])
    s["records"] = torch.where(live.transpose(1, 3)[:, :, 0], fresh, s["records"])
    k, v = _rows(s["records"])
    kv = torch.stack((k, v), 2).transpose(1, 3).to(s["dt"])
    s["arrived"] = torch.where(live, kv, s["arrived"])
    return s["arrived"]


def _linear(s):
    n, k, group = s["n"], s["k"], s["group"]
    code = torch.stack((s["w"] & 15, s["w"] >> 4), -1).view(n, k // group, group).float() - 8.0
    w = (code * s["scales"].float()[..., None]).view(n, k)
    y = s["a"].float() @ w.t()
    if s["epilogue"] == "residual":
        y = y + s["residual"].float()
    if s["epilogue"] == "swiglu":  # rows of w come as blocks of 16: up, gate, up, gate, ...
        y = y.view(-1, n // 32, 2, 16)
        up, gate = y[:, :, 0], y[:, :, 1]
        y = (up * gate / (1.0 + torch.exp(-gate))).reshape(-1, n // 2)
    return y.to(s["dt"])


def _logprobs(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1)
    log_total = torch.log(total)
    given = x.gather(1, s["tokens"][:, None])[:, 0] - top[:, 0] - log_total
    entropy = log_total - (e * (x - top)).sum(-1) / total
    if not s["top"]:
        return given, entropy
    # Unique keys, so that equal values go to the lowest index.
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 4294967296
    key = key + (4294967295 - torch.arange(x.shape[1], device=x.device))
    ids = 4294967295 - (key.topk(s["top"]).values & 4294967295)
    return given, entropy, x.gather(1, ids) - top - log_total[:, None], ids


def run(state):
    s = state
    if own:
        from hexgen2_b200 import ops

        if s["kind"] == "step":
            q = ops.rotary_cache_write_q4(s["qkv"], s["batch"], 1, s["heads"], s["heads_kv"],
                                          s["head_dim"], s["pos"], s["cos"], s["sin"], s["cache"])
            q = q.view(s["batch"], s["heads"], s["head_dim"])
            out = ops.decode_attention_q4(q, s["cache"], s["seqlens"], s["heads_kv"], s["longest"],
                                          s["scale"])
            # The updated state: the rows that were written, as the values they stand for.
            return q, out, ops.dequantize_cache_q4(s["cache"], s["ones"], s["rows"], starts=s["pos"])
        if s["kind"] == "handoff":
            ops.quantize_cache_q4(s["cache"], s["counts"], s["records"])
            return ops.dequantize_cache_q4(s["records"], s["counts"], s["arrived"])
        if s["kind"] == "linear":
            epilogue = {"none": ops.HX_EPI_NONE, "residual": ops.HX_EPI_RESIDUAL,
                        "swiglu": ops.HX_EPI_SWIGLU}[s["epilogue"]]
            return ops.gemm_q4(s["a"], s["w"], s["scales"], epilogue, residual=s["residual"])
        got = ops.token_logprobs(s["logits"], s["tokens"], top_k=s["top"], entropy=True)
        return got[:4] if s["top"] else got[:2]
    return {"step": _step, "handoff": _handoff, "linear": _linear, "logprobs": _logprobs}[s["kind"]](s)


# ------------------------------------------------------------------------------------ work
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "step":
        b, hq, hk, d = case["batch"], case["heads"], case["heads_kv"], case["head_dim"]
        live = sum(_lengths(case))
        # records read once, the new ones written and given back as rows; the packed projection, the
        # tables' rows, q and the output
        return {"bytes": (live + b) * hk * (d + 16) + b * size * ((3 * hq + 4 * hk) * d + d) + 8 * b,
                "flops": 4 * hq * d * live}
    if case["kind"] == "handoff":
        rows = sum(_lengths(case)) * case["heads_kv"]
        return {"bytes": rows * (4 * case["head_dim"] * size + case["head_dim"] + 16),
                "flops": 12 * rows * case["head_dim"]}
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        out = m * (n // 2 if case["epilogue"] == "swiglu" else n) * size
        return {"bytes": n * k // 2 + n * (k // case["group"]) * size + m * k * size + out
                + (out if case["epilogue"] == "residual" else 0), "flops": 2 * m * n * k}
    r, v = case["rows"], case["vocab"]
    return {"bytes": r * v * size + r * 16 + r * case["top"] * 12, "flops": 5 * r * v}


# ------------------------------------------------------------------------------------ in 64 bits
def _stored64(x):
    """What rows x (f64 copies of stored values) stand for once they are records, in f64. The
    codes and the scale go by f32, as the format says; the values they stand for do not round."""
    x32 = x.float()
    hi, lo = x32.max(-1, keepdim=True).values, x32.min(-1, keepdim=True).values
    span = hi - lo
    dead = span < 2.0 ** -100
    # f64 quotients of f32 values, rounded once more to f32, are the f32 quotients.
    rate = (15.0 / span.masked_fill(dead, 1.0).double()).float()
    code = ((x32 - lo) * rate).round().double().clamp(0, 15)
    return torch.where(dead, lo.double(), lo.double() + (span.double() / 15.0).float().double() * code)


def _record64(rec, at, d):
    """K (at 0) or V (at 1) rows of records in f64."""
    raw = rec[..., at * d // 2:(at + 1) * d // 2].long()
    code = torch.empty(*raw.shape[:-1], d, dtype=torch.float64, device=rec.device)
    code[..., 0::2], code[..., 1::2] = (raw % 16).double(), (raw // 16).double()
    tail = rec[..., d + 8 * at:d + 8 * at + 8].contiguous().view(torch.float32).double()
    return code * tail[..., :1] + tail[..., 1:]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "step":
        b, hq, hk, d = case["batch"], case["heads"], case["heads_kv"], case["head_dim"]
        x = s["qkv"].double().view(b, hq + 2 * hk, d)
        qs, outs, rows = [], [], []
        for i, n in enumerate(_lengths(case)):
            z = torch.complex(s["cos"][n - 1].double(), s["sin"][n - 1].double())
            turned = torch.view_as_real(torch.view_as_complex(x[i, :hq + hk].reshape(-1, d // 2, 2)) * z).flatten(1)
            qs.append(turned[:hq])
            q = turned[:hq].to(s["dt"]).double()  # attention reads q in the activation type
            new_k = _stored64(turned[hq:].to(s["dt"]).double())
            new_v = _stored64(x[i, hq + hk:])
            rows.append(torch.stack((new_k, new_v))[None])
            head = []
            for h in range(hk):
                rec = s["cache"][i, h, :n - 1]
                k = torch.cat((_record64(rec, 0, d), new_k[h:h + 1]))
                v = torch.cat((_record64(rec, 1, d), new_v[h:h + 1]))
                w = torch.softmax(q[h * (hq // hk):(h + 1) * (hq // hk)] @ k.t() * d ** -0.5, -1)
                head.append(w @ v)
            outs.append(torch.cat(head))
        return torch.stack(qs), torch.stack(outs), torch.stack(rows)
    if case["kind"] == "handoff":
        out = torch.zeros(s["cache"].shape, dtype=torch.float64, device="cuda")
        for i, n in enumerate(_lengths(case)):
            out[i, :n] = _stored64(s["cache"][i, :n].double())
        return out
    if case["kind"] == "linear":
        m, n, k, group = case["rows"], case["n"], case["k"], case["group"]
        y = torch.empty(m, n, dtype=torch.float64, device="cuda")
        for i in range(0, n, 2048):
            raw = s["w"][i:i + 2048].long()
            w = torch.empty(raw.shape[0], k, dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = (raw % 16).double() - 8, (raw // 16).double() - 8
            w *= s["scales"][i:i + 2048].double().repeat_interleave(group, 1)
            y[:, i:i + 2048] = s["a"].double() @ w.t()
        if case["epilogue"] == "residual":
            y += s["residual"].double()
        if case["epilogue"] == "swiglu":
            which = torch.arange(n, device="cuda") // 16 % 2
            y = y[:, which == 0] * torch.nn.functional.silu(y[:, which == 1])
        return y
    x = s["logits"].double()
    logp = torch.log_softmax(x, -1)
    given = logp.gather(1, s["tokens"][:, None])[:, 0]
    entropy = -(logp.exp() * logp).sum(-1)
    if not case["top"]:
        return given, entropy
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
    return given, entropy, logp.gather(1, order), order
