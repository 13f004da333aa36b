"""token_logprobs on the GPU against 64-bit log_softmax: values, entropy and the top list with ties,
masked, infinite and NaN logits, odd and strided rows."""
import pytest
import torch

from hexgen2_b200 import ops

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def plain(x, tokens, k):
    """64-bit values; the top list by (value, lowest index), NaN first."""
    logp = torch.log_softmax(x.double(), -1)
    p = logp.exp()
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(-1)
    order = torch.argsort(x.double().nan_to_num(nan=float("inf"), posinf=1e30, neginf=float("-inf")), dim=-1,
                          descending=True, stable=True)[:, :k]
    return logp.gather(1, tokens[:, None])[:, 0], entropy, logp.gather(1, order), order


def check(x, tokens, k, got):
    given, entropy, top, ids = plain(x, tokens, k)
    # A sum of V terms in f32 by a tree over at most 2^10 long partial sums, exp within 2 ulp, and
    # x - m, log Z rounded to f32 each: 2^-18 absolute covers log probabilities of up to 2^4 in size
    # per 2^-20 of relative rounding.
    def near(a, b):
        a = a.cpu().double()
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.isinf(), b.isinf())
        ok = b.isfinite()
        assert ((a - b)[ok].abs() <= 2.0 ** -20 * (16 + b[ok].abs())).all(), (a - b)[ok].abs().max()
    near(got.logprobs, given)
    near(got.entropy, entropy)
    if k:
        assert torch.equal(got.top_tokens.cpu(), ids)
        near(got.top_logprobs, top)
    else:
        assert got.top_logprobs is None and got.top_tokens is None


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (2, 2, 2), (3, 33, 32), (1, 1000, 0), (5, 1001, 5), (2, 4096, 20),
                                          (1, 32000, 20), (7, 32003, 1), (200, 513, 3), (400, 777, 32),
                                          (2, 150001, 32), (3, 300000, 7)])
def test_token_logprobs(dtype, rows, vocab, k):
    g = torch.Generator().manual_seed(rows + vocab)
    x = (3 * torch.randn(rows, vocab, generator=g)).to(DT[dtype])
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    got = ops.token_logprobs(x.cuda(), tokens.cuda(), top_k=k, entropy=True)
    check(x, tokens, k, got)
    again = ops.token_logprobs(x.cuda(), tokens.cuda(), top_k=k, entropy=True)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("vocab", [40, 5000, 40000])
def test_ties_go_to_the_lowest_index(vocab):
    """Rows of one value, of two values, ascending and descending rows, and equal zeros of both signs."""
    x = torch.zeros(6, vocab)
    x[1, ::3] = 1.0
    x[2] = torch.arange(vocab)
    x[3] = -torch.arange(vocab)
    x[4, ::2] = -0.0
    x[5] = float("-inf")
    x[5, vocab - 25:] = 2.0
    tokens = torch.zeros(6, dtype=torch.long)
    tokens[5] = vocab - 1
    for dt in (torch.float32, torch.bfloat16):
        check(x.to(dt), tokens, 20, ops.token_logprobs(x.to(dt).cuda(), tokens.cuda(), top_k=20, entropy=True))


@pytest.mark.parametrize("vocab", [64, 33001])
def test_masked_infinite_and_nan_rows(vocab):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(7, vocab, generator=g)
    x[0, 5:] = float("-inf")  # five tokens left
    x[1, 1:] = float("-inf")  # one left: certain
    x[2] = float("-inf")      # none left
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    x[5, 3], x[5, 4], x[5, 11] = float("nan"), float("nan"), float("inf")
    tokens = torch.tensor([6, 0, 1, 2, 9, 3, 1])
    got = ops.token_logprobs(x.cuda(), tokens.cuda(), top_k=8, entropy=True)
    assert got.logprobs[0].item() == float("-inf") and got.logprobs[1].item() == 0 and got.entropy[1].item() == 0
    assert got.logprobs[2:6].isnan().all() and got.entropy[2:6].isnan().all()
    assert got.top_logprobs[2:6].isnan().all()
    assert (got.top_logprobs[0, 5:] == float("-inf")).all()
    assert got.top_tokens[2].tolist() == list(range(8)) and got.top_tokens[3, 0].item() == 7
    assert got.top_tokens[4, 0].item() == 9 and got.top_tokens[5, :3].tolist() == [3, 4, 11]
    check(x, tokens, 8, got)


def test_tokens_outside_the_vocabulary_and_parts():
    x = torch.randn(4, 100).cuda()
    tokens = torch.tensor([-1, 100, 99, -100]).cuda()
    got = ops.token_logprobs(x, tokens)
    assert got.logprobs.isnan().tolist() == [True, True, False, True]
    assert got.entropy is None and got.top_tokens is None
    only = ops.token_logprobs(x, top_k=3)
    assert only.logprobs is None and torch.equal(only.top_tokens, x.topk(3).indices)
    assert torch.equal(ops.token_logprobs(x, entropy=True).entropy,
                       ops.token_logprobs(x, tokens, top_k=2, entropy=True).entropy)
    none = ops.token_logprobs(x[:0], tokens[:0], top_k=2, entropy=True)
    assert none.logprobs.shape == (0,) and none.top_tokens.shape == (0, 2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shift,extra", [(0, 7), (1, 0), (3, 5), (8, 8)])
def test_strided_and_unaligned_rows(dtype, shift, extra):
    """Rows at odd strides and starts; what lies between them must not count."""
    rows, vocab = 5, 2001
    g = torch.Generator().manual_seed(shift + extra)
    wide = torch.full((rows, shift + vocab + extra), 1000.0)
    wide[:, shift:shift + vocab] = torch.randn(rows, vocab, generator=g)
    wide = wide.to(DT[dtype])
    x = wide[:, shift:shift + vocab]
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    check(x, tokens, 6, ops.token_logprobs(wide.cuda()[:, shift:shift + vocab], tokens.cuda(), top_k=6, entropy=True))


@pytest.mark.parametrize("scale,offset", [(1e-3, 0.0), (100.0, 0.0), (3.0, 60000.0), (30.0, -60000.0)])
def test_flat_peaked_and_far_rows(scale, offset):
    """Nearly uniform rows, rows with one certain token, and logits far from zero (all f32)."""
    g = torch.Generator().manual_seed(1)
    x = scale * torch.randn(3, 9000, generator=g) + offset
    tokens = torch.tensor([0, 4500, 8999])
    check(x, tokens, 5, ops.token_logprobs(x.cuda(), tokens.cuda(), top_k=5, entropy=True))


MASKS = {  # which logits of a row of v are masked
    "leading half": lambda i, v: i < v // 2,  # whole slices of a cluster
    "all but three": lambda i, v: i < v - 3,
    "all but one in front": lambda i, v: i > 0,
    "every other run of 64": lambda i, v: i // 64 % 2 == 0,
    "half of the threads": lambda i, v: i // 8 % 128 < 64,  # by 16-byte vectors of 16-bit logits
    "one in seven left": lambda i, v: i % 7 != 0,
}


@pytest.mark.parametrize("dtype,mask", [("f32", -1000.0), ("f32", -1e9), ("f32", -1e35), ("f32", -1e38), ("f32", "min"),
                                        ("bf16", -1e35), ("bf16", "min"), ("f16", "min")])
@pytest.mark.parametrize("rows,vocab", [(6, 40), (6, 777), (6, 4096), (12, 33001), (1302, 2100)])
def test_logits_masked_with_low_finite_values(dtype, mask, rows, vocab):
    """Masked logits of the type's lowest value, or any other low one, leave finite sums: each pattern in its own
    rows, and rows of masked logits alone (equal logits: the entropy is log vocab)."""
    dt = DT[dtype]
    low = torch.finfo(dt).min if mask == "min" else mask
    g = torch.Generator().manual_seed(rows + vocab)
    x = torch.randn(rows + 1, vocab, generator=g)
    i = torch.arange(vocab)
    for r, pattern in zip(range(rows), list(MASKS.values()) * rows):
        x[r, pattern(i, vocab)] = low
    x[rows] = low
    x = x.to(dt)
    tokens = torch.randint(0, vocab, (rows + 1,), generator=g)
    got = ops.token_logprobs(x.cuda(), tokens.cuda(), top_k=5, entropy=True)
    assert got.entropy.isfinite().all() and got.logprobs.isfinite().all()
    check(x, tokens, 5, got)


def test_rows_beyond_32_bits():
    """Logits of more than 2^32 bytes and 2^31 elements: the last rows as in a small batch."""
    rows, vocab = 17000, 131077
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(3)
    x[-3:] = torch.randn(3, vocab, generator=g).bfloat16().cuda()
    tokens = torch.full((rows,), vocab - 1, device="cuda")
    got = ops.token_logprobs(x, tokens, top_k=4, entropy=True)
    check(x[-3:].cpu(), tokens[-3:].cpu(), 4, ops.TokenLogprobs(*(t[-3:] for t in got)))
