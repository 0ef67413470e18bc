"""``token_logprobs`` against log-softmax in 64 bits.

A log probability is x - m - ln Z.  Its terms' roundings are below 2^-24 of
|x|, |m| and ln Z, and Z's relative error below 2^-20 (a few roundings to a term
and per-thread sums of at most some hundred of them), so 2e-6 plus 2.5e-7 of
the largest |logit| bounds it; the entropy's weighted sum has the relative
error of Z times the size of the differences: 2e-6 of 1 + max|x - m| where
p counts, bounded here by 1e-5 (1 + ln vocab).  Ranked tokens must be equal.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _check(logits, tokens, top):
    from polar_pack_b200.scoring import token_logprobs
    r = token_logprobs(logits, tokens, top=top)
    x = logits.double()
    lp = torch.log_softmax(x, 1)
    tol = 2e-6 + 2.5e-7 * float(x[torch.isfinite(x)].abs().max())
    ok = tokens >= 0
    want = torch.where(ok, lp.gather(1, tokens.clamp(min=0).long()[:, None])[:, 0], 0.0)
    same = (r.logprob.double() == want)
    assert (same | ((r.logprob.double() - want).abs() <= tol)).all()
    ent = -(lp.exp() * lp.masked_fill(lp == -math.inf, 0.0)).sum(1)
    assert ((r.entropy.double() - ent).abs() <= 1e-5 * (1 + math.log(logits.shape[1]))).all()
    order = torch.sort(x, dim=1, descending=True, stable=True)
    assert torch.equal(r.top_ids.long(), order.indices[:, :top])
    got, want = r.top_logprobs.double(), lp.gather(1, order.indices[:, :top])
    assert ((got == want) | ((got - want).abs() <= tol)).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 33, 32), (2, 1000, 7), (4, 151936, 20),
                                            (300, 4099, 5), (1, 152064, 32), (700, 257, 0), (9, 40001, 1)])
def test_scores(cuda, dtype, rows, vocab, top):
    g = torch.Generator(device=cuda)
    g.manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, generator=g, device=cuda) * 3).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=cuda, dtype=torch.int32)
    _check(x, t, top)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_layouts(cuda, dtype):
    """Rows at odd offsets and strides, and rows that share their storage."""
    g = torch.Generator(device=cuda)
    g.manual_seed(1)
    big = (torch.randn(6, 3001, generator=g, device=cuda) * 3).to(dtype)
    t = torch.tensor([0, 5, -1, 2990, 1500, -100], dtype=torch.int32, device=cuda)
    for first in range(1, 9):
        _check(big[:, first:first + 2991], t, 9)
    _check(big[:1].expand(6, 3001), t, 4)


@pytest.mark.parametrize("shape", ["constant", "steps", "ascending", "descending", "bunched", "spike", "huge"])
def test_orders(cuda, shape):
    """Ties, sorted rows, the largest values side by side, one certain token."""
    V = 50_021
    i = torch.arange(V, device=cuda, dtype=torch.float32)
    x = {"constant": i * 0 + 2.0, "steps": (i % 7), "ascending": i / V * 8, "descending": -i / V * 8,
         "bunched": (i // 1024 == 17).float() * (5 + (i % 13)), "spike": (i == 30_000).float() * 60,
         "huge": (i % 11) * 5000.0}[shape]
    for dtype in (torch.float16, torch.float32):
        rows = torch.stack([x, x.flip(0), x.roll(4097)]).to(dtype)
        _check(rows, torch.tensor([30_000, 0, V - 1], dtype=torch.int32, device=cuda), 32)


@pytest.mark.parametrize("top", [1, 20])
def test_many_rows_of_ties(cuda, top):
    """Rows that list more logits than there is room for, on every SM at once."""
    V = 20_003
    i = torch.arange(V, device=cuda, dtype=torch.float32)
    x = torch.stack([i * 0 - 1.5, (i / V * 8), i % 3, (i > 2500).float() * 4]).repeat(250, 1).half()
    _check(x, torch.full((1000,), 5, dtype=torch.int32, device=cuda), top)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_masked_rows(cuda, dtype):
    """-inf entries and rows of nothing else, the type's lowest value, NaN, +inf, -0."""
    from polar_pack_b200.scoring import token_logprobs
    V = 9001
    g = torch.Generator(device=cuda)
    g.manual_seed(2)
    x = torch.randn(8, V, generator=g, device=cuda).to(dtype)
    x[0, 1:] = -math.inf
    x[1, ::2] = -math.inf
    x[2] = -math.inf
    x[3] = torch.finfo(dtype).min
    x[4, 77] = math.nan
    x[5, 78] = math.inf
    x[6] = -1
    x[6, 40], x[6, 20] = 0.0, -0.0
    x[7, :-1] = torch.finfo(dtype).min
    t = torch.tensor([0, 1, 5, 8, 3, 78, 40, V - 1], dtype=torch.int32, device=cuda)
    plain = [0, 1, 3, 6, 7]
    _check(x[0:2], t[0:2], 1)
    _check(x[plain], t[plain], 3)
    r = token_logprobs(x, t, top=2)
    assert r.logprob[2] == -math.inf and r.entropy[2] == 0
    assert r.top_ids[2].tolist() == [0, 1] and (r.top_logprobs[2] == -math.inf).all()
    assert r.top_ids[6].tolist() == [20, 40]
    assert torch.isnan(r.logprob[4]) and torch.isnan(r.entropy[4]) and r.top_ids[4, 0] == 77
    assert torch.isnan(r.logprob[5]) and torch.isnan(r.entropy[5])
    assert r.top_ids[5, 0] == 78 and r.top_logprobs[5, 1] == -math.inf
    assert r.top_ids[0].tolist() == [0, 1] and r.top_logprobs[0, 1] == -math.inf


def test_tokens_and_status(cuda):
    from polar_pack_b200.scoring import token_logprobs
    x = torch.randn(4, 100, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    r = token_logprobs(x, torch.tensor([-1, 5, -100, 99], dtype=torch.int32, device=cuda), status=status)
    assert r.logprob[0] == 0 and r.logprob[2] == 0 and int(status) == 0 and r.top_ids.shape == (4, 0)
    r = token_logprobs(x, torch.tensor([1, 100, 2, 3], dtype=torch.int32, device=cuda), status=status)
    assert torch.isnan(r.logprob[1]) and torch.isfinite(r.logprob[[0, 2, 3]]).all() and int(status) == 4
    assert torch.isfinite(r.entropy).all()
    r = token_logprobs(x[:0], torch.zeros(0, dtype=torch.int32, device=cuda), top=3)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)


def test_refusals(cuda):
    from polar_pack_b200.scoring import token_logprobs
    x = torch.randn(4, 100, device=cuda)
    t = torch.zeros(4, dtype=torch.int32, device=cuda)
    for args in ((x.double(), t), (x.t(), t), (x[0], t), (x, t.long()), (x, t[:3]), (x[:, ::2], t)):
        with pytest.raises(ValueError):
            token_logprobs(*args)
    for top in (-1, 33):
        with pytest.raises(ValueError):
            token_logprobs(x, t, top=top)
    with pytest.raises(ValueError):
        token_logprobs(x[:, :5], t, top=6)
    with pytest.raises(RuntimeError):
        token_logprobs(x.cpu(), t)


def test_side_stream(cuda):
    from polar_pack_b200.scoring import token_logprobs
    x = torch.randn(64, 5000, device=cuda)
    t = torch.zeros(64, dtype=torch.int32, device=cuda)
    want = token_logprobs(x, t, top=4)
    s = torch.cuda.Stream(cuda)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        y = x * 1.0
        got = token_logprobs(y, t, top=4)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_equal_terms(cuda, dtype):
    """Many equal logits below the maximum: their sum's roundings must not add up."""
    x = torch.full((4, 150001), -0.3, device=cuda, dtype=dtype)
    x[:, 1::512] = 0.25
    x[1] *= 3
    x[2, ::7] = -math.inf
    _check(x, torch.tensor([0, 1, 5, 513], dtype=torch.int32, device=cuda), 2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_lowest_beside_nothing(cuda, dtype):
    """Rows of the type's lowest value and -inf, in any order, odd lengths and starts."""
    g = torch.Generator(device=cuda)
    g.manual_seed(11)
    wide = torch.full((6, 20011), torch.finfo(dtype).min, device=cuda).to(dtype)
    wide[torch.rand(wide.shape, generator=g, device=cuda) < 0.5] = -math.inf
    wide[3:, 7000] = torch.tensor([1.0, 1e4, -5.0], device=cuda).to(dtype)
    for x in (wide, wide[:, 3:10002]):
        t = torch.tensor([int(torch.isfinite(r).nonzero()[0]) for r in x], dtype=torch.int32, device=cuda)
        _check(x, t, 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1300, 1001, 32), (1300, 4001, 5), (1300, 9000, 32), (40, 300, 32),
                                            (3, 2047, 32), (1200, 31, 31), (2000, 1, 1), (1250, 16383, 8)])
def test_short_rows(cuda, dtype, rows, vocab, top):
    """Rows of a few KB, of which a CTA of two warps takes one; ties and rows of nothing among them."""
    g = torch.Generator(device=cuda)
    g.manual_seed(rows * 7 + vocab)
    x = (torch.randn(rows, vocab, generator=g, device=cuda) * 3).to(dtype)
    x[1::3] = (x[1::3] * 2).round() / 2
    x[2] = torch.finfo(dtype).min if dtype == torch.float16 else -1.0
    t = torch.randint(0, vocab, (rows,), generator=g, device=cuda, dtype=torch.int32)
    _check(x, t, top)


@pytest.mark.parametrize("top", [0, 2])
def test_more_rows_than_a_grid(cuda, top):
    """More rows than a launch has CTAs for (2^24): a CTA takes one row after another."""
    from polar_pack_b200.scoring import token_logprobs
    rows, vocab = (1 << 24) + 5001, 6
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB of device memory")
    g = torch.Generator(device=cuda)
    g.manual_seed(21)
    x = (torch.randn(rows, vocab, generator=g, device=cuda) * 3).half()
    t = torch.randint(0, vocab, (rows,), generator=g, device=cuda, dtype=torch.int32)
    r = token_logprobs(x, t, top=top)
    some = torch.cat([torch.arange(0, 6000, device=cuda), torch.arange(rows - 6000, rows, device=cuda)])
    lp = torch.log_softmax(x[some].double(), 1)
    tol = 2e-6 + 2.5e-7 * float(x.abs().max())
    assert ((r.logprob[some] - lp.gather(1, t[some].long()[:, None])[:, 0]).abs() <= tol).all()
    assert ((r.entropy[some] + (lp.exp() * lp).sum(1)).abs() <= 1e-5 * (1 + math.log(vocab))).all()
    order = torch.sort(x[some].double(), dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(r.top_ids[some].long(), order)
    assert ((r.top_logprobs[some] - lp.gather(1, order)).abs() <= tol).all()
