"""token_logprobs on the GPU against float64.

Tolerance of a log probability and of the entropy, from the FP32 arithmetic: a lane
sums vocab / 256 + 64 terms one after the other (2^-24 of the sum each), a term's
exponent is off by 2^-23 of |m - z| < 32 in the terms that matter (2^-18), the cap's
reciprocal form by 2^-21 cap in z; the log and the difference by 2^-23 of their
size."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _tol(vocab: int, cap: float, size: torch.Tensor) -> torch.Tensor:
    return (vocab / 256 + 64) * 2.0 ** -24 + 2.0 ** -18 + cap * 2.0 ** -20 + 2.0 ** -22 * size.abs()


def _check(logits, tokens, top, cap):
    from se12_amd.logprobs import token_logprobs

    r = token_logprobs(logits, tokens, top=top, softcap=cap)
    x, t = logits.cpu().double(), tokens.cpu()
    z = cap * torch.tanh(x / cap) if cap else x
    z = z - z.amax(1, keepdim=True)      # (64 bits hold no log of a sum beside 3e38 either)
    lp = z - torch.logsumexp(z, 1, keepdim=True)
    vocab = x.shape[1]
    want = lp[torch.arange(x.shape[0]), t]
    assert ((r.logprobs.cpu().double() - want).abs() <= _tol(vocab, cap, want)).all()
    ent = torch.special.entr(lp.exp()).sum(1)
    # W / S is a weighted mean of m - z: the relative errors of a sum apply to it, up to log(vocab)
    assert ((r.entropy.cpu().double() - ent).abs() <= 2 * (1 + math.log(vocab)) * _tol(vocab, cap, ent)).all()
    assert r.top_ids.shape == (x.shape[0], top) and r.top_ids.dtype == torch.int64
    ids = torch.stack([torch.tensor(sorted(range(vocab), key=lambda i: (-row[i], i))[:top], dtype=torch.int64) for row in x.tolist()]) \
        if vocab * x.shape[0] < 40_000 else torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(r.top_ids.cpu(), ids)
    want = lp.gather(1, ids)
    got = r.top_logprobs.cpu().double()
    fine = want.isfinite()
    assert torch.equal(fine, got.isfinite()) and ((got - want).abs()[fine] <= _tol(vocab, cap, want[fine])).all()


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _logits(gpu, rows, vocab, dtype, seed, scale=4.0):
    g = torch.Generator()
    g.manual_seed(seed)
    x = (torch.randn((rows, vocab), generator=g) * scale).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g)
    return x.to(gpu), t.to(gpu)


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 31, 0), (2, 33, 32), (1, 255, 7), (4, 1023, 20), (3, 1025, 32),
                                            (2, 4097, 5), (7, 9001, 20), (1, 256000, 20), (300, 5003, 1)])
def test_logprobs(gpu, rows, vocab, top, dtype, cap):
    x, t = _logits(gpu, rows, vocab, dtype, rows * 1000 + vocab)
    _check(x, t, top, cap)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_begin_anywhere(gpu, dtype):
    """Strided rows, of an odd length, from an odd offset: 16-byte pieces cross both ends of a row."""
    big, _ = _logits(gpu, 6, 5000, dtype, 1)
    for first, vocab in ((1, 4001), (3, 4093), (7, 999), (5, 8)):
        _check(big[:, first:first + vocab], torch.tensor([0, vocab - 1, vocab // 2, 1, 2, 3], device=gpu) % vocab, 8, 0.0)


def test_the_largest_cap(gpu):
    x, t = _logits(gpu, 3, 5000, torch.float32, 7)
    _check(x, t, 6, 1024.0)


@pytest.mark.parametrize("rows,vocab", [(3, 5000), (2, 40_007), (1100, 2111)])
@pytest.mark.parametrize("cap", [65.0, 300.0, 1024.0])
def test_a_large_cap_leaves_small_logits_their_digits(gpu, cap, rows, vocab):
    """z is off by a few units of 2^-24 of itself (the quotient, a hyperbolic tangent good to 2 units, the product), not
    of the cap: logits of up to 8 here, so 2^-24 * 4 * 8 = 2^-19 beside the sums' own roundings."""
    from se12_amd.logprobs import token_logprobs

    x, t = _logits(gpu, rows, vocab, torch.float32, 9, scale=1.5)
    x = x.clamp(-8, 8)
    r = token_logprobs(x, t, top=3, softcap=cap)
    z = cap * torch.tanh(x.cpu().double() / cap)
    lp = z - torch.logsumexp(z, 1, keepdim=True)
    want, ent = lp.gather(1, t.cpu()[:, None])[:, 0], torch.special.entr(lp.exp()).sum(1)
    tol = lambda size: _tol(vocab, 0.0, size) + 2.0 ** -18      # noqa: E731  (of a logit and of those in the sum)
    assert ((r.logprobs.cpu().double() - want).abs() <= tol(want)).all()
    assert ((r.top_logprobs.cpu().double() - lp.gather(1, r.top_ids.cpu())).abs() <= tol(lp.gather(1, r.top_ids.cpu()))).all()
    assert ((r.entropy.cpu().double() - ent).abs() <= 2 * (1 + math.log(vocab)) * tol(ent)).all()


@pytest.mark.parametrize("cap", [20.0, 30.0, 64.0, 1000.0])
def test_two_capped_logits_keep_their_digits(gpu, cap):
    """Rows of two logits of up to 4: each z is off by 3 units of 2^-24 of itself at most (2 of its form, one of rounding),
    their difference d by 2^-24 * 24, log p = -log(1 + e^d) by no more and a few units of its own. Rows of larger ones,
    up to 1.5 caps: 4 units of the cap's half each (the quotient counts once more beyond cap / 2)."""
    from se12_amd.logprobs import token_logprobs

    for scale, off in ((1.0, 24 * 2.0 ** -24), (cap, 8 * cap * 2.0 ** -24)):
        x = (torch.rand((4096, 2), generator=_gen(10)) * 2 - 1) * (4.0 if scale == 1.0 else 1.5 * cap)
        t = torch.randint(0, 2, (4096,), generator=_gen(11))
        r = token_logprobs(x.to(gpu), t.to(gpu), top=2, softcap=cap)
        lp = torch.log_softmax(cap * torch.tanh(x.double() / cap), 1)
        want, ent = lp.gather(1, t[:, None])[:, 0], torch.special.entr(lp.exp()).sum(1)
        tol = off + 2.0 ** -22 * (1 + want.abs())
        assert ((r.logprobs.cpu().double() - want).abs() <= tol).all(), ((r.logprobs.cpu().double() - want).abs() / tol).max()
        assert (r.logprobs <= 0).all() and (r.entropy >= 0).all()
        # (the entropy's derivative by d is d p (1 - p), below 1/2)
        assert ((r.entropy.cpu().double() - ent).abs() <= off + 2.0 ** -21).all()


@pytest.mark.parametrize("cap", [2.0 ** -60, 2.0 ** -15, 2.0 ** -14, 1e-3, 1.0])
def test_small_caps(gpu, cap):
    """Both sides of the least cap whose coefficients FP32 holds, and the least of all."""
    from se12_amd.logprobs import token_logprobs

    x, t = _logits(gpu, 3, 5000, torch.float32, 12)
    x[1] *= cap
    x[2, :2500] *= cap / 8
    r = token_logprobs(x, t, top=4, softcap=cap)
    z = cap * torch.tanh(x.cpu().double() / cap)
    lp = z - torch.logsumexp(z, 1, keepdim=True)
    want = lp.gather(1, t.cpu()[:, None])[:, 0]
    assert ((r.logprobs.cpu().double() - want).abs() <= _tol(5000, 0.0, want)).all()
    ent = torch.special.entr(lp.exp()).sum(1)
    assert ((r.entropy.cpu().double() - ent).abs() <= 2 * (1 + math.log(5000)) * _tol(5000, 0.0, ent)).all()
    ids = torch.sort(x.cpu(), dim=1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(r.top_ids.cpu(), ids)


def test_more_rows_than_blocks_fill_the_card(gpu):
    x, t = _logits(gpu, 1500, 2100, torch.bfloat16, 2)
    _check(x, t, 3, 0.0)


def test_equal_logits_go_by_the_lower_index(gpu):
    for vocab in (64, 5000, 70000):
        x = torch.zeros((2, vocab), device=gpu)
        x[1, ::3] = 1.0
        x[0, 1::2] = -0.0
        _check(x, torch.tensor([0, 1], device=gpu), 32, 0.0)
        _check(x.to(torch.bfloat16), torch.tensor([0, 1], device=gpu), 32, 5.0)
    # ascending and descending: every chunk, or only the first, passes the bar
    x = torch.arange(30000, device=gpu).float()[None] / 1000
    _check(torch.cat([x, x.flip(1)]), torch.tensor([29999, 0], device=gpu), 20, 0.0)


def test_masked_logits(gpu):
    x, t = _logits(gpu, 8, 20000, torch.float32, 3)
    allowed = torch.rand((8, 20000), device=gpu) < 0.01
    allowed[3] = False
    allowed[3, 17] = True                       # one token is certain
    allowed[4] = False
    allowed[4, :2] = True
    t[3], t[4] = 17, 1
    allowed.scatter_(1, t[:, None], True)
    _check(x.masked_fill(~allowed, float("-inf")), t, 20, 0.0)
    # the type's lowest value is a logit like others: a row of it alone is uniform
    low = torch.full((2, 3000), torch.finfo(torch.float32).min, device=gpu)
    low[1, 5] = 3.0
    _check(low, torch.tensor([7, 5], device=gpu), 4, 0.0)
    low = torch.full((1, 3000), torch.finfo(torch.bfloat16).min, device=gpu, dtype=torch.bfloat16)
    _check(low, torch.tensor([7], device=gpu), 4, 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_best_are_zeros(gpu, dtype):
    """0 and -0 tie; they are above every number below, the smallest ones too."""
    x, t = _logits(gpu, 3, 20_000, dtype, 6)
    x = -x.relu()
    x[1] = torch.where(x[1] == 0, -1e-38, x[1])
    x[1, ::37] = torch.where(x[1, ::37] > -1, 0.0, x[1, ::37])
    x[2, :9_000] = -1.0
    x[2, 9_003] = -0.0
    x[2, 15_000] = 0.0
    _check(x, t, 7, 0.0)


@pytest.mark.parametrize("rows,cap", [(400, 0.0), (1100, 0.0), (400, 30.0)])
def test_a_peak_that_comes_late_in_a_row(gpu, rows, cap):
    """Two logits hold the row: one in a wave's first chunk, the peak up to 8 above it in its second. The sums are S = 1 +
    e^-gap and W = gap e^-gap on the peak's reference: a few roundings of 2^-24 each (of the sums, a term's exponent at
    most 8 2^-23, under the cap z by 2^-21 of it), so nothing of the size of the gap's own rounding is left in results
    near 0. None is above 0 as a logarithm, or below as an entropy."""
    from se12_amd.logprobs import token_logprobs

    gap = torch.rand(rows, generator=_gen(8)) * 8
    x = torch.full((rows, 9007), -1e4)
    x[:, 5], x[:, 1500] = 3.0, 3.0 + gap
    for order in (x, x.flip(1)):
        r = token_logprobs(order.to(gpu), order.argmax(1).to(gpu), top=2, softcap=cap)
        z = order.double()
        z = cap * torch.tanh(z / cap) if cap else z
        lp = z - torch.logsumexp(z, 1, keepdim=True)
        want, ent = lp.amax(1), torch.special.entr(lp.exp()).sum(1)
        tol = 2.0 ** -22 + (cap * 2.0 ** -21 + 2.0 ** -20) * (1 - want.exp()) + 2.0 ** -22 * want.abs()
        assert (r.logprobs <= 0).all() and (r.entropy >= 0).all() and (r.top_logprobs <= 0).all()
        assert ((r.logprobs.cpu().double() - want).abs() <= tol).all()
        assert ((r.top_logprobs[:, 0].cpu().double() - want).abs() <= tol).all()
        assert ((r.entropy.cpu().double() - ent).abs() <= 9 * tol).all()


def test_rows_without_a_distribution(gpu):
    from se12_amd.logprobs import token_logprobs

    for vocab in (40, 9000):
        x, _ = _logits(gpu, 6, vocab, torch.float32, 4)
        x[0] = float("-inf")
        x[1, 33] = float("nan")
        x[2, 7] = float("inf")
        x[3] = float("nan")
        x[4] = float("-inf")
        x[4, 9] = float("nan")
        t = torch.tensor([3, 2, 1, 0, 0, vocab], device=gpu)
        r = token_logprobs(x, t, top=5)
        assert r.logprobs[0] == float("-inf") and r.entropy[0] == 0 and (r.top_logprobs[0] == float("-inf")).all()
        assert r.top_ids[0].tolist() == [0, 1, 2, 3, 4] and r.top_ids[3].tolist() == [0, 1, 2, 3, 4]
        assert r.top_ids[4].tolist() == [0, 1, 2, 3, 4]
        for i in (1, 2, 3, 4):
            assert r.logprobs[i].isnan() and r.entropy[i].isnan() and r.top_logprobs[i].isnan().all()
        row = x[1].clone()
        row[33] = float("-inf")
        assert r.top_ids[1].tolist() == torch.sort(row, descending=True, stable=True).indices[:5].tolist()
        assert r.top_ids[2][0] == 7
        # a token that there is not
        assert r.logprobs[5] == float("-inf") and r.entropy[5].isfinite()
        assert token_logprobs(x[5:], torch.tensor([-100], device=gpu)).logprobs[0] == float("-inf")


def test_no_rows_and_a_graph(gpu):
    from se12_amd.logprobs import token_logprobs

    r = token_logprobs(torch.empty((0, 50), device=gpu), torch.empty(0, dtype=torch.int64, device=gpu), top=3)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 3)
    x, t = _logits(gpu, 2, 30000, torch.float32, 5)
    token_logprobs(x, t, top=4)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        r = token_logprobs(x, t, top=4, softcap=20.0)
    for i in range(4):
        x.copy_(_logits(gpu, 2, 30000, torch.float32, 6 + i)[0])
        graph.replay()
        e = token_logprobs(x, t, top=4, softcap=20.0)
        assert torch.equal(r.logprobs, e.logprobs) and torch.equal(r.top_ids, e.top_ids) and torch.equal(r.entropy, e.entropy)
        assert torch.equal(r.top_logprobs, e.top_logprobs)
