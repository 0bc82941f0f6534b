"""Paged key/value cache on the GPU: PagedKvCache.append and .attend against the
64-bit forms of tests/paged_oracle.py.

Tolerances. A rounding to BF16 is off by at most 2^-8 of the value (half of
torch.finfo(bfloat16).eps), one to E4M3 by 2^-4 or, below its smallest normal
2^-6, by half its least step, 2^-10 (both in units of the scale). Rotation: the
angle's fraction of a turn is rounded to FP32 (2^-24 of at most pi), sine, cosine
and the two products and their sum a few units of 2^-24 each: within 2^-20 of |a| +
|b|. Attention: a weight is rounded to BF16 (2^-8 of its share of sum w |v|), the
scores are FP32 sums of head_dim products (head_dim 2^-24 of sum |q k| scaling, at
most 40 here: 2^-11 for the weight's exponent, twice for numerator and
denominator), the output once more to BF16."""

from __future__ import annotations

import pytest
import torch

import paged_oracle as o

pytestmark = pytest.mark.gpu

E4M3, BF16 = torch.float8_e4m3fn, torch.bfloat16


def _codes(t: torch.Tensor) -> torch.Tensor:
    return t.cpu().float().double()


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _table(seqs: int, columns: int, pages: int, seed: int) -> list[list[int]]:
    order = torch.randperm(pages, generator=_gen(seed)).tolist()
    return [order[i * columns:(i + 1) * columns] for i in range(seqs)]


def _cache(gpu, pages, page, kvh, d, dtype, seed, scale_exponents=(-8, -2), garbage=None):
    """A pool of other sequences' leftovers: random values (or `garbage` bytes in every slot), random scales."""
    from se12_amd.paged import PagedKvCache

    g = _gen(seed)
    c = PagedKvCache(pages, page, kvh, d, dtype=dtype, device=gpu)
    if dtype == E4M3:
        for t in (c.k, c.v):
            t.copy_((torch.randn(t.shape, generator=g) * 60).clamp(-448, 448).to(E4M3))
        for t in (c.k_scale, c.v_scale):
            t.copy_(torch.exp2(torch.randint(*scale_exponents, t.shape, generator=g).float()))
    else:
        for t in (c.k, c.v):
            t.copy_(torch.randn(t.shape, generator=g).to(BF16))
    return c


def _batch(gpu, table, lengths, new, max_new=None):
    from se12_amd.paged import PagedBatch

    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    as32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    return PagedBatch(as32(table), as32(lengths), as32(starts), max_new=max_new or max(new)), starts


def _state(c):
    return (_codes(c.k), _codes(c.v), None if c.k_scale is None else c.k_scale.cpu().clone(),
            None if c.v_scale is None else c.v_scale.cpu().clone())


def _check_append(c, before, batch, lengths, starts, table, k, v, inv_freq, q=None, got_q=None):
    """The cache after an append against the oracle's, from the state before."""
    kp, vp, ks, vs = before
    e4m3 = ks is not None
    f = None if inv_freq is None else inv_freq.cpu()
    q_ref, written = o.append(kp, vp, ks, vs, table, lengths, starts, k.cpu(), v.cpu(), f, batch.max_new, None if q is None else q.cpu())
    if q is not None:
        n = starts[-1]
        size = q.cpu().double().abs()[:n]
        err = (got_q.cpu().double()[:n] - q_ref[:n]).abs()
        assert (err <= 2.0 ** -8 * q_ref[:n].abs() + 2.0 ** -20 * (size + size.amax(-1, keepdim=True))).all()
    slots = written[:, None, :, None].expand_as(kp)
    got_k, got_v = _codes(c.k), _codes(c.v)
    if e4m3:
        assert torch.equal(c.k_scale.cpu(), ks) and torch.equal(c.v_scale.cpu(), vs)
        # v is not rotated: its codes are exact, NaN where NaN was
        assert torch.equal(got_v.nan_to_num(1000.0), vp.nan_to_num(1000.0))
        # k: an element whose rotated value lies within 2^-20 of a rounding border may go either way (a step: 2^-3)
        same = (got_k == kp) | (got_k.isnan() & kp.isnan())
        assert same[~slots].all()
        assert ((got_k - kp).abs()[~same] <= 2.0 ** -3 * kp.abs()[~same] + 2.0 ** -9).all()
        assert (~same).sum() <= 1 + 1e-4 * slots.sum()
    else:
        assert torch.equal(got_v, vp.to(BF16).double())
        tol = torch.where(slots, 2.0 ** -8 * kp.abs() + 2.0 ** -20 * 2 * kp.abs().amax(-1, keepdim=True), torch.zeros_like(kp))
        assert ((got_k - kp).abs() <= tol).all()


@pytest.mark.parametrize("x_dtype", [torch.float32, BF16])
@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("d,page,kvh,heads,rotary,lengths,new", [
    (256, 64, 4, 8, 256, [0, 63, 64, 200], [1, 1, 1, 1]),                 # decode: first slot, last slot, new page
    (128, 16, 2, 14, 128, [0, 5, 31, 16], [40, 3, 17, 1]),                # pages of 16, seven heads to one
    (64, 32, 1, 1, 32, [7, 0, 100], [0, 70, 5]),                          # half of a head rotated; a sequence with nothing
    (256, 128, 2, 2, 256, [100, 1], [300, 127]),                          # pages of 128 begun and left inside
    (64, 64, 3, 9, 0, [3, 3, 3], [16, 15, 2]),                            # no rotation
])
def test_append(gpu, x_dtype, dtype, d, page, kvh, heads, rotary, lengths, new):
    total = sum(new)
    columns = max((a + b + page - 1) // page for a, b in zip(lengths, new)) + 1
    table = _table(len(new), columns, len(new) * columns + 2, 1)
    c = _cache(gpu, len(new) * columns + 2, page, kvh, d, dtype, 2)
    batch, starts = _batch(gpu, table, lengths, new)
    g = _gen(3)
    # views of one product's rows, as a fused projection gives them, and rows behind the last sequence
    x = (torch.randn((total + 3, (heads + 2 * kvh) * d), generator=g) * 2).to(x_dtype).to(gpu)
    q, k, v = (t.view(total + 3, -1, d) for t in x.split([heads * d, kvh * d, kvh * d], 1))
    inv = (10000.0 ** (-torch.arange(0, rotary, 2).float() / rotary)).to(gpu) if rotary else None
    before = _state(c)
    out = torch.full((total + 3, heads, d), 7.0, dtype=BF16, device=gpu)
    got = c.append(batch, k, v, q=q, inv_freq=inv, out=out)
    assert got is out and (out[total:] == 7.0).all()
    _check_append(c, before, batch, lengths, starts, table, k, v, inv, q, got)


def test_append_rotates_q_in_place(gpu):
    c = _cache(gpu, 4, 32, 2, 128, E4M3, 70)
    batch, _ = _batch(gpu, [[0, 1], [2, 3]], [20, 3], [30, 1])
    q = torch.randn((31, 8, 128), generator=_gen(71)).to(BF16).to(gpu)
    k, v = (torch.randn((31, 2, 128), generator=_gen(72 + i)).to(BF16).to(gpu) for i in range(2))
    inv = (10000.0 ** (-torch.arange(0, 64).float() / 64)).to(gpu)
    apart = c.append(batch, k, v, q=q, inv_freq=inv)
    assert c.append(batch, k, v, q=q, inv_freq=inv, out=q) is q and torch.equal(q, apart)


def test_one_token_in_rows_of_any_distance(gpu):
    """A single token's heads transposed, its row of an odd length: as a copy of it gives."""
    c, d = _cache(gpu, 4, 32, 4, 128, E4M3, 73), 128
    batch, _ = _batch(gpu, [[0, 1]], [20], [1])
    g = _gen(74)
    for dtype in (torch.float32, BF16):
        x = torch.randn((1, 16, 1, d), generator=g).to(dtype).to(gpu)
        rows = torch.randn((2, 16 * d + 3), generator=g).to(dtype).to(gpu)
        for t in (x.transpose(1, 2)[0], rows[:1, :16 * d].view(1, 16, d), rows[1:, 3:].view(1, 16, d)):
            q, k, v = t.split([8, 4, 4], 1)
            got = c.append(batch, k, v, q=q)
            state = _state(c)
            assert torch.equal(got, c.append(batch, k.clone(), v.clone(), q=q.clone())) and torch.equal(got, q.to(BF16))
            for a, b in zip(state, _state(c)):
                assert torch.equal(a, b)
            q = q.to(BF16) if dtype == BF16 else got
            assert torch.equal(c.attend(batch, q, 0.1), c.attend(batch, q.clone(memory_format=torch.contiguous_format), 0.1))


def test_calls_without_tokens(gpu):
    for dtype in (E4M3, BF16):
        c = _cache(gpu, 2, 16, 2, 64, dtype, 75)
        batch, _ = _batch(gpu, [[0], [1]], [3, 0], [0, 0], max_new=1)
        before = _state(c)
        k, q = torch.empty((0, 2, 64), device=gpu), torch.empty((0, 8, 64), device=gpu)
        assert c.append(batch, k, k) is None
        assert c.append(batch, k, k, q=q).shape == (0, 8, 64) and c.attend(batch, q.to(BF16), 0.125).shape == (0, 8, 64)
        out = torch.empty((0, 8, 64), dtype=BF16, device=gpu)
        assert c.append(batch, k, k, q=q, out=out) is out and c.attend(batch, q.to(BF16), 0.125, out=out) is out
        for a, b in zip(before, _state(c)):
            assert a is b is None or torch.equal(a, b)


def test_append_without_q_and_with_a_far_position(gpu):
    """Positions where an FP32 angle has lost every digit behind the point of a turn's hundredth."""
    lengths, new = [250_000, 131_071], [3, 2]
    table = [[-1] * 16000 for _ in new]
    pages, page = 5, 16
    for s, (a, n) in enumerate(zip(lengths, new)):
        for j in range(a // page, (a + n - 1) // page + 1):
            table[s][j] = 2 * s + j - a // page
    c = _cache(gpu, pages, page, 2, 128, BF16, 5)
    batch, starts = _batch(gpu, table, lengths, new)
    k, v = (torch.randn((5, 2, 128), generator=_gen(6 + i)).to(gpu) for i in range(2))
    inv = (10000.0 ** (-torch.arange(0, 128, 2).float() / 128)).to(gpu)
    before = _state(c)
    assert c.append(batch, k, v, inv_freq=inv) is None
    _check_append(c, before, batch, lengths, starts, table, k, v, inv)


def test_rotations_are_as_close_as_fp32_sines_of_64_bit_angles(gpu):
    """Of 42 million turned values, rounded to BF16, those that are not the exact rotation's: no more than of FP32
    arithmetic with sines and cosines rounded from 64 bits, which rounds once more (a product) per value."""
    c, d, heads = _cache(gpu, 40, 64, 8, 256, BF16, 77), 256, 8
    lengths, new = [0, 40_000, 3], [300, 500, 224]
    batch, starts = _batch(gpu, [[-1] * 700] * 3, lengths, new)
    inv = (10000.0 ** (-torch.arange(0, d, 2).float() / d)).to(gpu)
    k = torch.zeros((1024, 8, d), device=gpu)
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(lengths, new)]).to(gpu)
    angle = pos.double()[:, None, None] * inv.double()
    far = [0, 0]
    for seed in range(20):
        q = torch.randn((1024, heads, d), generator=_gen(78 + seed)).to(gpu)
        a, b = q[..., :128], q[..., 128:]
        exact = torch.cat([a.double() * angle.cos() - b.double() * angle.sin(), b.double() * angle.cos() + a.double() * angle.sin()], -1)
        cos, sin = angle.cos().float(), angle.sin().float()
        plain = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        got = c.append(batch, k, k, q=q, inv_freq=inv)
        want = exact.to(BF16)
        far[0] += (got != want).sum().item()
        far[1] += (plain.to(BF16) != want).sum().item()
    assert far[0] <= far[1], far


def test_scales_grow_and_older_tokens_are_rounded_again(gpu):
    page, kvh, d = 16, 2, 64
    c = _cache(gpu, 4, page, kvh, d, E4M3, 7)
    table, length = [[2, 0, 3]], 0
    sizes = [1e-3, 1e-3, 0.5, 0.0, 300.0, 1e-30, 1e4, 3e37, 1e-6, 1.0, 0.25, 1e-38, 2.0, 448.0, 449.0, 5.0, 1e-3, 1e-3, 1e-2]
    for i, size in enumerate(sizes):
        batch, starts = _batch(gpu, table, [length], [1])
        k, v = (torch.randn((1, kvh, d), generator=_gen(50 + 2 * i + j)).mul_(size).to(gpu) for j in range(2))
        if size in (448.0, 449.0):
            v[0, 0, 0] = size * 2.0 ** 30       # the largest value at, and just over, what a scale holds
        before = _state(c)
        c.append(batch, k, v)
        _check_append(c, before, batch, [length], starts, table, k, v, None)
        length += 1


def test_values_that_are_no_numbers_are_held_as_nan(gpu):
    c = _cache(gpu, 2, 16, 1, 64, E4M3, 8)
    batch, starts = _batch(gpu, [[1]], [0], [3])
    k, v = (torch.randn((3, 1, 64), generator=_gen(80 + i)).to(gpu) for i in range(2))
    k[0, 0, 3], k[1, 0, 5], v[2, 0, 7], v[0, 0, :] = float("nan"), float("inf"), float("-inf"), float("nan")
    before = _state(c)
    c.append(batch, k, v)
    _check_append(c, before, batch, [0], starts, [[1]], k, v, None)
    assert _codes(c.k)[1, 0, 0, 3].isnan() and _codes(c.k)[1, 0, 1, 5].isnan() and _codes(c.v)[1, 0, 7, 2].isnan()


def test_tokens_without_a_page_are_held_nowhere(gpu):
    """Pages outside the pool, positions outside the table, more new tokens than max_new."""
    for dtype in (E4M3, BF16):
        c = _cache(gpu, 3, 16, 2, 64, dtype, 9)
        table, lengths, new = [[-1, 1], [0, 3], [2, 1 << 30], [-5, -5]], [10, 14, 31, 32], [9, 5, 4, 2]
        batch, starts = _batch(gpu, table, lengths, new, max_new=6)
        k, v = (torch.randn((sum(new), 2, 64), generator=_gen(90 + i)).to(gpu) for i in range(2))
        q = torch.randn((sum(new), 4, 64), generator=_gen(92)).to(gpu)
        before = _state(c)
        out = c.append(batch, k, v, q=q, out=torch.zeros((sum(new), 4, 64), dtype=BF16, device=gpu))
        kp, vp, ks, vs = (None if t is None else t.clone() for t in before)
        _check_append(c, before, batch, lengths, starts, table, k, v, None)
        assert (out[6:9] == 0).all() and torch.equal(out[:6], q[:6].to(BF16))
        assert torch.equal(_codes(c.k)[2], kp[2])      # pages no token reached
        del kp, vp, ks, vs


def test_append_beyond_32_bit_offsets(gpu):
    """A pool whose last pages lie past 2^32 elements."""
    from se12_amd.paged import PagedKvCache

    page, kvh, d = 128, 8, 256
    pages = 2 ** 32 // (page * kvh * d) + 3
    c = PagedKvCache(pages, page, kvh, d, device=gpu)
    table, lengths, new = [[pages - 1, 0], [pages - 2, 1]], [100, 3], [40, 1]
    batch, starts = _batch(gpu, table, lengths, new)
    k, v = (torch.randn((41, kvh, d), generator=_gen(100 + i)).to(gpu) for i in range(2))
    c.append(batch, k, v)
    ids = [pages - 1, 0, pages - 2, 1]
    kp, vp = torch.zeros((4, kvh, page, d), dtype=torch.float64), torch.zeros((4, kvh, d, page), dtype=torch.float64)
    ks, vs = torch.ones((4, kvh)), torch.ones((4, kvh))
    o.append(kp, vp, ks, vs, [[0, 1], [2, 3]], lengths, starts, k.cpu(), v.cpu(), None, 40)
    assert torch.equal(_codes(c.k[ids]), kp) and torch.equal(_codes(c.v[ids]), vp)
    assert torch.equal(c.k_scale[ids].cpu(), ks)
    q = torch.randn((41, 16, d), generator=_gen(102)).to(BF16).to(gpu)
    got = c.attend(batch, q, 0.0625)
    # the keys before the new tokens are zeros of an unused pool, scale 1 or the page's
    ref, size, _ = o.attend(kp, vp, ks, vs, [[0, 1], [2, 3]], lengths, starts, q.cpu(), 0.0625, 0.0, 0, 40)
    _close(got, ref, size)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def _close(got, ref, size, rows=slice(None)):
    err = (got.cpu().double() - ref).abs()[rows]
    tol = (2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -10) * size + 1e-30)[rows]
    assert (err <= tol).all(), (err / tol).max()


def _poison(c, table, keys, page):
    """NaN in every slot that no sequence of the call holds."""
    held = torch.zeros((c.pages, page), dtype=torch.bool)
    for s, n in enumerate(keys):
        for j in range(n):
            if j // page < len(table[s]) and 0 <= table[s][j // page] < c.pages:
                held[table[s][j // page], j % page] = True
    held = held.to(c.device)
    nan = torch.tensor(float("nan"), device=c.device)
    for t, m in ((c.k, held[:, None, :, None]), (c.v, held[:, None, None, :])):
        t.copy_(torch.where(m, t.float(), nan).to(t.dtype))
    if c.k_scale is not None:
        empty = ~held.any(1)
        c.k_scale[empty], c.v_scale[empty] = float("nan"), float("nan")


def test_pages_behind_the_window_may_be_anything(gpu):
    """Pages no query sees any more went to others: their values and scales are NaN, or the table names no page."""
    for new in (1, 40):
        c, batch, q, before = _attend_case(gpu, E4M3, 128, 16, 4, 1, [200], [new], 0.0, 60, seed=7, extra=0)
        gone = (200 - 60 + 1) // 16
        ids = batch.page_table[0, :gone].long()
        c.k.view(torch.uint8)[ids] = 127
        c.v.view(torch.uint8)[ids] = 127
        c.k_scale[ids], c.v_scale[ids] = float("nan"), float("inf")
        assert torch.equal(c.attend(batch, q, 128 ** -0.5, window=60), before)
        batch.page_table[0, :gone] = torch.tensor([-1, 1 << 30] * 8, dtype=torch.int32, device=gpu)[:gone]
        assert torch.equal(c.attend(batch, q, 128 ** -0.5, window=60), before)


def _attend_case(gpu, dtype, d, page, heads, kvh, lengths, new, softcap, window, seed=0, max_new=None, extra=2, scales=(-7, -4)):
    columns = max((a + b + page - 1) // page for a, b in zip(lengths, new)) + 1
    pages = len(new) * columns + 1
    table = _table(len(new), columns, pages, seed + 1)
    c = _cache(gpu, pages, page, kvh, d, dtype, seed + 2, scale_exponents=scales)
    _poison(c, table, [a + b for a, b in zip(lengths, new)], page)
    batch, starts = _batch(gpu, table, lengths, new, max_new)
    total = starts[-1] + extra
    x = torch.randn((total, (heads + 3) * d), generator=_gen(seed + 3)).to(BF16).to(gpu)
    q = x[:, d:(heads + 1) * d].view(total, heads, d)
    out = torch.full((total, heads, d), 3.0, dtype=BF16, device=gpu)
    assert c.attend(batch, q, d ** -0.5, softcap=softcap, window=window, out=out) is out
    kp, vp, ks, vs = _state(c)
    ref, size, mine = o.attend(kp, vp, ks, vs, table, lengths, starts, q.cpu(), d ** -0.5, softcap, window, batch.max_new)
    _close(out, ref, size, mine)
    assert (out.cpu()[~mine] == 3.0).all()
    return c, batch, q, out


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("d,page,heads,kvh,lengths,new,softcap,window", [
    (256, 64, 8, 4, [0, 1, 63, 64, 300], [1, 1, 1, 1, 1], 50.0, 0),       # decode, from the first token
    (256, 32, 16, 8, [130, 31, 640], [1, 1, 1], 50.0, 100),              # a window that begins inside a page
    (128, 16, 28, 4, [700, 16, 15], [1, 1, 1], 0.0, 0),                  # seven heads to one, pages of 16
    (64, 128, 5, 1, [0, 127, 1000], [1, 1, 1], 0.0, 1),                  # one key seen
    (128, 32, 6, 2, [0, 33, 200, 8], [5, 1, 9, 0], 0.0, 0),              # drafted tokens; 27 columns; a sequence with none
    (256, 16, 4, 4, [3, 0, 90], [40, 65, 33], 50.0, 17),                 # prompts under a window shorter than they are
    (64, 64, 24, 1, [50, 0], [3, 130], 0.0, 64),                         # more heads than a unit's columns
    (256, 64, 8, 4, [700, 1500, 0, 33], [70, 1, 129, 40], 50.0, 0),       # prompts beside a decode step
    (128, 32, 8, 1, [2100], [60], 0.0, 0),                               # few columns, many keys: a unit's keys in parts
    (128, 16, 6, 2, [500, 3], [200, 64], 30.0, 100),                     # a window over columns that share a block
    (64, 16, 8, 8, [0, 2000], [65, 129], 0.0, 0),                        # one column into the second, third block
])
def test_attend(gpu, dtype, d, page, heads, kvh, lengths, new, softcap, window):
    _attend_case(gpu, dtype, d, page, heads, kvh, lengths, new, softcap, window)


def test_attend_many_sequences(gpu):
    """More sequences than a wave scans at once, most of them short, some empty."""
    lengths = [(i * 37) % 90 for i in range(150)]
    _attend_case(gpu, E4M3, 64, 16, 2, 1, lengths, [1 if i % 7 else 0 for i in range(150)], 0.0, 0)


def _again(c, batch, q, d, softcap, window, bound=2.0 ** -10):
    """The call once more, on what the cache and the batch hold now; `bound`: of the weights' exponents."""
    kp, vp, ks, vs = _state(c)
    table, lengths, starts = batch.page_table.tolist(), batch.lengths.tolist(), batch.starts.tolist()
    ref, size, mine = o.attend(kp, vp, ks, vs, table, lengths, starts, q.cpu(), d ** -0.5, softcap, window, batch.max_new)
    err = (c.attend(batch, q, d ** -0.5, softcap=softcap, window=window).cpu().double() - ref).abs()[mine]
    assert (err <= (2.0 ** -8 * ref.abs() + (2.0 ** -8 + bound) * size + 1e-30)[mine]).all()


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("d,page,heads,kvh,softcap,window", [(64, 32, 16, 8, 0.0, 0), (64, 16, 8, 8, 30.0, 333), (128, 64, 28, 4, 0.0, 500),
                                                             (256, 32, 8, 4, 50.0, 490)])
def test_many_tiles_to_a_wave(gpu, dtype, d, page, heads, kvh, softcap, window):
    """More key tiles than the card has waves: a wave's run goes from tile to tile and over the ends of sequences, from
    tiles that a window or a missing page cuts into whole ones."""
    lengths = [(i * 271) % 1100 for i in range(48)]
    c, batch, q, _ = _attend_case(gpu, dtype, d, page, heads, kvh, lengths, [1] * 48, softcap, window, seed=30, extra=0)
    gone = torch.rand(batch.page_table.shape, generator=_gen(31)) < 0.3
    batch.page_table[gone.to(gpu)] = -1
    _again(c, batch, q, d, softcap, window)


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("seqs,new,max_new,length,window", [(600, (1, 1, 0), 1, 150, 0), (150, (1, 2, 1, 0), 200, 700, 0), (90, (1, 7, 25), 40, 300, 60),
                                                            (600, (1,), 1, 20, 0), (900, (1,), 1, 90, 0)])
def test_more_units_than_waves(gpu, dtype, seqs, new, max_new, length, window):
    """Units that several waves share are joined by those that begin them."""
    lengths = [(i * 271) % length for i in range(seqs)]
    news = [new[i % len(new)] for i in range(seqs)]
    if max_new == 200:
        news[77], lengths[5] = 100, 6000
    _attend_case(gpu, dtype, 64, 16, 8, 4 if seqs < 100 else 2, lengths, news, 0.0, window, seed=36, max_new=max_new)


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("window", [0, 90])
def test_prompts_among_more_sequences_than_a_wave_scans(gpu, dtype, window):
    """Units of prompts in the second 64 sequences too, decode steps and sequences with nothing between them."""
    new = [(0, 1, 1, 1, 5)[i % 5] for i in range(100)]
    new[3], new[70], new[71], new[99] = 40, 33, 90, 70
    lengths = [(i * 53) % 150 for i in range(100)]
    _attend_case(gpu, dtype, 64, 16, 4, 2, lengths, new, 0.0, window, seed=60)


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("d,window", [(64, 1000), (256, 700)])
def test_parts_of_a_units_keys_under_a_window(gpu, dtype, d, window):
    _attend_case(gpu, dtype, d, 32, 4, 1, [2600, 900], [70, 35], 0.0, window, seed=61)


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("heads,kvh,lengths,new", [(4, 1, [2600, 900], [70, 35]), (4, 2, [300, 70], [1, 1])])
def test_a_window_of_the_largest_number_hides_nothing(gpu, dtype, heads, kvh, lengths, new):
    c, batch, q, out = _attend_case(gpu, dtype, 64, 32, heads, kvh, lengths, new, 0.0, 2 ** 31 - 1, seed=67, extra=0)
    for window in (0, 2 ** 31 - 40, 1 << 30):
        assert torch.equal(c.attend(batch, q, 64 ** -0.5, window=window), out)


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_more_query_heads_to_one_than_columns_of_a_block(gpu, dtype):
    _attend_case(gpu, dtype, 64, 16, 160, 1, [100, 5, 0], [1, 3, 1], 0.0, 0, seed=62)
    _attend_case(gpu, dtype, 64, 16, 80, 1, [300, 5], [1, 2], 0.0, 70, seed=63)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_first_tiles_of_prompts_from_bf16_pages(gpu, d):
    """Keys of the tile after next go over those of the first: many units of one, two, three and four tiles of 32 keys,
    a few times, all with the same result. (A wave ahead of the others must not overwrite what they still read.)"""
    lengths, new = [0, 20, 31, 0, 60, 3], [32, 40, 65, 33, 60, 90]
    c, batch, q, out = _attend_case(gpu, BF16, d, 16, 32, 16, lengths, new, 0.0, 0, seed=71, extra=0)
    for _ in range(20):
        assert torch.equal(c.attend(batch, q, d ** -0.5), out)


def test_more_allowed_new_tokens_than_there_are(gpu):
    """max_new is a bound: decode steps beside kernels for prompts that find nothing to do."""
    _attend_case(gpu, E4M3, 128, 32, 8, 2, [100, 33, 0], [1, 1, 1], 0.0, 0, seed=64, max_new=500)
    _attend_case(gpu, BF16, 64, 16, 2, 2, [100] * 80, [1] * 80, 0.0, 20, seed=65, max_new=100)


def test_sequences_that_share_pages(gpu):
    """The same pages under two sequences, and one page twice in a row, are read like others."""
    for dtype in (E4M3, BF16):
        c, batch, q, _ = _attend_case(gpu, dtype, 128, 32, 4, 2, [200, 170, 90], [1, 3, 40], 0.0, 0, seed=66, extra=0)
        batch.page_table[1, :5] = batch.page_table[0, :5]
        batch.page_table[2, 1] = batch.page_table[2, 0]
        _again(c, batch, q, 128, 0.0, 0)


@pytest.mark.parametrize("cap", [2.0 ** -60, 0.01])
@pytest.mark.parametrize("new", [1, 50])
def test_small_caps(gpu, cap, new):
    for dtype in (E4M3, BF16):
        _attend_case(gpu, dtype, 64, 32, 4, 2, [600, 3], [new, 1], cap, 0, seed=51, extra=0)


@pytest.mark.parametrize("new", [1, 50])
def test_the_largest_cap(gpu, new):
    """A score is held to 2^-22 of the cap, here 2^-12, twice in a quotient of sums."""
    c, batch, q, _ = _attend_case(gpu, E4M3, 128, 32, 4, 2, [600, 3], [new, 1], 0.0, 0, seed=50, extra=0)
    _again(c, batch, q, 128, 1024.0, 0, bound=2.0 ** -10 + 2.0 ** -11)


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("d,heads,kvh", [(128, 4, 4), (256, 8, 4)])
def test_the_maximum_moves_within_a_waves_run(gpu, dtype, d, heads, kvh):
    """Keys grow along the sequences; scores reach 2^7, so the bound on the weights' exponents is 2^-24 d 2^7 or less."""
    lengths = [(i * 271) % 1100 for i in range(48)]
    c, batch, q, _ = _attend_case(gpu, dtype, d, 64, heads, kvh, lengths, [1] * 48, 0.0, 0, seed=40, extra=0)
    for row in batch.page_table.tolist():
        for j, pid in enumerate(row):
            if dtype == E4M3:
                c.k_scale[pid] = 2.0 ** (-9 + j // 3)
            else:
                c.k[pid] = (c.k[pid].float() * 2.0 ** (-3 + j // 3)).to(BF16)
    _again(c, batch, q, d, 0.0, 0, bound=2.0 ** -6)


def test_attend_scales_that_are_no_powers_of_two(gpu):
    c, batch, q, _ = _attend_case(gpu, E4M3, 128, 32, 8, 4, [100, 7], [2, 1], 30.0, 0)
    for t in (c.k_scale, c.v_scale):
        t.mul_(1.37)
    kp, vp, ks, vs = _state(c)
    table, lengths, starts = batch.page_table.tolist(), batch.lengths.tolist(), batch.starts.tolist()
    ref, size, mine = o.attend(kp, vp, ks, vs, table, lengths, starts, q.cpu(), 128 ** -0.5, 30.0, 0, 2)
    _close(c.attend(batch, q, 128 ** -0.5, softcap=30.0), ref, size, mine)


@pytest.mark.parametrize("many", [20, 70])
@pytest.mark.parametrize("dtype,bad", [(E4M3, float("nan")), (BF16, float("nan")), (BF16, float("inf")), (BF16, float("-inf"))])
def test_what_a_query_may_not_see_has_no_part_in_its_row(gpu, dtype, bad, many):
    """A later token of the call, and one behind the window, hold values that are no numbers: rows that do not see them
    stay as they are, the others have them in exactly the columns they are in."""
    d, page, lengths, new, window = 128, 16, [40, 9], [12, many], 24
    c, batch, q, before = _attend_case(gpu, dtype, d, page, 4, 2, lengths, new, 0.0, window, seed=5, extra=0)
    table = batch.page_table.tolist()
    bad_keys = {0: (47, 20), 1: (17, 0)}
    for s, keys in bad_keys.items():
        for j in keys:
            c.k[table[s][j // page], 0, j % page, 3] = float("nan")      # a NaN score in head 0 only ..
            c.v[table[s][j // page], 1, 5 + s, j % page] = bad           # .. and one value of head 1
    got, before = c.attend(batch, q, d ** -0.5, window=window).cpu(), before.cpu()
    r = 0
    for s, (a, n) in enumerate(zip(lengths, new)):
        for p in range(a, a + n):
            sees = any(p - window < j <= p for j in bad_keys[s])
            assert got[r, :2].isnan().all() if sees else torch.equal(got[r, :2], before[r, :2])
            at = got[r, 2:, 5 + s]
            if sees:
                assert at.isnan().all() if bad != bad else (at == bad).all()
            others = [i for i in range(d) if i != 5 + s]
            assert torch.equal(got[r, 2:][:, others], before[r, 2:][:, others])
            if not sees:
                assert torch.equal(at, before[r, 2:, 5 + s])
            r += 1


@pytest.mark.parametrize("new", [8, 50])
def test_infinities_of_both_signs_meet_in_a_nan(gpu, new):
    c, batch, q, _ = _attend_case(gpu, BF16, 64, 16, 2, 1, [10], [new], 0.0, 0, seed=6, extra=0)
    page = batch.page_table[0, 0].item()
    c.v[page, 0, 9, 12], c.v[page, 0, 9, 14] = float("inf"), float("-inf")
    got = c.attend(batch, q, 0.125).cpu()[:, 0, 9]
    assert got[:2].isfinite().all() and (got[2:4] == float("inf")).all() and got[4:].isnan().all()


def test_pages_outside_the_pool_hold_nothing(gpu):
    d, page = 64, 16
    c = _cache(gpu, 6, page, 2, d, E4M3, 11)
    table, lengths, new = [[3, -1, 5], [6, 1 << 30, 2], [-1, -1, -1]], [40, 35, 10], [3, 1, 2]
    batch, starts = _batch(gpu, table, lengths, new)
    q = torch.randn((6, 4, d), generator=_gen(12)).to(BF16).to(gpu)
    kp, vp, ks, vs = _state(c)
    ref, size, _ = o.attend(kp, vp, ks, vs, table, lengths, starts, q.cpu(), 0.125, 0.0, 0, 3)
    got = c.attend(batch, q, 0.125)
    _close(got, ref, size)
    assert (got[4:] == 0).all()


def test_lengths_that_do_not_fit_the_table_stay_inside_it(gpu):
    """Lengths below zero and beyond the table, starts outside the rows: answers are of no use, but nothing outside is
    touched (the kernels hold every index inside the call's memory)."""
    from se12_amd.paged import PagedBatch

    c = _cache(gpu, 4, 16, 1, 64, E4M3, 13)
    as32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    batch = PagedBatch(as32([[0, 1], [2, 3]]), as32([-7, 2 ** 31 - 1]), as32([-3, 2, 2 ** 31 - 1]), max_new=3)
    guard = torch.full((4 + 4, 2, 64), 9.0, dtype=BF16, device=gpu)
    x = torch.randn((4, 2, 64), generator=_gen(14)).to(gpu)
    c.append(batch, x[:, :1], x[:, 1:], q=x, out=guard[:4])
    c.attend(batch, x.to(BF16), 0.125, out=guard[:4])
    torch.cuda.synchronize()
    assert (guard[4:] == 9.0).all()


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("lengths,new", [([40, 30, 100, 5], [2, 4, 3, 1]), ([20, 32, 90, 1000], [70, 40, 33, 1])])
@pytest.mark.parametrize("window", [0, 20, 64, 80])
def test_positions_beyond_the_table_are_what_they_are(gpu, dtype, lengths, new, window):
    """Tokens behind the table's last column are held nowhere, but their queries stand where they stand: turned by their
    position, and a window reaches back from there."""
    page, kvh, d, heads = 16, 2, 64, 4
    table = _table(4, 2, 9, 15)
    c = _cache(gpu, 9, page, kvh, d, dtype, 16)
    batch, starts = _batch(gpu, table, lengths, new)
    k, v = (torch.randn((sum(new), kvh, d), generator=_gen(17 + i)).to(gpu) for i in range(2))
    q = torch.randn((sum(new), heads, d), generator=_gen(19)).to(gpu)
    inv = (10000.0 ** (-torch.arange(0, d, 2).float() / d)).to(gpu)
    before = _state(c)
    turned = c.append(batch, k, v, q=q, inv_freq=inv)
    _check_append(c, before, batch, lengths, starts, table, k, v, inv, q, turned)
    kp, vp, ks, vs = _state(c)
    ref, size, _ = o.attend(kp, vp, ks, vs, table, lengths, starts, turned.cpu(), 0.125, 0.0, window, max(new))
    got = c.attend(batch, turned, 0.125, window=window)
    _close(got, ref, size)
    if window == 20:
        assert (got[starts[2]:starts[3]] == 0).all()      # (from 90 on nothing held is within 20)


@pytest.mark.parametrize("d,lengths,new,window", [(128, [1500, 40], [1, 1], 0), (64, [3000, 0, 700], [70, 90, 1], 0), (256, [900], [40], 300)])
@pytest.mark.parametrize("size", [2.0 ** 127, 2.0 ** 100, 2.0 ** -70])
def test_any_finite_values_of_bf16_pages_stay_finite(gpu, d, lengths, new, window, size):
    """Weights add up to less than one, as weights that are normalised first: sums of the type's largest values are no
    infinities, and keys that grow along the sequence move the maximum."""
    c, batch, q, _ = _attend_case(gpu, BF16, d, 32, 4, 2, lengths, new, 0.0, window, seed=76, extra=0)
    page_scale = torch.exp2(torch.arange(batch.page_table.shape[1]).float() / 8 - 3).to(gpu)
    for row in batch.page_table.long():
        c.k[row] = (c.k[row].float() * page_scale[:, None, None, None]).to(BF16)
    c.v.copy_((c.v.float().sign() * (1 + c.v.float().abs().fmod(0.9))).mul(size).to(BF16))
    kp, vp, ks, vs = _state(c)
    table, starts = batch.page_table.tolist(), batch.starts.tolist()
    ref, ref_size, _ = o.attend(kp, vp, ks, vs, table, lengths, starts, q.cpu(), d ** -0.5, 0.0, window, batch.max_new)
    got = c.attend(batch, q, d ** -0.5, window=window).cpu().double()
    # (scores reach 2^8 here, as bounded for keys that grow: 2^-24 * 256 * 2^8 in the weights' exponents)
    assert ((got - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -6) * ref_size).all()


def test_attend_with_sharp_scores_and_far_apart_tiles(gpu):
    """The maximum moves in many tiles: keys grow along the sequence; and one key holds all the weight."""
    for dtype in (E4M3, BF16):
        c, batch, q, _ = _attend_case(gpu, dtype, 128, 64, 4, 2, [1500], [1], 0.0, 0, seed=20, extra=0)
        table = batch.page_table.tolist()
        if dtype == E4M3:
            for j, pid in enumerate(table[0]):
                c.k_scale[pid] = 2.0 ** (-9 + j // 3)
        else:
            for j, pid in enumerate(table[0]):
                c.k[pid] = (c.k[pid].float() * 2.0 ** (-3 + j // 3)).to(BF16)
        kp, vp, ks, vs = _state(c)
        # scores reach 2^8 here: the bound on them grows with them, 2^-24 * 128 * sum |q k| scaling <= 2^-7
        ref, size, _ = o.attend(kp, vp, ks, vs, table, [1500], [0, 1], q.cpu(), 128 ** -0.5, 0.0, 0, 1)
        err = (c.attend(batch, q, 128 ** -0.5).cpu().double() - ref).abs()
        assert (err <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -6) * size).all()


def test_workspace_and_streams(gpu):
    c, batch, q, out = _attend_case(gpu, E4M3, 256, 64, 8, 4, [900, 20, 400], [1, 1, 1], 50.0, 0, seed=30, extra=0)
    n = c.attend_workspace(batch, 3, 8)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=gpu)           # its contents do not matter
    assert torch.equal(c.attend(batch, q, 0.0625, softcap=50.0, workspace=ws), out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = c.attend(batch, q, 0.0625, softcap=50.0)
    s.synchronize()
    assert torch.equal(again, out)
    from se12_amd._native import Se12Error

    with pytest.raises(Se12Error, match="workspace"):
        c.attend(batch, q, 0.0625, workspace=ws[:n - 256])


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("d,heads,kvh,lengths,new,window", [
    (256, 8, 4, [900, 20, 400, 3000], [1, 90, 1, 70], 0),                          # long units in parts, decode steps beside
    (128, 28, 4, [5000, 1], [64, 1], 0),                                           # one sequence, seven heads to one
    (64, 4, 2, [(i * 53) % 150 for i in range(100)], [90 if i in (3, 70, 99) else i % 3 for i in range(100)], 0),
    (64, 4, 2, [(i * 253) % 1500 for i in range(130)], [90 if i in (3, 70, 129) else i % 3 for i in range(130)], 1200),
])
def test_what_the_workspace_of_prompts_held_does_not_matter(gpu, dtype, d, heads, kvh, lengths, new, window):
    """Records of units, parts and statistics are all written before they are read, and none lies outside: a workspace of
    exactly the bytes asked for, of ones or zeros, with guards around it, and used again for fewer tokens."""
    c, batch, q, out = _attend_case(gpu, dtype, d, 64, heads, kvh, lengths, new, 0.0, window, seed=32, extra=0)
    n = c.attend_workspace(batch, q.shape[0], heads)
    for fill in (255, 0):
        guarded = torch.full((n + 2048,), fill, dtype=torch.uint8, device=gpu)
        guarded[:1024], guarded[1024 + n:] = 90, 90
        ws = guarded[1024:1024 + n]
        assert torch.equal(c.attend(batch, q, d ** -0.5, window=window, workspace=ws), out)
        assert (guarded[:1024] == 90).all() and (guarded[1024 + n:] == 90).all()
        few = [min(x, 1) for x in new]
        step, starts = _batch(gpu, batch.page_table.tolist(), lengths, few, max_new=max(new))
        rows = torch.tensor([s for s, x in zip(batch.starts.tolist(), new) if x], device=gpu)
        first = c.attend(step, q[rows], d ** -0.5, window=window, workspace=ws)
        assert torch.equal(c.attend(step, q[rows], d ** -0.5, window=window), first)
        kp, vp, ks, vs = _state(c)
        ref, size, _ = o.attend(kp, vp, ks, vs, batch.page_table.tolist(), lengths, starts, q[rows].cpu(), d ** -0.5, 0.0, window, 1)
        _close(first, ref, size)
        assert (guarded[:1024] == 90).all() and (guarded[1024 + n:] == 90).all()


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_captured_prompts_follow_lengths_and_starts(gpu, dtype):
    """One captured call over other divisions of the same rows at every replay: prompts, decode steps, nothing; two
    graphs with a workspace of their own in turn, eager calls between them."""
    d, page, heads, kvh = 128, 32, 8, 2
    c, batch, q, out = _attend_case(gpu, dtype, d, page, heads, kvh, [500, 900, 20, 3], [100, 1, 60, 39], 0.0, 0, seed=35, extra=0)
    # (slots that nobody held are read below: numbers in place of the NaN there)
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        if t is not None:
            t.copy_(t.float().nan_to_num(0.125).to(t.dtype))
    kp, vp, ks, vs = _state(c)
    calls = []
    for window in (0, 300):
        ws = torch.full((c.attend_workspace(batch, 200, heads),), 255, dtype=torch.uint8, device=gpu)
        y = torch.empty_like(out)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            c.attend(batch, q, d ** -0.5, window=window, out=y, workspace=ws)
        calls.append((window, graph, y, ws))      # (what a graph writes to lives as long as it)
    for lengths, starts in (([500, 900, 20, 3], [0, 100, 101, 161, 200]), ([500, 800, 20, 3], [0, 1, 101, 102, 102]),
                            ([10, 890, 40, 2], [0, 33, 34, 134, 200]), ([599, 900, 79, 41], [0, 1, 2, 3, 4]),
                            ([500, 900, 20, 3], [0, 100, 101, 161, 200])):
        batch.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        batch.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        for window, graph, y, _ in calls:
            y.fill_(5.0)
            graph.replay()
            eager = c.attend(batch, q, d ** -0.5, window=window, out=torch.full_like(out, 5.0))
            torch.cuda.synchronize()
            assert torch.equal(y, eager) and (y[starts[-1]:] == 5.0).all()
            ref, size, mine = o.attend(kp, vp, ks, vs, batch.page_table.tolist(), lengths, starts, q.cpu(), d ** -0.5, 0.0, window, 100)
            _close(y, ref, size, mine)
    assert torch.equal(calls[0][2], out)


@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("lengths,new,window", [
    ([0, 6000, 0, 40], [64, 64, 33, 200], 0),                  # one unit is most of the work
    ([2500, 10, 10, 10, 10, 10], [33, 33, 40, 50, 60, 70], 0),
    ([4000, 10, 2000], [100, 200, 129], 1500),
])
def test_few_prompts_of_very_different_lengths(gpu, dtype, lengths, new, window):
    _attend_case(gpu, dtype, 64, 16, 4, 2, lengths, new, 0.0, window, seed=33)


@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_prompts_with_scales_that_are_no_powers_of_two(gpu, softcap):
    """The values' scale goes into the weight's exponent: its logarithm, of 6 at most here, is off by 2^-22."""
    c, batch, q, _ = _attend_case(gpu, E4M3, 128, 32, 8, 4, [100, 7, 1500], [70, 1, 40], softcap, 0, seed=34, extra=0)
    for t in (c.k_scale, c.v_scale):
        t.mul_(1.37)
    _again(c, batch, q, 128, softcap, 0)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_prompt_then_captured_decode_steps(gpu, dtype):
    """Prompts of different lengths, then decode steps replayed from one graph whose lengths move on the device: every
    step against the oracle on the cache as it is, and against the same calls made one by one."""
    from se12_amd.paged import PagedBatch

    d, page, heads, kvh = 64, 16, 4, 2
    prompts, columns = [37, 1, 16], 5
    table = _table(3, columns, 3 * columns + 1, 40)
    inv = (10000.0 ** (-torch.arange(0, d, 2).float() / d)).to(gpu)
    as32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    outs = []
    for captured in (False, True):
        c = _cache(gpu, 3 * columns + 1, page, kvh, d, dtype, 41)
        lengths, step_starts = as32([0, 0, 0]), as32([0, 1, 2, 3])
        batch, starts = _batch(gpu, table, [0, 0, 0], prompts)
        g = _gen(42)
        x = torch.randn((sum(prompts), heads + 2 * kvh, d), generator=g).to(gpu)
        q, k, v = x.split([heads, kvh, kvh], 1)
        qr = c.append(batch, k, v, q=q, inv_freq=inv)
        got = c.attend(batch, qr, d ** -0.5, softcap=50.0)
        kp, vp, ks, vs = _state(c)
        ref, size, _ = o.attend(kp, vp, ks, vs, table, [0, 0, 0], starts, qr.cpu(), d ** -0.5, 50.0, 0, max(prompts))
        _close(got, ref, size)
        lengths += as32(prompts)
        batch = PagedBatch(as32(table), lengths, step_starts)
        x = torch.empty((3, heads + 2 * kvh, d), device=gpu)
        q_out, y = torch.empty((3, heads, d), dtype=BF16, device=gpu), torch.empty((3, heads, d), dtype=BF16, device=gpu)

        def step():
            c.append(batch, x[:, heads:heads + kvh], x[:, heads + kvh:], q=x[:, :heads], inv_freq=inv, out=q_out)
            c.attend(batch, q_out, d ** -0.5, softcap=50.0, out=y)
            lengths.add_(1)

        graph = None
        if captured:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                step()
        at = list(prompts)
        for i in range(20):
            x.copy_(torch.randn(x.shape, generator=g))
            if captured:
                graph.replay()
            else:
                step()
            kp, vp, ks, vs = _state(c)
            ref, size, _ = o.attend(kp, vp, ks, vs, table, at, [0, 1, 2, 3], q_out.cpu(), d ** -0.5, 50.0, 0, 1)
            _close(y, ref, size)
            at = [a + 1 for a in at]
            assert lengths.tolist() == at
            outs.append(y.cpu().clone())
    for a, b in zip(outs[:20], outs[20:]):
        assert torch.equal(a, b)


def test_a_decode_step_through_the_layer_ends_in_log_probabilities(gpu):
    """Two sequences of different lengths through a small layer: projection (the library's product), append, attend,
    output product, log probabilities; against the same in float64 from the cache's values."""
    from se12_amd.hip import RawBf16MatVecKernel
    from se12_amd.logprobs import token_logprobs

    d, page, heads, kvh, hidden, vocab = 64, 16, 4, 2, 256, 700
    g = _gen(60)
    w = {n: (torch.randn(s, generator=g) * 0.05).to(BF16).to(gpu)
         for n, s in (("qkv", ((heads + 2 * kvh) * d, hidden)), ("head", (vocab, heads * d)))}
    qkv, head = RawBf16MatVecKernel(w["qkv"]), RawBf16MatVecKernel(w["head"])
    lengths, new = [20, 3], [1, 1]
    c = _cache(gpu, 6, page, kvh, d, E4M3, 61)
    table = [[4, 1], [0, 2]]
    batch, starts = _batch(gpu, table, lengths, new)
    inv = (10000.0 ** (-torch.arange(0, d, 2).float() / d)).to(gpu)
    x = torch.randn((2, hidden), generator=g).to(BF16).to(gpu)
    y = qkv.multiply(x).view(2, heads + 2 * kvh, d)
    q = c.append(batch, y[:, heads:heads + kvh], y[:, heads + kvh:], q=y[:, :heads], inv_freq=inv)
    a = c.attend(batch, q, d ** -0.5)
    logits = head.multiply(a.view(2, -1))
    r = token_logprobs(logits, torch.tensor([5, 699], device=gpu), top=4, softcap=30.0)
    kp, vp, ks, vs = _state(c)
    ref, size, _ = o.attend(kp, vp, ks, vs, table, lengths, starts, q.cpu(), d ** -0.5, 0.0, 0, 1)
    _close(a, ref, size)
    z = 30.0 * torch.tanh(a.view(2, -1).cpu().double() @ w["head"].cpu().double().T / 30.0)
    lp = z - torch.logsumexp(z, 1, keepdim=True)
    got = torch.cat([r.logprobs[:, None], r.top_logprobs], 1).cpu().double()
    want = torch.cat([lp[[0, 1], [5, 699]][:, None], lp.sort(1, descending=True).values[:, :4]], 1)
    assert (got - want).abs().max() <= 1e-4       # FP32 products of 256 values of at most 1: 256 * 2^-24 * 16 and the cap's 2^-20 * 30
