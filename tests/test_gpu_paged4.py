"""A paged cache of 4 bits (E2M1) on the GPU: append, read and attend, and rotate_heads,
against the 64-bit forms of tests/e2m1_oracle.py and tests/paged_oracle.py.

Tolerances. BF16 rounds off by at most 2^-8 of the value. A key is its norm (a factor
rounded three times: the root, the weight, their product), two products, a sum and
the roundings of sine and cosine, each 2^-24 of itself: within 8 * 2^-24 < 2^-20 of |a| +
|b|, a and b the normed pair. A held digit is then the exact one's unless the exact
quotient lies as near to a border between two digits. Attention: a weight is rounded to
FP16 (2^-11 of its share of sum w |v|), scores are FP32 sums of head_dim products
(head_dim 2^-24 of sum |q k| scaling, 40 at most here: 2^-11 for a weight's exponent, twice
for numerator and denominator), the output once to BF16."""

from __future__ import annotations

import pytest
import torch

import e2m1_oracle as e
import paged_oracle as o
from test_gpu_paged import _batch, _gen, _table

pytestmark = pytest.mark.gpu

BF16, FP4 = torch.bfloat16, torch.float4_e2m1fn_x2


def _cache(gpu, pages, page, kvh, d, seed, scales=(96, 130)):
    """A pool of other sequences' leftovers: random codes, scales of 2^-3 to 2 and some that are none."""
    from se12_amd.paged import PagedKvCache

    c, g = PagedKvCache(pages, page, kvh, d, dtype=FP4, device=gpu), _gen(seed)
    for t in (c.k, c.v):
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.randint(*scales, t.shape, generator=g, dtype=torch.uint8))
    return c


def _snapshot(c):
    return [t.view(torch.uint8).cpu().clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]


def _check_append(c, before, batch, lengths, starts, table, q, k, v, got_q, turn):
    """The cache after an append of turned rows, from the bytes before; which slots were written."""
    page, kvh, d = c.page_size, c.kv_heads, c.head_dim
    was = type("Held", (), dict(zip(("k", "v", "k_scale", "v_scale"), before)))
    codes_k, codes_v, bytes_k, bytes_v = e.held_codes(c)
    old = e.held_codes(was)
    written = torch.zeros((c.pages, page), dtype=torch.bool)
    q_turn = {n: x for n, x in turn.items() if n not in ("q_norm", "k_norm")}
    for s in range(len(lengths)):
        for i in range(min(starts[s + 1] - starts[s], batch.max_new)):
            pos, r = lengths[s] + i, starts[s] + i
            if q is not None:
                size = e.turned(q[r].cpu(), 0, None, w=turn.get("q_norm"), offset=turn.get("offset", 0.0)).abs().amax()
                ref = e.turned(q[r].cpu(), pos, w=turn.get("q_norm"), **q_turn)
                assert ((got_q[r].cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -19 * size * turn.get("scale", 1.0)).all()
            if not (pos // page < len(table[s]) and 0 <= table[s][pos // page] < c.pages):
                continue
            pid, slot = table[s][pos // page], pos % page
            written[pid, slot] = True
            exact_v, byte_v = e.quantised(v[r].cpu())
            # (FP32 quotients, correctly rounded: a tie that is none lies within 2^-24 of its border)
            near = ((_quotient(v[r].cpu(), byte_v)[..., None] - e.BORDERS).abs() <= 2.0 ** -23 * e.BORDERS).any(-1)
            assert torch.equal(bytes_v[pid, :, slot], byte_v)
            fine = (byte_v != 255).repeat_interleave(32, -1)
            assert ((codes_v[pid, :, slot] == exact_v) | near | ~fine).all()
            x = e.turned(k[r].cpu(), pos, w=turn.get("k_norm"), **q_turn)
            off = 2.0 ** -19 * turn.get("scale", 1.0) * e.turned(k[r].cpu(), 0, None, w=turn.get("k_norm"), offset=turn.get("offset", 0.0)).abs().amax(-1, keepdim=True)
            _, byte_k = e.quantised(x)
            got = bytes_k[pid, :, slot]
            sixth = x.unflatten(-1, (-1, 32)).abs().amax(-1) / 6
            fine = byte_k != 255
            assert torch.equal(got == 255, ~fine)
            middle = e.MIDDLES[torch.minimum(got, byte_k).clamp(max=e.LAST - 1)]
            assert ((got == byte_k) | ((got - byte_k).abs() == 1) & ((sixth - middle).abs() <= off / 6))[fine].all()
            y = _quotient(x, got)
            want = e.VALUES[e.nearest(y.abs().nan_to_num(), e.BORDERS)] * torch.sign(y)
            s32 = e.scale_of(got).repeat_interleave(32, -1)
            near = ((y.abs()[..., None] - e.BORDERS).abs() * s32[..., None] <= off[..., None] + 2.0 ** -23).any(-1)
            assert ((codes_k[pid, :, slot] == want) | near | ~fine.repeat_interleave(32, -1)).all()
    rest = ~written
    for now, then in zip((codes_k, codes_v, bytes_k, bytes_v), old):
        assert torch.equal(now.transpose(1, 2)[rest].nan_to_num(99.0), then.transpose(1, 2)[rest].nan_to_num(99.0))
    return written


def _quotient(x, byte):
    s = e.scale_of(byte).repeat_interleave(32, -1)
    return torch.where(s > 0, x.double() / s.clamp(min=2.0 ** -17), torch.zeros_like(x.double()))


APPENDS = [
    # d, page, kvh, heads, rotary, interleaved, norm, lengths, new
    (256, 64, 4, 8, 256, False, None, [0, 63, 64, 200], [1, 1, 1, 1]),             # decode: first slot, last slot, new page
    (128, 16, 2, 14, 128, False, BF16, [0, 5, 31, 16], [40, 3, 17, 1]),            # pages of 16, seven heads to one
    (64, 32, 1, 1, 32, True, torch.float32, [7, 0, 100], [0, 70, 5]),              # half of a head; a sequence with nothing
    (256, 128, 2, 2, 128, True, BF16, [100, 1], [150, 127]),                       # pages of 128 begun and left inside
    (64, 64, 3, 9, 0, False, None, [3, 3, 3], [16, 15, 2]),                        # no rotation
    (128, 32, 2, 4, 24, False, torch.float32, [40, 9], [33, 20]),                  # pairs that no 8 columns hold
    (128, 32, 2, 4, 120, True, None, [15, 16, 17], [2, 1, 16]),
]


@pytest.mark.parametrize("x_dtype", [torch.float32, BF16])
@pytest.mark.parametrize("d,page,kvh,heads,rotary,interleaved,norm,lengths,new", APPENDS)
def test_append(gpu, x_dtype, d, page, kvh, heads, rotary, interleaved, norm, lengths, new):
    total = sum(new)
    columns = max((a + b + page - 1) // page for a, b in zip(lengths, new)) + 1
    table = _table(len(new), columns, len(new) * columns + 2, 1)
    c = _cache(gpu, len(new) * columns + 2, page, kvh, d, 2)
    batch, starts = _batch(gpu, table, lengths, new)
    g = _gen(3)
    # views of one product's rows, as a fused projection gives them, and rows behind the last sequence
    x = (torch.randn((total + 3, (heads + 2 * kvh) * d), generator=g) * 2).to(x_dtype).to(gpu)
    q, k, v = (t.view(total + 3, -1, d) for t in x.split([heads * d, kvh * d, kvh * d], 1))
    inv = (10000.0 ** (-torch.arange(0, rotary, 2).float() / rotary)).to(gpu) if rotary else None
    w = [None, None] if norm is None else [(torch.randn(d, generator=g) * 0.3).to(norm).to(gpu) for _ in range(2)]
    before = _snapshot(c)
    out = torch.full((total + 3, heads, d), 7.0, dtype=BF16, device=gpu)
    got = c.append(batch, k, v, q=q, inv_freq=inv, out=out, interleaved=interleaved, rotary_scale=1.25, q_norm=w[0], k_norm=w[1],
                   norm_offset=1.0)
    assert got is out and (out[total:] == 7.0).all()
    turn = dict(inv_freq=inv, interleaved=interleaved, scale=1.25 if rotary else 1.0, q_norm=w[0], k_norm=w[1], offset=1.0)
    _check_append(c, before, batch, lengths, starts, table, q, k, v, got, turn)
    # what is held, read back: exact
    kk, vv = c.read(batch, total + 3, out=(out[:, :kvh].contiguous(), out[:, :kvh].clone()))
    pk, pv = e.pools(c)
    for s, (a, n) in enumerate(zip(lengths, new)):
        for i in range(n):
            pid, slot, r = table[s][(a + i) // page], (a + i) % page, starts[s] + i
            assert torch.equal(kk[r].cpu().double(), pk[pid, :, slot]) and torch.equal(vv[r].cpu().double(), pv[pid, :, :, slot])


def _held_cache(gpu, d, page, kvh, lengths, new, seed):
    """A cache whose tokens are random values quantised, everything else codes with scales that are none."""
    columns = max((a + b + page - 1) // page for a, b in zip(lengths, new)) + 1
    pages = len(new) * columns + 1
    table = _table(len(new), columns, pages, seed + 1)
    c = _cache(gpu, pages, page, kvh, d, seed + 2)
    held = torch.zeros((pages, page), dtype=torch.bool)
    for row, n in zip(table, [a + b for a, b in zip(lengths, new)]):
        for j in range(n):
            held[row[j // page], j % page] = True
    for t in (c.k_scale, c.v_scale):
        x = t.cpu()
        x.permute(0, 3, 1, 2)[~held] = 255
        t.copy_(x)
    return c, table


def _close(out, ref, size, mine, vmax, bound=2.0 ** -10):
    err = (out.cpu().double() - ref).abs()[mine]
    assert (err <= (2.0 ** -8 * ref.abs() + (2.0 ** -11 + bound) * size + 2.0 ** -20 * vmax)[mine]).all(), err.max()


def _oracle(c, table, lengths, starts, q, scaling, softcap, window, max_new):
    k, v = e.pools(c)
    return (*o.attend(k, v, None, None, table, lengths, starts, q.cpu(), scaling, softcap, window, max_new), v.nan_to_num().abs().max().item())


def _attend_case(gpu, d, page, heads, kvh, lengths, new, softcap, window, seed=0, max_new=None, extra=2):
    c, table = _held_cache(gpu, d, page, kvh, lengths, new, seed)
    batch, starts = _batch(gpu, table, lengths, new, max_new)
    total = starts[-1] + extra
    x = torch.randn((total, (heads + 3) * d), generator=_gen(seed + 3)).to(BF16).to(gpu)
    q = x[:, d:(heads + 1) * d].view(total, heads, d)
    out = torch.full((total, heads, d), 3.0, dtype=BF16, device=gpu)
    assert c.attend(batch, q, d ** -0.5 / 4, softcap=softcap, window=window, out=out) is out
    ref, size, mine, vmax = _oracle(c, table, lengths, starts, q, d ** -0.5 / 4, softcap, window, batch.max_new)
    _close(out, ref, size, mine, vmax)
    assert (out.cpu()[~mine] == 3.0).all()
    return c, batch, q, out


ATTENDS = [
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
    (128, 128, 8, 4, [0, 700], [200, 90], 0.0, 0),
]


@pytest.mark.parametrize("d,page,heads,kvh,lengths,new,softcap,window", ATTENDS)
def test_attend(gpu, d, page, heads, kvh, lengths, new, softcap, window):
    _attend_case(gpu, d, page, heads, kvh, lengths, new, softcap, window)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------


def _one_page(gpu, x, dtype, heads=1):
    """Rows x [tokens, 64] as the values (and keys, unrotated) of one sequence from its start: what the cache holds."""
    tokens = x.shape[0]
    pages = (tokens + 15) // 16
    c = _cache(gpu, pages, 16, heads, 64, 4)
    batch, _ = _batch(gpu, [list(range(pages))], [0], [tokens])
    t = x.to(dtype).to(gpu).view(tokens, heads, 64)
    c.append(batch, t, t.clone())
    codes_k, codes_v, bytes_k, bytes_v = (y.transpose(1, 2).flatten(0, 1)[:tokens] for y in e.held_codes(c))
    assert torch.equal(codes_k, codes_v) and torch.equal(bytes_k, bytes_v)
    return t.cpu().double(), codes_k, bytes_k, c, batch


def test_every_bf16_size_is_held_as_its_nearest(gpu):
    """Every finite BF16 value as the largest of 32, small ones beside it: scales from 0 to the last, ties of scales and of
    digits among them, signs, zeros; against the definition in 64 bits, digit for digit."""
    bits = torch.arange(0, 0x7F80, dtype=torch.int32)
    top = (bits << 16).view(torch.float32)
    g = _gen(50)
    x = torch.rand((len(top), 32), generator=g) * 2 - 1
    x[:, 1::4] = torch.randint(-96, 97, (len(top), 8), generator=g) / 96.0       # multiples that ties are made of
    x = (x * top[:, None]).to(BF16)
    x[:, 0] = top.to(BF16)
    x[:, 5] = 0
    x = torch.cat([x, x.flip(1).neg()], 1)
    for lo in range(0, len(x), 8192):
        ref, codes, byte, _, _ = _one_page(gpu, x[lo:lo + 8192], BF16)
        want, want_byte = e.quantised(ref)
        assert torch.equal(byte, want_byte)
        assert torch.equal(codes, want)


def test_fp32_rows_at_the_borders_of_scales_and_digits(gpu):
    """FP32 values at ties, and one step of FP32 beside them. The quotient is rounded to FP32 before its digit is: beside a
    tie, within 2^-24 of it, the even digit may be taken."""
    scales = e.SCALES[[1, 3, 8, 9, 100, 119, 120, 121, 225, 226]]
    rows = []
    for s in scales:
        for b in e.BORDERS:
            for step in (-1, 0, 1):
                v = (b * s).float()
                v = torch.nextafter(v, v + step) if step else v
                rows.append(torch.cat([torch.tensor([6 * float(s)]), v.repeat(31)]))
    for m in e.MIDDLES[::7]:
        for step in (-1, 0, 1):
            v = (6 * m).float()
            v = torch.nextafter(v, v + step) if step else v
            rows.append(torch.cat([v[None], v.repeat(31) / 3]))
    x = torch.stack(rows)
    ref, codes, byte, _, _ = _one_page(gpu, torch.cat([x, -x], 1), torch.float32)
    want, want_byte = e.quantised(ref)
    assert torch.equal(byte, want_byte)
    near = ((_quotient(ref, byte).abs()[..., None] - e.BORDERS).abs() <= 2.0 ** -23 * e.BORDERS).any(-1)
    assert ((codes == want) | near).all()
    exact = (_quotient(ref, byte).abs()[..., None] == e.BORDERS).any(-1)
    assert exact.any() and torch.equal(codes[exact], want[exact])


def test_values_beyond_what_is_held_and_no_numbers(gpu):
    x = torch.zeros((9, 64))
    x[0, 3], x[0, 4], x[0, 5] = 61440.0, 3e38, -70000.0                # beyond the last scale: the largest, by sign
    x[1, 0], x[1, 1] = 1e-6, -1e-7                                     # below the least scale: zeros
    x[2, 31], x[2, 32] = float("nan"), 1.0                             # a NaN takes its 32 columns, not the next
    x[3, 40], x[3, 41], x[3, 2] = float("inf"), 2.0, 5.0
    x[4, 33], x[4, 7] = float("-inf"), 3.0
    x[5] = float("nan")
    x[7, :32] = 2.0 ** -14 * torch.linspace(-6, 6, 32)                 # subnormal scales
    x[8, 9], x[8, 10] = float("inf"), float("nan")
    ref, codes, byte, c, batch = _one_page(gpu, x, torch.float32)
    want, want_byte = e.quantised(ref)
    assert torch.equal(byte, want_byte)
    fine = (byte != 255).repeat_interleave(32, -1)
    assert torch.equal(codes[fine], want[fine])
    k, v = c.read(batch, 9)
    for got in (k[:, 0].cpu().double(), v[:, 0].cpu().double()):
        assert torch.equal(got.isnan(), ~fine[:, 0])
        assert got[0, 3:6].tolist() == [61440.0, 61440.0, -61440.0] and (got[1] == 0).all()
        assert torch.equal(got[fine[:, 0]], e.values(want, byte)[:, 0][fine[:, 0]])


@pytest.mark.parametrize("interleaved", [False, True])
def test_a_token_is_held_alike_however_it_comes(gpu, interleaved):
    """One call, calls of a few tokens each, and one token at a time: the same bytes, and the same q."""
    d, page, kvh, heads, n = 128, 32, 2, 6, 75
    g = _gen(51)
    x = torch.randn((n, heads + 2 * kvh, d), generator=g).to(gpu)
    inv = (10000.0 ** (-torch.arange(0, 96, 2).float() / 96)).to(gpu)
    w = [torch.rand(d, generator=g).to(gpu) + 0.5 for _ in range(2)]
    kw = dict(inv_freq=inv, interleaved=interleaved, rotary_scale=1.1, q_norm=w[0], k_norm=w[1])
    held = []
    for sizes in ([75], [1] * 75, [16, 5, 30, 1, 23], [3] * 25, [8, 60, 7]):
        c = _cache(gpu, 30, page, kvh, d, 52)
        qs, at = [], 0
        for m in sizes:
            batch, _ = _batch(gpu, [[7, 3, 12, 0, 5, 6, 8, 9, 10, 11, 13, 14]], [250 + at], [m])
            q, k, v = x[at:at + m].split([heads, kvh, kvh], 1)
            qs.append(c.append(batch, k, v, q=q, **kw))
            at += m
        held.append([torch.cat(qs).cpu(), *_snapshot(c)])
    for other in held[1:]:
        for a, b in zip(held[0], other):
            assert torch.equal(a, b)


def test_append_in_place_without_q_and_one_row_of_any_distance(gpu):
    c = _cache(gpu, 4, 32, 2, 128, 70)
    batch, _ = _batch(gpu, [[0, 1], [2, 3]], [20, 3], [30, 1])
    g = _gen(71)
    q, k, v = (torch.randn((31, h, 128), generator=g).to(BF16).to(gpu) for h in (8, 2, 2))
    inv = (10000.0 ** (-torch.arange(0, 64).float() / 64)).to(gpu)
    w = torch.rand(128, generator=g).to(BF16).to(gpu)
    apart = c.append(batch, k, v, q=q, inv_freq=inv, q_norm=w)
    state = _snapshot(c)
    assert c.append(batch, k, v, q=q, inv_freq=inv, q_norm=w, out=q) is q and torch.equal(q, apart)
    assert c.append(batch, k, v, inv_freq=inv) is None
    for a, b in zip(state, _snapshot(c)):
        assert torch.equal(a, b)
    one, _ = _batch(gpu, [[0, 1]], [20], [1])
    rows = torch.randn((2, 12 * 128 + 3), generator=g).to(gpu)
    q, k, v = rows[1:, 3:].view(1, 12, 128).split([8, 2, 2], 1)
    a = c.append(one, k, v, q=q, inv_freq=inv)
    state = _snapshot(c)
    assert torch.equal(a, c.append(one, k.clone(), v.clone(), q=q.clone(), inv_freq=inv))
    for x, y in zip(state, _snapshot(c)):
        assert torch.equal(x, y)


def test_far_positions_and_tokens_without_a_page(gpu):
    """Positions beyond 2^20 under interleaved pairs; pages outside the pool, a table that ends, hold nothing; q is turned
    all the same."""
    d, page = 64, 16
    lengths, new = [1_500_000, 131_071, 30], [3, 20, 40]
    table = [[-1] * 100_000 for _ in new]
    for s, (a, n) in enumerate(zip(lengths, new)):
        for j in range(a // page, (a + n - 1) // page + 1):
            table[s][j] = (3 * s + j - a // page) if j % 2 == 0 or s < 2 else (1 << 30 if j == 3 else -1)
    c = _cache(gpu, 9, page, 2, d, 5)
    batch, starts = _batch(gpu, table, lengths, new)
    g = _gen(6)
    q, k, v = (torch.randn((63, h, d), generator=g).to(gpu) for h in (4, 2, 2))
    inv = (10000.0 ** (-torch.arange(0, d, 2).float() / d)).to(gpu)
    before = _snapshot(c)
    got = c.append(batch, k, v, q=q, inv_freq=inv, interleaved=True)
    _check_append(c, before, batch, lengths, starts, table, q, k, v, got, dict(inv_freq=inv, interleaved=True))
    kk, vv = c.read(batch, 63)
    for s, (a, n) in enumerate(zip(lengths, new)):
        for i in range(n):
            p = table[s][(a + i) // page] if (a + i) // page < len(table[s]) else -1
            if not 0 <= p < 9:
                assert (kk[starts[s] + i] == 0).all() and (vv[starts[s] + i] == 0).all()


def test_beyond_32_bit_offsets(gpu):
    """Pages beyond 4 GiB of codes: written, read and attended to."""
    d, page, kvh = 256, 128, 8
    pages = (5 << 30) // (kvh * page * d // 2)
    from se12_amd.paged import PagedKvCache

    c = PagedKvCache(pages, page, kvh, d, dtype=FP4, device=gpu)
    table, lengths, new = [[pages - 1, 3], [pages - 2, 2]], [100, 0], [40, 3]
    batch, starts = _batch(gpu, table, lengths, new)
    g = _gen(53)
    q, k, v = (torch.randn((43, h, d), generator=g).to(gpu) for h in (8, 8, 8))
    qr = c.append(batch, k, v, q=q)
    small = PagedKvCache(4, page, kvh, d, dtype=FP4, device=gpu)
    near, _ = _batch(gpu, [[0, 1], [2, 3]], lengths, new)
    assert torch.equal(qr, small.append(near, k, v, q=q))
    for a, b in zip(c.read(batch, 43), small.read(near, 43)):
        assert torch.equal(a, b)
    assert torch.equal(c.attend(batch, qr, 0.0625), small.attend(near, qr, 0.0625))
    assert (c.k.view(torch.uint8)[4:pages - 2].view(torch.int64) == 0).all()


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norms_and_pairs_for_caches_of_other_types(gpu, dtype, interleaved):
    """append of a cache of BF16 or E4M3 with norms, pairs and a scale: as of keys and queries made so before."""
    from se12_amd.paged import PagedKvCache

    d, kvh, heads = 128, 2, 4
    lengths, new = [5, 30], [40, 3]
    g = _gen(54)
    x = torch.randn((43, heads + 2 * kvh, d), generator=g).to(gpu)
    inv = (10000.0 ** (-torch.arange(0, 64, 2).float() / 64)).to(gpu)
    w = [torch.rand(d, generator=g).to(BF16).to(gpu) for _ in range(2)]
    c = PagedKvCache(8, 32, kvh, d, dtype=dtype, device=gpu)
    batch, starts = _batch(gpu, [[0, 1], [2, 3]], lengths, new)
    for t in (x, x.to(BF16)):
        q, k, v = t.split([heads, kvh, kvh], 1)
        out = torch.empty((43 * heads * d + 4,), dtype=BF16, device=gpu)[4:].view(43, heads, d)      # 8-byte aligned
        got = c.append(batch, k, v, q=q, inv_freq=inv, out=out, interleaved=interleaved, rotary_scale=1.2, q_norm=w[0], k_norm=w[1], norm_offset=1.0)
        assert got is out
        kk, vv = c.read(batch, 43)
        for s, (a, n) in enumerate(zip(lengths, new)):
            for i in range(n):
                r = starts[s] + i
                ref = [e.turned(y[r].cpu(), a + i, inv, interleaved, 1.2, z, offset=1.0) for y, z in ((q, w[0]), (k, w[1]))]
                assert ((got[r].cpu().double() - ref[0]).abs() <= 2.0 ** -8 * ref[0].abs() + 2.0 ** -19 * ref[0].abs().amax()).all()
                # (E4M3: half a step is 2^-4 of a value, below 2^-6 of the page's scale 2^-10 of that scale. The scale of a page
                # with older tokens, 5 and 30 here, is never less than it was, and a new cache's is 1; these values, below 448,
                # ask for no more: 2^-10. BF16 holds codes times a power of two as they are. FP32 before: 2^-19 of the largest)
                step, least = (2.0 ** -8, 0.0) if dtype == BF16 else (2.0 ** -4, 2.0 ** -10)
                for y, z in ((kk[r], ref[1]), (vv[r], v[r].cpu().double())):
                    assert z.abs().max() < 448
                    assert ((y.cpu().double() - z).abs() <= step * z.abs() + least + 2.0 ** -19 * max(8.0, z.abs().max().item())).all()


# ---------------------------------------------------------------------------
# reading back
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [FP4, torch.float8_e4m3fn, BF16])
@pytest.mark.parametrize("d,page,kvh,lengths,new", [
    (64, 16, 1, [0, 5, 0], [100, 30, 1]), (128, 128, 3, [0, 0], [1, 300]), (256, 32, 2, [17, 0, 40, 0], [1, 64, 0, 47]),
])
def test_read(gpu, dtype, d, page, kvh, lengths, new):
    """Exactly what is held, of rows that a sequence has; the others stay, and zeros stand for tokens held nowhere."""
    from se12_amd.paged import PagedKvCache
    from test_gpu_paged import _cache as other_cache

    columns = max((a + b + page - 1) // page for a, b in zip(lengths, new))
    pages = len(new) * columns + 1
    table = _table(len(new), columns, pages, 55)
    table[0][0] = -1
    c = _cache(gpu, pages, page, kvh, d, 56) if dtype == FP4 else other_cache(gpu, pages, page, kvh, d, dtype, 56)
    if dtype == FP4:
        k_pool, v_pool = e.pools(c)
    else:
        k_pool, v_pool = c.k.cpu().double(), c.v.cpu().double()
        if c.k_scale is not None:
            k_pool, v_pool = k_pool * c.k_scale.cpu().double()[..., None, None], v_pool * c.v_scale.cpu().double()[..., None, None]
    total = sum(new)
    for max_new in (None, 5000):
        batch, starts = _batch(gpu, table, lengths, new, max_new)
        out = [torch.full((total + 2, kvh, d), 7.0, dtype=BF16, device=gpu) for _ in range(2)]
        k, v = c.read(batch, total + 2, out=tuple(out))
        assert k is out[0] and v is out[1] and (k[total:] == 7.0).all() and (v[total:] == 7.0).all()
        for s, (a, n) in enumerate(zip(lengths, new)):
            for i in range(n):
                pid, slot = table[s][(a + i) // page], (a + i) % page
                want = [torch.zeros(kvh, d).double()] * 2 if pid < 0 else [k_pool[pid, :, slot], v_pool[pid, :, :, slot]]
                assert torch.equal(k[starts[s] + i].cpu().double(), want[0]) and torch.equal(v[starts[s] + i].cpu().double(), want[1])
        again = c.read(batch, total)
        assert torch.equal(again[0], k[:total]) and torch.equal(again[1], v[:total])


def test_calls_without_tokens(gpu):
    c = _cache(gpu, 2, 16, 2, 64, 75)
    batch, _ = _batch(gpu, [[0], [1]], [3, 0], [0, 0], max_new=1)
    before = _snapshot(c)
    k, q = torch.empty((0, 2, 64), device=gpu), torch.empty((0, 8, 64), device=gpu)
    assert c.append(batch, k, k) is None and c.append(batch, k, k, q=q).shape == (0, 8, 64)
    assert c.attend(batch, q.to(BF16), 0.125).shape == (0, 8, 64)
    assert [t.shape for t in c.read(batch, 0)] == [(0, 2, 64)] * 2
    from se12_amd.paged import rotate_heads

    assert [t.shape for t in rotate_heads(batch, q, k)] == [(0, 8, 64), (0, 2, 64)]
    for a, b in zip(before, _snapshot(c)):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# rotation by itself
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("x_dtype", [torch.float32, BF16])
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("d,heads,kvh,rotary,interleaved,norm,lengths,new", [
    (128, 8, 2, 128, False, BF16, [0, 900, 3], [1, 1, 1]),
    (256, 3, 1, 128, True, torch.float32, [70_000, 0], [5, 9]),
    (96, 5, 5, 96, False, BF16, [7, 0, 11], [40, 0, 3]),
    (8, 1, 3, 8, True, None, [3], [17]),
    (200, 2, 2, 24, False, torch.float32, [0, 5], [3, 4]),
    (64, 70, 1, 0, False, BF16, [1], [6]),
    (40, 4, 0, 32, False, None, [9], [33]),
])
def test_rotate_heads(gpu, x_dtype, dtype, d, heads, kvh, rotary, interleaved, norm, lengths, new):
    from se12_amd.paged import rotate_heads

    total = sum(new)
    batch, starts = _batch(gpu, [[0]] * len(new), lengths, new)
    g = _gen(57)
    x = (torch.randn((total + 2, (heads + kvh) * d + 8), generator=g) * 2).to(x_dtype).to(gpu)
    q, k = x[:, :heads * d].view(total + 2, heads, d), x[:, heads * d:(heads + kvh) * d].view(total + 2, kvh, d) if kvh else None
    inv = (10000.0 ** (-torch.arange(0, rotary, 2).float() / rotary)).to(gpu) if rotary else None
    w = [None, None] if norm is None else [(torch.randn(d, generator=g) * 0.3).to(norm).to(gpu) for _ in range(2)]
    out = tuple(torch.full((total + 2, h, d), 7.0, dtype=dtype, device=gpu) if h else None for h in (heads, kvh))
    got = rotate_heads(batch, q, k, inv, interleaved=interleaved, rotary_scale=1.25, q_norm=w[0], k_norm=w[1] if kvh else None, norm_offset=0.5,
                       dtype=dtype, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    for t, y, z in ((q, got[0], w[0]), (k, got[1], w[1])):
        if t is None:
            continue
        assert (y[total:] == 7.0).all()
        for s, (a, n) in enumerate(zip(lengths, new)):
            for i in range(n):
                r = starts[s] + i
                ref = e.turned(t[r].cpu(), a + i, inv, interleaved, 1.25 if rotary else 1.0, z, offset=0.5)
                size = e.turned(t[r].cpu(), 0, None, w=z, offset=0.5).abs().amax(-1, keepdim=True)
                # (2^-20 of |a| + |b|, times the scale)
                assert ((y[r].cpu().double() - ref).abs() <= (2.0 ** -8 if dtype == BF16 else 2.0 ** -24) * ref.abs() + 2.5 * 2.0 ** -20 * size).all()


def test_rotate_heads_in_place_and_as_append_does(gpu):
    """Over its inputs; the same q as an append's, whose angles are worked out from their run's first (of BF16 one in 2^16
    may differ by a step); many tokens, four to a block, as few."""
    from se12_amd.paged import rotate_heads

    d, heads, kvh, n = 128, 4, 2, 5000
    batch, _ = _batch(gpu, [[0] * 200], [100], [n])
    g = _gen(58)
    q, k = (torch.randn((n, h, d), generator=g).to(BF16).to(gpu) for h in (heads, kvh))
    inv = (10000.0 ** (-torch.arange(0, d, 2).float() / d)).to(gpu)
    w = torch.rand(d, generator=g).to(gpu)
    kw = dict(inv_freq=inv, q_norm=w, k_norm=w)
    a, b = rotate_heads(batch, q, k, **kw)
    c = _cache(gpu, 4, 128, kvh, d, 59)
    other = c.append(batch, k, k, q=q, **kw)
    assert (other != a).sum() <= 2.0 ** -16 * a.numel() and (other.float() - a.float()).abs().max() <= 2.0 ** -7 * a.float().abs().max()
    for i in (0, 17, 4990):
        few, _ = _batch(gpu, [[0]], [100 + i], [10])
        x, y = rotate_heads(few, q[i:i + 10], k[i:i + 10], **kw)
        assert torch.equal(x, a[i:i + 10]) and torch.equal(y, b[i:i + 10])
    x, y = rotate_heads(batch, q, k, out=(q, k), **kw)
    assert x is q and y is k and torch.equal(q, a) and torch.equal(k, b)


def test_norms_of_zero_rows_and_large_values(gpu):
    """x rsqrt(mean(x^2) + eps) where the squares leave FP32, and where there is nothing."""
    from se12_amd.paged import rotate_heads

    batch, _ = _batch(gpu, [[0]], [0], [5])
    x = torch.zeros((5, 1, 64))
    x[1], x[2] = 1e-30, 3e25 * torch.linspace(-1, 1, 64)
    x[3, 0, 0] = float("inf")
    x[4, 0, 5] = float("nan")
    w = torch.ones(64, device=gpu)
    for eps in (0.0, 1e-6):
        y, _ = rotate_heads(batch, x.to(gpu), q_norm=w, norm_eps=eps, dtype=torch.float32)
        y = y.cpu().double()[:, 0]
        z = x.double()[:, 0]
        ref = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + eps)
        assert torch.equal(y.isnan(), ref.isnan())
        # (three roundings to FP32; below its normals by their step)
        fine = ~ref.isnan()
        assert ((y - ref).abs()[fine] <= 3 * 2.0 ** -24 * ref.abs()[fine] + 2.0 ** -149).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def _again(c, batch, q, scaling, softcap=0.0, window=0, bound=2.0 ** -10):
    """The call once more, on what the cache and the batch hold now; `bound`: of the weights' exponents, twice."""
    table, lengths, starts = batch.page_table.tolist(), batch.lengths.tolist(), batch.starts.tolist()
    ref, size, mine, vmax = _oracle(c, table, lengths, starts, q, scaling, softcap, window, batch.max_new)
    got = c.attend(batch, q, scaling, softcap=softcap, window=window)
    _close(got, ref, size, mine, vmax, bound)
    return got


def test_attend_many_sequences(gpu):
    lengths = [(i * 37) % 90 for i in range(150)]
    _attend_case(gpu, 64, 16, 2, 1, lengths, [1 if i % 7 else 0 for i in range(150)], 0.0, 0)


@pytest.mark.parametrize("d,page,heads,kvh,softcap,window", [(64, 32, 16, 8, 0.0, 0), (64, 16, 8, 8, 30.0, 333), (128, 64, 28, 4, 0.0, 500),
                                                             (256, 32, 8, 4, 50.0, 490)])
def test_many_tiles_to_a_wave(gpu, d, page, heads, kvh, softcap, window):
    """A wave's run goes from tile to tile and over the ends of sequences, some pages named nowhere."""
    lengths = [(i * 271) % 1100 for i in range(48)]
    c, batch, q, _ = _attend_case(gpu, d, page, heads, kvh, lengths, [1] * 48, softcap, window, seed=30, extra=0)
    gone = torch.rand(batch.page_table.shape, generator=_gen(31)) < 0.3
    batch.page_table[gone.to(gpu)] = -1
    _again(c, batch, q, d ** -0.5 / 4, softcap, window)


@pytest.mark.parametrize("seqs,new,max_new,length,window", [(600, (1, 1, 0), 1, 150, 0), (150, (1, 2, 1, 0), 200, 700, 0), (90, (1, 7, 25), 40, 300, 60),
                                                            (900, (1,), 1, 90, 0)])
def test_more_units_than_waves(gpu, seqs, new, max_new, length, window):
    lengths = [(i * 271) % length for i in range(seqs)]
    news = [new[i % len(new)] for i in range(seqs)]
    if max_new == 200:
        news[77], lengths[5] = 100, 6000
    _attend_case(gpu, 64, 16, 8, 4 if seqs < 100 else 2, lengths, news, 0.0, window, seed=36, max_new=max_new)


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("window", [0, 90])
def test_prompts_among_more_sequences_than_a_wave_scans(gpu, d, window):
    new = [(0, 1, 1, 1, 5)[i % 5] for i in range(100)]
    new[3], new[70], new[71], new[99] = 40, 33, 90, 70
    _attend_case(gpu, d, 16, 4, 2, [(i * 53) % 150 for i in range(100)], new, 0.0, window, seed=60)


@pytest.mark.parametrize("d,lengths,new,window", [
    (64, [2600, 900], [70, 35], 1000), (256, [2600, 900], [70, 35], 700), (128, [0, 6000, 0, 40], [64, 64, 33, 200], 0),
    (256, [2500, 10, 10, 10, 10, 10], [33, 33, 40, 50, 60, 70], 0), (128, [4000, 10, 2000], [100, 200, 129], 1500),
])
def test_a_units_keys_in_parts(gpu, d, lengths, new, window):
    _attend_case(gpu, d, 32, 4, 1, lengths, new, 0.0, window, seed=61)


@pytest.mark.parametrize("heads,kvh,lengths,new", [(4, 1, [2600, 900], [70, 35]), (4, 2, [300, 70], [1, 1])])
def test_a_window_of_the_largest_number_hides_nothing(gpu, heads, kvh, lengths, new):
    c, batch, q, out = _attend_case(gpu, 64, 32, heads, kvh, lengths, new, 0.0, 2 ** 31 - 1, seed=67, extra=0)
    for window in (0, 2 ** 31 - 40, 1 << 30):
        assert torch.equal(c.attend(batch, q, 64 ** -0.5 / 4, window=window), out)


def test_more_query_heads_to_one_than_columns_of_a_block(gpu):
    _attend_case(gpu, 64, 16, 160, 1, [100, 5, 0], [1, 3, 1], 0.0, 0, seed=62)
    _attend_case(gpu, 256, 16, 80, 1, [300, 5], [1, 2], 0.0, 70, seed=63)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_first_tiles_of_prompts(gpu, d):
    """Many units of one, two and three tiles of 64 keys, a few times, all with the same result."""
    lengths, new = [0, 20, 31, 0, 60, 100], [32, 40, 65, 33, 60, 90]
    c, batch, q, out = _attend_case(gpu, d, 16, 32, 16, lengths, new, 0.0, 0, seed=71, extra=0)
    for _ in range(20):
        assert torch.equal(c.attend(batch, q, d ** -0.5 / 4), out)


def test_more_allowed_new_tokens_than_there_are(gpu):
    _attend_case(gpu, 128, 32, 8, 2, [100, 33, 0], [1, 1, 1], 0.0, 0, seed=64, max_new=500)
    _attend_case(gpu, 256, 16, 2, 2, [100] * 80, [1] * 80, 0.0, 20, seed=65, max_new=100)


def test_sequences_that_share_pages(gpu):
    c, batch, q, _ = _attend_case(gpu, 128, 32, 4, 2, [200, 170, 90], [1, 3, 40], 0.0, 0, seed=66, extra=0)
    batch.page_table[1, :5] = batch.page_table[0, :5]
    batch.page_table[2, 1] = batch.page_table[2, 0]
    _again(c, batch, q, 128 ** -0.5 / 4)


@pytest.mark.parametrize("new", [1, 50])
def test_caps(gpu, new):
    """The largest cap: a score is held to 2^-22 of it, here 2^-12, twice in a quotient of sums."""
    for cap in (2.0 ** -60, 0.01):
        _attend_case(gpu, 64, 32, 4, 2, [600, 3], [new, 1], cap, 0, seed=51, extra=0)
    c, batch, q, _ = _attend_case(gpu, 128, 32, 4, 2, [600, 3], [new, 1], 0.0, 0, seed=50, extra=0)
    _again(c, batch, q, 128 ** -0.5 / 4, 1024.0, bound=2.0 ** -10 + 2.0 ** -11)


@pytest.mark.parametrize("d,heads,kvh,new", [(128, 4, 4, 1), (256, 8, 4, 1), (256, 4, 2, 50), (64, 4, 2, 70)])
def test_the_maximum_moves_within_a_run(gpu, d, heads, kvh, new):
    """Keys grow along the sequences, one in 16 tokens by a factor: |q k| scaling sums to 2^9 at most here (asserted), so a
    score is off by d 2^-24 2^9 <= 2^-7, twice in a quotient of sums."""
    lengths = [(i * 271) % 1100 for i in range(24 if new == 1 else 4)]
    c, batch, q, _ = _attend_case(gpu, d, 64, heads, kvh, lengths, [new] * len(lengths), 0.0, 0, seed=40, extra=0)
    for row in batch.page_table.tolist():
        for j, pid in enumerate(row):
            c.k_scale[pid] = min(60 + 8 * (j // 3) + 3 * (j % 3), 112)
    kp = e.pools(c)[0]
    assert q.float().abs().amax().item() * kp.nan_to_num().abs().sum(-1).max().item() * d ** -0.5 / 4 <= 2.0 ** 9
    _again(c, batch, q, d ** -0.5 / 4, bound=2.0 ** -6)


@pytest.mark.parametrize("d,lengths,new,window", [(128, [1500, 40], [1, 1], 0), (64, [1500, 0, 700], [70, 90, 1], 0), (256, [900, 3], [40, 2], 300)])
@pytest.mark.parametrize("byte", [226, 1, 0])
def test_the_largest_and_least_values(gpu, d, lengths, new, window, byte):
    """Values of up to 61440 (and of the least scale, and none): sums stay numbers."""
    c, batch, q, _ = _attend_case(gpu, d, 32, 4, 2, lengths, new, 0.0, window, seed=76, extra=0)
    c.v_scale.copy_(torch.where(c.v_scale == 255, c.v_scale, byte))
    got = _again(c, batch, q, d ** -0.5 / 4, window=window)
    assert got.isfinite().all()


@pytest.mark.parametrize("d,new", [(64, 1), (128, 7), (256, 40), (128, 60)])
def test_queries_of_any_size(gpu, d, new):
    """Powers of two of q against the scaling change nothing; zeros see all keys alike; a row with no number is one alone."""
    c, batch, q, out = _attend_case(gpu, d, 32, 4, 2, [90, 300], [new, 1], 0.0, 0, seed=77, extra=0)
    for x in (2.0 ** 100, 2.0 ** -90):
        assert torch.equal(c.attend(batch, (q.float() * x).to(BF16), d ** -0.5 / 4 / x), out)
    y = q.clone()
    y[0, 1] = 0
    y[-1, 0, 3], y[-1, 2, 5] = float("nan"), float("inf")
    got = c.attend(batch, y, d ** -0.5 / 4)
    assert got[-1, 0].isnan().all() and got[-1, 2].isnan().all()
    table, starts = batch.page_table.tolist(), batch.starts.tolist()
    y[-1, 0], y[-1, 2] = q[-1, 0], q[-1, 2]
    ref, size, mine, vmax = _oracle(c, table, [90, 300], starts, y, d ** -0.5 / 4, 0.0, 0, new)
    got[-1, 0], got[-1, 2] = out[-1, 0], out[-1, 2]
    _close(got, ref, size, mine, vmax)
    assert torch.equal(got[1:], out[1:]) and torch.equal(got[0, [0, 2, 3]], out[0, [0, 2, 3]])


@pytest.mark.parametrize("d,many", [(128, 7), (64, 60), (256, 50), (256, 5), (128, 70)])
def test_what_a_query_may_not_see_has_no_part_in_its_row(gpu, d, many):
    """A later token of the call, and one behind the window, are held as no numbers: rows that do not see them stay as they
    are, the others have them in exactly their 32 columns (a key's: in all)."""
    page, lengths, new, window = 16, [40, 9], [12, many], 24
    c, batch, q, before = _attend_case(gpu, d, page, 4, 2, lengths, new, 0.0, window, seed=5, extra=0)
    table = batch.page_table.tolist()
    bad_keys = {0: (47, 20), 1: (17, 0)}
    for s, keys in bad_keys.items():
        for j in keys:
            c.k_scale[table[s][j // page], 0, 1, j % page] = 255
            c.v_scale[table[s][j // page], 1, s, j % page] = 255
    got, before = c.attend(batch, q, d ** -0.5 / 4, window=window).cpu(), before.cpu()
    r = 0
    for s, (a, n) in enumerate(zip(lengths, new)):
        for p in range(a, a + n):
            sees = any(p - window < j <= p for j in bad_keys[s])
            assert got[r, :2].isnan().all() if sees else torch.equal(got[r, :2], before[r, :2])
            at = slice(32 * s, 32 * s + 32)
            assert got[r, 2:, at].isnan().all() if sees else torch.equal(got[r, 2:, at], before[r, 2:, at])
            others = [i for i in range(d) if not 32 * s <= i < 32 * s + 32]
            assert torch.equal(got[r, 2:][:, others], before[r, 2:][:, others])
            r += 1


@pytest.mark.parametrize("d,new", [(64, 1), (256, 1), (128, 9), (64, 60), (256, 60)])
def test_values_that_are_no_numbers_are_seen_whatever_their_weight(gpu, d, new):
    """A key of great size beside the others: its weight is all or nothing, by the sign of its score."""
    c, batch, q, _ = _attend_case(gpu, d, 16, 8, 2, [150, 3], [new, 1], 0.0, 0, seed=84, extra=0)
    page = batch.page_table[0, 4].item()
    c.k_scale[page, :, :, 3] = 200                       # (2^10: scores of thousands)
    before = c.attend(batch, q, d ** -0.5 / 4)
    k = e.pools(c)[0][page, :, 3]
    scores = q[:new].cpu().double().view(new, 2, 4, d) @ k[None, :, :, None]
    assert (scores > 1000).any() and (scores < -1000).any() and before.isfinite().all()
    c.v_scale[page, :, 1, 3] = 255
    got = c.attend(batch, q, d ** -0.5 / 4)
    assert got[:new, :, 32:64].isnan().all()
    assert torch.equal(got[:new, :, :32], before[:new, :, :32]) and torch.equal(got[:new, :, 64:], before[:new, :, 64:])
    assert torch.equal(got[new:], before[new:])


@pytest.mark.parametrize("d,lengths,new,window", [(64, [200, 13], [1, 1], 60), (256, [200, 13], [40, 5], 60), (128, [77], [70], 0), (64, [0, 130], [65, 3], 20)])
def test_slots_that_are_not_seen_may_hold_any_bytes(gpu, d, lengths, new, window):
    page = 32
    c, batch, q, before = _attend_case(gpu, d, page, 4, 2, lengths, new, 0.0, window, seed=78, extra=0)
    seen = torch.zeros((c.pages, page), dtype=torch.bool)
    for row, a, n in zip(batch.page_table.tolist(), lengths, new):
        for j in range(max(0, a - window + 1) if window else 0, a + n):
            seen[row[j // page], j % page] = True
    assert not seen.all()
    for fill in (lambda s: torch.full(s, 255, dtype=torch.uint8), lambda s: torch.randint(0, 256, s, generator=_gen(79), dtype=torch.uint8)):
        for t in (c.k_scale, c.v_scale):
            x = t.cpu()
            x.permute(0, 3, 1, 2)[~seen] = fill(x.permute(0, 3, 1, 2)[~seen].shape)
            t.copy_(x)
        k = c.k.view(torch.uint8).cpu()
        k.permute(0, 2, 1, 3)[~seen] = fill(k.permute(0, 2, 1, 3)[~seen].shape)
        c.k.view(torch.uint8).copy_(k)
        assert torch.equal(c.attend(batch, q, d ** -0.5 / 4, window=window), before)


def test_pages_outside_the_pool_hold_nothing(gpu):
    for d, many in ((64, 3), (128, 70), (256, 70)):
        c = _cache(gpu, 6, 16, 2, d, 11)
        table, lengths, new = [[3, -1, 5, 0, 1], [6, 1 << 30, 2, 4, -5], [-1] * 5], [40 if many == 3 else 3, 35, 10], [many, 1, 2]
        batch, starts = _batch(gpu, table, lengths, new)
        q = torch.randn((sum(new), 4, d), generator=_gen(12)).to(BF16).to(gpu)
        ref, size, mine, vmax = _oracle(c, table, lengths, starts, q, d ** -0.5 / 4, 0.0, 0, many)
        got = c.attend(batch, q, d ** -0.5 / 4)
        _close(got, ref, size, mine, vmax)
        assert (got[starts[2]:] == 0).all()


def test_lengths_that_do_not_fit_the_table_stay_inside_it(gpu):
    from se12_amd.paged import PagedBatch, rotate_heads

    c = _cache(gpu, 4, 16, 1, 64, 13)
    as32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    batch = PagedBatch(as32([[0, 1], [2, 3]]), as32([-7, 2 ** 31 - 1]), as32([-3, 2, 2 ** 31 - 1]), max_new=3)
    guard = torch.full((2, 4 + 4, 2, 64), 9.0, dtype=BF16, device=gpu)
    x = torch.randn((4, 2, 64), generator=_gen(14)).to(gpu)
    inv = (10000.0 ** (-torch.arange(0, 64, 2).float() / 64)).to(gpu)
    c.append(batch, x[:, :1], x[:, 1:], q=x, inv_freq=inv, out=guard[0, :4])
    c.attend(batch, x.to(BF16), 0.125, out=guard[0, :4])
    rotate_heads(batch, x, x, inv, out=(guard[0, :4], guard[1, :4]))
    c.read(batch, 4, out=(guard[0, :2].view(4, 1, 64), guard[1, :2].view(4, 1, 64)))
    torch.cuda.synchronize()
    assert (guard[:, 4:] == 9.0).all()


@pytest.mark.parametrize("d,lengths,new", [(64, [40, 30, 100, 5], [2, 4, 3, 1]), (256, [20, 32, 90, 1000], [70, 40, 33, 1])])
@pytest.mark.parametrize("window", [0, 20, 64, 80])
def test_positions_beyond_the_table_are_what_they_are(gpu, d, lengths, new, window):
    page, kvh, heads = 16, 2, 4
    table = _table(4, 2, 9, 15)
    c = _cache(gpu, 9, page, kvh, d, 16)
    batch, starts = _batch(gpu, table, lengths, new)
    k, v = (torch.randn((sum(new), kvh, d), generator=_gen(17 + i)).to(gpu) for i in range(2))
    q = torch.randn((sum(new), heads, d), generator=_gen(19)).to(gpu)
    inv = (10000.0 ** (-torch.arange(0, d, 2).float() / d)).to(gpu)
    before = _snapshot(c)
    turned = c.append(batch, k, v, q=q, inv_freq=inv)
    _check_append(c, before, batch, lengths, starts, table, q, k, v, turned, dict(inv_freq=inv))
    got = _again(c, batch, turned, d ** -0.5 / 4, window=window)
    if window == 20:
        assert (got[starts[2]:starts[3]] == 0).all()      # (from 90 on nothing held is within 20)


@pytest.mark.parametrize("d,heads,kvh,lengths,new,window", [
    (256, 8, 4, [900, 20, 400, 3000], [1, 90, 1, 70], 0),                          # long units in parts, decode steps beside
    (128, 28, 4, [5000, 1], [64, 1], 0),                                           # one sequence, seven heads to one
    (256, 8, 4, [900, 20, 400], [1, 1, 1], 0),
    (64, 4, 2, [(i * 253) % 1500 for i in range(130)], [90 if i in (3, 70, 129) else i % 3 for i in range(130)], 1200),
])
def test_what_the_workspace_held_does_not_matter(gpu, d, heads, kvh, lengths, new, window):
    """A workspace of exactly the bytes asked for, of ones or zeros, with guards around it, used again for fewer tokens;
    and another stream."""
    c, batch, q, out = _attend_case(gpu, d, 64, heads, kvh, lengths, new, 0.0, window, seed=32, extra=0)
    n = c.attend_workspace(batch, q.shape[0], heads)
    for fill in (255, 0):
        guarded = torch.full((n + 2048,), fill, dtype=torch.uint8, device=gpu)
        guarded[:1024], guarded[1024 + n:] = 90, 90
        ws = guarded[1024:1024 + n]
        assert torch.equal(c.attend(batch, q, d ** -0.5 / 4, window=window, workspace=ws), out)
        few = [min(x, 1) for x in new]
        step, starts = _batch(gpu, batch.page_table.tolist(), lengths, few, max_new=max(new))
        rows = torch.tensor([s for s, x in zip(batch.starts.tolist(), new) if x], device=gpu)
        first = c.attend(step, q[rows], d ** -0.5 / 4, window=window, workspace=ws)
        ref, size, mine, vmax = _oracle(c, batch.page_table.tolist(), lengths, starts, q[rows], d ** -0.5 / 4, 0.0, window, 1)
        _close(first, ref, size, mine, vmax)
        assert (guarded[:1024] == 90).all() and (guarded[1024 + n:] == 90).all()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = c.attend(batch, q, d ** -0.5 / 4, window=window)
    s.synchronize()
    assert torch.equal(again, out)


@pytest.mark.parametrize("d", [128, 256])
def test_captured_prompts_follow_lengths_and_starts(gpu, d):
    """One captured call over other divisions of the same rows at every replay; two graphs with a workspace of their own
    in turn, eager calls between them."""
    page, heads, kvh = 32, 8, 2
    c, batch, q, out = _attend_case(gpu, d, page, heads, kvh, [500, 900, 20, 3], [100, 1, 60, 39], 0.0, 0, seed=35, extra=0)
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.where(t == 255, 100, t))
    calls = []
    for window in (0, 300):
        ws = torch.full((c.attend_workspace(batch, 200, heads),), 255, dtype=torch.uint8, device=gpu)
        y = torch.empty_like(out)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            c.attend(batch, q, d ** -0.5 / 4, window=window, out=y, workspace=ws)
        calls.append((window, graph, y, ws))
    for lengths, starts in (([500, 900, 20, 3], [0, 100, 101, 161, 200]), ([500, 800, 20, 3], [0, 1, 101, 102, 102]),
                            ([10, 890, 40, 2], [0, 33, 34, 134, 200]), ([599, 900, 79, 41], [0, 1, 2, 3, 4]),
                            ([500, 900, 20, 3], [0, 100, 101, 161, 200])):
        batch.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        batch.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        for window, graph, y, _ in calls:
            y.fill_(5.0)
            graph.replay()
            eager = c.attend(batch, q, d ** -0.5 / 4, window=window, out=torch.full_like(out, 5.0))
            torch.cuda.synchronize()
            assert torch.equal(y, eager) and (y[starts[-1]:] == 5.0).all()
            ref, size, mine, vmax = _oracle(c, batch.page_table.tolist(), lengths, starts, q, d ** -0.5 / 4, 0.0, window, 100)
            _close(y, ref, size, mine, vmax)
    assert torch.equal(calls[0][2], out)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("d,interleaved", [(64, False), (256, True)])
def test_prompt_then_captured_decode_steps_then_read(gpu, d, interleaved):
    """Prompts of different lengths, normed and rotated, then decode steps replayed from one graph whose lengths move on the
    device: every step against the oracle on the cache as it is, and against the same calls made one by one; then all read
    back, and drafts of four tokens over it."""
    from se12_amd.paged import PagedBatch, rotate_heads

    page, heads, kvh = 16, 4, 2
    prompts, columns = [37, 1, 16], 5
    table = _table(3, columns, 3 * columns + 1, 40)
    inv = (10000.0 ** (-torch.arange(0, d, 2).float() / d)).to(gpu)
    w = [(torch.rand(d, generator=_gen(43 + i)) + 0.5).to(BF16).to(gpu) for i in range(2)]
    turn = dict(inv_freq=inv, interleaved=interleaved, q_norm=w[0], k_norm=w[1])
    as32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    outs, reads = [], []
    for captured in (False, True):
        c = _cache(gpu, 3 * columns + 1, page, kvh, d, 41)
        lengths, step_starts = as32([0, 0, 0]), as32([0, 1, 2, 3])
        batch, starts = _batch(gpu, table, [0, 0, 0], prompts)
        g = _gen(42)
        x = torch.randn((sum(prompts), heads + 2 * kvh, d), generator=g).to(gpu)
        q, k, v = x.split([heads, kvh, kvh], 1)
        qr = c.append(batch, k, v, q=q, **turn)
        _again(c, batch, qr, d ** -0.5 / 4, 50.0)
        lengths += as32(prompts)
        batch = PagedBatch(as32(table), lengths, step_starts)
        x = torch.empty((3, heads + 2 * kvh, d), device=gpu)
        q_out, y, q_by_itself = (torch.empty((3, heads, d), dtype=BF16, device=gpu) for _ in range(3))

        def step():
            q, k, v = x.split([heads, kvh, kvh], 1)
            c.append(batch, k, v, q=q, out=q_out, **turn)
            rotate_heads(batch, q, None, inv, interleaved=interleaved, q_norm=w[0], out=(q_by_itself, None))
            c.attend(batch, q_out, d ** -0.5 / 4, softcap=50.0, out=y)
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
            ref, size, mine, vmax = _oracle(c, table, at, [0, 1, 2, 3], q_out, d ** -0.5 / 4, 50.0, 0, 1)
            _close(y, ref, size, mine, vmax)
            assert (q_by_itself.float() - q_out.float()).abs().max() <= 2.0 ** -7 * q_out.float().abs().max()
            at = [a + 1 for a in at]
            assert lengths.tolist() == at
            outs.append(y.cpu().clone())
        whole, starts = _batch(gpu, table, [0, 0, 0], at)
        reads.append([t.cpu() for t in c.read(whole, starts[-1])])
        k_pool, v_pool = e.pools(c)
        for s, n in enumerate(at):
            for i in range(n):
                assert torch.equal(reads[-1][0][starts[s] + i].double(), k_pool[table[s][i // page], :, i % page])
                assert torch.equal(reads[-1][1][starts[s] + i].double(), v_pool[table[s][i // page], :, :, i % page])
        drafts, _ = _batch(gpu, table, at, [4, 4, 4])
        x = torch.randn((12, heads + 2 * kvh, d), generator=g).to(gpu)
        q, k, v = x.split([heads, kvh, kvh], 1)
        _again(c, drafts, c.append(drafts, k, v, q=q, **turn), d ** -0.5 / 4, 50.0)
    for a, b in zip(outs[:20], outs[20:]):
        assert torch.equal(a, b)
    for a, b in zip(*reads):
        assert torch.equal(a, b)


def test_rows_beyond_32_bit_offsets(gpu):
    """Rows 2^30 values apart; and outputs of more than 2^31 values, of one sequence that holds two pages over and over."""
    from se12_amd.paged import rotate_heads

    d, heads, kvh = 64, 4, 2
    x = torch.empty((4, 1 << 30), dtype=BF16, device=gpu)
    near = torch.randn((4, (heads + 2 * kvh) * d), generator=_gen(80)).to(BF16).to(gpu)
    x[:, :near.shape[1]] = near
    inv = (10000.0 ** (-torch.arange(0, d, 2).float() / d)).to(gpu)
    w = torch.rand(d, generator=_gen(81)).to(gpu)
    got = []
    for rows in (x, near):
        q, k, v = rows[:, :near.shape[1]].unflatten(1, (heads + 2 * kvh, d)).split([heads, kvh, kvh], 1)
        c = _cache(gpu, 4, 16, kvh, d, 82)
        batch, _ = _batch(gpu, [[0, 1], [2, 3]], [3, 15], [2, 2])
        got.append([c.append(batch, k, v, q=q, inv_freq=inv, q_norm=w), *_snapshot(c), c.attend(batch, q, 0.125), *rotate_heads(batch, q, k, inv)])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    del x, q, k, v, rows
    d, kvh, page, n = 256, 8, 128, 1_050_000
    c = _cache(gpu, 2, page, kvh, d, 83)
    columns = (n + page - 1) // page
    batch, _ = _batch(gpu, [[j % 2 for j in range(columns)]], [0], [n])
    k, v = c.read(batch, n)
    k_pool, v_pool = e.pools(c)
    for r in (0, page, n // 2, 1_048_575, 1_048_576, n - 1):
        assert torch.equal(k[r].cpu().double(), k_pool[r // page % 2, :, r % page]) and torch.equal(v[r].cpu().double(), v_pool[r // page % 2, :, :, r % page])
    inv = (10000.0 ** (-torch.arange(0, d, 2).float() / d)).to(gpu)
    turned, _ = rotate_heads(batch, k, None, inv)
    for r in (0, 1_048_575, 1_048_576, n - 4, n - 1):
        one, _ = _batch(gpu, [[0]], [r], [1])
        assert torch.equal(rotate_heads(one, k[r:r + 1], None, inv)[0], turned[r:r + 1])


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, BF16])
def test_norms_for_caches_of_other_types_in_a_graph(gpu, dtype):
    """Steps of a cache that norms before it appends, replayed with eager work between, against the same one by one."""
    from se12_amd.paged import PagedBatch, PagedKvCache

    d, kvh, heads = 64, 2, 4
    inv = (10000.0 ** (-torch.arange(0, d, 2).float() / d)).to(gpu)
    w = (torch.rand(d, generator=_gen(90)) + 0.5).to(gpu)
    as32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    outs = []
    for captured in (False, True):
        c = PagedKvCache(6, 16, kvh, d, dtype=dtype, device=gpu)
        lengths = as32([14, 0])
        batch = PagedBatch(as32([[0, 2, 4], [1, 3, 5]]), lengths, as32([0, 1, 2]))
        x, y, g = torch.empty((2, heads + 2 * kvh, d), dtype=BF16, device=gpu), torch.empty((2, heads, d), dtype=BF16, device=gpu), _gen(91)

        def step():
            q, k, v = x.split([heads, kvh, kvh], 1)
            c.attend(batch, c.append(batch, k, v, q=q, inv_freq=inv, interleaved=True, q_norm=w, k_norm=w), 0.125, out=y)
            lengths.add_(1)

        if captured:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                step()
        for _ in range(6):
            x.copy_(torch.randn(x.shape, generator=g))
            graph.replay() if captured else step()
            outs.append((y.cpu(), c.k.float().cpu(), c.v.float().cpu()))
            torch.randn(1000, device=gpu).sum().item()
    for a, b in zip(outs[:6], outs[6:]):
        for s, t in zip(a, b):
            assert torch.equal(s, t)


@pytest.mark.parametrize("d,page,kvh,heads,rotary,interleaved,norm,lengths,new", [
    (256, 64, 3, 3, 256, False, BF16, [5, 130], [40, 17]),                 # heads in pairs, one left
    (128, 16, 5, 10, 64, True, torch.float32, [0, 33], [70, 12]),
    (64, 32, 3, 12, 56, False, None, [1], [100]),
    (256, 128, 1, 2, 248, False, BF16, [9], [31]),                         # one head; pairs apart by no multiple of 8
    (64, 16, 2, 2, 8, False, torch.float32, [3, 14], [33, 20]),
    (128, 64, 7, 7, 0, False, BF16, [60], [75]),
])
def test_append_of_odd_numbers_of_heads(gpu, d, page, kvh, heads, rotary, interleaved, norm, lengths, new):
    columns = max((a + n + page - 1) // page for a, n in zip(lengths, new))
    pages = len(new) * columns + 1
    table = _table(len(new), columns, pages, 92)
    c = _cache(gpu, pages, page, kvh, d, 93)
    batch, starts = _batch(gpu, table, lengths, new)
    g = _gen(94)
    x = torch.randn((starts[-1], heads + 2 * kvh, d), generator=g).to(BF16).to(gpu)
    q, k, v = x.split([heads, kvh, kvh], 1)
    inv = (10000.0 ** (-torch.arange(0, rotary, 2).float() / rotary)).to(gpu) if rotary else None
    w = [None, None] if norm is None else [(torch.rand(d, generator=g) + 0.5).to(norm).to(gpu) for _ in range(2)]
    before = _snapshot(c)
    got = c.append(batch, k, v, q=q, inv_freq=inv, interleaved=interleaved, q_norm=w[0], k_norm=w[1])
    _check_append(c, before, batch, lengths, starts, table, q, k, v, got, dict(inv_freq=inv, interleaved=interleaved, q_norm=w[0], k_norm=w[1]))


def test_a_cache_in_the_callers_tensors_and_values_at_odd_addresses(gpu):
    """from_tensors holds them in place; frequencies and weights need not be aligned."""
    from se12_amd.paged import PagedKvCache, rotate_heads

    c = _cache(gpu, 4, 16, 2, 64, 95)
    other = PagedKvCache.from_tensors(c.k, c.v, c.k_scale, c.v_scale)
    batch, _ = _batch(gpu, [[0, 2], [1, 3]], [3, 0], [20, 1])
    g = _gen(96)
    q, k, v = (torch.randn((21, h, 64), generator=g).to(gpu) for h in (4, 2, 2))
    inv = 10000.0 ** (-torch.arange(0, 64, 2).float() / 64)
    w = torch.rand(64, generator=g)
    odd = [torch.cat([torch.zeros(1), t]).to(gpu)[1:] for t in (inv, w)]
    assert all(t.data_ptr() % 16 for t in odd)
    a = other.append(batch, k, v, q=q, inv_freq=odd[0], q_norm=odd[1], k_norm=odd[1])
    state = _snapshot(c)
    b = c.append(batch, k, v, q=q, inv_freq=inv.to(gpu), q_norm=w.to(gpu), k_norm=w.to(gpu))
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(state, _snapshot(c)))
    assert torch.equal(other.attend(batch, a, 0.125), c.attend(batch, a, 0.125))
    for x, y in zip(rotate_heads(batch, q, k, odd[0], q_norm=odd[1]), rotate_heads(batch, q, k, inv.to(gpu), q_norm=w.to(gpu))):
        assert torch.equal(x, y)


def test_the_plain_append_entry_serves_4_bits_too(gpu):
    import ctypes

    from se12_amd import _native as nat

    batch, _ = _batch(gpu, [[0, 2], [1, 3]], [3, 0], [20, 1])
    q, k, v = (torch.randn((21, h, 64), generator=_gen(97)).to(gpu) for h in (4, 2, 2))
    inv = (10000.0 ** (-torch.arange(0, 32, 2).float() / 32)).to(gpu)
    a, b = _cache(gpu, 4, 16, 2, 64, 98), _cache(gpu, 4, 16, 2, 64, 98)
    out = torch.empty((21, 4, 64), dtype=BF16, device=gpu)
    nat.step_check(nat.lib().se12_step_paged_append(a._struct, batch._struct(21), q.data_ptr(), k.data_ptr(), v.data_ptr(), nat.STEP_F32, 256, 128, 128, 4,
                                                    inv.data_ptr(), 32, out.data_ptr(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert torch.equal(out, b.append(batch, k, v, q=q, inv_freq=inv))
    assert all(torch.equal(x, y) for x, y in zip(_snapshot(a), _snapshot(b)))


@pytest.mark.parametrize("d,new", [(64, 1), (128, 7), (256, 1), (64, 70), (128, 60), (256, 50)])
@pytest.mark.parametrize("scaling,softcap", [(2.0 ** 100, 0.0), (-2.0 ** 100, 0.0), (2.0 ** 100, 50.0)])
def test_scores_beyond_fp32(gpu, d, new, scaling, softcap):
    """Queries and a scaling whose product FP32 does not hold: the largest score has all the weight (those alike share it; of
    capped ones all above 0), and a key of zeros a score of 0. Sums of whole numbers up to 3 times codes times scales of 4
    bits: exact."""
    c, batch, q, _ = _attend_case(gpu, d, 32, 4, 2, [90, 300], [new, 1], 0.0, 0, seed=87, extra=0)
    table = batch.page_table.tolist()
    for s, slot in ((0, 3), (1, 40)):
        c.k_scale[table[s][slot // 32], :, :, slot % 32] = 0
    y = (torch.randint(-3, 4, q.shape, generator=_gen(88)) * 2.0 ** 100).to(BF16).to(gpu)
    y[-1, 2] = 0
    got = _again(c, batch, y, scaling, softcap)
    assert got.isfinite().all()
    # (where nothing is above 0 but the key of zeros, it is the largest)
    pid = table[1][1]
    one = _batch(gpu, [[pid]], [9], [1])[0]
    k = c.k.view(torch.uint8)
    k[pid, :, :10] = 0x22
    k[pid, :, 8] = 0
    c.k_scale[pid, :, :, :10] = 120
    c.v_scale[pid, :, :, :10] = 120
    down = torch.full((1, 4, d), -2.0 ** 100, dtype=BF16, device=gpu)
    got = c.attend(one, down, abs(scaling))
    _, v = c.read(_batch(gpu, [[pid]], [8], [1])[0], 1)
    assert torch.equal(got, v.repeat_interleave(2, 1))


@pytest.mark.parametrize("interleaved", [False, True])
def test_angles_of_any_size(gpu, interleaved):
    """Frequencies up to FP32's largest: a rotation keeps a pair's length whatever its angle, and below 2^51 quarter turns it
    is that of the angle in 64 bits."""
    from se12_amd.paged import rotate_heads

    d, heads, kvh = 64, 4, 2
    inv = 2.0 ** torch.linspace(-20, 127, 32)
    inv[-1] = torch.finfo(torch.float32).max
    lengths, new = [0, 1001, 1 << 29], [20, 3, 17]
    batch, starts = _batch(gpu, [[0] * 70, [1] * 70, [2] * 70], lengths, new)
    g = _gen(89)
    q, k, v = (torch.randn((40, h, d), generator=g).to(gpu) for h in (heads, kvh, kvh))
    turned = rotate_heads(batch, q, k, inv.to(gpu), interleaved=interleaved, dtype=torch.float32)
    c = _cache(gpu, 9, 16, kvh, d, 90)
    appended = c.append(batch, k, v, q=q, inv_freq=inv.to(gpu), interleaved=interleaved)
    pairs = (lambda t: t.unflatten(-1, (32, 2))) if interleaved else (lambda t: t.unflatten(-1, (2, 32)).transpose(-2, -1))
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(lengths, new)]).double()
    small = pos[:, None] * inv.double() < 2.0 ** 51
    for got, x, step in ((turned[0], q, 0.0), (turned[1], k, 0.0), (appended, q, 2.0 ** -8)):
        got, x = got.cpu().double(), x.cpu()
        a, b = pairs(got), pairs(x.double())
        # (FP32: a cosine, a sine, two products and a sum, each 2^-24 of itself: 2^-21 of |a| + |b|)
        size = b.abs().sum(-1)
        assert ((a.square().sum(-1).sqrt() - b.square().sum(-1).sqrt()).abs() <= (2 * step + 2.0 ** -20) * size).all()
        ref = pairs(torch.stack([e.turned(x[r], pos[r].item(), inv, interleaved) for r in range(40)]))
        off = (a - ref).abs() <= step * ref.abs() + 2.0 ** -20 * size[..., None]
        assert off.transpose(1, 2).flatten(2)[small].all()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompts_beyond_32_bit_offsets(gpu, d):
    """More than 64 columns to a KV head, of one unit alone and of keys in parts: pages beyond 4 GiB of codes as near ones, and
    queries 2^30 values apart as side by side."""
    from se12_amd.paged import PagedKvCache

    page, kvh, heads, new = 128, 8, 24, [40, 23, 30]
    g = _gen(91)
    columns = 12
    pages = (9 << 29) // (kvh * page * d // 2)      # 4.5 GiB of codes
    q, k, v = (torch.randn((1593, h, d), generator=g).to(BF16).to(gpu) for h in (heads, kvh, kvh))
    got = []
    for count in (pages, 3 * columns):
        c = PagedKvCache(count, page, kvh, d, dtype=FP4, device=gpu)
        table = [[count - 1 - columns * s - j for j in range(columns)] for s in range(3)]
        before, _ = _batch(gpu, table, [0] * 3, [100, 0, 1493])
        c.append(before, k, v)
        batch, _ = _batch(gpu, table, [100, 0, 1493], new)
        turned = c.append(batch, k[:93], v[:93], q=q[:93])
        got.append(c.attend(batch, turned, d ** -0.5))
        del c
    assert torch.equal(*got) and got[0].isfinite().all()
    c = _cache(gpu, 8, page, 1, d, 92)
    batch, _ = _batch(gpu, [[4, 1, 3, 0, 2, 5, 7, 6]], [700], [3])
    near = q[:3].reshape(3, heads * d)
    far = torch.empty((3, 1 << 30), dtype=BF16, device=gpu)
    far[:, :heads * d] = near
    assert torch.equal(c.attend(batch, far[:, :heads * d].view(3, heads, d), d ** -0.5), c.attend(batch, near.view(3, heads, d), d ** -0.5))
