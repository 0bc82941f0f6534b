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
