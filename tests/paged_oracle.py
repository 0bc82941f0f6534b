"""The paged cache's operators in plain 64-bit form, a sequence, page and head at a
time on the CPU: what se12_step_paged_append and se12_step_paged_attention are
compared with."""

from __future__ import annotations

import torch

MIN_EXPONENT = -100


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest E4M3 values, ties to even, as float64 (|x| <= 448; NaN and infinities give NaN)."""
    fine = torch.isfinite(x)
    y = torch.where(fine, x, torch.zeros_like(x)).double()
    step = torch.exp2(torch.frexp(y)[1].double().sub(4).clamp(min=-9))
    return torch.where(fine, torch.round(y / step) * step, torch.full_like(y, float("nan")))


def scale_for(x: torch.Tensor) -> float:
    """The least 2^e, e >= MIN_EXPONENT, with the finite |x| <= 448 * 2^e."""
    top = x[torch.isfinite(x)].abs().max().item() if torch.isfinite(x).any() else 0.0
    e = MIN_EXPONENT
    while top > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def turned(x: torch.Tensor, pos: int, inv_freq: torch.Tensor | None) -> torch.Tensor:
    """x [heads, head_dim] of one token, rotated to its position."""
    x = x.double().clone()
    if inv_freq is None:
        return x
    h = inv_freq.numel()
    angle = pos * inv_freq.double()
    a, b = x[:, :h].clone(), x[:, h:2 * h].clone()
    x[:, :h] = a * angle.cos() - b * angle.sin()
    x[:, h:2 * h] = b * angle.cos() + a * angle.sin()
    return x


def append(k_pool, v_pool, k_scale, v_scale, table, lengths, starts, k, v, inv_freq, max_new, q=None):
    """Pools as float64 of the held codes ([pages, heads, page, d] and [pages, heads, d, page]), changed in place;
    scales None for a BF16 cache (whose values stay unrounded here). Returns q rotated and the slots written
    [pages, page]."""
    pages, heads, page, _ = k_pool.shape
    written = torch.zeros((pages, page), dtype=torch.bool)
    q_out = None if q is None else q.double().clone()
    for s in range(len(lengths)):
        n = min(starts[s + 1] - starts[s], max_new)
        rows = {}
        for i in range(n):
            pos, r = lengths[s] + i, starts[s] + i
            if q is not None:
                q_out[r] = turned(q[r], pos, inv_freq)
            if pos // page < len(table[s]) and 0 <= table[s][pos // page] < pages:
                rows.setdefault(pos // page, []).append((pos % page, turned(k[r], pos, inv_freq), v[r].double()))
        for c, tokens in rows.items():
            pid, first = table[s][c], tokens[0][0]
            for pool, scale, which in ((k_pool, k_scale, 1), (v_pool.transpose(2, 3), v_scale, 2)):
                for h in range(heads):
                    x = torch.stack([t[which][h] for t in tokens])
                    if scale is None:
                        pool[pid, h, first:first + len(tokens)] = x
                        continue
                    was, now = scale[pid, h].item(), scale_for(x)
                    if first:
                        now = max(now, was)
                        if now != was:
                            pool[pid, h, :first] = e4m3(pool[pid, h, :first] * (was / now))
                    pool[pid, h, first:first + len(tokens)] = e4m3(x / now)
                    scale[pid, h] = now
            written[pid, first:first + len(tokens)] = True
    return q_out, written


def attend(k_pool, v_pool, k_scale, v_scale, table, lengths, starts, q, scaling, softcap, window, max_new):
    """Per query and head what it sees, exactly: (out, sum of weights times |v|) [tokens, heads, d], float64, and the
    rows that belong to a sequence. Pools float64 codes; scales None: 1."""
    pages, kvh, page, d = k_pool.shape
    tokens, heads, _ = q.shape
    g = heads // kvh
    out, size = torch.zeros((tokens, heads, d), dtype=torch.float64), torch.zeros((tokens, heads, d), dtype=torch.float64)
    mine = torch.zeros(tokens, dtype=torch.bool)
    for s in range(len(lengths)):
        n = min(starts[s + 1] - starts[s], max_new)
        keys = min(lengths[s] + n, len(table[s]) * page)
        for i in range(n):
            pos, r = lengths[s] + i, starts[s] + i
            mine[r] = True
            lo = max(0, pos - window + 1) if window else 0
            seen = [j for j in range(lo, min(pos + 1, keys)) if 0 <= table[s][j // page] < pages]
            if not seen:
                continue
            pid, slot = torch.tensor([table[s][j // page] for j in seen]), torch.tensor([j % page for j in seen])
            for h in range(kvh):
                k, v = k_pool[pid, h, slot], v_pool[pid, h, :, slot]
                if k_scale is not None:
                    k, v = k * k_scale[pid, h, None].double(), v * v_scale[pid, h, None].double()
                sc = q[r, h * g:(h + 1) * g].double() @ k.T * scaling
                if softcap:
                    sc = softcap * torch.tanh(sc / softcap)
                w = torch.softmax(sc, -1)
                out[r, h * g:(h + 1) * g] = w @ v
                size[r, h * g:(h + 1) * g] = w @ v.abs()
    return out, size, mine
