"""The operators a program that serves many sequences at once calls besides the
products: a key/value cache in pages, the attention that reads it, and what is
reported of the logits. Each in its plain form, and through the package.

A case is a dict with an "op" and its sizes:

  append    q and k rotated to their tokens' positions, k and v written to the
            pages of their sequences (PagedKvCache.append); a cache of E4M3 has
            one power-of-two scale per page and head, which grows with what is
            appended
  attend    attention of the new tokens over their sequences' pages
            (PagedKvCache.attend): one token per sequence in a decode step,
            several where drafted tokens are checked, many for a prompt
  logprobs  log probabilities of given tokens, entropy and the most likely
            alternatives of every row of logits (token_logprobs)

"held" tokens are in the cache before the call, up to "new" more come with it.
With "ragged" the sequences differ in both. The pages of a sequence lie anywhere
in the pool, and what lies behind its last token is left over from others.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0
MIN_EXPONENT = -100          # scales are 2^MIN_EXPONENT or more


def listed() -> list[dict]:
    return [
        # one user, one new token, Gemma-2-2B's heads: the smallest call
        {"name": "append_2b_b1", "op": "append", "seqs": 1, "held": 777, "new": 1, "ragged": False, "heads": 8,
         "kv_heads": 4, "head_dim": 256, "page": 64, "cache": "e4m3", "x": "f32", "rotary": 256},
        # a decode step of 48 sequences, Gemma-2-9B's heads
        {"name": "append_9b_b48", "op": "append", "seqs": 48, "held": 900, "new": 1, "ragged": True, "heads": 16,
         "kv_heads": 8, "head_dim": 256, "page": 32, "cache": "e4m3", "x": "f32", "rotary": 256},
        # prompts of different lengths written behind what is there
        {"name": "append_prompts", "op": "append", "seqs": 7, "held": 500, "new": 1999, "ragged": True, "heads": 16,
         "kv_heads": 8, "head_dim": 256, "page": 64, "cache": "e4m3", "x": "bf16", "rotary": 256},
        # one user, a thousand tokens back: latency
        {"name": "attend_2b_b1", "op": "attend", "seqs": 1, "held": 1023, "new": 1, "ragged": False, "heads": 8,
         "kv_heads": 4, "head_dim": 256, "page": 64, "cache": "e4m3", "softcap": 50.0, "window": 0},
        # a decode step of 32 sequences of different lengths, Gemma-2-9B's heads
        {"name": "attend_9b_b32", "op": "attend", "seqs": 32, "held": 4095, "new": 1, "ragged": True, "heads": 16,
         "kv_heads": 8, "head_dim": 256, "page": 64, "cache": "e4m3", "softcap": 50.0, "window": 0},
        # the same without loss: a BF16 cache, and a window
        {"name": "attend_bf16_b24", "op": "attend", "seqs": 24, "held": 5000, "new": 1, "ragged": True, "heads": 8,
         "kv_heads": 4, "head_dim": 256, "page": 32, "cache": "bf16", "softcap": 50.0, "window": 4096},
        # three long documents, seven query heads to a key head
        {"name": "attend_long_b3", "op": "attend", "seqs": 3, "held": 65000, "new": 1, "ragged": True, "heads": 28,
         "kv_heads": 4, "head_dim": 128, "page": 128, "cache": "e4m3", "softcap": 0.0, "window": 0},
        # five drafted tokens of each of 12 sequences are checked at once
        {"name": "attend_draft_b12", "op": "attend", "seqs": 12, "held": 2500, "new": 5, "ragged": True, "heads": 16,
         "kv_heads": 8, "head_dim": 128, "page": 16, "cache": "e4m3", "softcap": 0.0, "window": 0},
        # prompts in chunks behind what is held
        {"name": "attend_prompts", "op": "attend", "seqs": 5, "held": 1500, "new": 1700, "ragged": True, "heads": 8,
         "kv_heads": 4, "head_dim": 256, "page": 64, "cache": "e4m3", "softcap": 50.0, "window": 0},
        # one sampled token with its twenty alternatives, Gemma-2's vocabulary
        {"name": "logprobs_b1", "op": "logprobs", "rows": 1, "vocab": 256000, "x": "f32", "top": 20, "softcap": 30.0,
         "masked": False},
        # a step of 40 sequences under a grammar that allows half of the tokens
        {"name": "logprobs_b40", "op": "logprobs", "rows": 40, "vocab": 100277, "x": "bf16", "top": 5, "softcap": 0.0,
         "masked": True},
        # every token of a prompt scored
        {"name": "logprobs_prompt", "op": "logprobs", "rows": 1024, "vocab": 256000, "x": "f32", "top": 5,
         "softcap": 30.0, "masked": False},
    ]


# ---------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------


def _log(rng, lo: float, hi: float) -> int:
    return max(int(lo), int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "logprobs", "logprobs"])
    if op == "logprobs":
        vocab = _log(rng, 300, 256000)
        rows = _log(rng, 1, max(2, min(4096, 100e6 / vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "x": rng.choice(["f32", "bf16"]), "top": rng.choice([0, 1, 5, 20, 32]),
                "softcap": rng.choice([0.0, 30.0]), "masked": rng.random() < 0.3}
    kv = rng.choice([1, 2, 3, 4, 8])
    case = {"op": op, "ragged": rng.random() < 0.7, "heads": kv * rng.choice([1, 2, 3, 4, 5, 7, 8]), "kv_heads": kv,
            "head_dim": rng.choice([64, 128, 256]), "page": rng.choice([16, 32, 64, 128]),
            "cache": rng.choice(["e4m3", "e4m3", "bf16"])}
    case["seqs"] = _log(rng, 1, 64.49)
    if op == "append":
        case["new"] = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 9, 4000)])
        while case["seqs"] * case["new"] * (case["heads"] + 2 * kv) * case["head_dim"] > 50e6:
            smaller = "seqs" if case["seqs"] > 1 else "new"
            case[smaller] //= 2
        case["held"] = rng.choice([0, _log(rng, 1, 3000), _log(rng, 1, 3000)])
        return {**case, "x": rng.choice(["f32", "bf16"]), "rotary": rng.choice([case["head_dim"], case["head_dim"] // 2])}
    case["new"] = rng.choice([1, 1, 1, _log(rng, 2, 8), _log(rng, 9, 1500)])
    case["held"] = rng.choice([0, _log(rng, 1, 16000), _log(rng, 1, 16000), _log(rng, 1, 16000)])
    while (case["seqs"] * (case["held"] + case["new"]) * kv * case["head_dim"] > 80e6
           or case["seqs"] * case["new"] * (case["held"] + case["new"]) * case["heads"] * case["head_dim"] > 15e9):
        smaller = "seqs" if case["seqs"] > 1 else "held" if case["held"] > case["new"] else "new"
        case[smaller] //= 2
    return {**case, "softcap": rng.choice([0.0, 0.0, 50.0]), "window": rng.choice([0, 0, 1024, 4096])}


def _tokens(case: dict) -> tuple[list[int], list[int]]:
    """Tokens held before the call and new ones, per sequence: "held" and "new" for the first sequence; where
    "ragged", an eighth of that up to all of it for the others."""
    held, new = [], []
    for i in range(case["seqs"]):
        a = 1.0 - (i * 0.6180339887) % 1.0 * 0.875 if case["ragged"] else 1.0
        b = 1.0 - (i * 0.7548776662) % 1.0 * 0.875 if case["ragged"] else 1.0
        held.append(int(case["held"] * a))
        new.append(max(1, int(case["new"] * b)))
    return held, new


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _gen(seed: int, salt: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1009 + salt)
    return g


def _int32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _randn(shape, seed: int, salt: int) -> torch.Tensor:
    return torch.randn(shape, generator=_gen(seed, salt), device=DEV)


def _held_pages(x: torch.Tensor, cache: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Pages [pages, kv_heads, ..] of values as the cache holds them, and their scales [pages, kv_heads]."""
    if cache == "bf16":
        return x.to(torch.bfloat16), torch.ones(x.shape[:2], device=DEV)
    amax = x.abs().amax((2, 3))
    scale = torch.exp2(torch.ceil(torch.log2(amax / E4M3_MAX)))
    return (x / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale


def prepare(case: dict, seed: int) -> dict:
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = _randn((rows, vocab), seed, 1).mul_(3.0)
        # a few tokens stand out, as in a model's logits
        at = torch.randint(0, vocab, (rows, 8), generator=_gen(seed, 2), device=DEV)
        x.scatter_add_(1, at, 10.0 + 2.0 * _randn((rows, 8), seed, 3))
        tokens = torch.where(torch.arange(rows, device=DEV) % 2 == 0, x.argmax(1),
                             torch.randint(0, vocab, (rows,), generator=_gen(seed, 4), device=DEV))
        if case["masked"]:
            allowed = torch.rand((rows, vocab), generator=_gen(seed, 5), device=DEV) < 0.5
            allowed.scatter_(1, tokens[:, None], True)
            x.masked_fill_(~allowed, float("-inf"))
        return {"case": case, "logits": x.to(torch.bfloat16) if case["x"] == "bf16" else x, "tokens": tokens}

    held, new = _tokens(case)
    kvh, d, page, seqs = case["kv_heads"], case["head_dim"], case["page"], case["seqs"]
    total = sum(new)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    need = [-(-(h + n) // page) for h, n in zip(held, new)]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=_gen(seed, 10), device=DEV).to(torch.int32)
    at = torch.tensor([sum(need[:i]) for i in range(seqs)], device=DEV)
    column = torch.arange(max(need), device=DEV)
    # entries behind a sequence's last page are never read
    table = torch.where(column < torch.tensor(need, device=DEV)[:, None],
                        order[(at[:, None] + column).clamp(max=pages - 1)], torch.full((), -1, dtype=torch.int32, device=DEV))
    k, k_scale = _held_pages(_randn((pages, kvh, page, d), seed, 11) * (0.5 + 1.5 * torch.rand(d, generator=_gen(seed, 12), device=DEV)),
                             case["cache"])
    v, v_scale = _held_pages(_randn((pages, kvh, d, page), seed, 13), case["cache"])
    state = {"case": case, "k": k, "v": v, "table": table, "lengths": _int32(held), "starts": _int32(starts), "max_new": max(new),
             "max_keys": max(h + n for h, n in zip(held, new)), "k_scale": k_scale if case["cache"] == "e4m3" else None,
             "v_scale": v_scale if case["cache"] == "e4m3" else None}
    if case["op"] == "append":
        t = torch.bfloat16 if case["x"] == "bf16" else torch.float32
        state["q_new"] = _randn((total, case["heads"], d), seed, 14).to(t)
        state["k_new"] = (1.3 * _randn((total, kvh, d), seed, 15)).to(t)
        state["v_new"] = _randn((total, kvh, d), seed, 16).to(t)
        r = case["rotary"]
        state["inv_freq"] = 10000.0 ** (-torch.arange(0, r, 2, device=DEV, dtype=torch.float32) / r)
    else:
        state["q"] = _randn((total, case["heads"], d), seed, 17).mul_(1.5).to(torch.bfloat16)
    if own:
        from se12_amd.paged import PagedBatch, PagedKvCache

        state["cache"] = PagedKvCache.from_tensors(k, v, state["k_scale"], state["v_scale"])
        state["batch"] = PagedBatch(table, state["lengths"], state["starts"], max_new=state["max_new"])
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _new_tokens(s: dict, total: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(sequence, position) of every new token."""
    t = torch.arange(total, device=DEV)
    starts = s["starts"].long()
    seq = (t[:, None] >= starts[None, 1:]).sum(1)
    return seq, s["lengths"].long()[seq] + t - starts[seq]


def _rotated(x: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor) -> torch.Tensor:
    angle = pos.double()[:, None] * inv_freq.double()       # the angle of a far position needs 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    h = inv_freq.numel()
    x = x.float()
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)


def _pages(pool: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
    """The pages' values (of E4M3: before their scale) in FP32."""
    if pool.dtype == torch.bfloat16:
        return pool[ids].float()
    return pool.view(torch.uint8)[ids].view(pool.dtype).float()


def _write(pool, scale, x, seq, pos, s, transposed: bool) -> None:
    """x [tokens, kv_heads, head_dim] into the pages; `transposed` pages hold a token as a column."""
    page_size = s["case"]["page"]
    page, slot = s["table"].long()[seq, pos // page_size], pos % page_size
    if scale is None:
        values = x.to(torch.bfloat16)
        if transposed:
            pool.transpose(2, 3)[page, :, slot] = values
        else:
            pool[page, :, slot] = values
        return
    # one scale per page and head: the least power of two that holds what is new, and never less than before
    # while older tokens share the page
    touched, group = torch.unique(page, return_inverse=True)
    heads = x.shape[1]
    amax = torch.zeros((touched.numel(), heads), device=DEV).scatter_reduce_(0, group[:, None].expand(-1, heads),
                                                                             x.abs().amax(2), "amax")
    first = torch.full((touched.numel(),), page_size, device=DEV).scatter_reduce_(0, group, slot, "amin")
    m, e = torch.frexp(amax)                                   # amax = m 2^e, 448 = 0.875 2^9
    need = torch.exp2((e - 9 + (m > 0.875).int()).float().clamp(min=MIN_EXPONENT))
    need = torch.where(amax > 0, need, torch.full_like(need, 2.0 ** MIN_EXPONENT))
    old = scale[touched]
    now = torch.where((first > 0)[:, None], torch.maximum(old, need), need)
    again = (_pages(pool, touched) * (old / now)[:, :, None, None]).to(torch.float8_e4m3fn)
    older = (torch.arange(page_size, device=DEV) < first[:, None])[:, None, None, :]
    older = older if transposed else older.transpose(2, 3)
    raw = pool.view(torch.uint8)
    held = torch.where(older, again.view(torch.uint8), raw[touched])
    values = (x / now[group][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    if transposed:
        held.transpose(2, 3)[group, :, slot] = values
    else:
        held[group, :, slot] = values
    raw[touched] = held
    scale[touched] = now


def _append(s: dict):
    seq, pos = _new_tokens(s, s["k_new"].shape[0])
    q = _rotated(s["q_new"], pos, s["inv_freq"]).to(torch.bfloat16)
    _write(s["k"], s["k_scale"], _rotated(s["k_new"], pos, s["inv_freq"]), seq, pos, s, False)
    _write(s["v"], s["v_scale"], s["v_new"].float(), seq, pos, s, True)
    return q


def _attend(s: dict) -> torch.Tensor:
    c = s["case"]
    seqs, kvh, d, g = c["seqs"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    used = -(-s["max_keys"] // c["page"])
    table = s["table"][:, :used].long().clamp(min=0)
    k, v = _pages(s["k"], table), _pages(s["v"], table)          # [seqs, pages, kvh, page, d], [.., d, page]
    if s["k_scale"] is not None:
        k *= s["k_scale"][table][..., None, None]
        v *= s["v_scale"][table][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(seqs, kvh, used * c["page"], d)
    v = v.permute(0, 2, 1, 4, 3).reshape(seqs, kvh, used * c["page"], d)
    seq, pos = _new_tokens(s, s["q"].shape[0])
    row = pos - s["lengths"].long()[seq]
    q = torch.zeros((seqs, s["max_new"], c["heads"], d), device=DEV)
    q[seq, row] = s["q"].float()
    q = q.view(seqs, -1, kvh, g, d).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, -1, d)
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
    if c["softcap"]:
        sc = torch.tanh(sc / c["softcap"]) * c["softcap"]
    at = s["lengths"].long()[:, None] + torch.arange(s["max_new"], device=DEV)      # positions of the (padded) queries
    key = torch.arange(used * c["page"], device=DEV)
    seen = key <= at[..., None]
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    sc = sc.masked_fill_(~seen.repeat_interleave(g, 1)[:, None], float("-inf"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.view(seqs, kvh, -1, g, d).permute(0, 2, 1, 3, 4).reshape(seqs, s["max_new"], c["heads"], d)
    return o[seq, row].to(torch.bfloat16)


def _logprobs(s: dict):
    c, x, tokens = s["case"], s["logits"].float(), s["tokens"]
    z = torch.tanh(x / c["softcap"]) * c["softcap"] if c["softcap"] else x
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    entropy = torch.log(total[:, 0]) + torch.where(e > 0, e * (m - z), torch.zeros_like(e)).sum(1) / total[:, 0]
    logprob = (z - m).gather(1, tokens[:, None])[:, 0] - torch.log(total[:, 0])
    if not c["top"]:
        return logprob, entropy, torch.empty((c["rows"], 0), device=DEV), torch.empty((c["rows"], 0), dtype=torch.int64, device=DEV)
    # by logit, then by index: one whole number that orders both
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = order * 2 ** 20 + (2 ** 20 - 1 - torch.arange(c["vocab"], device=DEV))
    ids = 2 ** 20 - 1 - (torch.topk(key, c["top"], 1).values & (2 ** 20 - 1))
    return logprob, entropy, (z - m).gather(1, ids) - torch.log(total), ids


def run(state: dict):
    op = state["case"]["op"]
    if op == "append":
        if own:
            q = state["cache"].append(state["batch"], state["k_new"], state["v_new"], q=state["q_new"], inv_freq=state["inv_freq"])
        else:
            q = _append(state)
        out = {"q": q, "k": state["k"], "v": state["v"]}
        return out if state["k_scale"] is None else {**out, "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    if op == "attend":
        c = state["case"]
        if own:
            return state["cache"].attend(state["batch"], state["q"], c["head_dim"] ** -0.5, softcap=c["softcap"], window=c["window"])
        return _attend(state)
    if own:
        from se12_amd.logprobs import token_logprobs

        r = token_logprobs(state["logits"], state["tokens"], top=state["case"]["top"], softcap=state["case"]["softcap"])
        return r.logprobs, r.entropy, r.top_logprobs, r.top_ids
    return _logprobs(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case: dict) -> dict:
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["x"] == "f32" else 2) + case["rows"] * (16 + 12 * case["top"]), "flops": 4 * n}
    held, new = _tokens(case)
    d, kvh, heads = case["head_dim"], case["kv_heads"], case["heads"]
    held_bytes = 1 if case["cache"] == "e4m3" else 2
    if case["op"] == "append":
        x, n = 4 if case["x"] == "f32" else 2, sum(new)
        return {"bytes": n * d * (heads * (x + 2) + 2 * kvh * (x + held_bytes)), "flops": 6 * n * d * (heads + kvh)}
    keys = pairs = 0
    for h, n in zip(held, new):
        w = case["window"] or h + n
        keys += h + n - max(0, h + 1 - w)                        # seen by any of the queries
        pairs += sum(min(h + i + 1, w) for i in range(n))
    return {"bytes": 2 * keys * kvh * d * held_bytes + 4 * sum(new) * heads * d, "flops": 4 * pairs * heads * d}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest E4M3 values, ties to even: 3 bits behind the leading one, no step below 2^-9."""
    step = torch.exp2(torch.frexp(x)[1].double().sub(4).clamp(min=-9))
    return torch.round(x / step) * step


def _turn(x: torch.Tensor, pos: int, freq: torch.Tensor) -> torch.Tensor:
    """x [.., head_dim] of tokens at pos, pos + 1, ..: each pair (i, i + h) turned by its angle."""
    p = torch.arange(pos, pos + x.shape[0], device=DEV, dtype=torch.float64)
    z = torch.polar(torch.ones((), device=DEV, dtype=torch.float64), p[:, None] * freq)[:, None, :]
    h = freq.numel()
    w = torch.complex(x[..., :h], x[..., h:2 * h]) * z
    return torch.cat([w.real, w.imag, x[..., 2 * h:]], -1)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        out = [[], [], []]
        for i in range(0, case["rows"], 64):
            z = s["logits"][i:i + 64].double()
            if case["softcap"]:
                z = case["softcap"] * torch.tanh(z / case["softcap"])
            lp = z - torch.logsumexp(z, 1, keepdim=True)
            out[0].append(lp[torch.arange(lp.shape[0], device=DEV), s["tokens"][i:i + 64]])
            out[1].append(torch.special.entr(lp.exp()).sum(1))
            out[2].append(lp.sort(1, descending=True).values[:, :case["top"]])
        return [*(torch.cat(o) for o in out), None]
    held, new = _tokens(case)
    page, d, h8 = case["page"], case["head_dim"], case["cache"] == "e4m3"
    table = s["table"].tolist()
    at = 0
    if case["op"] == "append":
        freq = s["inv_freq"].double()
        k, v = s["k"].double(), s["v"].double()
        scales = {"k": s["k_scale"].double(), "v": s["v_scale"].double()} if h8 else {}
        q_out = []
        for i, (h, n) in enumerate(zip(held, new)):
            q_out.append(_turn(s["q_new"][at:at + n].double(), h, freq))
            kk, vv = _turn(s["k_new"][at:at + n].double(), h, freq), s["v_new"][at:at + n].double()
            at += n
            for p in range(h // page, (h + n - 1) // page + 1):
                lo, hi = max(h, p * page), min(h + n, (p + 1) * page)
                pid, first = table[i][p], lo - p * page
                for name, pool, x in (("k", k[pid], kk), ("v", v[pid].transpose(1, 2), vv)):
                    x = x[lo - h:hi - h].transpose(0, 1)                                # [kv_heads, tokens, d]
                    if not h8:
                        pool[:, first:first + hi - lo] = x
                        continue
                    top = x.abs().amax((1, 2))
                    need = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)).clamp(min=MIN_EXPONENT))
                    was = scales[name][pid]
                    now = torch.maximum(was, need) if first else need
                    pool[:, :first] = _e4m3(pool[:, :first] * (was / now)[:, None, None])
                    pool[:, first:first + hi - lo] = _e4m3(x / now[:, None, None])
                    scales[name][pid] = now
        out = {"q": torch.cat(q_out), "k": k, "v": v}
        return {**out, "k_scale": scales["k"], "v_scale": scales["v"]} if h8 else out
    g, out, k_pool, v_pool = case["heads"] // case["kv_heads"], [], s["k"].double(), s["v"].double()
    for i, (h, n) in enumerate(zip(held, new)):
        ids = torch.tensor(table[i][:-(-(h + n) // page)], device=DEV)
        q = s["q"][at:at + n].double()
        at += n
        o = torch.empty_like(q)
        for j in range(case["kv_heads"]):
            k, v = k_pool[ids, j], v_pool[ids, j].transpose(1, 2)
            if h8:
                k, v = k * s["k_scale"][ids, j].double()[:, None, None], v * s["v_scale"][ids, j].double()[:, None, None]
            k, v = k.reshape(-1, d)[:h + n], v.reshape(-1, d)[:h + n]
            for u in range(0, n, 256):
                qq = q[u:u + 256, j * g:(j + 1) * g]
                sc = (qq.reshape(-1, d) @ k.T).view(qq.shape[0], g, -1) / math.sqrt(d)
                if case["softcap"]:
                    sc = case["softcap"] * torch.tanh(sc / case["softcap"])
                gap = (h + u + torch.arange(qq.shape[0], device=DEV))[:, None] - torch.arange(h + n, device=DEV)
                hidden = (gap < 0) | (gap >= case["window"]) if case["window"] else gap < 0
                w = torch.softmax(sc.masked_fill(hidden[:, None], float("-inf")), -1)
                o[u:u + 256, j * g:(j + 1) * g] = (w.view(-1, h + n) @ v).view(qq.shape[0], g, d)
        out.append(o)
    return torch.cat(out)
