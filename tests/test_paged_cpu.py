"""What the paged cache, its attention and the log probabilities refuse before any
launch: the C entries with made-up pointers (never followed: each call has something
wrong with it), and the Python wrappers with tensors on the CPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import paged_oracle as o
from se12_amd import _native as nat

P = 4096      # a pointer no call reads


def _pages(**kw):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, dtype=nat.STEP_E4M3, pages=10, page_size=64, kv_heads=4, head_dim=128)
    f.update(kw)
    return nat.StepPages(*f.values())


def _batch(**kw):
    f = dict(page_table=P, table_stride=8, lengths=P, starts=P, table_width=8, sequences=3, tokens=3, max_new=1)
    f.update(kw)
    return nat.StepBatch(*f.values())


BAD_SHARED = [
    (dict(k=None), {}, "NULL cache"), (dict(dtype=1), {}, "BF16 or E4M3"), (dict(k_scale=None), {}, "needs scales"),
    (dict(page_size=48), {}, "page_size"), (dict(page_size=8), {}, "page_size"), (dict(head_dim=96), {}, "head_dim"),
    (dict(pages=0), {}, "cache shape"), (dict(kv_heads=0), {}, "cache shape"), (dict(kv_heads=3), {}, "multiple of kv_heads"),
    (dict(k=P + 8), {}, "16-byte aligned"), (dict(v_scale=P + 2), {}, "misaligned"),
    ({}, dict(page_table=None), "NULL batch"), ({}, dict(lengths=None), "NULL batch"), ({}, dict(starts=None), "NULL batch"),
    ({}, dict(sequences=0), "batch shape"), ({}, dict(sequences=65537), "batch shape"), ({}, dict(tokens=-1), "batch shape"),
    ({}, dict(max_new=0), "batch shape"), ({}, dict(table_stride=7), "batch shape"), ({}, dict(starts=P + 1), "misaligned"),
    ({}, dict(table_width=2 ** 25, table_stride=2 ** 25), "2^30"),
]


@pytest.mark.parametrize("pages,batch,message", BAD_SHARED)
def test_both_calls_refuse_bad_caches_and_batches(pages, batch, message):
    lib, p, b = nat.lib(), _pages(**pages), _batch(**batch)
    for call in (lambda: lib.se12_step_paged_append(ctypes.byref(p), ctypes.byref(b), P, P, P, nat.STEP_F32, 1024, 512, 512, 8, P, 128, P,
                                                    None),
                 lambda: lib.se12_step_paged_attention(ctypes.byref(p), ctypes.byref(b), P, 1024, P, 8, 0.1, 0.0, 0, P, 1 << 30, None),
                 lambda: lib.se12_step_paged_attention_workspace(ctypes.byref(p), ctypes.byref(b), 8)):
        with pytest.raises(nat.Se12Error, match=message.replace("^", r"\^")):
            nat.step_check(call())


@pytest.mark.parametrize("change,message", [
    (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(q_out=None), "NULL"), (dict(inv=None), "NULL"), (dict(dtype=2), "BF16 or FP32"),
    (dict(rotary=12), "rotary"), (dict(rotary=136), "rotary"), (dict(rotary=-8), "rotary"), (dict(ks=510), "multiple of 4"),
    (dict(vs=508), "hold all heads"), (dict(qs=1020), "hold all heads"), (dict(heads=6), "kv_heads"), (dict(k=P + 8), "misaligned"),
    (dict(q_out=P + 4), "misaligned"), (dict(inv=P + 4), "misaligned"),
])
def test_append_refuses(change, message):
    f = dict(q=P, k=P, v=P, dtype=nat.STEP_F32, qs=1024, ks=512, vs=512, heads=8, inv=P, rotary=128, q_out=P)
    f.update(change)
    with pytest.raises(nat.Se12Error, match=message):
        nat.step_check(nat.lib().se12_step_paged_append(ctypes.byref(_pages()), ctypes.byref(_batch()), *f.values(), None))


Q = 16 * P     # 3 rows of 8 heads of 128, in BF16 6,144 bytes


@pytest.mark.parametrize("change", [
    dict(dtype=nat.STEP_F32, q_out=Q),                                   # of another type than q
    dict(q_out=Q + 8), dict(q_out=Q - 8), dict(q_out=Q + 6136), dict(q_out=Q - 6136),
    dict(qs=2048, q_out=Q),                                              # q's rows apart, the output's not
    dict(dtype=nat.STEP_F32, q_out=Q + 12280), dict(k=Q + 16 * P, q_out=Q + 16 * P + 3064), dict(v=Q + 16 * P, q_out=Q + 16 * P - 6136),
    dict(k=Q, ks=4096),
])
def test_append_refuses_an_output_over_its_inputs(change):
    """Blocks read and write in any order, so only q itself, value for value, may be written over."""
    f = dict(q=Q, k=2 * Q, v=3 * Q, dtype=nat.STEP_BF16, qs=1024, ks=512, vs=512, heads=8, inv=P, rotary=128, q_out=Q)
    f.update(change)
    with pytest.raises(nat.Se12Error, match="overlaps"):
        nat.step_check(nat.lib().se12_step_paged_append(ctypes.byref(_pages()), ctypes.byref(_batch()), *f.values(), None))


@pytest.mark.parametrize("change,message", [
    (dict(q=None), "NULL"), (dict(out=None), "NULL"), (dict(qs=1016), "hold all heads"), (dict(qs=1028), "multiple of 8"),
    (dict(cap=-1.0), "softcap"), (dict(cap=float("nan")), "softcap"), (dict(cap=1025.0), "softcap"),
    (dict(window=-1), "window"), (dict(q=P + 8), "misaligned"),
    (dict(out=P + 4), "misaligned"), (dict(ws=None), "workspace"), (dict(ws=P + 128), "workspace"), (dict(size=100), "workspace"),
    (dict(heads=7), "kv_heads"), (dict(out=P + 3 * 2048 - 16), "overlaps"), (dict(q=P + 3 * 2048 - 16), "overlaps"), (dict(), "overlaps"),
])
def test_attention_refuses(change, message):
    f = dict(q=P, qs=1024, out=P, heads=8, scaling=0.1, cap=0.0, window=0, ws=P, size=1 << 30)
    f.update(change)
    with pytest.raises(nat.Se12Error, match=message):
        nat.step_check(nat.lib().se12_step_paged_attention(ctypes.byref(_pages()), ctypes.byref(_batch()), *f.values(), None))


@pytest.mark.parametrize("batch,message", [
    (dict(tokens=1 << 30, max_new=1 << 20), "too many sequences, tokens"), (dict(tokens=1 << 28, sequences=65536), "too many"),
    (dict(sequences=64, table_width=1 << 24, table_stride=1 << 24), "too long a table"),
])
def test_attention_refuses_what_one_launch_does_not_hold(batch, message):
    lib, p, b = nat.lib(), _pages(kv_heads=8), _batch(**batch)
    for call in (lambda: lib.se12_step_paged_attention(ctypes.byref(p), ctypes.byref(b), P, 1 << 14, P, 128, 0.1, 0.0, 0, P, 1 << 60, None),
                 lambda: lib.se12_step_paged_attention_workspace(ctypes.byref(p), ctypes.byref(b), 128)):
        with pytest.raises(nat.Se12Error, match=message):
            nat.step_check(call())


def _workspace(heads=16, pages=None, **batch):
    f = dict(sequences=64, tokens=64, max_new=1, table_width=128, table_stride=128)
    f.update(batch)
    n = nat.lib().se12_step_paged_attention_workspace(ctypes.byref(_pages(**{"kv_heads": 8, "head_dim": 256, **(pages or {})})),
                                                      ctypes.byref(_batch(**f)), heads)
    if n < 0:
        nat.step_check(n)
    return n


@pytest.mark.parametrize("batch", [
    dict(max_new=512), dict(tokens=96, max_new=33), dict(sequences=1024, tokens=1535, max_new=512),
    dict(tokens=64 + 511, max_new=512), dict(sequences=4096, tokens=4160, max_new=65, table_width=1024, table_stride=1024),
    dict(tokens=6400, max_new=6400), dict(sequences=1, tokens=512, max_new=512), dict(sequences=65536, tokens=65536, max_new=4096),
])
@pytest.mark.parametrize("dtype", [nat.STEP_E4M3, nat.STEP_BF16])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_the_workspace_of_few_prompts_among_many_sequences(batch, dtype, head_dim):
    """Parts of two rounds of blocks (512 of 128 columns at 256 values and two statistics, 1,024 at half as many), the
    waves' parts of short sequences (2,048 of 16 columns), and records: a sequence of one new token adds nothing."""
    columns = 2048 * 16 + (1 if head_dim == 256 or (head_dim == 128 and dtype == nat.STEP_BF16) else 2) * 512 * 128
    records = (2 * batch["tokens"] // 128 + 2 * batch["tokens"] // 65 + 1600) * 48 if "tokens" in batch else 1 << 20
    assert _workspace(pages=dict(dtype=dtype, head_dim=head_dim), **batch) <= columns * (head_dim + 2) * 4 + records + 1024


@pytest.mark.parametrize("heads,kv_heads", [(16, 8), (28, 4), (8, 8), (160, 1), (7, 7)])
@pytest.mark.parametrize("sequences,width", [(1, 2000), (64, 100), (300, 4), (5, 1)])
@pytest.mark.parametrize("page_size,dtype", [(64, nat.STEP_E4M3), (16, nat.STEP_BF16)])
def test_a_workspace_for_more_tokens_serves_fewer(heads, kv_heads, sequences, width, page_size, dtype):
    pages, last = dict(kv_heads=kv_heads, page_size=page_size, dtype=dtype, head_dim=128), 0
    for max_new in (1, 2, 9, 40, 1 << 20):
        f = dict(sequences=sequences, table_width=width, table_stride=width, max_new=max_new)
        sizes = [_workspace(heads, pages, tokens=n, **f) for n in [*range(1, 200), *range(200, 20_000, 97), 100_000, 1_000_000]]
        assert sizes == sorted(sizes) and sizes[-1] >= last
        last = sizes[-1]


@pytest.mark.parametrize("change,message", [
    (dict(vocab=0), "bad shape"), (dict(rows=-1), "bad shape"), (dict(top=33), "top"), (dict(top=-1), "top"), (dict(vocab=4, top=5), "top"),
    (dict(logits=None), "NULL"), (dict(tokens=None), "NULL"), (dict(tl=None), "NULL"), (dict(dtype=2), "BF16 or FP32"),
    (dict(stride=999), "overlap"), (dict(cap=-1.0), "softcap"), (dict(cap=1025.0), "softcap"),
    (dict(logits=P + 2), "misaligned"), (dict(tokens=P + 4), "misaligned"),
    (dict(vocab=50000, stride=50000, ws=None), "workspace"), (dict(vocab=50000, stride=50000, size=8), "workspace"),
])
def test_logprobs_refuse(change, message):
    f = dict(logits=P, dtype=nat.STEP_F32, stride=1000, rows=2, vocab=1000, cap=0.0, tokens=P, top=5, lp=P, ent=P, tl=P, ti=P, ws=P,
             size=1 << 30)
    f.update(change)
    with pytest.raises(nat.Se12Error, match=message):
        nat.step_check(nat.lib().se12_step_logprobs(*f.values(), None))


def test_calls_without_tokens_or_rows_do_nothing():
    lib, p, b = nat.lib(), _pages(), _batch(tokens=0)
    assert lib.se12_step_paged_append(ctypes.byref(p), ctypes.byref(b), P, P, P, nat.STEP_F32, 1024, 512, 512, 8, P, 128, P, None) == 0
    assert lib.se12_step_paged_attention(ctypes.byref(p), ctypes.byref(b), P, 1024, P, 8, 0.1, 0.0, 0, None, 0, None) == 0
    assert lib.se12_step_paged_attention_workspace(ctypes.byref(p), ctypes.byref(b), 8) == 0
    assert lib.se12_step_logprobs(None, 0, 10, 0, 10, 0.0, None, 0, None, None, None, None, None, 0, None) == 0


def test_calls_without_tokens_need_no_memory():
    """Tensors of no rows have no memory: NULL."""
    lib, p, b = nat.lib(), _pages(), _batch(tokens=0)
    for q_out in (None, P):
        assert lib.se12_step_paged_append(ctypes.byref(p), ctypes.byref(b), None, None, None, nat.STEP_F32, 1024, 512, 512, 8, P, 128,
                                          q_out, None) == 0
    assert lib.se12_step_paged_attention(ctypes.byref(p), ctypes.byref(b), None, 1024, None, 8, 0.1, 0.0, 0, None, 0, None) == 0


def test_wrappers_refuse_tensors_on_the_cpu_and_bad_shapes():
    from se12_amd.logprobs import token_logprobs
    from se12_amd.paged import PagedBatch, PagedKvCache

    i32 = torch.zeros((2, 3), dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        PagedBatch(i32, i32[0, :2], i32[0])
    with pytest.raises(ValueError, match="int32"):
        PagedBatch(i32.long(), i32[0, :2], i32[0])
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="HIP device"):
        PagedKvCache.from_tensors(k, torch.zeros((4, 2, 64, 16), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="v must be"):
        PagedKvCache.from_tensors(k, k)
    with pytest.raises(ValueError, match="needs k_scale"):
        PagedKvCache.from_tensors(k.to(torch.float8_e4m3fn), torch.zeros((4, 2, 64, 16), dtype=torch.float8_e4m3fn))
    with pytest.raises(ValueError, match="page_size"):
        PagedKvCache.from_tensors(k[:, :, :8], k)
    with pytest.raises(ValueError, match="goes with"):
        PagedKvCache.from_tensors(k, torch.zeros((4, 2, 64, 16), dtype=torch.bfloat16), torch.ones((4, 2)), torch.ones((4, 2)))
    with pytest.raises(ValueError, match="HIP device"):
        token_logprobs(torch.zeros((2, 5)), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        token_logprobs(torch.zeros((2, 5), dtype=torch.float16), torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("multiple", [4, 8])
def test_the_distance_of_a_single_row_to_the_next_does_not_matter(multiple):
    """torch calls [1, heads, head_dim] contiguous whatever its first stride is, and contiguous() leaves it."""
    from se12_amd.paged import PagedKvCache

    c = PagedKvCache.__new__(PagedKvCache)
    c.head_dim, c.device, c._index = 64, torch.device("cpu"), -1
    whole = torch.arange(8 * 64 + 3.0)
    for x in (whole[:512].view(1, 8, 1, 64).transpose(1, 2)[0],                  # the heads of one token, transposed
              torch.cat([whole[:513], whole[:513]]).view(2, 513)[:1, :512].view(1, 8, 64),      # a row of an odd length
              whole[3:515].view(1, 8, 64),                                       # from an odd offset
              whole[:512].view(8, 64).expand(1, 8, 64), whole[:64].view(1, 1, 64).expand(1, 8, 64)):
        r = c._rows(x, "x", 8, None, None, multiple)
        assert torch.equal(r, x) and r.stride()[1:] == (64, 1)
        assert r.stride(0) >= 512 and r.stride(0) % multiple == 0 and r.data_ptr() % (4 * multiple) == 0


@pytest.mark.parametrize("max_new", [0, -1, 1.5, 2 ** 31, 2 ** 32 + 1])
def test_a_batch_refuses_a_max_new_that_32_bits_or_whole_numbers_do_not_hold(max_new):
    from se12_amd.paged import PagedBatch

    i32 = torch.zeros((2, 3), dtype=torch.int32)
    with pytest.raises(ValueError, match="max_new"):
        PagedBatch(i32, i32[0, :2], i32[0], max_new=max_new)


def test_sizes_beyond_32_bits_are_refused():
    """Not cut to their low 32 bits on the way to the C entries (tensors without memory)."""
    from se12_amd.logprobs import token_logprobs
    from se12_amd.paged import PagedBatch, PagedKvCache

    table = torch.empty((1, 2 ** 32 + 1), dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="columns"):
        PagedBatch(table, torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    for shape in ((1, 2 ** 32 + 5), (2 ** 32 + 1, 1), (1, 2 ** 30 + 1)):
        with pytest.raises(ValueError, match="2\\^30"):
            token_logprobs(torch.empty(shape, device="meta"), torch.empty(shape[0], dtype=torch.int64, device="meta"))
    batch = PagedBatch.__new__(PagedBatch)
    batch.device, batch.max_new, batch._fields, batch._last = torch.device("cpu"), 1, (P, 8, P, P, 8, 3), (-1, None)
    c = PagedKvCache.__new__(PagedKvCache)
    c.device, c._struct = batch.device, ctypes.byref(_pages())
    assert c.attend_workspace(batch, 3, 8) > 0
    for tokens, heads in ((2 ** 32 + 3, 8), (3, 2 ** 32 + 8), (2 ** 31, 8)):
        with pytest.raises(ValueError, match="tokens"):
            c.attend_workspace(batch, tokens, heads)


def test_grids_of_more_threads_than_32_bits_count_are_refused():
    """Before the first launch of a call, not by the last."""
    lib, p = nat.lib(), _pages(kv_heads=1024, pages=1 << 20)
    b = _batch(sequences=65536, tokens=65536, max_new=1)
    with pytest.raises(nat.Se12Error, match="too many"):
        nat.step_check(lib.se12_step_paged_append(ctypes.byref(p), ctypes.byref(b), None, P, P, nat.STEP_F32, 0, 1 << 17, 1 << 17, 1024, None,
                                                  0, None, None))
    b = _batch(sequences=65536, tokens=1 << 25, max_new=1 << 20)
    with pytest.raises(nat.Se12Error, match="too many sequences, tokens"):
        nat.step_check(lib.se12_step_paged_attention_workspace(ctypes.byref(p), ctypes.byref(b), 1024))
    with pytest.raises(nat.Se12Error, match="too many rows"):
        nat.step_check(lib.se12_step_logprobs(P, nat.STEP_F32, 10, 1 << 24, 10, 0.0, P, 0, P, P, None, None, None, 0, None))


@pytest.mark.parametrize("cap,scaling,message", [
    (1e-40, 0.1, "softcap"), (2.0 ** -61, 0.1, "softcap"), (0.0, float("inf"), "scaling"), (0.0, float("nan"), "scaling"),
    (0.0, 1.5 * 2.0 ** 127, "scaling"), (2.0 ** -60, 2.0 ** 70, "scaling"),
])
def test_caps_and_scalings_whose_factors_32_bits_do_not_hold_are_refused(cap, scaling, message):
    """0 times an infinite factor would be a NaN."""
    lib = nat.lib()
    with pytest.raises(nat.Se12Error, match=message):
        nat.step_check(lib.se12_step_paged_attention(ctypes.byref(_pages()), ctypes.byref(_batch()), P, 1024, P, 8, scaling, cap, 0, P,
                                                     1 << 30, None))
    if message == "softcap":
        with pytest.raises(nat.Se12Error, match=message):
            nat.step_check(lib.se12_step_logprobs(P, nat.STEP_F32, 1000, 2, 1000, cap, P, 5, P, P, P, P, P, 1 << 30, None))


@pytest.mark.parametrize("cap", [-1.0, 1e-300, 1e-40, 2.0 ** -61, 1025.0, float("nan")])
def test_wrappers_refuse_caps_before_32_bits_make_them_none(cap):
    """(1e-300 is 0 in FP32, which stands for no cap.)"""
    from se12_amd.paged import check_softcap

    with pytest.raises(ValueError, match="softcap"):
        check_softcap(cap)
    for fine in (0, 0.0, 2.0 ** -60, 30.0, 1024):
        check_softcap(fine)


def test_the_oracle_rounds_as_the_type_does():
    """Every E4M3 value, every midpoint between two of them and its neighbours, against torch's conversion on the CPU."""
    values = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (values[1:] + values[:-1]) / 2
    x = torch.cat([values, mid, mid * (1 + 1e-6), mid * (1 - 1e-6)])
    x = torch.cat([x, -x])
    assert torch.equal(o.e4m3(x), x.float().to(torch.float8_e4m3fn).double())
    assert o.scale_for(torch.tensor([448.0])) == 1.0 and o.scale_for(torch.tensor([448.1])) == 2.0
    assert o.scale_for(torch.tensor([0.0, float("nan")])) == 2.0 ** -100 and o.scale_for(torch.tensor([1e30, float("inf")])) == 2.0 ** 91
