"""What the paged cache of 4 bits, reading back and rotate_heads refuse before any launch:
the C entries with made-up pointers (never followed: each call has something wrong with
it), and the Python wrappers with tensors on the CPU. And the oracle's rounding against
its definition, and rotary_frequencies."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import e2m1_oracle as e
from se12_amd import _native as nat
from test_paged_cpu import P, Q, _batch, _pages

FP4 = torch.float4_e2m1fn_x2


def _pages4(**kw):
    return _pages(**{"dtype": nat.STEP_E2M1, **kw})


def _turn(**kw):
    f = dict(inv_freq=P, q_norm=P, k_norm=P, scale=1.0, eps=1e-6, offset=0.0, norm_dtype=nat.STEP_BF16, rotary=128, interleaved=0)
    f.update(kw)
    return nat.StepRotation(*f.values())


def _refused(message, call):
    with pytest.raises(nat.Se12Error, match=message):
        nat.step_check(call())


@pytest.mark.parametrize("pages,batch,message", [
    (dict(k=None), {}, "NULL cache"), (dict(dtype=4), {}, "BF16 or E4M3"), (dict(dtype=-1), {}, "BF16 or E4M3"), (dict(k_scale=None), {}, "needs scales"),
    (dict(v_scale=None), {}, "needs scales"), (dict(k_scale=P + 8), {}, "scales of an E2M1"), (dict(v_scale=P + 4), {}, "scales of an E2M1"),
    (dict(page_size=48), {}, "page_size"), (dict(head_dim=96), {}, "head_dim"), (dict(head_dim=32), {}, "head_dim"), (dict(pages=0), {}, "cache shape"),
    (dict(kv_heads=3), {}, "multiple of kv_heads"), (dict(v=P + 8), {}, "16-byte aligned"),
    ({}, dict(page_table=None), "NULL batch"), ({}, dict(sequences=65537), "batch shape"), ({}, dict(tokens=-1), "batch shape"),
    ({}, dict(max_new=0), "batch shape"), ({}, dict(table_stride=7), "batch shape"), ({}, dict(lengths=P + 1), "misaligned"),
    ({}, dict(table_width=2 ** 25, table_stride=2 ** 25), r"2\^30"),
])
def test_calls_refuse_bad_caches_and_batches(pages, batch, message):
    lib, p, b, r = nat.lib(), _pages4(**pages), _batch(**batch), _turn()
    calls = [lambda: lib.se12_step_paged_append(ctypes.byref(p), ctypes.byref(b), P, P, P, nat.STEP_F32, 1024, 512, 512, 8, P, 128, P, None),
             lambda: lib.se12_step_paged_append_rotated(ctypes.byref(p), ctypes.byref(b), P, P, P, nat.STEP_F32, 1024, 512, 512, 8, ctypes.byref(r), P,
                                                        None),
             lambda: lib.se12_step_paged_attention(ctypes.byref(p), ctypes.byref(b), P, 1024, P, 8, 0.1, 0.0, 0, P, 1 << 30, None),
             lambda: lib.se12_step_paged_attention_workspace(ctypes.byref(p), ctypes.byref(b), 8)]
    if "kv_heads" not in pages:
        calls.append(lambda: lib.se12_step_paged_read(ctypes.byref(p), ctypes.byref(b), P, 2 * P, None))
    for call in calls:
        _refused(message, call)


@pytest.mark.parametrize("change,message", [
    (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(q_out=None), "NULL"), (dict(dtype=2), "BF16 or FP32"), (dict(ks=510), "multiple of 4"),
    (dict(vs=508), "hold all heads"), (dict(qs=1020), "hold all heads"), (dict(heads=6), "kv_heads"), (dict(k=P + 8), "misaligned"),
    (dict(q_out=P + 4), "misaligned"), (dict(q_out=Q + 12280), "overlaps"), (dict(q_out=Q), "overlaps"), (dict(k=4 * Q, q_out=4 * Q + 3064), "overlaps"),
])
def test_append_refuses(change, message):
    f = dict(q=Q, k=2 * Q, v=3 * Q, dtype=nat.STEP_F32, qs=1024, ks=512, vs=512, heads=8, r=ctypes.byref(_turn()), q_out=8 * Q)
    f.update(change)
    _refused(message, lambda: nat.lib().se12_step_paged_append_rotated(ctypes.byref(_pages4()), ctypes.byref(_batch()), *f.values(), None))


def test_append_of_this_form_is_for_caches_of_4_bits():
    for dtype in (nat.STEP_E4M3, nat.STEP_BF16):
        _refused("must be E2M1", lambda: nat.lib().se12_step_paged_append_rotated(
            ctypes.byref(_pages(dtype=dtype)), ctypes.byref(_batch()), P, P, P, nat.STEP_F32, 1024, 512, 512, 8, ctypes.byref(_turn()), P, None))


@pytest.mark.parametrize("change,message", [
    (dict(rotary=12), "rotary"), (dict(rotary=136), "rotary"), (dict(rotary=-8), "rotary"), (dict(inv_freq=None), "NULL"),
    (dict(norm_dtype=2), "norm weights"), (dict(scale=math.inf), "finite"), (dict(scale=math.nan), "finite"), (dict(eps=-1e-9), "finite"),
    (dict(eps=math.nan), "finite"), (dict(eps=math.inf), "finite"), (dict(offset=math.inf), "finite"), (dict(inv_freq=P + 8), "misaligned"),
    (dict(q_norm=P + 2), "misaligned"), (dict(k_norm=P + 8), "misaligned"),
])
def test_rotations_are_checked(change, message):
    lib, b, r = nat.lib(), _batch(), _turn(**change)
    _refused(message, lambda: lib.se12_step_paged_append_rotated(ctypes.byref(_pages4()), ctypes.byref(b), P, P, P, nat.STEP_F32, 1024, 512, 512, 8,
                                                                 ctypes.byref(r), P, None))
    _refused(message, lambda: lib.se12_step_rotate_heads(ctypes.byref(b), Q, 2 * Q, nat.STEP_BF16, 1024, 512, 8, 4, 128, ctypes.byref(r), 3 * Q, 4 * Q,
                                                         nat.STEP_BF16, None))
    _refused("NULL", lambda: lib.se12_step_paged_append_rotated(ctypes.byref(_pages4()), ctypes.byref(b), P, P, P, nat.STEP_F32, 1024, 512, 512, 8,
                                                                None, P, None))
    _refused("NULL", lambda: lib.se12_step_rotate_heads(ctypes.byref(b), Q, 2 * Q, nat.STEP_BF16, 1024, 512, 8, 4, 128, None, 3 * Q, 4 * Q,
                                                        nat.STEP_BF16, None))


@pytest.mark.parametrize("k,v,message", [(None, P, "NULL"), (P, None, "NULL"), (P + 8, Q, "misaligned"), (P, Q + 2, "misaligned"), (P, P, "overlaps"),
                                         (Q, Q + 3056, "overlaps"), (Q + 3056, Q, "overlaps")])
def test_read_refuses(k, v, message):
    for pages in (_pages4(), _pages(), _pages(dtype=nat.STEP_BF16)):
        _refused(message, lambda: nat.lib().se12_step_paged_read(ctypes.byref(pages), ctypes.byref(_batch()), k, v, None))
    _refused("NULL", lambda: nat.lib().se12_step_paged_read(None, ctypes.byref(_batch()), P, Q, None))
    _refused("too many", lambda: nat.lib().se12_step_paged_read(
        ctypes.byref(_pages4(kv_heads=1024)), ctypes.byref(_batch(tokens=1 << 30, max_new=1 << 30)), 1 << 20, 1 << 52, None))


@pytest.mark.parametrize("change,message", [
    (dict(q=None), "NULL"), (dict(k=None), "NULL"), (dict(q_out=None), "NULL"), (dict(k_out=None), "NULL"), (dict(dtype=2), "BF16 or FP32"),
    (dict(out_dtype=3), "BF16 or FP32"), (dict(head_dim=12), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(heads=0), "head counts"), (dict(heads=65536), "head counts"), (dict(kv=-1), "head counts"), (dict(kv=65536), "head counts"),
    (dict(qs=1022), "multiple of 4"), (dict(qs=1020), "hold all heads"), (dict(ks=508), "hold all heads"), (dict(q=Q + 4), "misaligned"),
    (dict(k_out=P + 8), "misaligned"), (dict(q_out=Q + 16), "overlaps"), (dict(q_out=2 * Q), "overlaps"), (dict(k_out=Q), "overlaps"),
    (dict(q_out=Q, qs=2048), "overlaps"), (dict(q_out=Q, out_dtype=nat.STEP_F32), "overlaps"), (dict(q_out=8 * Q, k_out=8 * Q + 6128), "overlaps"),
])
def test_rotate_heads_refuses(change, message):
    f = dict(q=Q, k=2 * Q, dtype=nat.STEP_BF16, qs=1024, ks=512, heads=8, kv=4, head_dim=128, r=ctypes.byref(_turn()), q_out=4 * Q, k_out=6 * Q,
             out_dtype=nat.STEP_BF16)
    f.update(change)
    _refused(message, lambda: nat.lib().se12_step_rotate_heads(ctypes.byref(_batch()), *f.values(), None))


@pytest.mark.parametrize("batch,message", [
    (dict(lengths=None), "NULL batch"), (dict(starts=None), "NULL batch"), (dict(sequences=0), "batch shape"), (dict(sequences=65537), "batch shape"),
    (dict(tokens=-1), "batch shape"), (dict(tokens=(1 << 30) + 1), "batch shape"), (dict(max_new=0), "batch shape"), (dict(starts=P + 2), "misaligned"),
    (dict(tokens=1 << 30, max_new=1 << 20), "too many"),
])
def test_rotate_heads_refuses_batches(batch, message):
    q, k, out = 1 << 20, 1 << 44, 1 << 46
    call = lambda b: nat.lib().se12_step_rotate_heads(b, q, k, nat.STEP_BF16, 1024, 512, 8, 4, 128, ctypes.byref(_turn()), out, 1 << 48,  # noqa: E731
                                                      nat.STEP_BF16, None)
    _refused(message, lambda: call(ctypes.byref(_batch(**batch))))
    _refused("NULL", lambda: call(None))


def test_calls_without_tokens_need_no_memory():
    lib, b, r = nat.lib(), _batch(tokens=0), _turn()
    p = _pages4()
    assert lib.se12_step_paged_append_rotated(ctypes.byref(p), ctypes.byref(b), None, None, None, nat.STEP_F32, 1024, 512, 512, 8, ctypes.byref(r),
                                              None, None) == 0
    assert lib.se12_step_paged_append(ctypes.byref(p), ctypes.byref(b), None, None, None, nat.STEP_F32, 1024, 512, 512, 8, None, 0, None, None) == 0
    assert lib.se12_step_paged_read(ctypes.byref(p), ctypes.byref(b), None, None, None) == 0
    assert lib.se12_step_paged_attention(ctypes.byref(p), ctypes.byref(b), None, 1024, None, 8, 0.1, 0.0, 0, None, 0, None) == 0
    assert lib.se12_step_rotate_heads(ctypes.byref(b), None, None, nat.STEP_BF16, 1024, 512, 8, 4, 128, ctypes.byref(r), None, None, nat.STEP_BF16,
                                      None) == 0


def test_blocks_of_prompts_are_twice_as_large_and_counted_so():
    lib, b = nat.lib(), _batch(sequences=200, tokens=1 << 27, max_new=1 << 20)
    assert lib.se12_step_paged_attention_workspace(ctypes.byref(_pages(kv_heads=1, head_dim=256)), ctypes.byref(b), 8) > 0
    p = _pages4(kv_heads=1, head_dim=256)
    _refused("too many", lambda: lib.se12_step_paged_attention_workspace(ctypes.byref(p), ctypes.byref(b), 8))
    _refused("too many", lambda: lib.se12_step_paged_attention(ctypes.byref(p), ctypes.byref(b), P, 1 << 14, P, 8, 0.1, 0.0, 0, P, 1 << 60, None))


@pytest.mark.parametrize("head_dim", [64, 128])
def test_blocks_of_prompts_of_smaller_heads_are_not(head_dim):
    """As many calls as over a cache of BF16, whose blocks have as many threads."""
    lib = nat.lib()
    for tokens in (1 << 27, 1 << 28, (1 << 28) - (1 << 16), 1 << 29):
        b, fits = _batch(sequences=200, tokens=tokens, max_new=1 << 20), []
        for p in (_pages4(kv_heads=1, head_dim=head_dim), _pages(kv_heads=1, head_dim=head_dim, dtype=nat.STEP_BF16)):
            fits.append(lib.se12_step_paged_attention_workspace(ctypes.byref(p), ctypes.byref(b), 8) > 0)
        assert fits[0] == fits[1]


@pytest.mark.parametrize("heads,kv_heads", [(8, 4), (16, 8), (28, 4), (1, 1), (160, 1)])
@pytest.mark.parametrize("sequences,width,page_size,head_dim", [(1, 6000, 16, 256), (64, 20, 64, 128), (300, 4, 128, 64), (3, 100, 32, 256)])
def test_a_workspace_for_more_tokens_serves_fewer(heads, kv_heads, sequences, width, page_size, head_dim):
    lib = nat.lib()
    p = _pages4(kv_heads=kv_heads, page_size=page_size, head_dim=head_dim)
    sizes = []
    for tokens in sorted({1, 2, 3, 5, 40, sequences, 2 * sequences + 1, 64 * sequences, 700, 9000}):
        b = _batch(sequences=sequences, tokens=tokens, max_new=9000, table_width=width, table_stride=width)
        sizes.append(lib.se12_step_paged_attention_workspace(ctypes.byref(p), ctypes.byref(b), heads))
    assert all(x > 0 for x in sizes) and sizes == sorted(sizes)


# ---------------------------------------------------------------------------
# the wrappers
# ---------------------------------------------------------------------------


def test_caches_of_wrong_tensors_are_refused():
    from se12_amd.paged import PagedKvCache

    k, v = torch.zeros((4, 2, 16, 32), dtype=torch.uint8).view(FP4), torch.zeros((4, 2, 1, 64, 8), dtype=torch.uint8).view(FP4)
    s = torch.zeros((4, 2, 2, 16), dtype=torch.uint8)
    make = PagedKvCache.from_tensors
    for args, message in (((k, v, s, s), "HIP device"), ((k, v), "needs k_scale"), ((k, v, s), "needs v_scale"), ((k, v, s.int(), s), "k_scale must be"),
                          ((k, v, s, s[:, :, :1]), "v_scale must be"), ((k, v, s, s.transpose(2, 3)), "v_scale must be"), ((k, k, s, s), "v must be"),
                          ((k, v.view(torch.uint8), s, s), "v must be"), ((k[:, :, :8], v, s, s), "page_size"), ((k[..., :16], v, s, s), "head_dim"),
                          ((k.view(torch.uint8), v, s, s), "k must be"), ((k.transpose(0, 1).contiguous().transpose(0, 1), v, s, s), "contiguous"),
                          ((torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((4, 2, 64, 16), dtype=torch.bfloat16), s, s), "goes with")):
        with pytest.raises(ValueError, match=message):
            make(*args)
    with pytest.raises(ValueError, match="HIP device"):
        PagedKvCache(4, 16, 2, 64, dtype=FP4, device="cpu")


def _on_cpu(kvh=2, d=64, dtype=FP4):
    """A cache and a batch as far as the wrappers' checks look (tensors on the CPU: index -1)."""
    from se12_amd.paged import PagedBatch, PagedKvCache

    c = PagedKvCache.__new__(PagedKvCache)
    c.device, c._index, c.dtype, c.kv_heads, c.head_dim, c.page_size, c.pages = torch.device("cpu"), -1, dtype, kvh, d, 16, 10
    c._struct = ctypes.byref(_pages4(kv_heads=kvh, head_dim=d, page_size=16))
    batch = PagedBatch.__new__(PagedBatch)
    batch.device, batch.max_new, batch._fields, batch._last = c.device, 1, (P, 8, P, P, 8, 3), (-1, None)
    batch.page_table = torch.zeros((3, 8), dtype=torch.int32)
    return c, batch


@pytest.mark.parametrize("change,message", [
    (dict(k=torch.zeros((3, 2, 64), dtype=torch.float16)), "bfloat16 or float32"), (dict(k=torch.zeros((3, 4, 64))), "k"),
    (dict(v=torch.zeros((2, 2, 64))), "v"), (dict(v=torch.zeros((3, 2, 64), dtype=torch.bfloat16)), "v must be"),
    (dict(q=torch.zeros((3, 3, 64))), "no multiple"), (dict(q=torch.zeros((3, 4, 32))), "q"), (dict(inv_freq=torch.zeros(6)), "inv_freq"),
    (dict(inv_freq=torch.zeros(36)), "at most 32"), (dict(inv_freq=torch.zeros(0)), "inv_freq"), (dict(inv_freq=torch.zeros(16, dtype=torch.float64)), "float32 vector"),
    (dict(inv_freq=torch.zeros(64)[::2]), "contiguous"), (dict(q_norm=torch.zeros(32)), "q_norm must be"), (dict(k_norm=torch.zeros(64, dtype=torch.float16)), "k_norm must be"),
    (dict(k_norm=torch.zeros(128)[::2]), "contiguous"), (dict(q_norm=torch.zeros(64), k_norm=torch.zeros(64, dtype=torch.bfloat16)), "one type"),
    (dict(rotary_scale=math.nan), "finite"), (dict(norm_eps=-1.0), "finite"), (dict(norm_offset=math.inf), "finite"), (dict(norm_offset=2.0 ** 127), "finite"),
    (dict(out=torch.zeros((3, 4, 64))), "out must be"), (dict(out=torch.zeros((2, 4, 64), dtype=torch.bfloat16)), "out must be"),
    (dict(q=None, out=torch.zeros((3, 4, 64), dtype=torch.bfloat16)), "goes with q"), (dict(q=None, q_norm=torch.zeros(64)), "goes with q"),
    (dict(batch=None), "PagedBatch"),
])
@pytest.mark.parametrize("dtype", [FP4, torch.bfloat16])
def test_append_wrapper_refuses(dtype, change, message):
    c, batch = _on_cpu(dtype=dtype)
    f = dict(batch=batch, k=torch.zeros((3, 2, 64)), v=torch.zeros((3, 2, 64)), q=torch.zeros((3, 4, 64)))
    f.update(change)
    with pytest.raises(ValueError, match=message):
        c.append(**f)


def test_append_of_other_caches_refuses_an_output_over_k_or_v():
    c, batch = _on_cpu(dtype=torch.bfloat16)
    x = torch.zeros(4096, dtype=torch.bfloat16)
    q, k, v, w = x[:768].view(3, 4, 64), x[768:1152].view(3, 2, 64), x[1152:1536].view(3, 2, 64), torch.zeros(64)
    for at in (400, 1000, 1400):
        with pytest.raises(ValueError, match="overlaps k or v"):
            c._append_turned(batch, q, k, v, x[at:at + 768].view(3, 4, 64), None, False, 1.0, w, None, 1e-6, 0.0)


@pytest.mark.parametrize("tokens,out,message", [
    (-1, None, "tokens"), (1.5, None, "tokens"), (2 ** 31, None, "tokens"), (3, (torch.zeros((3, 2, 64)),) * 2, "out must be"),
    (3, (torch.zeros((3, 2, 64), dtype=torch.bfloat16), torch.zeros((3, 2, 32), dtype=torch.bfloat16)), "out must be"),
    (3, (torch.zeros((3, 2, 128), dtype=torch.bfloat16)[..., ::2],) * 2, "contiguous"), (3, (None, None), "out must be"),
    (3, (torch.zeros(385, dtype=torch.bfloat16)[1:].view(3, 2, 64),) * 2, "aligned"),
])
def test_read_wrapper_refuses(tokens, out, message):
    c, batch = _on_cpu()
    with pytest.raises(ValueError, match=message):
        c.read(batch, tokens, out=out)
    with pytest.raises(ValueError, match="PagedBatch"):
        c.read(None, 3)


@pytest.mark.parametrize("change,message", [
    (dict(batch=None), "PagedBatch"), (dict(q=torch.zeros((3, 4, 60))), "multiple of 8"), (dict(q=torch.zeros((3, 4, 264))), "up to 256"),
    (dict(q=torch.zeros((3, 0, 64))), "heads"), (dict(q=torch.zeros((3, 256))), "q must be"), (dict(q=torch.zeros((3, 4, 64), dtype=torch.float16)), "q must be"),
    (dict(k=torch.zeros((2, 2, 64))), "rows"), (dict(k=torch.zeros((3, 0, 64))), "heads"), (dict(k=torch.zeros((3, 2, 32))), "k"),
    (dict(k=torch.zeros((3, 2, 64), dtype=torch.bfloat16)), "k must be"), (dict(dtype=torch.float16), "dtype"), (dict(k=None, k_norm=torch.zeros(64)), "go with k"),
    (dict(k=None, out=(None, torch.zeros((3, 2, 64), dtype=torch.bfloat16))), "go with k"), (dict(out=(torch.zeros((3, 4, 64)), None)), "out must hold"),
    (dict(out=(None, torch.zeros((2, 2, 64), dtype=torch.bfloat16))), "out must hold"), (dict(inv_freq=torch.zeros(36)), "inv_freq"),
    (dict(q_norm=torch.zeros(60)), "q_norm"), (dict(norm_eps=math.nan), "finite"),
    (dict(out=(torch.zeros(769, dtype=torch.bfloat16)[1:].view(3, 4, 64), None)), "aligned"),
])
def test_rotate_heads_wrapper_refuses(change, message):
    from se12_amd.paged import rotate_heads

    f = dict(batch=_on_cpu()[1], q=torch.zeros((3, 4, 64)), k=torch.zeros((3, 2, 64)))
    f.update(change)
    with pytest.raises(ValueError, match=message):
        rotate_heads(**f)


# ---------------------------------------------------------------------------
# the oracle, and the frequencies
# ---------------------------------------------------------------------------


def test_scales_are_fp16_numbers_cut_to_three_bits():
    """Every byte; and the digits, as torch numbers them."""
    for byte in range(e.LAST + 1):
        bits = torch.tensor([byte << 7], dtype=torch.int32).to(torch.int16)
        assert bits.view(torch.float16).double().item() == e.SCALES[byte].item()
    assert e.SCALES[e.LAST] == 10240 and (e.SCALES[1:] > e.SCALES[:-1]).all()
    assert e.codes_of(torch.arange(256, dtype=torch.uint8)[:, None])[0x7A].tolist() == [-1.0, 6.0]


def test_the_oracle_takes_the_nearest_and_of_two_the_even():
    """Every midpoint between two digits and two scales, and beside it, by search over all of them."""
    for values, middles in ((e.VALUES, e.BORDERS), (e.SCALES, e.MIDDLES)):
        x = torch.cat([values, middles, middles * (1 + 2.0 ** -40), middles * (1 - 2.0 ** -40), values[-1:] * 3])
        got = e.nearest(x, middles)
        d = (x[:, None] - values).abs()
        least = d.min(1, keepdim=True).values
        for i in range(len(x)):
            near = (d[i] == least[i]).nonzero()[:, 0].tolist()
            assert got[i].item() == (near[0] if len(near) == 1 else next(j for j in near if j % 2 == 0))


def test_the_oracle_turns_and_norms():
    x = torch.tensor([[3.0, 4.0, 0.0, 0.0, 1.0, 2.0, 3.0, 4.0]])
    inv = torch.tensor([0.5])
    c, s = math.cos(1.5), math.sin(1.5)
    for interleaved in (False, True):
        y = e.turned(x, 3, inv, interleaved, scale=2.0)
        assert torch.allclose(y[0], torch.tensor([2 * (3 * c - 4 * s), 2 * (4 * c + 3 * s), 0, 0, 1, 2, 3, 4], dtype=torch.float64), rtol=0, atol=1e-14)
    inv = torch.tensor([0.5, 0.25])
    y = e.turned(x, 2, inv, True)
    assert torch.allclose(y[0, 2:4], torch.zeros(2).double()) and torch.equal(y[0, 4:], x[0, 4:].double())
    y = e.turned(x, 0, None, w=torch.full((8,), 0.5), eps=0.0, offset=1.0)
    assert torch.allclose(y, 1.5 * x.double() / math.sqrt(55 / 8))


def test_frequencies_for_contexts_of_any_length():
    from se12_amd.rotary import rotary_frequencies

    plain, one = rotary_frequencies(128, 10000.0)
    ref = torch.tensor([10000.0 ** (-2 * i / 128) for i in range(64)], dtype=torch.float64)
    assert one == 1.0 and plain.dtype == torch.float32 and torch.equal(plain, ref.float())
    linear, one = rotary_frequencies(128, 10000.0, "linear", 4.0)
    assert one == 1.0 and torch.equal(linear, (ref / 4).float())
    base, one = rotary_frequencies(128, 10000.0, "base", 8.0)
    # (one rounding of FP32, and powers in 64 bits)
    assert one == 1.0 and base[0] == 1.0 and abs(base[-1].item() / ref[-1].item() * 8 - 1) <= 2.0 ** -24 + 1e-12
    parts, scale = rotary_frequencies(128, 10000.0, "parts", 16.0, context=4096)
    turns = 4096 * ref / (2 * math.pi)
    assert abs(scale - (0.1 * math.log(16.0) + 1)) <= 1e-15
    assert torch.equal(parts[turns > 32], plain[turns > 32]) and torch.equal(parts[turns < 1], (ref[turns < 1] / 16).float())
    between = (turns >= 1) & (turns <= 32)
    share = (turns[between] - 1) / 31
    assert between.any() and ((parts[between].double() - ref[between] * (share + (1 - share) / 16)).abs() <= 2.0 ** -24 * ref[between]).all()
    for method in ("linear", "base", "parts"):
        same, scale = rotary_frequencies(64, 500000.0, method, 1.0)
        assert scale == 1.0 and torch.equal(same, rotary_frequencies(64, 500000.0)[0])


@pytest.mark.parametrize("args,message", [
    ((12,), "multiple of 8"), ((0,), "multiple of 8"), ((8.5,), "multiple of 8"), ((64, 1.0), "base"), ((64, math.inf), "base"),
    ((64, 1e4, "other"), "method"), ((64, 1e4, "linear", 0.5), "factor"), ((64, 1e4, "linear", math.nan), "factor"),
    ((64, 1e4, "parts", 2.0, 0), "context"), ((64, 1e4, "parts", 2.0, 4096, 32.0, 1.0), "slow below fast"),
])
def test_frequencies_refuse(args, message):
    from se12_amd.rotary import rotary_frequencies

    with pytest.raises(ValueError, match=message):
        rotary_frequencies(*args)


def test_the_other_caches_need_no_torch_with_types_of_4_bits(monkeypatch):
    import importlib.util

    from se12_amd import paged

    monkeypatch.delattr(torch, "float4_e2m1fn_x2")
    spec = importlib.util.spec_from_file_location("se12_amd.paged_of_8_bits", paged.__file__)
    other = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(other)
    k, v, s = torch.zeros((4, 2, 16, 64)), torch.zeros((4, 2, 64, 16)), torch.ones((4, 2))
    for dtype, scales in ((torch.bfloat16, ()), (torch.float8_e4m3fn, (s, s))):
        with pytest.raises(ValueError, match="HIP device"):
            other.PagedKvCache.from_tensors(k.to(dtype), v.to(dtype), *scales)
    with pytest.raises(ValueError, match="k must be"):
        other.PagedKvCache.from_tensors(k, v)
    with pytest.raises(ValueError, match="k must be"):
        other.PagedKvCache(4, 16, 2, 64, dtype=None, device="cpu")


def test_rotations_go_to_the_kernels_as_the_struct_they_are():
    values = (1 << 40, 1 << 41, 1 << 42, 1.25, 1e-6, 0.5, nat.STEP_F32, 120, 1)
    assert nat.pack_rotation(*values) == bytes(nat.StepRotation(*values))


@pytest.mark.parametrize("scale", [1e39, -1e300, 2.0 ** 127])
def test_a_factor_that_fp32_does_not_hold_is_refused(scale):
    from se12_amd.paged import rotate_heads

    lib, b, r = nat.lib(), _batch(), _turn(scale=scale)
    _refused("finite", lambda: lib.se12_step_paged_append_rotated(ctypes.byref(_pages4()), ctypes.byref(b), P, P, P, nat.STEP_F32, 1024, 512, 512, 8,
                                                                  ctypes.byref(r), None, None))
    _refused("finite", lambda: lib.se12_step_rotate_heads(ctypes.byref(b), Q, 2 * Q, nat.STEP_BF16, 1024, 512, 8, 4, 128, ctypes.byref(r), Q + 16, 4 * Q,
                                                          nat.STEP_BF16, None))
    with pytest.raises(ValueError, match="finite"):
        rotate_heads(_on_cpu()[1], torch.zeros((3, 4, 64)), rotary_scale=scale)


@pytest.mark.parametrize("base,factor", [(1e4, 1e308), (1e300, 1e30), (1e308, 2.0)])
def test_a_base_that_64_bits_do_not_hold_is_refused(base, factor):
    from se12_amd.rotary import rotary_frequencies

    with pytest.raises(ValueError, match="base"):
        rotary_frequencies(8, base, "base", factor)
