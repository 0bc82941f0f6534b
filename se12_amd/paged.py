"""A key/value cache in pages, for programs that decode sequences of different
lengths in one batch: any page of a pool holds any part of any sequence, in BF16,
in 8 bits (E4M3) with one power-of-two scale per page and KV head, or in 4 bits
(E2M1) with an 8-bit scale per 32 columns of a token. (The static cache of
`gemma2.Gemma2Decoder` has one length for the whole batch.)

    cache = PagedKvCache(pages=4096, page_size=64, kv_heads=4, head_dim=256, device=dev)  # one per layer
    batch = PagedBatch(page_table, lengths, starts, max_new=1)      # shared by the layers
    q = cache.append(batch, k, v, q=q, inv_freq=inv_freq)           # rotates q and k, writes k and v
    y = cache.attend(batch, q, scaling, softcap=50.0)
    ...                                                             # after the last layer
    lengths += starts.diff()

`append` norms q and k per head and rotates them in either layout of pairs;
`rotate_heads` does that by itself; `PagedKvCache.read` gives back what is held.

All calls run on the current stream of the cache's device, read the batch's
tensors when their kernels run (a captured call follows what they hold at its
replay) and never wait for the device. No counterpart in the reference, whose
runtime leaves the cache to the framework. Kernels: se12_step_paged_append,
se12_step_paged_append_rotated, se12_step_paged_attention, se12_step_paged_read and
se12_step_rotate_heads (include/se12_step.h).
"""

from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from . import _native as nat

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)
_E2M1 = getattr(torch, "float4_e2m1fn_x2", object())      # (a torch without the type: equal to none)
_DTYPES = {torch.bfloat16: nat.STEP_BF16, torch.float8_e4m3fn: nat.STEP_E4M3, _E2M1: nat.STEP_E2M1}
_KINDS = {torch.bfloat16: nat.STEP_BF16, torch.float32: nat.STEP_F32}
_NO_GUARD = contextlib.nullcontext()


def _on(device: torch.device):
    """The device's guard where it is not the current one."""
    return _NO_GUARD if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    """The handle of the device's current stream."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _row_view(t, name: str, head_dim: int, index: int, device, heads: int | None, tokens: int | None, dtype: torch.dtype | None,
              multiple: int, owner: str = "the cache") -> torch.Tensor:
    """t [tokens, heads, head_dim] with heads side by side and rows `multiple` elements apart: itself, or a copy."""
    shape = t.shape if isinstance(t, torch.Tensor) else ()
    if len(shape) != 3 or shape[2] != head_dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {head_dim}]")
    if tokens is not None and shape[0] != tokens:
        raise ValueError(f"{name} has {shape[0]} rows, k has {tokens}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, {owner} on {device}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    (row, head, one), width = t.stride(), shape[1] * head_dim
    apart = row >= width and row % multiple == 0
    if (one != 1 or (head != head_dim and shape[1] > 1) or not (apart or shape[0] <= 1)
            or t.data_ptr() % (multiple * t.element_size())):
        t, apart = t.contiguous(), False
        if t.data_ptr() % (multiple * t.element_size()):
            t = t.clone()
    # (of a single row any first stride is contiguous to torch)
    return t if apart else t.as_strided(shape, (width, head_dim, 1))


def _norm_weight(w, name: str, head_dim: int, index: int, device) -> tuple[torch.Tensor, int]:
    """(w, its address)"""
    if not (isinstance(w, torch.Tensor) and w.get_device() == index and w.dtype in (torch.bfloat16, torch.float32) and w.shape == (head_dim,)
            and w.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous bfloat16 or float32 [{head_dim}] tensor on {device}")
    at = w.data_ptr()
    if at % 16:
        w = w.clone()
        at = w.data_ptr()
    return w, at


def _frequencies(inv_freq, head_dim: int, index: int, device) -> tuple[torch.Tensor, int, int]:
    """(inv_freq, its address, the columns it turns)"""
    if not (isinstance(inv_freq, torch.Tensor) and inv_freq.get_device() == index and inv_freq.dtype == torch.float32 and inv_freq.dim() == 1
            and inv_freq.is_contiguous()):
        raise ValueError(f"inv_freq must be a contiguous float32 vector on {device}")
    rotary = 2 * inv_freq.numel()
    if rotary % 8 or not 0 < rotary <= head_dim:
        raise ValueError(f"inv_freq must hold a multiple of 4, at most {head_dim // 2} frequencies, got {inv_freq.numel()}")
    at = inv_freq.data_ptr()
    if at % 16:
        inv_freq = inv_freq.clone()
        at = inv_freq.data_ptr()
    return inv_freq, at, rotary


def _rotation(head_dim: int, index: int, device, at: int, rotary: int, interleaved, rotary_scale, q_norm, k_norm, norm_eps, norm_offset):
    """A se12_step_rotation's bytes, and the weights that it points to."""
    q_at, k_at, dtype = 0, 0, torch.bfloat16
    if q_norm is not None:
        q_norm, q_at = _norm_weight(q_norm, "q_norm", head_dim, index, device)
        dtype = q_norm.dtype
    if k_norm is not None:
        k_norm, k_at = _norm_weight(k_norm, "k_norm", head_dim, index, device)
        if q_norm is not None and k_norm.dtype != dtype:
            raise ValueError("q_norm and k_norm must be of one type")
        dtype = k_norm.dtype
    if not (abs(rotary_scale) < 2.0 ** 127 and math.isfinite(norm_eps) and norm_eps >= 0 and abs(norm_offset) < 2.0 ** 127):
        raise ValueError("rotary_scale, norm_eps and norm_offset must be finite (the first and last below 2^127), norm_eps not below 0")
    return nat.pack_rotation(at, q_at, k_at, rotary_scale, norm_eps, norm_offset, _KINDS[dtype], rotary, 1 if interleaved else 0), (q_norm, k_norm)


def _int32(t: torch.Tensor, name: str, shape: tuple, device: torch.device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device:
        raise ValueError(f"{name} must be an int32 tensor on {device}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    return t


def check_softcap(softcap: float) -> None:
    """0 for none, or 2^-60 to 1024 (FP32 holds the factors of these)."""
    if not (softcap == 0 or 2.0 ** -60 <= softcap <= 1024.0):
        raise ValueError(f"softcap must be 0, or 2^-60 to 1024, got {softcap}")


class PagedBatch:
    """The new tokens of a call: sequence s holds lengths[s] tokens, rows starts[s]
    .. starts[s + 1] - 1 of q, k and v are its next ones, and its token j lies in
    slot j % page_size of page page_table[s, j // page_size].

    page_table int32 [sequences, columns], lengths int32 [sequences], starts int32
    [sequences + 1], ascending from 0, all on one device and used in place: a
    program changes what they hold between calls. max_new: the most new tokens of
    a sequence in any call with this batch (1 for decode steps). Entries behind a
    sequence's last page are not read; a token whose page is outside the pool, or
    whose position is outside the table, is held nowhere. Rows of q, k and v from
    starts[sequences] on are neither read nor written."""

    def __init__(self, page_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor, max_new: int = 1) -> None:
        if not isinstance(page_table, torch.Tensor) or page_table.dtype != torch.int32 or page_table.dim() != 2:
            raise ValueError("page_table must be an int32 [sequences, columns] tensor")
        n, width = page_table.shape
        if not 1 <= n <= 65536 or not 1 <= width <= 2 ** 30:
            raise ValueError(f"page_table must have 1 to 65536 rows and 1 to 2^30 columns, got {list(page_table.shape)}")
        if page_table.stride(1) != 1 and width > 1 or n > 1 and page_table.stride(0) < width:
            raise ValueError("page_table's rows must be contiguous and not overlap")
        if int(max_new) != max_new or not 1 <= max_new < 2 ** 31:
            raise ValueError(f"max_new must be a whole number from 1 to 2^31 - 1, got {max_new}")
        if not page_table.is_cuda:
            raise ValueError("page_table must be on a HIP device")
        self.device = page_table.device
        self.page_table = page_table
        self.lengths = _int32(lengths, "lengths", (n,), self.device)
        self.starts = _int32(starts, "starts", (n + 1,), self.device)
        if not (self.lengths.is_contiguous() and self.starts.is_contiguous()):
            raise ValueError("lengths and starts must be contiguous")
        self.sequences, self.max_new = n, int(max_new)
        self._fields = (page_table.data_ptr(), max(page_table.stride(0), width), lengths.data_ptr(), starts.data_ptr(), width, n)
        self._last = (-1, None)

    def _struct(self, tokens: int):
        """The C struct of a call with so many rows, by reference; the layers of a step share it."""
        last = self._last
        if last[0] != tokens:
            if tokens >= 2 ** 31:
                raise ValueError(f"a call holds below 2^31 tokens, got {tokens}")
            last = self._last = (tokens, ctypes.byref(nat.StepBatch(*self._fields, tokens, self.max_new)))
        return last[1]


class PagedKvCache:
    """One layer's cache: `k` [pages, kv_heads, page_size, head_dim] and `v` [pages,
    kv_heads, head_dim, page_size] (a value column's tokens side by side, as the
    attention's matrix operands take them), dtype float8_e4m3fn or bfloat16; with
    float8_e4m3fn `k_scale` and `v_scale` FP32 [pages, kv_heads], positive numbers by
    which a held value is multiplied. page_size 16, 32, 64 or 128, head_dim 64, 128 or 256.

    dtype float4_e2m1fn_x2 (two values to an element, the first in the low half): `k`
    [pages, kv_heads, page_size, head_dim / 2], `v` [pages, kv_heads, page_size / 16,
    head_dim, 8] (16 tokens of a column side by side), `k_scale` and `v_scale` uint8
    [pages, kv_heads, head_dim / 32, page_size], one to 32 columns of a token: an FP16
    number's bits 14 .. 7 (5 of exponent, 3 of fraction), 0 to 226; 255 stands for no number."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.float8_e4m3fn,
                 device=None) -> None:
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if dtype == _E2M1:
            shapes = ((pages, kv_heads, page_size, head_dim // 2), (pages, kv_heads, page_size // 16, head_dim, 8))
            k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for shape in shapes)
            scales = [torch.zeros((pages, kv_heads, head_dim // 32, page_size), dtype=torch.uint8, device=device) for _ in range(2)]
        else:
            k = torch.zeros((pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
            v = torch.zeros((pages, kv_heads, head_dim, page_size), dtype=dtype, device=device)
            scales = [torch.ones((pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2)] \
                if dtype == torch.float8_e4m3fn else [None, None]
        self._bind(k, v, *scales)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None) -> "PagedKvCache":
        """A cache in the caller's tensors (used in place)."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k, v, k_scale, v_scale) -> None:
        if not isinstance(k, torch.Tensor) or k.dim() != 4 or k.dtype not in _DTYPES:
            raise ValueError("k must be a float4_e2m1fn_x2, float8_e4m3fn or bfloat16 [pages, kv_heads, page_size, head_dim] tensor")
        pages, kv_heads, page_size, head_dim = k.shape
        e2m1, e4m3 = k.dtype == _E2M1, k.dtype == torch.float8_e4m3fn
        head_dim *= 2 if e2m1 else 1
        if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}, got {page_size}, {head_dim}")
        if pages < 1 or not 1 <= kv_heads <= 1024 or pages > 2 ** 31 - 1:
            raise ValueError("the cache needs a page and 1 to 1024 heads")
        v_shape = (pages, kv_heads, page_size // 16, head_dim, 8) if e2m1 else (pages, kv_heads, head_dim, page_size)
        if not isinstance(v, torch.Tensor) or v.dtype != k.dtype or tuple(v.shape) != v_shape:
            raise ValueError(f"v must be {k.dtype} {list(v_shape)}")
        scaled, kind = e2m1 or e4m3, "an E2M1" if e2m1 else "an E4M3"
        scale_shape, scale_dtype = ((pages, kv_heads, head_dim // 32, page_size), torch.uint8) if e2m1 else ((pages, kv_heads), torch.float32)
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if (t is not None) != scaled:
                raise ValueError(f"{name} goes with an E4M3 or E2M1 cache" if t is not None else f"{kind} cache needs {name}")
            if scaled and (t.dtype != scale_dtype or tuple(t.shape) != scale_shape):
                raise ValueError(f"{name} must be {scale_dtype} {list(scale_shape)}")
        tensors = [t for t in (k, v, k_scale, v_scale) if t is not None]
        if any(not t.is_contiguous() for t in tensors):
            raise ValueError("a cache's tensors must be contiguous")
        if any(not t.is_cuda or t.device != k.device for t in tensors):
            raise ValueError("a cache's tensors must be on one HIP device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.dtype, self._index = k.device, k.dtype, k.get_device()
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, kv_heads, page_size, head_dim
        self._struct = ctypes.byref(nat.StepPages(k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if scaled else None,
                                     v_scale.data_ptr() if scaled else None, _DTYPES[k.dtype], pages, page_size, kv_heads, head_dim))

    def _rows(self, t: torch.Tensor, name: str, heads: int | None, tokens: int | None, dtype: torch.dtype | None,
              multiple: int) -> torch.Tensor:
        return _row_view(t, name, self.head_dim, self._index, self.device, heads, tokens, dtype, multiple)

    def _check(self, batch: PagedBatch) -> None:
        if not isinstance(batch, PagedBatch):
            raise ValueError("batch must be a PagedBatch")
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")

    def append(self, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None,
               inv_freq: torch.Tensor | None = None, out: torch.Tensor | None = None, *, interleaved: bool = False,
               rotary_scale: float = 1.0, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
               norm_eps: float = 1e-6, norm_offset: float = 0.0) -> torch.Tensor | None:
        """Writes the new tokens' k and v [tokens, kv_heads, head_dim] to their pages, k rotated to its position, and
        returns q [tokens, heads, head_dim] rotated, in BF16 (into `out` if given, which may be q, or shares no memory with
        q, k and v; None without q). BF16 or FP32, all of one type; rows may be strided (views of one product's output).
        The rotation turns the pairs (i, i + len(inv_freq)) by position * inv_freq[i], FP32 inv_freq of up to head_dim / 2
        frequencies, a multiple of 4 (the elements behind the pairs stay; None: no rotation), as
        se12_step_prefill_attention pairs them; or the pairs (2 i, 2 i + 1) where `interleaved`; sine and cosine times
        `rotary_scale`. With `q_norm` and `k_norm` [head_dim] (BF16 or FP32) q's and k's heads are normed before: x
        rsqrt(mean(x^2) + norm_eps) (norm_offset + w). (`rotary.rotary_frequencies` stretches inv_freq to longer contexts.)

        An E2M1 cache holds 32 columns of a token as codes times the 8-bit scale nearest to a sixth of their largest
        value, 10240 at most (so values up to 61440), each value as the nearest code; 32 columns with a NaN or an infinity
        as NaN. What a token is held as depends on that token alone.

        (Norms, interleaved pairs and a scale for a cache of BF16 or E4M3 take a launch more for each of q and k, one that
        widens BF16 v, memory for k and v in FP32, and a copy of `out` there and back where it is not 16-byte aligned.)
        An E4M3 page and head's scale is the least power of two (2^-100 or more) that holds its new values; with older
        tokens in the page at least what it was, and if it grows the older ones are rounded again. NaN and infinities
        are held as NaN. A page that two entries of the table name must not be written by a call."""
        self._check(batch)
        if not isinstance(k, torch.Tensor) or k.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("k must be a bfloat16 or float32 tensor")
        head_dim, index, device, dtype = self.head_dim, self._index, self.device, k.dtype
        k = _row_view(k, "k", head_dim, index, device, self.kv_heads, None, None, 4)
        tokens = k.shape[0]
        v = _row_view(v, "v", head_dim, index, device, self.kv_heads, tokens, dtype, 4)
        inv_freq, inv_at, rotary = (None, 0, 0) if inv_freq is None else _frequencies(inv_freq, head_dim, index, device)
        heads, q_stride, q_at, out_at = self.kv_heads, 0, None, None
        if q is not None:
            q = _row_view(q, "q", head_dim, index, device, None, tokens, dtype, 4)
            heads, q_stride, q_at = q.shape[1], q.stride(0), q.data_ptr()
            if heads % self.kv_heads or heads == 0:
                raise ValueError(f"q's {heads} heads are no multiple of the cache's {self.kv_heads}")
            out = self._out(out, tokens, heads)
            out_at = out.data_ptr()
        elif out is not None:
            raise ValueError("out goes with q")
        elif q_norm is not None:
            raise ValueError("q_norm goes with q")
        e2m1 = self.dtype == _E2M1
        plain = q_norm is None and k_norm is None and not interleaved and rotary_scale == 1.0
        if e2m1 or not plain or norm_eps != 1e-6 or norm_offset != 0.0:
            rotation, held = _rotation(head_dim, index, device, inv_at, rotary, interleaved, rotary_scale, q_norm, k_norm, norm_eps, norm_offset)
        lib, new, kind = nat.lib(), batch._struct(tokens), _KINDS[dtype]
        with _on(device):
            if e2m1:
                nat.step_check(lib.se12_step_paged_append_rotated(
                    self._struct, new, q_at, k.data_ptr(), v.data_ptr(), kind, q_stride, k.stride(0), v.stride(0), heads, rotation, out_at,
                    _stream(device)))
                return out
            if not plain:
                return self._append_turned(batch, q, k, v, out, inv_freq, interleaved, rotary_scale, *held, norm_eps, norm_offset)
            nat.step_check(lib.se12_step_paged_append(
                self._struct, new, q_at, k.data_ptr(), v.data_ptr(), kind, q_stride, k.stride(0), v.stride(0), heads, inv_at or None, rotary,
                out_at, _stream(device)))
        return out

    def _append_turned(self, batch, q, k, v, out, inv_freq, interleaved, rotary_scale, q_norm, k_norm, norm_eps, norm_offset):
        """append for a cache of BF16 or E4M3 whose kernel does not norm: q and k turned before, k kept in FP32."""
        if q is not None:
            spans = [(t.data_ptr(), t.data_ptr() + t.element_size() * ((t.shape[0] - 1) * t.stride(0) + t.shape[1] * t.shape[2]))
                     for t in (out, k, v) if t.shape[0]]
            if any(lo < spans[0][1] and spans[0][0] < hi for lo, hi in spans[1:]):
                raise ValueError("out overlaps k or v")
        turn = dict(interleaved=interleaved, rotary_scale=rotary_scale, norm_eps=norm_eps, norm_offset=norm_offset)
        turned, _ = rotate_heads(batch, k, None, inv_freq, q_norm=k_norm, dtype=torch.float32, **turn)
        if q is not None:
            # (q's kernel writes 16 bytes at once)
            fits = out.data_ptr() % 16 == 0
            got, _ = rotate_heads(batch, q, None, inv_freq, q_norm=q_norm, out=(out if fits else out.clone(), None), **turn)
            if not fits:
                out.copy_(got)
        self.append(batch, turned, v.float())
        return out

    def read(self, batch: PagedBatch, tokens: int, out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds of the batch's tokens, in BF16: (k, v) [tokens, kv_heads, head_dim], rows starts[s] ..
        starts[s + 1] - 1 of positions lengths[s] .. (lengths of zero and starts that add the sequences' tokens up: whole
        sequences; max_new the longest). Into `out` if given, two tensors apart. Rounded once: E2M1, BF16 and E4M3 under
        power-of-two scales are exact. A token held nowhere gives zeros; rows of no sequence are not written."""
        self._check(batch)
        if int(tokens) != tokens or not 0 <= tokens < 2 ** 31:
            raise ValueError(f"tokens must be a whole number from 0 to 2^31 - 1, got {tokens}")
        shape = (int(tokens), self.kv_heads, self.head_dim)
        if out is None:
            k, v = torch.empty((2, *shape), dtype=torch.bfloat16, device=self.device).unbind()
        else:
            k, v = out
        for t in () if out is None else (k, v):
            if not isinstance(t, torch.Tensor) or t.device != self.device or t.dtype != torch.bfloat16 or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"out must be two contiguous bfloat16 {list(shape)} tensors on {self.device}")
            if t.data_ptr() % 16:
                raise ValueError("out must be 16-byte aligned")
        with _on(self.device):
            nat.step_check(nat.lib().se12_step_paged_read(self._struct, batch._struct(shape[0]), k.data_ptr(), v.data_ptr(), _stream(self.device)))
        return k, v

    def attend(self, batch: PagedBatch, q: torch.Tensor, scaling: float, softcap: float = 0.0, window: int = 0,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the new tokens' q [tokens, heads, head_dim] (BF16, rotated; rows may be strided) over their
        sequences' pages, the tokens of this call appended before: softmax(cap(q . k scaling)) . v over the keys max(0,
        p - window + 1) .. p of the query's position p, cap(s) = softcap tanh(s / softcap) where softcap > 0 (2^-60 to 1024),
        window 0 = all. Returns BF16 [tokens, heads, head_dim] (`out` if given, apart from q; rows of no sequence are not
        written). No gradients.

        FP32 scores and sums; weights rounded to BF16 (over an E2M1 cache to FP16). A query that sees nothing gives zeros. `workspace`: uint8 of at
        least `attend_workspace()` bytes for callers that must not allocate; calls that share one must not overlap, and
        one that a captured call was given lives, as its other tensors, as long as the graph."""
        self._check(batch)
        q = self._rows(q, "q", None, None, torch.bfloat16, 8)
        tokens, heads = q.shape[0], q.shape[1]
        if heads % self.kv_heads or heads == 0:
            raise ValueError(f"q's {heads} heads are no multiple of the cache's {self.kv_heads}")
        check_softcap(softcap)
        if int(window) != window or not 0 <= window < 2 ** 31:
            raise ValueError("window must be a whole number, 0 or more")
        out = self._out(out, tokens, heads)
        if tokens == 0:
            return out
        lib = nat.lib()
        pages, new = self._struct, batch._struct(tokens)
        with _on(self.device):
            if workspace is None:
                n = lib.se12_step_paged_attention_workspace(pages, new, heads)
                if n < 0:
                    nat.step_check(n)
                workspace = torch.empty(n, dtype=torch.uint8, device=self.device)
            elif workspace.dtype != torch.uint8 or workspace.device != self.device or not workspace.is_contiguous():
                raise ValueError(f"workspace must be a contiguous uint8 tensor on {self.device}")
            nat.step_check(lib.se12_step_paged_attention(
                pages, new, q.data_ptr(), q.stride(0), out.data_ptr(), heads, float(scaling), float(softcap), int(window),
                workspace.data_ptr(), workspace.numel(), _stream(self.device)))
        return out

    def attend_workspace(self, batch: PagedBatch, tokens: int, heads: int) -> int:
        """Bytes of `attend`'s workspace for calls of so many tokens; enough for fewer as well."""
        self._check(batch)
        if not 0 <= tokens < 2 ** 31 or not 0 < heads < 2 ** 31:
            raise ValueError(f"tokens and heads must be below 2^31, got {tokens}, {heads}")
        n = nat.lib().se12_step_paged_attention_workspace(self._struct, batch._struct(tokens), heads)
        if n < 0:
            nat.step_check(n)
        return int(n)

    def _out(self, out: torch.Tensor | None, tokens: int, heads: int) -> torch.Tensor:
        shape = (tokens, heads, self.head_dim)
        if out is None:
            return torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        if out.device != self.device or out.dtype != torch.bfloat16 or tuple(out.shape) != shape or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous bfloat16 {list(shape)} tensor on {self.device}")
        if out.data_ptr() % 8:
            raise ValueError("out must be 8-byte aligned")
        return out


def rotate_heads(batch: PagedBatch, q: torch.Tensor, k: torch.Tensor | None = None, inv_freq: torch.Tensor | None = None, *,
                 interleaved: bool = False, rotary_scale: float = 1.0, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None, norm_eps: float = 1e-6, norm_offset: float = 0.0,
                 dtype: torch.dtype = torch.bfloat16, out: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The batch's q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] (BF16 or FP32, both of one type; rows
    may be strided) normed and rotated to their positions as `PagedKvCache.append` does, in `dtype` (bfloat16 or float32):
    (q, k), k None without k (in BF16 one value in 2^16 may be a step from `append`'s). Into `out` = (q, k) if given; each may be its own input, and is apart from the rest
    otherwise. head_dim a multiple of 8 up to 256. The batch's page table is not read; rows of no sequence are
    not written. No gradients."""
    if not isinstance(batch, PagedBatch):
        raise ValueError("batch must be a PagedBatch")
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.dtype not in _KINDS:
        raise ValueError("q must be a bfloat16 or float32 [tokens, heads, head_dim] tensor")
    shape, kind = q.shape, q.dtype
    tokens, heads, head_dim = shape
    if head_dim % 8 or not 8 <= head_dim <= 256 or not 1 <= heads <= 65535:
        raise ValueError(f"q must have 1 to 65535 heads and a head_dim of a multiple of 8 up to 256, got {heads}, {head_dim}")
    if dtype not in _KINDS:
        raise ValueError(f"dtype must be bfloat16 or float32, got {dtype}")
    index, device = batch.page_table.get_device(), batch.device
    q = _row_view(q, "q", head_dim, index, device, None, None, None, 4, "the batch")
    q_out, k_out = (None, None) if out is None else out
    q_out = _turned_out(q_out, shape, dtype, device)
    kv_heads = k_stride = 0
    k_at = k_out_at = None
    if k is not None:
        if isinstance(k, torch.Tensor) and k.dim() == 3:
            shape = k.shape
            kv_heads = shape[1]
            if not 1 <= kv_heads <= 65535:
                raise ValueError(f"k must have 1 to 65535 heads, got {kv_heads}")
            if shape[0] != tokens:
                raise ValueError(f"k has {shape[0]} rows, q has {tokens}")
        k = _row_view(k, "k", head_dim, index, device, None, None, kind, 4, "the batch")
        k_out = _turned_out(k_out, shape, dtype, device)
        k_stride, k_at, k_out_at = k.stride(0), k.data_ptr(), k_out.data_ptr()
    elif k_norm is not None or k_out is not None:
        raise ValueError("k_norm and out's second tensor go with k")
    inv_freq, inv_at, rotary = (None, 0, 0) if inv_freq is None else _frequencies(inv_freq, head_dim, index, device)
    rotation, held = _rotation(head_dim, index, device, inv_at, rotary, interleaved, rotary_scale, q_norm, k_norm, norm_eps, norm_offset)
    with _on(device):
        nat.step_check(nat.lib().se12_step_rotate_heads(
            batch._struct(tokens), q.data_ptr(), k_at, _KINDS[kind], q.stride(0), k_stride, heads, kv_heads, head_dim, rotation, q_out.data_ptr(),
            k_out_at, _KINDS[dtype], _stream(device)))
    del inv_freq, held      # (until the call has been made)
    return q_out, k_out


def _turned_out(out, shape, dtype: torch.dtype, device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if not isinstance(out, torch.Tensor) or out.device != device or out.dtype != dtype or out.shape != shape or not out.is_contiguous():
        raise ValueError(f"out must hold contiguous {dtype} tensors of q's and k's shapes on {device}")
    if out.data_ptr() % 16:
        raise ValueError("out must be 16-byte aligned")
    return out
