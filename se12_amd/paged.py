"""A key/value cache in pages, for programs that decode sequences of different
lengths in one batch: any page of a pool holds any part of any sequence, in BF16
or in 8 bits (E4M3) with one power-of-two scale per page and KV head. (The static
cache of `gemma2.Gemma2Decoder` has one length for the whole batch.)

    cache = PagedKvCache(pages=4096, page_size=64, kv_heads=4, head_dim=256, device=dev)  # one per layer
    batch = PagedBatch(page_table, lengths, starts, max_new=1)      # shared by the layers
    q = cache.append(batch, k, v, q=q, inv_freq=inv_freq)           # rotates q and k, writes k and v
    y = cache.attend(batch, q, scaling, softcap=50.0)
    ...                                                             # after the last layer
    lengths += starts.diff()

Both calls run on the current stream of the cache's device, read the batch's
tensors when their kernels run (a captured call follows what they hold at its
replay) and never wait for the device. No counterpart in the reference, whose
runtime leaves the cache to the framework. Kernels: se12_step_paged_append and
se12_step_paged_attention (include/se12_step.h).
"""

from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _native as nat

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)
_NO_GUARD = contextlib.nullcontext()


def _on(device: torch.device):
    """The device's guard where it is not the current one."""
    return _NO_GUARD if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    """The handle of the device's current stream."""
    return torch._C._cuda_getCurrentRawStream(device.index)


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
    which a held value is multiplied. page_size 16, 32, 64 or 128, head_dim 64, 128 or 256."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.float8_e4m3fn,
                 device=None) -> None:
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        k = torch.zeros((pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        scales = [torch.ones((pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2)] \
            if dtype == torch.float8_e4m3fn else [None, None]
        self._bind(k, torch.zeros((pages, kv_heads, head_dim, page_size), dtype=dtype, device=device), *scales)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None) -> "PagedKvCache":
        """A cache in the caller's tensors (used in place)."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k, v, k_scale, v_scale) -> None:
        if not isinstance(k, torch.Tensor) or k.dim() != 4 or k.dtype not in (torch.float8_e4m3fn, torch.bfloat16):
            raise ValueError("k must be a float8_e4m3fn or bfloat16 [pages, kv_heads, page_size, head_dim] tensor")
        pages, kv_heads, page_size, head_dim = k.shape
        if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}, got {page_size}, {head_dim}")
        if pages < 1 or not 1 <= kv_heads <= 1024 or pages > 2 ** 31 - 1:
            raise ValueError("the cache needs a page and 1 to 1024 heads")
        if not isinstance(v, torch.Tensor) or v.dtype != k.dtype or tuple(v.shape) != (pages, kv_heads, head_dim, page_size):
            raise ValueError(f"v must be {k.dtype} {[pages, kv_heads, head_dim, page_size]}")
        e4m3 = k.dtype == torch.float8_e4m3fn
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if (t is not None) != e4m3:
                raise ValueError(f"{name} goes with an E4M3 cache" if t is not None else f"an E4M3 cache needs {name}")
            if e4m3 and (t.dtype != torch.float32 or tuple(t.shape) != (pages, kv_heads)):
                raise ValueError(f"{name} must be float32 {[pages, kv_heads]}")
        tensors = [t for t in (k, v, k_scale, v_scale) if t is not None]
        if any(not t.is_contiguous() for t in tensors):
            raise ValueError("a cache's tensors must be contiguous")
        if any(not t.is_cuda or t.device != k.device for t in tensors):
            raise ValueError("a cache's tensors must be on one HIP device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.dtype, self._index = k.device, k.dtype, k.get_device()
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, kv_heads, page_size, head_dim
        self._struct = ctypes.byref(nat.StepPages(k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if e4m3 else None,
                                     v_scale.data_ptr() if e4m3 else None, nat.STEP_E4M3 if e4m3 else nat.STEP_BF16, pages,
                                     page_size, kv_heads, head_dim))

    def _rows(self, t: torch.Tensor, name: str, heads: int | None, tokens: int | None, dtype: torch.dtype | None,
              multiple: int) -> torch.Tensor:
        """t [tokens, heads, head_dim] with heads side by side and rows `multiple` elements apart: itself, or a copy."""
        shape = t.shape if isinstance(t, torch.Tensor) else ()
        if len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {self.head_dim}]")
        if tokens is not None and shape[0] != tokens:
            raise ValueError(f"{name} has {shape[0]} rows, k has {tokens}")
        if t.get_device() != self._index:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        if dtype is not None and t.dtype != dtype:
            raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
        (row, head, one), width = t.stride(), shape[1] * self.head_dim
        apart = row >= width and row % multiple == 0
        if (one != 1 or (head != self.head_dim and shape[1] > 1) or not (apart or shape[0] <= 1)
                or t.data_ptr() % (multiple * t.element_size())):
            t, apart = t.contiguous(), False
            if t.data_ptr() % (multiple * t.element_size()):
                t = t.clone()
        # (of a single row any first stride is contiguous to torch)
        return t if apart else t.as_strided(shape, (width, self.head_dim, 1))

    def _check(self, batch: PagedBatch) -> None:
        if not isinstance(batch, PagedBatch):
            raise ValueError("batch must be a PagedBatch")
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")

    def append(self, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None,
               inv_freq: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor | None:
        """Writes the new tokens' k and v [tokens, kv_heads, head_dim] to their pages, k rotated to its position, and
        returns q [tokens, heads, head_dim] rotated, in BF16 (into `out` if given, which may be q, or shares no memory with
        q, k and v; None without q). BF16 or FP32, all of one type; rows may be strided (views of one product's output).
        The rotation turns the pairs (i, i + len(inv_freq)) by position * inv_freq[i], FP32 inv_freq of up to head_dim / 2
        frequencies, a multiple of 4 (the elements behind the pairs stay; None: no rotation), as
        se12_step_prefill_attention pairs them.

        An E4M3 page and head's scale is the least power of two (2^-100 or more) that holds its new values; with older
        tokens in the page at least what it was, and if it grows the older ones are rounded again. NaN and infinities
        are held as NaN. A page that two entries of the table name must not be written by a call."""
        self._check(batch)
        if not isinstance(k, torch.Tensor) or k.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("k must be a bfloat16 or float32 tensor")
        k = self._rows(k, "k", self.kv_heads, None, None, 4)
        tokens = k.shape[0]
        v = self._rows(v, "v", self.kv_heads, tokens, k.dtype, 4)
        rotary = 0
        if inv_freq is not None:
            if inv_freq.device != self.device or inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
                raise ValueError(f"inv_freq must be a contiguous float32 vector on {self.device}")
            rotary = 2 * inv_freq.numel()
            if rotary % 8 or not 0 < rotary <= self.head_dim:
                raise ValueError(f"inv_freq must hold a multiple of 4, at most {self.head_dim // 2} frequencies, got {inv_freq.numel()}")
            if inv_freq.data_ptr() % 16:
                inv_freq = inv_freq.clone()
        heads, q_stride = self.kv_heads, 0
        if q is not None:
            q = self._rows(q, "q", None, tokens, k.dtype, 4)
            heads, q_stride = q.shape[1], q.stride(0)
            if heads % self.kv_heads or heads == 0:
                raise ValueError(f"q's {heads} heads are no multiple of the cache's {self.kv_heads}")
            out = self._out(out, tokens, heads)
        elif out is not None:
            raise ValueError("out goes with q")
        with _on(self.device):
            nat.step_check(nat.lib().se12_step_paged_append(
                self._struct, batch._struct(tokens), None if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(),
                nat.STEP_F32 if k.dtype == torch.float32 else nat.STEP_BF16, q_stride, k.stride(0), v.stride(0), heads,
                None if inv_freq is None else inv_freq.data_ptr(), rotary, None if q is None else out.data_ptr(),
                _stream(self.device)))
        return out

    def attend(self, batch: PagedBatch, q: torch.Tensor, scaling: float, softcap: float = 0.0, window: int = 0,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the new tokens' q [tokens, heads, head_dim] (BF16, rotated; rows may be strided) over their
        sequences' pages, the tokens of this call appended before: softmax(cap(q . k scaling)) . v over the keys max(0,
        p - window + 1) .. p of the query's position p, cap(s) = softcap tanh(s / softcap) where softcap > 0 (2^-60 to 1024),
        window 0 = all. Returns BF16 [tokens, heads, head_dim] (`out` if given, apart from q; rows of no sequence are not
        written). No gradients.

        FP32 scores and sums; weights rounded to BF16. A query that sees nothing gives zeros. `workspace`: uint8 of at
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
