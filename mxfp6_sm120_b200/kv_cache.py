"""Paged 8-bit KV cache: write, read, attention; and rotary positions with several axes.

The reference leaves attention to its serving runtime (docs/runtime-integration.md:13-22); these
are the operators that stand between the QKV projection and the output projection of a decoder
whose linears run W6A8.  The cache is held in the number format of the W6A8 activations - E4M3
values under power-of-two UE8M0 scales - with one scale per block of 32 tokens and head.

Every operator takes the same description of a batch:

``block_table``  ``[batch, width]`` int32, page of every ``page_size`` tokens of a sequence;
                 an id outside the cache names no page (its tokens are neither written nor seen)
``seq_lens``     ``[batch]`` int32, tokens of each sequence INCLUDING the rows of this call
``cu_seqlens``   ``[batch + 1]`` int32, rows ``cu_seqlens[b] : cu_seqlens[b + 1]`` of the token
                 tensors are the last positions of sequence ``b``; None: one row per sequence

All three live on the device and are read there while the call runs (they must not change
meanwhile), so a captured CUDA graph follows them; rows behind ``cu_seqlens[batch]`` are left as
they were.

These are serving operators without a backward pass: results carry no gradient, whatever their
inputs require.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from ._loader import check, library
from .ops import SCALE_VECTOR_SIZE, _DTYPE_CODE, _refuse, _require_sm100

KV_HEAD_DIMS = (64, 128, 256)
KV_PAGE_SIZES = (32, 64, 128)


_BF16, _F16 = torch.bfloat16, torch.float16
_SM100_SEEN: set[int] = set()


def _raw_stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _launch(device: torch.device, function, *args) -> None:
    """Call a C entry on ``device`` and its current stream.

    These operators run several times per decoder layer with microseconds of GPU work each, so the
    argument rules above the call are plain comparisons whose messages are only built to be raised,
    the device is switched only when it is not the current one, and the stream is asked for by its
    handle (0.1 us; as an object 1.3 us).
    """
    index = device.index
    if index not in _SM100_SEEN:
        if device.type != "cuda":
            raise ValueError(f"the tensors must be on a CUDA device; got {device}")
        _require_sm100(device)
        _SM100_SEEN.add(index)
    if torch._C._cuda_getDevice() == index:
        status = function(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = function(*args, _raw_stream(index))
    if status != 0:
        check(status)


@dataclass(frozen=True)
class PagedKVCache:
    """Keys and values of one layer in pages of 8-bit numbers.

    ``k_values`` / ``v_values``: uint8 E4M3 codes ``[pages, kv_heads, page_size, head_dim]``;
    ``k_scales`` / ``v_scales``: uint8 UE8M0 codes ``[pages, kv_heads, page_size // 32]``, one per
    32 tokens of a page and head: a value is ``code * 2**(scale - 127)``.  Scale codes of blocks that
    hold tokens are 0 to 254 (:func:`kv_cache_write` makes 28 to 253); 255 is no number.
    """

    k_values: torch.Tensor
    v_values: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor

    def __post_init__(self) -> None:
        k, v, ks, vs = self.k_values, self.v_values, self.k_scales, self.v_scales
        shape = k.shape
        if len(shape) != 4:
            raise ValueError(f"k_values must be [pages, kv_heads, page_size, head_dim]; got {tuple(shape)}")
        pages, heads, page, dim = shape
        if page not in KV_PAGE_SIZES:
            raise ValueError(f"page_size must be one of {KV_PAGE_SIZES}; got {page}")
        if dim not in KV_HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {KV_HEAD_DIMS}; got {dim}")
        if pages < 1 or heads < 1:
            raise ValueError("the cache needs at least one page and one head")
        if v.shape != shape:
            raise ValueError("v_values must have the shape of k_values")
        want = (pages, heads, page // SCALE_VECTOR_SIZE)
        if ks.shape != want or vs.shape != want:
            raise ValueError(f"k_scales and v_scales must be {list(want)}")
        u8 = torch.uint8
        if k.dtype != u8 or v.dtype != u8 or ks.dtype != u8 or vs.dtype != u8:
            raise TypeError("cache tensors must be uint8")
        device = k.device
        if v.device != device or ks.device != device or vs.device != device:
            raise ValueError("cache tensors must be on one device")
        if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
            raise ValueError("cache tensors must be contiguous")
        object.__setattr__(self, "device", device)
        object.__setattr__(self, "_extents", (pages, heads, page, dim))

    def _arguments(self) -> tuple:
        """What every call passes on."""
        return (self.k_values.data_ptr(), self.v_values.data_ptr(), self.k_scales.data_ptr(),
                self.v_scales.data_ptr(), *self._extents)

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, page_size: int, head_dim: int,
                 device: torch.device | str | int = "cuda") -> "PagedKVCache":
        """A zeroed cache of ``pages`` pages (scale codes 127: factors of one)."""
        shape = (pages, kv_heads, page_size, head_dim)
        blocks = (pages, kv_heads, page_size // SCALE_VECTOR_SIZE)
        return cls(torch.zeros(shape, dtype=torch.uint8, device=device),
                   torch.zeros(shape, dtype=torch.uint8, device=device),
                   torch.full(blocks, 127, dtype=torch.uint8, device=device),
                   torch.full(blocks, 127, dtype=torch.uint8, device=device))

    @property
    def pages(self) -> int:
        return self._extents[0]

    @property
    def kv_heads(self) -> int:
        return self._extents[1]

    @property
    def page_size(self) -> int:
        return self._extents[2]

    @property
    def head_dim(self) -> int:
        return self._extents[3]

    def nbytes(self) -> int:
        """Bytes of the values and scales."""
        return 2 * (self.k_values.numel() + self.k_scales.numel())


def _check_batch(cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                 cu_seqlens: torch.Tensor | None, tokens: int) -> tuple:
    """The batch description's argument rules; returns its C arguments."""
    if not isinstance(cache, PagedKVCache):
        raise TypeError("cache must be a PagedKVCache instance")
    device = cache.device
    if block_table.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("block_table and seq_lens must be int32")
    shape = block_table.shape
    if len(shape) != 2 or shape[1] < 1 or (shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError("block_table must be [batch, width] with contiguous rows")
    batch, width = shape
    if batch < 1:
        raise ValueError("the batch must hold at least one sequence")
    if seq_lens.shape != (batch,) or not seq_lens.is_contiguous():
        raise ValueError(f"seq_lens must be contiguous [{batch}]")
    if block_table.device != device or seq_lens.device != device:
        raise ValueError("block_table and seq_lens must be on the cache's device")
    offsets = None
    if cu_seqlens is None:
        if tokens != batch:
            raise ValueError(f"without cu_seqlens every sequence has one row; got {tokens} rows for "
                             f"{batch} sequences")
    else:
        if cu_seqlens.dtype != torch.int32:
            raise TypeError("cu_seqlens must be int32")
        if cu_seqlens.shape != (batch + 1,) or not cu_seqlens.is_contiguous():
            raise ValueError(f"cu_seqlens must be contiguous [{batch + 1}]")
        if cu_seqlens.device != device:
            raise ValueError("cu_seqlens must be on the cache's device")
        offsets = cu_seqlens.data_ptr()
    return (block_table.data_ptr(), seq_lens.data_ptr(), offsets, block_table.stride(0), tokens, width,
            batch)


def _check_rows(tensor: torch.Tensor, name: str, heads: int | None, dim: int,
                device: torch.device) -> tuple:
    """Rules of ``[tokens, heads, dim]`` rows of 16-bit numbers; returns the strides."""
    dtype = tensor.dtype
    if dtype is not _BF16 and dtype is not _F16:
        raise TypeError(f"{name} must have dtype torch.float16 or torch.bfloat16; got {dtype}")
    shape = tensor.shape
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {dim}]; got "
                         f"{tuple(shape)}")
    strides = tensor.stride()
    if strides[2] != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    if tensor.device != device:
        raise ValueError(f"{name} must be on {device}; got {tensor.device}")
    return strides


def _check_output_rows(tensor: torch.Tensor, name: str, like: torch.Tensor,
                       device: torch.device) -> tuple:
    """Rules of an output of ``like``'s shape and dtype, whose rows share no memory."""
    tokens, heads, dim = like.shape
    strides = _check_rows(tensor, name, heads, dim, device)
    if tensor.shape[0] != tokens or tensor.dtype != like.dtype:
        raise ValueError(f"{name} must match its input's shape and dtype")
    token_stride, head_stride, _ = strides
    bad = (heads > 1 and head_stride < dim) or (tokens > 1 and token_stride < dim)
    if not bad and tokens > 1 and heads > 1:
        inner, outer = sorted(((head_stride, heads), (token_stride, tokens)))
        bad = outer[0] < inner[0] * (inner[1] - 1) + dim
    if bad:
        raise ValueError(f"{name} must not overlap itself")
    return strides


def kv_cache_write(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor,
                   block_table: torch.Tensor, seq_lens: torch.Tensor,
                   cu_seqlens: torch.Tensor | None = None) -> None:
    """Quantise new keys and values ``[tokens, kv_heads, head_dim]`` into the cache's pages.

    The scale of a block of 32 tokens and head is the smallest power of two that takes the largest
    finite magnitude written to it to 448 or less (at least 2^-99).  Where a call adds tokens to a
    block that already holds some, the scale only grows, and the codes already there are rounded
    once more to it; writing a block's first token starts it anew.  Values round to nearest even
    and saturate (infinities too); NaN stays NaN.  Positions below zero (``seq_lens[b]`` smaller
    than the sequence's rows) and positions behind the block table are not written.  No page may
    be named by two sequences, or twice by one, for positions that the call writes.
    """
    if k.ndim != 3:
        raise ValueError(f"k must be [tokens, kv_heads, head_dim]; got {tuple(k.shape)}")
    batch = _check_batch(cache, block_table, seq_lens, cu_seqlens, k.shape[0])
    device = cache.device
    _, heads, _, dim = cache._extents
    k_strides = _check_rows(k, "k", heads, dim, device)
    v_strides = _check_rows(v, "v", heads, dim, device)
    if v.shape != k.shape or v.dtype is not k.dtype:
        raise ValueError("k and v must have one shape and dtype")
    _launch(device, library().mxfp6_kv_cache_write, *cache._arguments(), *batch, k.data_ptr(), v.data_ptr(),
            _DTYPE_CODE[k.dtype], k_strides[0], k_strides[1], v_strides[0], v_strides[1])


def kv_cache_read(cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  cu_seqlens: torch.Tensor | None = None, *, tokens: int | None = None,
                  dtype: torch.dtype = torch.bfloat16,
                  out: tuple[torch.Tensor, torch.Tensor] | None = None,
                  ) -> tuple[torch.Tensor, torch.Tensor]:
    """The last ``cu_seqlens[b + 1] - cu_seqlens[b]`` tokens of every sequence as 16-bit rows.

    Returns ``(k, v)`` of ``[tokens, kv_heads, head_dim]``; ``out`` gives the two (contiguous)
    buffers, else ``tokens`` rows of ``dtype`` are allocated (default: one per sequence).  Rows
    whose position is below zero or on no page are zero.  Every value is ``code * scale`` rounded
    once: exact in BF16.
    """
    if not isinstance(cache, PagedKVCache):
        raise TypeError("cache must be a PagedKVCache instance")
    device = cache.device
    _, heads, _, dim = cache._extents
    if out is None:
        if dtype not in _DTYPE_CODE:
            raise TypeError(f"dtype must be torch.float16 or torch.bfloat16; got {dtype}")
        if tokens is None and cu_seqlens is not None:
            raise ValueError("tokens (rows in all) is needed with cu_seqlens when out is not given")
        rows = block_table.shape[0] if tokens is None else int(tokens)
        if rows < 0:
            raise ValueError(f"tokens must not be negative; got {rows}")
        out = (torch.empty((rows, heads, dim), dtype=dtype, device=device),
               torch.empty((rows, heads, dim), dtype=dtype, device=device))
    k, v = out
    if k.ndim != 3:
        raise ValueError("out must be two [tokens, kv_heads, head_dim] tensors")
    rows = k.shape[0]
    if tokens is not None and rows != tokens:
        raise ValueError("out must have `tokens` rows")
    batch = _check_batch(cache, block_table, seq_lens, cu_seqlens, rows)
    _check_rows(k, "out[0]", heads, dim, device)
    _check_rows(v, "out[1]", heads, dim, device)
    if not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("out's tensors must be contiguous")
    if v.shape != k.shape or v.dtype is not k.dtype:
        raise ValueError("the outputs must have one shape and dtype")
    _launch(device, library().mxfp6_kv_cache_read, *cache._arguments(), *batch, k.data_ptr(), v.data_ptr(),
            _DTYPE_CODE[k.dtype])
    return k, v


def kv_cache_attention(q: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor,
                       seq_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *,
                       max_query_len: int | None = None, scale: float | None = None,
                       causal: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """Grouped-query attention of ``q`` ``[tokens, q_heads, head_dim]`` over the cache.

    Row ``i`` of sequence ``b`` stands at position ``seq_lens[b] - rows + i`` and sees the cached
    tokens up to and including its own position (``causal``) or all ``seq_lens[b]`` of them;
    query head ``h`` reads key head ``h // (q_heads // kv_heads)``.  A row that sees no token is
    zero.  ``scale`` multiplies the scores (default ``head_dim ** -0.5``).  ``max_query_len``: an
    upper bound of the rows of any sequence (default: 1 without ``cu_seqlens``, else all rows); a
    tight one picks the better kernel, and rows of a sequence that has more may be left unwritten.
    Write the rows' own keys and values first (:func:`kv_cache_write` takes the same
    ``block_table``, ``seq_lens`` and ``cu_seqlens``).  ``out`` must not overlap ``q``.  Sums are
    32-bit: keys and values up to 2^80 in magnitude overflow none of them while the scores fit 32
    bits.  A block table that names at most 1024 tokens a sequence takes a form for short ones.
    """
    if q.ndim != 3:
        raise ValueError(f"q must be [tokens, q_heads, head_dim]; got {tuple(q.shape)}")
    tokens, q_heads, dim = q.shape
    batch = _check_batch(cache, block_table, seq_lens, cu_seqlens, tokens)
    device = cache.device
    _, heads, page_size, head_dim = cache._extents
    q_strides = _check_rows(q, "q", None, head_dim, device)
    if q_heads < 1 or q_heads % heads != 0:
        raise ValueError(f"q_heads ({q_heads}) must be a multiple of the cache's {heads} heads")
    if max_query_len is None:
        max_query_len = 1 if cu_seqlens is None else max(1, tokens)
    elif max_query_len < 1:
        raise ValueError(f"max_query_len must be positive; got {max_query_len}")
    if scale is None:
        scale = dim ** -0.5
    elif not math.isfinite(scale):
        raise ValueError(f"scale must be finite; got {scale}")
    if out is None:
        out = torch.empty((tokens, q_heads, dim), dtype=q.dtype, device=device)
        out_strides = (q_heads * dim, dim)
    else:
        out_strides = _check_output_rows(out, "out", q, device)
    lib = library()
    code = _DTYPE_CODE[q.dtype]
    need = lib.mxfp6_kv_cache_attention_workspace(batch[6], tokens, max_query_len, q_heads, heads, dim,
                                                  code, batch[5] * page_size)
    # Scratch of this call alone: the allocator keeps it apart between streams and graphs.
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
    _launch(device, lib.mxfp6_kv_cache_attention, *cache._arguments(), *batch, q.data_ptr(), out.data_ptr(), code,
            q_heads, q_strides[0], q_strides[1], out_strides[0], out_strides[1], max_query_len, scale,
            1 if causal else 0, None if workspace is None else workspace.data_ptr(), need)
    return out


# --------------------------------------------------------------------------- rotary positions


@dataclass(frozen=True)
class RotaryFrequencies:
    """``inv_freq``: float64 ``[rotary_dim / 2]``, radians per position of every pair;
    ``axis``: int32 ``[rotary_dim / 2]``, the row of ``positions`` that turns it;
    ``adjacent``: pairs are ``(2i, 2i + 1)`` instead of ``(i, i + rotary_dim / 2)``;
    ``axes``: rows that ``positions`` must have, the largest ``axis`` and one, so that a call with
    fewer is refused without reading the device (:func:`rotary_frequencies` knows it; None: a pair
    whose axis has no row becomes NaN)."""

    inv_freq: torch.Tensor
    axis: torch.Tensor
    adjacent: bool = False
    axes: int | None = None

    def __post_init__(self) -> None:
        inv, axis = self.inv_freq, self.axis
        half = inv.shape[0] if inv.ndim == 1 else -1
        if half < 8 or half % 8 != 0 or half > 128:
            raise ValueError("inv_freq must be [rotary_dim / 2] with rotary_dim a multiple of 16 up to "
                             f"256; got {tuple(inv.shape)}")
        if inv.dtype != torch.float64:
            raise TypeError("inv_freq must be float64")
        if axis.dtype != torch.int32:
            raise TypeError("axis must be int32")
        if axis.shape != (half,):
            raise ValueError("axis must have the shape of inv_freq")
        if axis.device != inv.device:
            raise ValueError("axis must be on inv_freq's device")
        if not (inv.is_contiguous() and axis.is_contiguous()):
            raise ValueError("inv_freq and axis must be contiguous")
        if self.axes is not None and not 1 <= self.axes <= 8:
            raise ValueError(f"axes must be 1 to 8; got {self.axes}")

    @property
    def rotary_dim(self) -> int:
        return 2 * self.inv_freq.shape[0]


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, sections: list[int] | None = None,
                       *, interleaved: bool = False, adjacent: bool = False,
                       device: torch.device | str | int = "cuda") -> RotaryFrequencies:
    """``theta ** (-2 i / rotary_dim)`` for the ``rotary_dim / 2`` pairs of a head, with their axes.

    ``sections`` gives the number of pairs that each position axis turns (they sum to
    ``rotary_dim / 2``; default: one axis).  Chunked: the first ``sections[0]`` pairs follow axis
    0, the next ``sections[1]`` axis 1, and so on.  ``interleaved``: pair ``i`` follows axis
    ``a = i % axes`` while ``i < axes * sections[a]``, else axis 0.
    """
    _refuse(rotary_dim < 16 or rotary_dim % 16 != 0 or rotary_dim > 256,
            f"rotary_dim must be a multiple of 16 up to 256; got {rotary_dim}")
    _refuse(not theta > 0.0, f"theta must be positive; got {theta}")
    half = rotary_dim // 2
    sections = [half] if sections is None else [int(n) for n in sections]
    _refuse(not 1 <= len(sections) <= 8 or min(sections) < 0 or sum(sections) != half,
            f"sections must be 1 to 8 counts that sum to {half}; got {sections}")
    axes = len(sections)
    if interleaved:
        axis = [i % axes if i < axes * sections[i % axes] else 0 for i in range(half)]
        _refuse([axis.count(a) for a in range(axes)] != sections,
                f"sections {sections} cannot be interleaved")
    else:
        axis = [a for a, count in enumerate(sections) for _ in range(count)]
    inv = [theta ** (-i / half) for i in range(half)]
    return RotaryFrequencies(torch.tensor(inv, dtype=torch.float64, device=device),
                             torch.tensor(axis, dtype=torch.int32, device=device), adjacent,
                             max(axis) + 1)


def rotary_multi_axis(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                      frequencies: RotaryFrequencies, *, q_out: torch.Tensor | None = None,
                      k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Turn the query heads ``q`` and key heads ``k`` ``[tokens, heads, head_dim]`` by their positions.

    ``positions``: int32 or int64 ``[axes, tokens]`` (or ``[tokens]`` for one axis); pair ``i`` of
    every head turns by ``positions[axis[i], token] * inv_freq[i]`` radians, computed in 64 bits.
    ``positions`` may have more rows than ``frequencies.axes``, not fewer.  Values behind
    ``rotary_dim`` are copied.  ``q_out`` / ``k_out`` may be ``q`` / ``k`` themselves (in place);
    other overlaps are not allowed.
    """
    if not isinstance(frequencies, RotaryFrequencies):
        raise TypeError("frequencies must be a RotaryFrequencies instance")
    device = q.device
    if q.ndim != 3:
        raise ValueError(f"q must be [tokens, heads, head_dim]; got {tuple(q.shape)}")
    tokens, q_heads, dim = q.shape
    q_strides = _check_rows(q, "q", None, dim, device)
    k_strides = _check_rows(k, "k", None, dim, device)
    if k.shape[0] != tokens or k.dtype is not q.dtype:
        raise ValueError("q and k must have one token count and dtype")
    inv_freq = frequencies.inv_freq
    half = inv_freq.shape[0]
    if dim % 8 != 0 or 2 * half > dim:
        raise ValueError(f"head_dim must be a multiple of 8 and at least rotary_dim ({2 * half}); got {dim}")
    if inv_freq.device != device:
        raise ValueError("frequencies must be on q's device")
    if positions.ndim == 1:
        positions = positions.unsqueeze(0)
    wide = positions.dtype == torch.int64
    if not wide and positions.dtype != torch.int32:
        raise TypeError("positions must be int32 or int64")
    shape = positions.shape
    if len(shape) != 2 or not 1 <= shape[0] <= 8 or shape[1] != tokens or (
            tokens > 1 and positions.stride(1) != 1):
        raise ValueError(f"positions must be [axes, {tokens}] with contiguous rows, 1 to 8 axes")
    if frequencies.axes is not None and shape[0] < frequencies.axes:
        raise ValueError(f"positions must have a row for each of the frequencies' {frequencies.axes} axes; "
                         f"got {shape[0]}")
    if positions.device != device:
        raise ValueError("positions must be on q's device")
    if q_out is None:
        q_out = torch.empty((tokens, q_heads, dim), dtype=q.dtype, device=device)
    if k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=device)
    q_out_strides = _check_output_rows(q_out, "q_out", q, device)
    k_out_strides = _check_output_rows(k_out, "k_out", k, device)
    q_at, k_at, q_out_at, k_out_at = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    if tokens > 0 and ((q_at == q_out_at and q_strides != q_out_strides)
                       or (k_at == k_out_at and k_strides != k_out_strides)):
        raise ValueError("an output overlaps its input with other strides")
    _launch(device, library().mxfp6_rotary_multi_axis, q_at, q_out_at, q_heads, q_strides[0], q_strides[1],
            q_out_strides[0], q_out_strides[1], k_at, k_out_at, k.shape[1], k_strides[0], k_strides[1],
            k_out_strides[0], k_out_strides[1], _DTYPE_CODE[q.dtype], tokens, dim, positions.data_ptr(),
            positions.stride(0), shape[0], 1 if wide else 0, inv_freq.data_ptr(),
            frequencies.axis.data_ptr(), half, 1 if frequencies.adjacent else 0)
    return q_out, k_out
