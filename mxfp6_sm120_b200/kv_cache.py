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

All three live on the device and are read there, so a captured CUDA graph follows them; rows
behind ``cu_seqlens[batch]`` are left as they were.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from ._loader import check, library
from .ops import SCALE_VECTOR_SIZE, _DTYPE_CODE, _ptr, _refuse, _require_sm100

KV_HEAD_DIMS = (64, 128, 256)
KV_PAGE_SIZES = (32, 64, 128)


class _on_device:
    """``torch.cuda.device`` that costs nothing when the device is the current one already."""

    __slots__ = ("index", "guard")

    def __init__(self, device: torch.device):
        self.index, self.guard = device.index, None

    def __enter__(self) -> int:
        if torch.cuda.current_device() != self.index:
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc) -> None:
        if self.guard is not None:
            self.guard.__exit__(*exc)


_SM100_SEEN: set[int] = set()


def _require_gpu(device: torch.device) -> None:
    _refuse(device.type != "cuda", f"the tensors must be on a CUDA device; got {device}")
    if device.index not in _SM100_SEEN:
        _require_sm100(device)
        _SM100_SEEN.add(device.index)


@dataclass(frozen=True)
class PagedKVCache:
    """Keys and values of one layer in pages of 8-bit numbers.

    ``k_values`` / ``v_values``: uint8 E4M3 codes ``[pages, kv_heads, page_size, head_dim]``;
    ``k_scales`` / ``v_scales``: uint8 UE8M0 codes ``[pages, kv_heads, page_size // 32]``, one per
    32 tokens of a page and head: a value is ``code * 2**(scale - 127)``.
    """

    k_values: torch.Tensor
    v_values: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor

    def __post_init__(self) -> None:
        values, scales = self.k_values, self.k_scales
        _refuse(values.ndim != 4, f"k_values must be [pages, kv_heads, page_size, head_dim]; got "
                                  f"{tuple(values.shape)}")
        pages, heads, page, dim = values.shape
        _refuse(page not in KV_PAGE_SIZES, f"page_size must be one of {KV_PAGE_SIZES}; got {page}")
        _refuse(dim not in KV_HEAD_DIMS, f"head_dim must be one of {KV_HEAD_DIMS}; got {dim}")
        _refuse(pages < 1 or heads < 1, "the cache needs at least one page and one head")
        _refuse(self.v_values.shape != values.shape, "v_values must have the shape of k_values")
        want = (pages, heads, page // SCALE_VECTOR_SIZE)
        _refuse(scales.shape != want or self.v_scales.shape != want,
                f"k_scales and v_scales must be {list(want)}")
        for tensor in (values, self.v_values, scales, self.v_scales):
            _refuse(tensor.dtype != torch.uint8, "cache tensors must be uint8", TypeError)
            _refuse(tensor.device != values.device, "cache tensors must be on one device")
            _refuse(not tensor.is_contiguous(), "cache tensors must be contiguous")

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
    def device(self) -> torch.device:
        return self.k_values.device

    @property
    def pages(self) -> int:
        return self.k_values.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k_values.shape[1]

    @property
    def page_size(self) -> int:
        return self.k_values.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k_values.shape[3]

    def nbytes(self) -> int:
        """Bytes of the values and scales."""
        return 2 * (self.k_values.numel() + self.k_scales.numel())

    def _pointers(self) -> tuple:
        return (self.k_values.data_ptr(), self.v_values.data_ptr(), self.k_scales.data_ptr(),
                self.v_scales.data_ptr(), *self.k_values.shape)


def _check_batch(cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                 cu_seqlens: torch.Tensor | None, tokens: int) -> tuple:
    """The batch description's argument rules; returns its C arguments."""
    _refuse(not isinstance(cache, PagedKVCache), "cache must be a PagedKVCache instance", TypeError)
    device = cache.device
    _refuse(block_table.dtype != torch.int32 or seq_lens.dtype != torch.int32,
            "block_table and seq_lens must be int32", TypeError)
    _refuse(block_table.ndim != 2 or block_table.shape[1] < 1
            or (block_table.shape[1] > 1 and block_table.stride(1) != 1),
            "block_table must be [batch, width] with contiguous rows")
    batch = block_table.shape[0]
    _refuse(batch < 1, "the batch must hold at least one sequence")
    _refuse(seq_lens.shape != (batch,) or not seq_lens.is_contiguous(),
            f"seq_lens must be contiguous [{batch}]")
    _refuse(block_table.device != device or seq_lens.device != device,
            "block_table and seq_lens must be on the cache's device")
    if cu_seqlens is None:
        _refuse(tokens != batch, f"without cu_seqlens every sequence has one row; got {tokens} rows "
                                 f"for {batch} sequences")
    else:
        _refuse(cu_seqlens.dtype != torch.int32, "cu_seqlens must be int32", TypeError)
        _refuse(cu_seqlens.shape != (batch + 1,) or not cu_seqlens.is_contiguous(),
                f"cu_seqlens must be contiguous [{batch + 1}]")
        _refuse(cu_seqlens.device != device, "cu_seqlens must be on the cache's device")
    return (block_table.data_ptr(), seq_lens.data_ptr(), _ptr(cu_seqlens), block_table.stride(0),
            tokens, block_table.shape[1], batch)


def _check_rows(tensor: torch.Tensor, name: str, heads: int | None, dim: int,
                device: torch.device) -> None:
    _refuse(tensor.dtype not in _DTYPE_CODE,
            f"{name} must have dtype torch.float16 or torch.bfloat16; got {tensor.dtype}", TypeError)
    _refuse(tensor.ndim != 3 or tensor.shape[2] != dim
            or (heads is not None and tensor.shape[1] != heads),
            f"{name} must be [tokens, {'heads' if heads is None else heads}, {dim}]; got "
            f"{tuple(tensor.shape)}")
    _refuse(tensor.stride(2) != 1, f"{name}'s last dimension must be contiguous")
    _refuse(tensor.device != device, f"{name} must be on {device}; got {tensor.device}")


def _no_overlap_within(tensor: torch.Tensor, name: str) -> None:
    """Refuse outputs whose rows share memory (expanded views)."""
    tokens, heads, dim = tensor.shape
    token_stride, head_stride, _ = tensor.stride()
    bad = (heads > 1 and head_stride < dim) or (tokens > 1 and token_stride < dim)
    if not bad and tokens > 1 and heads > 1:
        inner, outer = sorted(((head_stride, heads), (token_stride, tokens)))
        bad = outer[0] < inner[0] * (inner[1] - 1) + dim
    _refuse(bad, f"{name} must not overlap itself")


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
    _refuse(k.ndim != 3, f"k must be [tokens, kv_heads, head_dim]; got {tuple(k.shape)}")
    batch = _check_batch(cache, block_table, seq_lens, cu_seqlens, k.shape[0])
    device = cache.device
    _check_rows(k, "k", cache.kv_heads, cache.head_dim, device)
    _check_rows(v, "v", cache.kv_heads, cache.head_dim, device)
    _refuse(v.shape != k.shape or v.dtype != k.dtype, "k and v must have one shape and dtype")
    _require_gpu(device)
    with _on_device(device) as stream:
        check(library().mxfp6_kv_cache_write(
            *cache._pointers(), *batch, k.data_ptr(), v.data_ptr(), _DTYPE_CODE[k.dtype],
            k.stride(0), k.stride(1), v.stride(0), v.stride(1), stream))


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
    _refuse(not isinstance(cache, PagedKVCache), "cache must be a PagedKVCache instance", TypeError)
    if out is None:
        _refuse(dtype not in _DTYPE_CODE,
                f"dtype must be torch.float16 or torch.bfloat16; got {dtype}", TypeError)
        _refuse(tokens is None and cu_seqlens is not None,
                "tokens (rows in all) is needed with cu_seqlens when out is not given")
        rows = block_table.shape[0] if tokens is None else int(tokens)
        _refuse(rows < 0, f"tokens must not be negative; got {rows}")
        shape = (rows, cache.kv_heads, cache.head_dim)
        out = (torch.empty(shape, dtype=dtype, device=cache.device),
               torch.empty(shape, dtype=dtype, device=cache.device))
    k, v = out
    _refuse(k.ndim != 3, "out must be two [tokens, kv_heads, head_dim] tensors")
    _refuse(tokens is not None and k.shape[0] != tokens, "out must have `tokens` rows")
    batch = _check_batch(cache, block_table, seq_lens, cu_seqlens, k.shape[0])
    for tensor, name in ((k, "out[0]"), (v, "out[1]")):
        _check_rows(tensor, name, cache.kv_heads, cache.head_dim, cache.device)
        _refuse(not tensor.is_contiguous(), f"{name} must be contiguous")
    _refuse(v.shape != k.shape or v.dtype != k.dtype, "the outputs must have one shape and dtype")
    _require_gpu(cache.device)
    with _on_device(cache.device) as stream:
        check(library().mxfp6_kv_cache_read(
            *cache._pointers(), *batch, k.data_ptr(), v.data_ptr(), _DTYPE_CODE[k.dtype], stream))
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
    tight one picks the better kernel.  Write the rows' own keys and values first
    (:func:`kv_cache_write` takes the same ``block_table``, ``seq_lens`` and ``cu_seqlens``).
    """
    _refuse(q.ndim != 3, f"q must be [tokens, q_heads, head_dim]; got {tuple(q.shape)}")
    tokens, q_heads, dim = q.shape
    batch = _check_batch(cache, block_table, seq_lens, cu_seqlens, tokens)
    _check_rows(q, "q", None, cache.head_dim, cache.device)
    _refuse(q_heads < 1 or q_heads % cache.kv_heads != 0,
            f"q_heads ({q_heads}) must be a multiple of the cache's {cache.kv_heads} heads")
    if max_query_len is None:
        max_query_len = 1 if cu_seqlens is None else max(1, tokens)
    _refuse(max_query_len < 1, f"max_query_len must be positive; got {max_query_len}")
    scale = dim ** -0.5 if scale is None else float(scale)
    _refuse(not math.isfinite(scale), f"scale must be finite; got {scale}")
    if out is None:
        out = torch.empty((tokens, q_heads, dim), dtype=q.dtype, device=q.device)
    else:
        _check_rows(out, "out", q_heads, dim, cache.device)
        _refuse(out.shape != q.shape or out.dtype != q.dtype, "out must match q's shape and dtype")
        _no_overlap_within(out, "out")
    _require_gpu(cache.device)
    with _on_device(cache.device) as stream:
        lib = library()
        need = lib.mxfp6_kv_cache_attention_workspace(
            batch[-1], tokens, max_query_len, q_heads, cache.kv_heads, dim, _DTYPE_CODE[q.dtype],
            batch[-2] * cache.page_size)
        # Scratch of this call alone: the allocator keeps it apart between streams and graphs.
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        check(lib.mxfp6_kv_cache_attention(
            *cache._pointers(), *batch, q.data_ptr(), out.data_ptr(), _DTYPE_CODE[q.dtype], q_heads,
            q.stride(0), q.stride(1), out.stride(0), out.stride(1), max_query_len, scale,
            1 if causal else 0, _ptr(workspace), need, stream))
    return out


# --------------------------------------------------------------------------- rotary positions


@dataclass(frozen=True)
class RotaryFrequencies:
    """``inv_freq``: float64 ``[rotary_dim / 2]``, radians per position of every pair;
    ``axis``: int32 ``[rotary_dim / 2]``, the row of ``positions`` that turns it;
    ``adjacent``: pairs are ``(2i, 2i + 1)`` instead of ``(i, i + rotary_dim / 2)``."""

    inv_freq: torch.Tensor
    axis: torch.Tensor
    adjacent: bool = False

    def __post_init__(self) -> None:
        half = self.inv_freq.shape[0] if self.inv_freq.ndim == 1 else -1
        _refuse(half < 8 or half % 8 != 0 or half > 128,
                "inv_freq must be [rotary_dim / 2] with rotary_dim a multiple of 16 up to 256; got "
                f"{tuple(self.inv_freq.shape)}")
        _refuse(self.inv_freq.dtype != torch.float64, "inv_freq must be float64", TypeError)
        _refuse(self.axis.dtype != torch.int32, "axis must be int32", TypeError)
        _refuse(self.axis.shape != (half,), "axis must have the shape of inv_freq")
        _refuse(self.axis.device != self.inv_freq.device, "axis must be on inv_freq's device")
        _refuse(not (self.inv_freq.is_contiguous() and self.axis.is_contiguous()),
                "inv_freq and axis must be contiguous")

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
                             torch.tensor(axis, dtype=torch.int32, device=device), adjacent)


def rotary_multi_axis(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                      frequencies: RotaryFrequencies, *, q_out: torch.Tensor | None = None,
                      k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Turn the query heads ``q`` and key heads ``k`` ``[tokens, heads, head_dim]`` by their positions.

    ``positions``: int32 or int64 ``[axes, tokens]`` (or ``[tokens]`` for one axis); pair ``i`` of
    every head turns by ``positions[axis[i], token] * inv_freq[i]`` radians, computed in 64 bits.
    Values behind ``rotary_dim`` are copied.  ``q_out`` / ``k_out`` may be ``q`` / ``k``
    themselves (in place); other overlaps are not allowed.
    """
    _refuse(not isinstance(frequencies, RotaryFrequencies),
            "frequencies must be a RotaryFrequencies instance", TypeError)
    device = q.device
    _refuse(q.ndim != 3, f"q must be [tokens, heads, head_dim]; got {tuple(q.shape)}")
    tokens, _, dim = q.shape
    _check_rows(q, "q", None, dim, device)
    _check_rows(k, "k", None, dim, device)
    _refuse(k.shape[0] != tokens or k.dtype != q.dtype, "q and k must have one token count and dtype")
    rotary_dim = frequencies.rotary_dim
    _refuse(dim % 8 != 0 or rotary_dim > dim,
            f"head_dim must be a multiple of 8 and at least rotary_dim ({rotary_dim}); got {dim}")
    _refuse(frequencies.inv_freq.device != device, "frequencies must be on q's device")
    if positions.ndim == 1:
        positions = positions.unsqueeze(0)
    _refuse(positions.dtype not in (torch.int32, torch.int64), "positions must be int32 or int64",
            TypeError)
    _refuse(positions.ndim != 2 or not 1 <= positions.shape[0] <= 8 or positions.shape[1] != tokens
            or (tokens > 1 and positions.stride(1) != 1),
            f"positions must be [axes, {tokens}] with contiguous rows, 1 to 8 axes")
    _refuse(positions.device != device, "positions must be on q's device")
    outs = []
    for x, y, name in ((q, q_out, "q_out"), (k, k_out, "k_out")):
        if y is None:
            y = torch.empty(x.shape, dtype=x.dtype, device=device)
        elif y is not x:
            _check_rows(y, name, x.shape[1], dim, device)
            _refuse(y.shape != x.shape or y.dtype != x.dtype,
                    f"{name} must match its input's shape and dtype")
        _no_overlap_within(y, name)
        _refuse(tokens > 0 and y.data_ptr() == x.data_ptr() and y.stride() != x.stride(),
                f"{name} overlaps its input with other strides")
        outs.append(y)
    q_out, k_out = outs
    _require_gpu(device)
    with _on_device(device) as stream:
        check(library().mxfp6_rotary_multi_axis(
            q.data_ptr(), q_out.data_ptr(), q.shape[1], q.stride(0), q.stride(1), q_out.stride(0),
            q_out.stride(1), k.data_ptr(), k_out.data_ptr(), k.shape[1], k.stride(0), k.stride(1),
            k_out.stride(0), k_out.stride(1), _DTYPE_CODE[q.dtype], tokens, dim,
            positions.data_ptr(), positions.stride(0), positions.shape[0],
            1 if positions.dtype == torch.int64 else 0, frequencies.inv_freq.data_ptr(),
            frequencies.axis.data_ptr(), rotary_dim // 2, 1 if frequencies.adjacent else 0, stream))
    return q_out, k_out
