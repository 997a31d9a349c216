"""GPU tests of the paged KV cache operators against their definitions in 64 bits."""

from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

from oracle import kv_oracle as kvo

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DTYPES = [torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Batch:
    """A random paged cache with ragged sequences; every byte that no token owns is arbitrary
    (NaN codes among them), and so are the table entries behind a sequence's last page."""

    def __init__(self, mx, seed, lens, news, heads=2, page=32, dim=64, spread=3, spare=2, finite=False):
        rng = random.Random(seed)
        self.lens, self.news, self.page = list(lens), list(news), page
        self.heads, self.dim = heads, dim
        counts = [-(-max(n, 0) // page) for n in lens]
        self.pages = sum(counts) + spare
        self.width = max(max(counts), 1) + 1
        order = list(range(self.pages))
        rng.shuffle(order)
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for b, count in enumerate(counts):
            self.table[b, :count] = order[at : at + count]
            for j in range(count, self.width):
                self.table[b, j] = rng.choice([-1, self.pages, 2**31 - 1, -(2**31)])
            at += count
        g = _gen(seed)
        shape = (self.pages, heads, page, dim)
        self.values = []
        for _ in range(2):
            v = (torch.randn(shape, generator=g) * 112).clamp(-448, 448).to(torch.float8_e4m3fn)
            self.values.append(v.view(torch.uint8).numpy().copy())
        self.scales = [torch.randint(127 - spread - 6, 127 - 6 + 1, (self.pages, heads, page // 32),
                                     generator=g, dtype=torch.uint8).numpy() for _ in range(2)]
        if not finite:
            owned = np.zeros((self.pages, page), bool)
            for b, n in enumerate(lens):
                for p in range(max(n, 0)):
                    owned[self.table[b, p // page], p % page] = True
            for v in self.values:
                junk = torch.randint(0, 256, v.shape, generator=g, dtype=torch.uint8).numpy()
                junk[:, :, ::3] = 0x7F
                keep = np.broadcast_to(owned[:, None, :, None], v.shape)
                np.copyto(v, np.where(keep, v, junk))
            blocks = owned.reshape(self.pages, page // 32, 32).any(-1)
            for s in self.scales:
                np.copyto(s, np.where(blocks[:, None, :], s, 255))
        self.cu = [0]
        for n in news:
            self.cu.append(self.cu[-1] + n)
        self.tokens = self.cu[-1]
        k, v = (torch.from_numpy(x).to(DEV) for x in self.values)
        ks, vs = (torch.from_numpy(x.copy()).to(DEV) for x in self.scales)
        self.cache = mx.PagedKVCache(k, v, ks, vs)
        self.dev = (torch.from_numpy(self.table).to(DEV), _i32(self.lens), _i32(self.cu))

    def oracle_attention(self, q, scale, causal):
        return kvo.attention(kvo.to_numpy(q), *self.values, *self.scales, self.table, self.lens, self.cu,
                             scale, causal)

    def weight_of(self, q, scale, causal):
        """sum_j p_j |v_j| / sum_j p_j: what a relative error of the weights is multiplied by."""
        mags = [v & 127 for v in self.values]
        return kvo.attention(kvo.to_numpy(q), self.values[0], mags[1], *self.scales, self.table, self.lens,
                             self.cu, scale, causal)


# ------------------------------------------------------------------------------ write


def _same_cache(batch, want_values, want_scales):
    got = [batch.cache.k_values, batch.cache.v_values]
    for g, w in zip(got, want_values):
        g = kvo.VALUES[g.cpu().numpy()]
        assert np.array_equal(g, kvo.VALUES[w], equal_nan=True)
    for g, w in zip([batch.cache.k_scales, batch.cache.v_scales], want_scales):
        assert np.array_equal(g.cpu().numpy(), w)


def _write_and_check(mx, batch, k, v, cu=True):
    values = [x.copy() for x in batch.values]
    scales = [x.copy() for x in batch.scales]
    for x, val, sc in zip((k, v), values, scales):
        kvo.write(val, sc, kvo.to_numpy(x), batch.table, batch.lens, batch.cu, batch.pages, batch.page)
    table, lens, dcu = batch.dev
    mx.kv_cache_write(batch.cache, k, v, table, lens, dcu if cu else None)
    _same_cache(batch, values, scales)
    batch.values, batch.scales = values, scales


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,dim,heads", [(32, 64, 1), (64, 128, 3), (128, 256, 2)])
def test_write_matches_definition(mx, dtype, page, dim, heads):
    lens = [1, 31, 32, 33, 64, 100, 7, 0, 260]
    news = [1, 31, 32, 2, 1, 100, 0, 0, 129]
    batch = Batch(mx, 11, lens, news, heads, page, dim)
    kv = torch.randn((batch.tokens, 2 * heads * dim), generator=_gen(5)) * 3
    kv[:, ::7] *= 20
    kv = kv.to(dtype).to(DEV)
    k = kv[:, : heads * dim].view(batch.tokens, heads, dim)      # strided rows
    v = kv[:, heads * dim :].view(batch.tokens, heads, dim)
    _write_and_check(mx, batch, k, v)
    # a second write of the same rows changes nothing
    before = [t.clone() for t in (batch.cache.k_values, batch.cache.v_values)]
    mx.kv_cache_write(batch.cache, k, v, *batch.dev)
    assert torch.equal(batch.cache.k_values, before[0]) and torch.equal(batch.cache.v_values, before[1])


def test_append_token_by_token_raises_the_scale_and_rerounds(mx):
    """Magnitudes that grow, shrink and jump within a block: the kept codes follow the scale."""
    heads, dim, page = 2, 64, 32
    factors = [1.0, 0.01, 3.0, 0.5, 40.0, 39.0, 1e4, 1e-6, 2e4] + [1.0] * 30 + [5.0, 700.0]
    batch = Batch(mx, 3, [len(factors)], [0], heads, page, dim)
    gen = _gen(8)
    for i, factor in enumerate(factors):
        batch.lens, batch.cu, batch.tokens = [i + 1], [0, 1], 1
        batch.dev = (batch.dev[0], _i32(batch.lens), _i32(batch.cu))
        k = (torch.randn((1, heads, dim), generator=gen) * factor).to(torch.bfloat16).to(DEV)
        v = (torch.randn((1, heads, dim), generator=gen) / factor).to(torch.bfloat16).to(DEV)
        _write_and_check(mx, batch, k, v, cu=i % 2 == 0)


def test_write_of_unaligned_strides_nan_and_infinities(mx):
    heads, dim = 3, 64
    batch = Batch(mx, 4, [40, 5], [40, 3], heads, 32, dim)
    raw = torch.randn((batch.tokens, heads * (dim + 1) + 3), generator=_gen(1)).to(torch.float16).to(DEV)
    k = raw[:, 1 : 1 + heads * (dim + 1)].view(batch.tokens, heads, dim + 1)[..., :dim]
    v = torch.randn((heads, batch.tokens, dim), generator=_gen(2)).to(torch.float16).to(DEV).transpose(0, 1)
    k[3, 1, 5], k[3, 1, 6], k[33, 2, 0] = math.nan, math.inf, -math.inf
    k[7] = 0
    v[:32, 2] = 0                      # a block of zeros takes the smallest scale
    v[41] = 65504.0                    # largest FP16
    v[42] = 2.0 ** -24                 # smallest FP16
    _write_and_check(mx, batch, k, v)


def test_write_ignores_what_has_no_place(mx):
    """Positions below zero, pages that the table does not name, rows behind the last sequence,
    lengths beyond the table."""
    batch = Batch(mx, 6, [3, 70, 50], [5, 10, 4], 2, 32, 64, finite=True)
    batch.table[1, 2] = -1                      # tokens 64..69 have no page
    batch.lens[2] = batch.width * 32 + 2        # the table ends inside the new rows
    batch.table[2, :] = -1
    free = [p for p in range(batch.pages) if p not in batch.table[:2]]
    batch.table[2, batch.width - 1] = free[0]
    batch.dev = (torch.from_numpy(batch.table).to(DEV), _i32(batch.lens), _i32(batch.cu))
    rows = torch.randn((batch.tokens + 7, 2, 64), generator=_gen(1)).to(torch.bfloat16).to(DEV)
    _write_and_check(mx, batch, rows, rows * 2)
    # rows that cu_seqlens does not reach, and offsets that make no sense, stay in bounds
    for cu in ([0, 0, 0, 0], [5, 3, 9, 2], [-4, -1, 10 ** 6, 2 ** 31 - 1]):
        other = Batch(mx, 6, [3, 70, 50], [5, 10, 4], 2, 32, 64)
        mx.kv_cache_write(other.cache, rows, rows, other.dev[0], other.dev[1], _i32(cu))
        torch.cuda.synchronize()


# ------------------------------------------------------------------------------- read


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,dim,heads", [(32, 64, 1), (64, 128, 3), (128, 256, 2)])
def test_read_matches_definition(mx, dtype, page, dim, heads):
    lens = [1, 31, 64, 0, 200, 130]
    news = [1, 31, 10, 0, 200, 1]
    batch = Batch(mx, 21, lens, news, heads, page, dim)
    where = [(b, n - new + i) for b, (n, new) in enumerate(zip(lens, news)) for i in range(new)]
    table, dlens, cu = batch.dev
    pad = 5
    out = [torch.full((batch.tokens + pad, heads, dim), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    got = mx.kv_cache_read(batch.cache, table, dlens, cu, out=tuple(out))
    fresh = mx.kv_cache_read(batch.cache, table, dlens, cu, tokens=batch.tokens, dtype=dtype)
    for g, f, val, sc in zip(got, fresh, batch.values, batch.scales):
        want = torch.from_numpy(kvo.read(val, sc, batch.table, where)).to(dtype)
        assert torch.equal(g[: batch.tokens].cpu(), want)
        assert torch.equal(f.cpu(), want)
        assert bool((g[batch.tokens :] == 7.0).all())   # rows behind the last sequence


def test_read_of_missing_pages_and_negative_positions_is_zero(mx):
    batch = Batch(mx, 22, [3, 40], [6, 40], 2, 32, 64)
    batch.table[1, 0] = batch.pages
    got = mx.kv_cache_read(batch.cache, torch.from_numpy(batch.table).to(DEV), *batch.dev[1:],
                           tokens=batch.tokens)
    where = [(0, p) for p in range(-3, 3)] + [(1, p) for p in range(40)]
    for g, val, sc in zip(got, batch.values, batch.scales):
        want = kvo.read(val, sc, batch.table, where)
        assert np.array_equal(kvo.to_numpy(g), want)
    assert bool((got[0][:3] == 0).all()) and bool((got[0][6:38] == 0).all())
    one = mx.kv_cache_read(batch.cache, batch.dev[0], batch.dev[1])    # the newest token of each
    assert one[0].shape == (2, 2, 64)


def test_write_then_read_stays_within_half_a_step(mx):
    """A round trip is off by at most half an E4M3 step at the block's scale: 2^-4 of the value,
    or half the smallest step (2^-10) times the scale for values in the subnormal range."""
    batch = Batch(mx, 23, [300], [300], 2, 64, 128)
    k = (torch.randn((300, 2, 128), generator=_gen(2)) * 5).to(torch.bfloat16).to(DEV)
    v = torch.randn((300, 2, 128), generator=_gen(3)).to(torch.bfloat16).to(DEV)
    mx.kv_cache_write(batch.cache, k, v, *batch.dev)
    got = mx.kv_cache_read(batch.cache, *batch.dev, tokens=300)
    for x, y in zip((k, v), got):
        x, y = kvo.to_numpy(x), kvo.to_numpy(y)
        for lo in range(0, 300, 32):
            for h in range(2):
                a, b = x[lo : lo + 32, h], y[lo : lo + 32, h]
                scale = 2.0 ** (kvo.needed_scale(np.abs(a).max()) - 127)
                assert np.all(np.abs(a - b) <= np.maximum(np.abs(a) * 2.0 ** -4, scale * 2.0 ** -10))


# -------------------------------------------------------------------------- attention


def _delta(dtype):
    """Relative error allowed to the weights.  They are held as E4M3 terms whose sum is off by at
    most 2^-9 (two terms, BF16) or 2^-14 (three, FP16); the same again covers the 32-bit scores
    (|score| < 40: 40 * 2^-24 * 24 sums) and exponentials, and for FP16 the weights pass through
    FP16 (2^-12)."""
    return 2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -11


def _check_attention(batch, q, got, scale, causal):
    want = batch.oracle_attention(q, scale, causal)
    weight = batch.weight_of(q, scale, causal)
    half = torch.finfo(q.dtype).eps / 2
    limit = half * np.abs(want) + _delta(q.dtype) * weight + 1e-7
    off = np.abs(kvo.to_numpy(got) - want)
    assert np.isfinite(off).all()
    worst = float((off - limit).max())
    assert worst <= 0, f"off by {worst} more than the rounding allows"


def _attend(mx, batch, q, **kwargs):
    return mx.kv_cache_attention(q, batch.cache, *batch.dev, **kwargs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,dim,heads,group", [
    (32, 64, 1, 1), (64, 64, 2, 8), (32, 128, 3, 4), (128, 128, 1, 7), (64, 256, 2, 6), (32, 256, 1, 16)])
def test_decode_matches_definition(mx, dtype, page, dim, heads, group):
    lens = [1, 2, 31, 32, 33, 127, 128, 129, 500, 0, 257]
    batch = Batch(mx, 31, lens, [1] * len(lens), heads, page, dim)
    wide = (torch.randn((len(lens), (heads * group + 2) * dim), generator=_gen(7)) * 2).to(dtype).to(DEV)
    q = wide[:, : heads * group * dim].view(len(lens), heads * group, dim)
    table, dlens, _ = batch.dev
    got = mx.kv_cache_attention(q, batch.cache, table, dlens)
    _check_attention(batch, q, got, dim ** -0.5, True)
    assert bool((got[9] == 0).all())                       # nothing cached: zeros
    again = mx.kv_cache_attention(q, batch.cache, table, dlens)
    assert torch.equal(got, again)                          # the same bits every time


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("page,dim,heads,group", [(32, 64, 2, 3), (64, 128, 1, 4), (128, 256, 1, 6)])
def test_several_rows_per_sequence(mx, dtype, causal, page, dim, heads, group):
    """Drafted tokens: a few rows a sequence, one sequence without rows, one with more rows than
    tokens (its first rows see nothing)."""
    lens = [5, 130, 64, 2, 300, 33]
    news = [5, 3, 0, 4, 5, 1]
    batch = Batch(mx, 32, lens, news, heads, page, dim)
    q = (torch.randn((batch.tokens, heads * group, dim), generator=_gen(9)) * 2).to(dtype).to(DEV)
    got = _attend(mx, batch, q, max_query_len=5, causal=causal)
    _check_attention(batch, q, got, dim ** -0.5, causal)
    if causal:
        assert bool((got[8:10] == 0).all())
    loose = _attend(mx, batch, q, causal=causal)           # a loose bound may take another kernel
    _check_attention(batch, q, loose, dim ** -0.5, causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("page,dim,heads,group", [(32, 64, 1, 2), (64, 128, 2, 3), (128, 256, 1, 5)])
def test_prompt_chunks(mx, dtype, causal, page, dim, heads, group):
    lens = [200, 131, 70, 1, 290]
    news = [200, 100, 1, 1, 40]
    batch = Batch(mx, 33, lens, news, heads, page, dim)
    q = (torch.randn((batch.tokens, heads * group, dim), generator=_gen(10)) * 2).to(dtype).to(DEV)
    got = _attend(mx, batch, q, max_query_len=200, causal=causal)
    _check_attention(batch, q, got, dim ** -0.5, causal)


@pytest.mark.parametrize("rows", [1, 3, 90])
def test_rows_behind_the_last_sequence_stay(mx, rows):
    batch = Batch(mx, 34, [100, 90], [rows, rows], 2, 32, 128)
    q = torch.randn((2 * rows + 9, 8, 128), generator=_gen(1)).to(torch.bfloat16).to(DEV)
    out = torch.full_like(q, 5.0)
    got = mx.kv_cache_attention(q, batch.cache, *batch.dev, max_query_len=rows, out=out)
    assert got.data_ptr() == out.data_ptr() and bool((out[2 * rows :] == 5.0).all())
    batch.tokens = 2 * rows
    _check_attention(batch, q[: 2 * rows], got[: 2 * rows], 128 ** -0.5, True)


@pytest.mark.parametrize("rows", [1, 40])
def test_missing_pages_are_not_seen(mx, rows):
    batch = Batch(mx, 35, [200, 64], [rows, rows], 2, 32, 64)
    batch.table[0, 2] = -1
    batch.table[1, :] = batch.pages + 5
    batch.dev = (torch.from_numpy(batch.table).to(DEV), *batch.dev[1:])
    q = torch.randn((2 * rows, 4, 64), generator=_gen(1)).to(torch.bfloat16).to(DEV)
    got = _attend(mx, batch, q, max_query_len=rows)
    _check_attention(batch, q, got, 64 ** -0.5, True)
    assert bool((got[rows:] == 0).all())


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_scale_and_output_views(mx, rows, dtype):
    """Head-major q, odd row strides, an output that is a slice of wider rows, another scale."""
    batch = Batch(mx, 36, [150, 80], [rows, rows], 2, 64, 128)
    heads = 6
    odd = torch.randn((2 * rows, heads * 129 + 1), generator=_gen(3)).to(dtype).to(DEV)
    q = odd[:, 1:].view(2 * rows, heads, 129)[..., :128]
    wide = torch.zeros((2 * rows, heads + 1, 128), dtype=dtype, device=DEV)
    got = _attend(mx, batch, q, max_query_len=rows, scale=0.31, out=wide[:, 1:])
    _check_attention(batch, q, got, 0.31, True)
    assert bool((wide[:, 0] == 0).all())
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd_out = torch.zeros((2 * rows, heads * 131), dtype=dtype, device=DEV)
    odd_out = odd_out.view(2 * rows, heads, 131)[..., 1:129]
    other = _attend(mx, batch, swapped, max_query_len=rows, scale=0.31, out=odd_out)
    assert torch.equal(other, got)


@pytest.mark.parametrize("rows", [1, 60])
def test_nan_and_infinity_reach_only_their_rows(mx, rows):
    """A NaN key poisons the rows that see it (in its head), a NaN value its column; an infinite
    query its own row."""
    n = 170
    batch = Batch(mx, 37, [n, n], [rows, rows], 2, 32, 64)
    where = (int(batch.table[0, 40 // 32]), 1, 40 % 32)
    batch.cache.k_values[where][3] = 0x7F
    spot = (int(batch.table[1, 10 // 32]), 0, 10 % 32)
    batch.cache.v_values[spot][5] = 0xFF
    q = torch.randn((2 * rows, 4, 64), generator=_gen(4)).to(torch.bfloat16).to(DEV)
    q[2 * rows - 1, 3, 0] = math.inf
    got = _attend(mx, batch, q, max_query_len=rows, causal=False).float().cpu()
    assert bool(got[:rows, 2:].isnan().all()) and bool(got[:rows, :2].isfinite().all())
    assert bool(got[rows:, :2, 5].isnan().all())
    rest = torch.cat([got[rows:, :2, :5], got[rows:, :2, 6:]], -1)
    assert bool(rest.isfinite().all()) and bool(got[rows : 2 * rows - 1, 2:].isfinite().all())
    assert not bool(got[2 * rows - 1, 3].isfinite().any()) and bool(got[2 * rows - 1, 2].isfinite().all())


@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_scores_and_scales(mx, rows, dtype):
    """Scores of hundreds (one token takes all the weight), blocks whose scales are far apart, and
    rising maxima along the sequence."""
    batch = Batch(mx, 38, [260, 260], [rows, rows], 1, 32, 64, spread=0)
    ks, vs = batch.scales
    for b, shift in enumerate((0, 5)):
        for j in range(-(-260 // 32)):
            page = batch.table[b, j]
            ks[page] = 121 + (j % 4) - shift
            vs[page] = 127 - 5 * j
    batch.cache.k_scales.copy_(torch.from_numpy(ks))
    batch.cache.v_scales.copy_(torch.from_numpy(vs))
    q = torch.randn((2 * rows, 2, 64), generator=_gen(5)).to(dtype).to(DEV)
    # |scores| stay below 40 (see the tolerance); the softmax is dominated by a few tokens
    scale = 30.0 / float(np.abs(kvo.read(batch.values[0], ks, batch.table, [(0, p) for p in range(260)])).max() * 8 * 8)
    got = _attend(mx, batch, q, max_query_len=rows, scale=scale)
    _check_attention(batch, q, got, scale, True)


def test_one_token_returns_its_value(mx):
    """A single visible token has weight one: the output is its value, rounded once."""
    for dim in (64, 128, 256):
        for dtype in DTYPES:
            batch = Batch(mx, 39, [1], [1], 2, 32, dim)
            q = torch.randn((1, 4, dim), generator=_gen(5)).to(dtype).to(DEV)
            got = mx.kv_cache_attention(q, batch.cache, batch.dev[0], batch.dev[1])
            want = kvo.read(batch.values[1], batch.scales[1], batch.table, [(0, 0)])
            want = torch.from_numpy(want).repeat_interleave(2, dim=1).to(dtype)
            assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("case", ["decode", "chunk"])
def test_graph_replay_follows_the_device_metadata(mx, case):
    """One captured call serves other lengths and page tables; two graphs of one pool replayed on
    two streams do not share scratch."""
    rows = 1 if case == "decode" else 48
    batch = Batch(mx, 40, [400, 300, 500], [rows] * 3, 2, 64, 128)
    q = torch.randn((3 * rows, 8, 128), generator=_gen(5)).to(torch.bfloat16).to(DEV)
    q2 = torch.randn((3 * rows, 8, 128), generator=_gen(6)).to(torch.bfloat16).to(DEV)
    table, lens, cu = (t.clone() for t in batch.dev)
    cu_arg = None if case == "decode" else cu
    call = lambda x: mx.kv_cache_attention(x, batch.cache, table, lens, cu_arg, max_query_len=rows)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for stream, x in zip(side, (q, q2)):
        with torch.cuda.stream(stream):
            call(x)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(call(x))
            graphs.append(graph)
    torch.cuda.synchronize()
    for new_lens in ([400, 300, 500], [rows, 77 + rows, 500], [129, 128, 127]):
        batch.lens = new_lens
        lens.copy_(_i32(new_lens))
        want = [call(q), call(q2)]
        torch.cuda.synchronize()
        for _ in range(3):
            for stream, graph in zip(side, graphs):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        _check_attention(batch, q, outs[0], 128 ** -0.5, True)


def test_calls_on_two_streams_at_once(mx):
    batch = Batch(mx, 41, [700, 900], [1, 1], 2, 64, 256)
    qs = [torch.randn((2, 12, 256), generator=_gen(i)).to(torch.bfloat16).to(DEV) for i in range(2)]
    want = [mx.kv_cache_attention(q, batch.cache, *batch.dev[:2]) for q in qs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(mx.kv_cache_attention(qs[i], batch.cache, *batch.dev[:2]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_long_context_and_long_cache(mx):
    """A context of many tiles against 64-bit torch on the GPU, and pages whose byte offsets pass
    2^32."""
    dim, heads, page = 128, 1, 128
    pages = (1 << 32) // (heads * page * dim) + 600
    g = torch.Generator(device=DEV).manual_seed(1)
    k = torch.zeros((pages, heads, page, dim), dtype=torch.uint8, device=DEV)
    v = torch.zeros_like(k)
    n = 500 * page - 37
    table = torch.arange(pages - 500, pages, dtype=torch.int32, device=DEV).flip(0).view(1, -1).contiguous()
    codes = (torch.randn((2, 500, heads, page, dim), device=DEV, generator=g) * 100).clamp(-448, 448)
    codes = codes.to(torch.float8_e4m3fn).view(torch.uint8)
    k[pages - 500 :], v[pages - 500 :] = codes[0], codes[1]
    ones = torch.full((pages, heads, page // 32), 121, dtype=torch.uint8, device=DEV)
    cache = mx.PagedKVCache(k, v, ones, ones.clone())
    for rows in (1, 100):
        q = (torch.randn((rows, 4, dim), device=DEV, generator=g) * 2).to(torch.bfloat16)
        cu = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
        got = mx.kv_cache_attention(q, cache, table, _i32([n]), cu, max_query_len=rows)
        keys = k[table[0].long()].view(torch.float8_e4m3fn).double().view(-1, dim)[:n] * 2.0 ** -6
        vals = v[table[0].long()].view(torch.float8_e4m3fn).double().view(-1, dim)[:n] * 2.0 ** -6
        s = torch.einsum("thd,nd->thn", q.double(), keys) * dim ** -0.5
        last = torch.arange(n - rows, n, device=DEV)
        s.masked_fill_(torch.arange(n, device=DEV)[None, None] > last[:, None, None], -math.inf)
        p = torch.softmax(s, -1)
        want, weight = p @ vals, p @ vals.abs()
        off = (got.double() - want).abs() - (2.0 ** -9 * want.abs() + 2.0 ** -8 * weight)
        assert float(off.max()) <= 0
    row = torch.randn((1, heads, dim), device=DEV, generator=g).to(torch.bfloat16)
    mx.kv_cache_write(cache, row, row, table, _i32([n]))
    back = mx.kv_cache_read(cache, table, _i32([n]))
    assert float((back[0] - row).abs().max()) <= float(row.abs().max()) * 2.0 ** -4


# ----------------------------------------------------------------------------- rotary


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,q_heads,k_heads,dim,rotary_dim,sections,interleaved,adjacent", [
    (1, 1, 1, 64, 64, [32], False, False),
    (5, 24, 4, 256, 64, [12, 10, 10], True, False),
    (33, 8, 2, 128, 128, [32, 16, 16], False, False),
    (300, 3, 1, 96, 32, [8, 4, 4], False, True),
    (2, 40, 8, 256, 256, [32, 32, 32, 32], True, True),
])
def test_rotary_matches_definition(mx, dtype, tokens, q_heads, k_heads, dim, rotary_dim, sections,
                                   interleaved, adjacent):
    """Off by the final rounding (half a step) and the 32-bit rotation: |x| * 2^-20 covers sine
    and cosine (2^-22 each) and two products."""
    f = mx.rotary_frequencies(rotary_dim, 1.0e6, sections, interleaved=interleaved, adjacent=adjacent,
                              device=DEV)
    wide = torch.randn((tokens, (q_heads + k_heads) * dim), generator=_gen(tokens)).to(dtype).to(DEV)
    q = wide[:, : q_heads * dim].view(tokens, q_heads, dim)
    k = wide[:, q_heads * dim :].view(tokens, k_heads, dim)
    far = torch.randint(-5, 1 << 20, (len(sections), tokens), generator=_gen(2))
    for positions in (far.to(DEV), far.to(torch.int32).to(DEV)):
        got = mx.rotary_multi_axis(q, k, positions, f)
        for x, y in zip((q, k), got):
            want = kvo.rotary(kvo.to_numpy(x), far.numpy(), f.inv_freq.cpu().numpy(), f.axis.cpu().numpy(),
                              adjacent)
            off = np.abs(kvo.to_numpy(y) - want)
            half = rotary_dim // 2
            xs = np.abs(kvo.to_numpy(x))
            size = xs.max(-1, keepdims=True)
            limit = np.abs(want) * torch.finfo(dtype).eps / 2 + size * 2.0 ** -20
            if dtype is torch.float16:
                limit = limit + 2.0 ** -25                 # half the smallest FP16 step
            assert np.all(off <= limit), float((off - limit).max())
            assert torch.equal(y[..., 2 * half :], x[..., 2 * half :])
    keep = wide.clone()
    mx.rotary_multi_axis(q, k, far.to(DEV), f, q_out=q, k_out=k)           # in place
    assert torch.equal(q, got[0]) and torch.equal(k, got[1])
    wide.copy_(keep)
    if len(sections) == 1:
        flat = mx.rotary_multi_axis(q, k, far[0].to(DEV), f)
        assert torch.equal(flat[0], got[0])


def test_rotary_of_odd_strides_and_no_tokens(mx):
    f = mx.rotary_frequencies(32, 1.0e4, device=DEV)
    odd = torch.randn((7, 3 * 65 + 1), generator=_gen(1)).to(torch.bfloat16).to(DEV)
    q = odd[:, 1:].view(7, 3, 65)[..., :64]
    k = q[:, :1]
    pos = torch.arange(7, device=DEV)
    got = mx.rotary_multi_axis(q, k, pos, f)
    want = mx.rotary_multi_axis(q.contiguous(), k.contiguous(), pos, f)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    empty = mx.rotary_multi_axis(q[:0], k[:0], pos[:0], f)
    assert empty[0].shape == (0, 3, 64)
    back = mx.rotary_multi_axis(*want, -pos, f)            # turning back restores the rows
    assert float((back[0].float() - q.float()).abs().max()) <= 2.0 ** -7 * float(q.abs().max()) * 2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [4, 150])
def test_nan_behind_a_row_does_not_reach_it(mx, rows, dim, dtype):
    """Causal: a NaN value reaches the rows at and behind its token, in its head and column, and a
    NaN key the rows at and behind it; the rows before stay as they were without them."""
    n = 300
    batch = Batch(mx, 42, [n, n], [rows, rows], 2, 64, dim, finite=True)
    q = torch.randn((2 * rows, 4, dim), generator=_gen(4)).to(dtype).to(DEV)
    clean = _attend(mx, batch, q, max_query_len=rows)
    def spot(b, position):
        return int(batch.table[b, position // 64]), position % 64
    first = n - rows
    at_v, at_k = first + rows // 2, first + rows // 2 + 1
    page, slot = spot(0, at_v)
    batch.cache.v_values[page, 1, slot, dim - 3] = 0xFF
    batch.cache.v_values[page, 1, slot, 0] = 0x7F
    page, slot = spot(1, at_k)
    batch.cache.k_values[page, 0, slot, 7] = 0x7F
    got = _attend(mx, batch, q, max_query_len=rows).cpu()
    want = clean.cpu().clone()
    for column in (dim - 3, 0):
        want[at_v - first : rows, 2:, column] = math.nan
    want[rows + at_k - first :, :2] = math.nan
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    assert torch.equal(got[ok], want[ok])


# ------------------------------------------------------- attention: sizes and scores at the edges


def _rescale_blocks(batch, exponent_of_tile, tiles=128):
    """Key scales of ``2**exponent`` per tile of tokens (scores of about that many nats)."""
    for b, n in enumerate(batch.lens):
        for p in range(0, n, 32):
            page, block = batch.table[b, p // batch.page], p % batch.page // 32
            batch.scales[0][page, :, block] = 120 + exponent_of_tile[p // tiles % len(exponent_of_tile)]
    batch.cache.k_scales.copy_(torch.from_numpy(batch.scales[0]))


def _check_large_scores(batch, q, got, scale, causal):
    """As _check_attention, with the rounding of the 32-bit scores written out.  A score is a sum of
    at most 24 matrix instructions (8 steps along head_dim, 3 terms), each of which may cut off the
    last bit, 2^-23, of a partial sum of at most S = sum_i |q_i k_i| * scale.  An error of e nats in
    the scores of numerator and denominator changes the output by at most 2 e of the weighted
    magnitudes: 2 * 24 * 2^-23 * S more than _delta."""
    want = batch.oracle_attention(q, scale, causal)
    weight = batch.weight_of(q, scale, causal)
    most = 0.0
    for b, n in enumerate(batch.lens):
        k = np.abs(kvo.read(batch.values[0], batch.scales[0], batch.table, [(b, p) for p in range(n)]))
        rows = np.abs(kvo.to_numpy(q[batch.cu[b] : batch.cu[b + 1]]))
        for h in range(q.shape[1]):
            most = max(most, float((rows[:, h] @ k[:, h // (q.shape[1] // batch.heads)].T).max()) * abs(scale))
    half = torch.finfo(q.dtype).eps / 2
    delta = _delta(q.dtype) + 2 * 24 * 2.0 ** -23 * most
    assert delta < 0.02                       # the check still tells right from wrong
    off = np.abs(kvo.to_numpy(got) - want)
    assert np.isfinite(off).all()
    assert float((off - (half * np.abs(want) + delta * weight + 1e-7)).max()) <= 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sequences,rows", [(1, 1), (90, 1), (2, 70)])
def test_maxima_that_jump_between_tiles(mx, sequences, rows, dtype):
    """Tiles whose largest scores are tens and hundreds of powers of two above and below the ones
    before them, in lists that are cut between CTAs and in lists that are not."""
    lens = [900 - 3 * b for b in range(sequences)]
    batch = Batch(mx, 51, lens, [rows] * sequences, 2, 32, 64, spread=0)
    _rescale_blocks(batch, [0, 2, 4, 6, 1, 6, 3, 5])
    q = torch.randn((batch.tokens, 4, 64), generator=_gen(52))
    q[:, 1] *= 0.125                          # a row of another range beside it
    q = q.to(dtype).to(DEV)
    got = _attend(mx, batch, q, max_query_len=rows)
    _check_large_scores(batch, q, got, 64 ** -0.5, True)


@pytest.mark.parametrize("dim,rows", [(128, 1), (128, 40), (256, 1), (256, 40)])
def test_maxima_that_jump_in_wide_heads(mx, dim, rows):
    batch = Batch(mx, 53, [700, 650], [rows, rows], 1, 64, dim, spread=0)
    _rescale_blocks(batch, [0, 4, 6, 2, 7, 1])
    q = torch.randn((batch.tokens, 4, dim), generator=_gen(54)).to(torch.bfloat16).to(DEV)
    got = _attend(mx, batch, q, max_query_len=rows)
    _check_large_scores(batch, q, got, dim ** -0.5, True)


@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("scale", [0.0, -0.125])
def test_scale_of_zero_and_below(mx, rows, scale):
    """Zero: the mean of the values that a row sees.  Negative: the smallest scores weigh most."""
    batch = Batch(mx, 55, [333, 80], [rows, rows], 2, 32, 64)
    q = torch.randn((2 * rows, 4, 64), generator=_gen(56)).to(torch.bfloat16).to(DEV)
    got = _attend(mx, batch, q, max_query_len=rows, scale=scale)
    _check_attention(batch, q, got, scale, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,group", [(64, 40), (128, 64), (256, 33)])
def test_many_query_heads_of_one_key_head(mx, dim, group, dtype):
    """One new token already has more rows than a few: sequences of one and of three tokens."""
    for news in ([1, 1, 1], [3, 1, 0]):
        batch = Batch(mx, 57, [300, 1, 45], news, 1, 64, dim)
        q = torch.randn((batch.tokens, group, dim), generator=_gen(58)).to(dtype).to(DEV)
        got = _attend(mx, batch, q, max_query_len=max(news))
        _check_attention(batch, q, got, dim ** -0.5, True)


@pytest.mark.parametrize("dim,page", [(64, 128), (128, 32), (256, 64)])
def test_large_ragged_batch_of_few_and_many_rows(mx, dim, page):
    """150 sequences: most with one new token, a few with chunks, some empty."""
    rng = random.Random(59)
    news = [rng.choice([1, 1, 1, 1, 0, 2, 45]) for _ in range(150)]
    lens = [max(n, rng.choice([1, 5, 40, 200])) for n in news]
    batch = Batch(mx, 60, lens, news, 1, page, dim)
    q = torch.randn((batch.tokens, 2, dim), generator=_gen(61)).to(torch.bfloat16).to(DEV)
    got = _attend(mx, batch, q, max_query_len=45)
    _check_attention(batch, q, got, dim ** -0.5, True)


def test_offsets_that_make_no_sense_stay_in_bounds(mx):
    """Descending, negative and too large row offsets; a bound that is too small; lengths below zero
    and behind the table: rows may be anything or unwritten, but nothing else is touched."""
    batch = Batch(mx, 62, [100, 64, 3], [30, 1, 2], 2, 32, 64)
    guard = torch.full((batch.tokens + 40, 6, 64), 9.0, dtype=torch.bfloat16, device=DEV)
    out = guard[20 : 20 + batch.tokens]
    q = torch.randn((batch.tokens, 6, 64), generator=_gen(63)).to(torch.bfloat16).to(DEV)
    for lens, cu, most in (([100, 64, 3], [30, 3, 33, 1], 40), ([100, 64, 3], [-5, -1, 10 ** 6, 2 ** 31 - 1], 40),
                           ([-7, 2 ** 31 - 1, 10 ** 6], batch.cu, 40), ([-2 ** 31, 64, 0], batch.cu, 40),
                           (batch.lens, [0, 0, 0, 0], 40), (batch.lens, [2, 33, 33, 33], 1)):
        mx.kv_cache_attention(q, batch.cache, batch.dev[0], _i32(lens), _i32(cu), max_query_len=most, out=out)
        assert bool((guard[:20] == 9.0).all()) and bool((guard[20 + batch.tokens :] == 9.0).all())
    # sequences within a bound that others exceed are right
    out.fill_(9.0)
    mx.kv_cache_attention(q, batch.cache, *batch.dev, max_query_len=2, out=out)
    assert bool((out[:30] == 9.0).all())
    whole = _attend(mx, batch, q, max_query_len=30)
    _check_attention(batch, q, whole, 64 ** -0.5, True)
    part = torch.cat([whole[:30], out[30:]])
    _check_attention(batch, q, part, 64 ** -0.5, True)


def test_calls_without_rows(mx):
    """No tokens in a call: nothing is read, written or launched."""
    batch = Batch(mx, 70, [40, 3], [0, 0], 2, 32, 64)
    before = [t.clone() for t in (batch.cache.k_values, batch.cache.k_scales)]
    empty = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=DEV)
    mx.kv_cache_write(batch.cache, empty, empty, *batch.dev)
    k, v = mx.kv_cache_read(batch.cache, *batch.dev, tokens=0)
    out = mx.kv_cache_attention(torch.empty((0, 6, 64), dtype=torch.bfloat16, device=DEV), batch.cache, *batch.dev)
    torch.cuda.synchronize()
    assert k.shape == v.shape == (0, 2, 64) and out.shape == (0, 6, 64)
    assert torch.equal(before[0], batch.cache.k_values) and torch.equal(before[1], batch.cache.k_scales)


@pytest.mark.parametrize("rows", [1, 60])
def test_a_cache_whose_memory_is_replaced(mx, rows):
    """A call uses the memory that the cache's tensors have when it is made."""
    batch = Batch(mx, 71, [150], [rows], 2, 32, 64)
    q = torch.randn((rows, 4, 64), generator=_gen(72)).to(torch.bfloat16).to(DEV)
    for t in (batch.cache.k_values, batch.cache.v_values, batch.cache.k_scales, batch.cache.v_scales):
        old = t.data
        t.data = old.clone()
        old.fill_(255)
    got = _attend(mx, batch, q, max_query_len=rows)
    _check_attention(batch, q, got, 64 ** -0.5, True)


def test_a_table_shared_by_all_sequences(mx):
    """Sequences that read the same pages (a row of the table expanded, stride zero), and a table
    whose rows are a slice of wider ones."""
    batch = Batch(mx, 73, [180], [1], 2, 32, 128)
    q = torch.randn((5, 4, 128), generator=_gen(74)).to(torch.bfloat16).to(DEV)
    lens = _i32([180, 100, 7, 33, 128])
    wide = torch.full((5, batch.width + 9), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
    wide[:, 4 : 4 + batch.width] = batch.dev[0]
    for table in (batch.dev[0].expand(5, -1), wide[:, 4 : 4 + batch.width]):
        got = mx.kv_cache_attention(q, batch.cache, table, lens)
        for b, n in enumerate((180, 100, 7, 33, 128)):
            batch.lens = [n]
            _check_attention(batch, q[b : b + 1], got[b : b + 1], 128 ** -0.5, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [7, 8, 9, 16, 17, 24, 25, 32, 33])
def test_row_counts_around_the_variants(mx, rows, dim, dtype):
    """New tokens x query heads per key head on both sides of every border between kernels, over
    sequences short and long enough to be cut."""
    group = next(g for g in (4, 3, 5, 1) if rows % g == 0) if rows != 7 else 7
    new = rows // group
    batch = Batch(mx, 75, [1200, new, 131], [new] * 3, 1, 128, dim)
    q = torch.randn((batch.tokens, group, dim), generator=_gen(76)).to(dtype).to(DEV)
    got = _attend(mx, batch, q, max_query_len=new)
    _check_attention(batch, q, got, dim ** -0.5, True)


@pytest.mark.parametrize("tokens,q_heads,k_heads,dim,rotary_dim", [
    (3, 5, 1, 72, 16),          # seven groups of eight behind the turned values: an odd one is left
    (1303, 2, 1, 24, 16),       # one group of eight, four tokens a CTA, three in the last
    (1303, 24, 4, 256, 64),     # several CTAs for four tokens
    (700, 9, 2, 160, 96),
])
def test_rotary_of_partial_heads(mx, tokens, q_heads, k_heads, dim, rotary_dim):
    half = rotary_dim // 2
    test_rotary_matches_definition(mx, torch.bfloat16, tokens, q_heads, k_heads, dim, rotary_dim,
                                   [half - half // 3, half // 3], False, tokens % 2 == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("adjacent", [False, True])
def test_pairs_without_a_row_of_positions_are_nan(mx, adjacent, dtype):
    """Frequencies whose axes the host does not know: pairs whose axis has no row become NaN, the
    others turn as ever and the values behind rotary_dim stay."""
    f = mx.rotary_frequencies(32, 1.0e4, [8, 8], adjacent=adjacent, device=DEV)
    axis = f.axis.clone()
    axis[[3, 4, 12]] = _i32([2, -1, 2 ** 31 - 1])
    q = torch.randn((5, 3, 48), generator=_gen(1)).to(dtype).to(DEV)
    pos = torch.randint(0, 1000, (2, 5), generator=_gen(2)).to(DEV)
    want = [t.clone() for t in mx.rotary_multi_axis(q, q[:, :1], pos, f)]
    got = mx.rotary_multi_axis(q, q[:, :1], pos, mx.RotaryFrequencies(f.inv_freq, axis, adjacent))
    lost = [i for pair in (3, 4, 12) for i in ((2 * pair, 2 * pair + 1) if adjacent else (pair, pair + 16))]
    for g, w in zip(got, want):
        w[..., lost] = math.nan
        assert torch.equal(g.isnan(), w.isnan())
        assert torch.equal(g.nan_to_num(), w.nan_to_num())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,group", [(64, 4), (128, 3), (256, 2)])
@pytest.mark.parametrize("rows", [4, 70])
def test_rows_that_see_nothing_are_zero_whatever_they_hold(mx, rows, dim, group, causal, dtype):
    """NaN and infinities in the query rows of a padded sequence, of positions below zero and of a
    sequence without pages; the other rows keep their bits."""
    batch = Batch(mx, 80, [0, rows - 1, 300, 2 * rows], [rows] * 4, 2, 32, dim)
    batch.table[3, :] = -1
    batch.dev = (torch.from_numpy(batch.table).to(DEV), *batch.dev[1:])
    q = torch.randn((batch.tokens, 2 * group, dim), generator=_gen(81)).to(dtype).to(DEV)
    want = _attend(mx, batch, q, max_query_len=rows, causal=causal)
    _check_attention(batch, q, want, dim ** -0.5, causal)
    blind = torch.tensor([*range(rows + (1 if causal else 0)), *range(3 * rows, 4 * rows)], device=DEV)
    q[blind[0::3], :, 7] = math.nan
    q[blind[1::3], :, 0] = math.inf
    q[blind[2::3]] = -math.inf
    got = _attend(mx, batch, q, max_query_len=rows, causal=causal)
    assert bool((got[blind] == 0).all())
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("rows", [1, 60])
def test_small_scales_of_large_keys(mx, rows, sign, dtype):
    """Keys of about 2^98 under a scale of 2^-101: ordinary scores, though the factor of a row's
    scores is below 2^-100."""
    batch = Batch(mx, 84, [333, 80], [rows, rows], 2, 32, 64)
    batch.scales[0] = np.where(batch.scales[0] == 255, 255, batch.scales[0].astype(np.int32) + 98).astype(np.uint8)
    batch.cache.k_scales.copy_(torch.from_numpy(batch.scales[0]))
    q = torch.randn((2 * rows, 4, 64), generator=_gen(85)).to(dtype).to(DEV)
    got = _attend(mx, batch, q, max_query_len=rows, scale=sign * 2.0 ** -101)
    _check_attention(batch, q, got, sign * 2.0 ** -101, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,dim,group", [(32, 64, 8), (128, 64, 3), (64, 128, 4), (32, 256, 6)])
def test_first_row_of_a_prompt_is_its_value(mx, page, dim, group, dtype):
    """The first row of a prompt sees one token, whose weight is one: its output is the token's value,
    rounded once.  Values have four significant bits, so both types hold them."""
    lens = [300, 64, 129, 45, 70]
    batch = Batch(mx, 82, lens, lens, 2, page, dim)
    for seed in (83, 84, 85):
        q = (torch.randn((batch.tokens, 2 * group, dim), generator=_gen(seed)) * 2).to(dtype).to(DEV)
        got = _attend(mx, batch, q, max_query_len=300)[batch.cu[:-1]]
        want = kvo.read(batch.values[1], batch.scales[1], batch.table, [(b, 0) for b in range(5)])
        want = torch.from_numpy(want).repeat_interleave(group, dim=1).to(dtype)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 60])
def test_weights_add_up_to_one(mx, rows, dim, dtype):
    """Values that are all one: whatever the weights were rounded to, their mean is one.  Sums of at
    most 400 weights in 32 bits, a reciprocal and a product are off by less than 2^-14, which rounds
    back to one in both types."""
    batch = Batch(mx, 86, [400, 77], [rows, rows], 2, 32, dim, finite=True)
    batch.cache.v_values.fill_(0x38)
    batch.cache.v_scales.fill_(127)
    q = (torch.randn((2 * rows, 6, dim), generator=_gen(87)) * 3).to(dtype).to(DEV)
    got = _attend(mx, batch, q, max_query_len=rows)
    assert bool((got == 1).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("rows", [1, 60])
def test_equal_scores_far_below_zero(mx, rows, dim, dtype):
    """Scores of about -2^115 (2^13 * 2^98 * dim / sqrt(dim)), the same for every token: the weights are
    equal, not all zero."""
    batch = Batch(mx, 88, [300, 70], [rows, rows], 1, 32, dim, finite=True)
    batch.values[0][:], batch.scales[0][:] = 0x38, 127 + 98
    batch.cache.k_values.fill_(0x38)
    batch.cache.k_scales.fill_(127 + 98)
    q = torch.full((2 * rows, 4, dim), -(2.0 ** 13), dtype=dtype, device=DEV)
    got = _attend(mx, batch, q, max_query_len=rows)
    _check_attention(batch, q, got, dim ** -0.5, True)


def _check_rounded_weights(batch, q, got, scale):
    """As _check_attention, from what the weights are held in.  Each is off by a factor 1 + d_j, |d_j| <= d,
    and the row is divided by the sum of the weights as they were rounded: with o the exact output,

        sum_j p_j (1 + d_j) v_j / sum_j p_j (1 + d_j) - o = sum_j p_j d_j (v_j - o) / (1 + sum_j p_j d_j)

    which is at most d / (1 - d) * sum_j p_j |v_j - o|.  d = 2^-11 for the rounding to FP16, and for BF16
    2^-9 more for the second E4M3 term; 2^-13 more covers 32-bit scores below 40 (24 sums of 2^-24 each)
    and exponentials, and the division.  Weights below 2^-3 (2^-7 with three terms) of the 181 and more
    that the largest of their block is scaled to are off by 2^-14 (2^-18) instead: less than 2^-21 (2^-25)
    of the sum a token, times twice the largest value.  The output is rounded once more, by half a step."""
    want = batch.oracle_attention(q, scale, True)
    rows = kvo.to_numpy(q)
    bf16 = q.dtype is torch.bfloat16
    d = 2.0 ** -11 + 2.0 ** -13 + (2.0 ** -9 if bf16 else 0.0)
    group = q.shape[1] // batch.heads
    for b, length in enumerate(batch.lens):
        where = [(b, p) for p in range(length)]
        k = kvo.read(batch.values[0], batch.scales[0], batch.table, where)
        v = kvo.read(batch.values[1], batch.scales[1], batch.table, where)
        n = batch.cu[b + 1] - batch.cu[b]
        for i in range(n):
            sees = length - n + i + 1
            for h in range(q.shape[1]):
                s = k[:sees, h // group] @ rows[batch.cu[b] + i, h] * scale
                p = np.exp(s - s.max())
                o, seen = want[batch.cu[b] + i, h], v[:sees, h // group]
                apart = (p[:, None] * np.abs(seen - o)).sum(0) / p.sum()
                few = sees * (2.0 ** -21 if bf16 else 2.0 ** -25) * 2 * np.abs(seen).max()
                limit = torch.finfo(q.dtype).eps / 2 * np.abs(o) + d / (1 - d) * apart + few
                off = np.abs(kvo.to_numpy(got[batch.cu[b] + i, h]) - o)
                assert np.all(off <= limit + 2.0 ** -25), (b, i, h, float((off - limit).max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,group", [(64, 129), (128, 200), (256, 256)])
def test_more_query_heads_than_a_tile_has_rows(mx, dim, group, dtype):
    """The query heads of one token fill a row tile and more; whole vectors and odd strides."""
    for news in ([1, 1, 1], [2, 5, 1]):
        batch = Batch(mx, 89, [300, 5, 45], news, 1, 64, dim)
        wide = torch.randn((batch.tokens, group * dim + 1), generator=_gen(90)).to(dtype).to(DEV)
        for q in (wide[:, :-1].contiguous().view(batch.tokens, group, dim),
                  wide[:, 1:].view(batch.tokens, group, dim)):
            got = _attend(mx, batch, q, max_query_len=max(news))
            _check_rounded_weights(batch, q, got, dim ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [2, 45])
def test_rows_within_what_their_weights_are_held_in(mx, rows, dim, dtype):
    batch = Batch(mx, 91, [260, rows, 97], [rows] * 3, 2, 32, dim)
    q = torch.randn((batch.tokens, 8, dim), generator=_gen(92)).to(dtype).to(DEV)
    got = _attend(mx, batch, q, max_query_len=rows)
    _check_rounded_weights(batch, q, got, dim ** -0.5)
