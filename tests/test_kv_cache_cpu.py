"""CPU tests of the paged KV cache operators: refusals, the oracle's own rounding, host tables."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import mxfp6_sm120_b200 as mx
from oracle import kv_oracle as kvo


def _cache(pages=4, heads=2, page=32, dim=64):
    return mx.PagedKVCache.allocate(pages, heads, page, dim, device="cpu")


def _batch(batch=2, width=2):
    return (torch.zeros((batch, width), dtype=torch.int32),
            torch.ones((batch,), dtype=torch.int32))


def test_oracle_rounding_agrees_with_torch():
    gen = torch.Generator().manual_seed(3)
    x = torch.cat([torch.randn(4000, generator=gen) * s for s in (0.002, 0.1, 30.0, 400.0)])
    x = torch.cat([x, torch.tensor([0.0, -0.0, 448.0, -448.0, 464.0, 1e9, 2.0 ** -10, 3 * 2.0 ** -10])])
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(kvo.encode(x.numpy()), want)
    assert [kvo.needed_scale(v) for v in (0.0, 448.0, 448.5, 896.0, 1e-40)] == [28, 127, 128, 128, 28]


def test_cache_container_refusals():
    good = _cache()
    assert (good.pages, good.kv_heads, good.page_size, good.head_dim) == (4, 2, 32, 64)
    assert good.nbytes() == 2 * (4 * 2 * 32 * 64 + 4 * 2)
    v, s = good.k_values, good.k_scales
    for kind, match, args in (
        (ValueError, "page_size", (v[:, :, :16], v[:, :, :16], s, s)),
        (ValueError, "head_dim", (v[..., :32], v[..., :32], s, s)),
        (ValueError, "at least one", (v[:0], v[:0], s[:0], s[:0])),
        (ValueError, "must be \\[pages", (v[0], v, s, s)),
        (ValueError, "shape of k_values", (v, v[:2], s, s)),
        (ValueError, "k_scales and v_scales", (v, v, s[:2], s)),
        (ValueError, "k_scales and v_scales", (v, v, s, s[..., :0])),
        (TypeError, "uint8", (v.to(torch.int8), v, s, s)),
        (TypeError, "uint8", (v, v, s, s.to(torch.int32))),
        (ValueError, "contiguous", (v.transpose(0, 1).contiguous().transpose(0, 1), v, s, s)),
        (ValueError, "one device", (v, v.to("meta"), s, s)),
    ):
        with pytest.raises(kind, match=match):
            mx.PagedKVCache(*args)


def test_batch_and_row_refusals():
    cache = _cache()
    table, lens = _batch()
    rows = torch.zeros((2, 2, 64), dtype=torch.bfloat16)

    def write(k=rows, v=rows, table=table, lens=lens, cu=None, cache=cache):
        mx.kv_cache_write(cache, k, v, table, lens, cu)

    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    for kind, match, kwargs in (
        (TypeError, "PagedKVCache", dict(cache=None)),
        (TypeError, "int32", dict(table=table.long())),
        (TypeError, "int32", dict(lens=lens.long())),
        (TypeError, "cu_seqlens must be int32", dict(cu=cu.long())),
        (ValueError, "cu_seqlens must be contiguous \\[3\\]", dict(cu=cu[:2])),
        (ValueError, "block_table must be", dict(table=table[0])),
        (ValueError, "block_table must be", dict(table=table[:, :0])),
        (ValueError, "contiguous rows", dict(table=table.t().contiguous().t())),
        (ValueError, "at least one sequence", dict(table=table[:0], lens=lens[:0], k=rows[:0], v=rows[:0])),
        (ValueError, "seq_lens must be", dict(lens=lens[:1])),
        (ValueError, "one row", dict(k=rows[:1], v=rows[:1])),
        (ValueError, "k must be \\[tokens", dict(k=rows[0])),
        (ValueError, "k must be \\[tokens, 2, 64\\]", dict(k=rows[:, :1])),
        (ValueError, "v must be \\[tokens, 2, 64\\]", dict(v=rows[..., :32])),
        (TypeError, "k must have dtype", dict(k=rows.float())),
        (ValueError, "one shape and dtype", dict(v=rows.half())),
        (ValueError, "last dimension", dict(k=torch.zeros((2, 64, 2), dtype=torch.bfloat16).transpose(1, 2))),
        (ValueError, "CUDA device", dict()),
    ):
        with pytest.raises(kind, match=match):
            write(**kwargs)


def test_read_refusals():
    cache = _cache()
    table, lens = _batch()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    out = torch.zeros((2, 2, 64), dtype=torch.float16)
    for kind, match, kwargs in (
        (TypeError, "dtype", dict(dtype=torch.float32)),
        (ValueError, "tokens \\(rows in all\\)", dict(cu_seqlens=cu)),
        (ValueError, "must not be negative", dict(cu_seqlens=cu, tokens=-1)),
        (ValueError, "`tokens` rows", dict(cu_seqlens=cu, tokens=3, out=(out, out.clone()))),
        (ValueError, "contiguous", dict(out=(out.transpose(0, 1).contiguous().transpose(0, 1), out))),
        (ValueError, "one shape and dtype", dict(out=(out, out.bfloat16()))),
        (ValueError, "CUDA device", dict(out=(out, out.clone()))),
    ):
        with pytest.raises(kind, match=match):
            mx.kv_cache_read(cache, table, lens, **kwargs)


def test_attention_refusals():
    cache = _cache()
    table, lens = _batch()
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    for kind, match, args, kwargs in (
        (ValueError, "q must be", (q[0],), {}),
        (ValueError, "multiple of the cache", (q[:, :3],), {}),
        (ValueError, "q must be", (torch.zeros((2, 4, 128), dtype=torch.bfloat16),), {}),
        (TypeError, "dtype", (q.float(),), {}),
        (ValueError, "max_query_len", (q,), dict(max_query_len=0)),
        (ValueError, "scale must be finite", (q,), dict(scale=math.inf)),
        (ValueError, "out must match", (q,), dict(out=q.half())),
        (ValueError, "out must be", (q,), dict(out=q[:, :2])),
        (ValueError, "overlap itself", (q,), dict(out=torch.zeros((1, 4, 64), dtype=torch.bfloat16).expand(2, 4, 64))),
        (ValueError, "CUDA device", (q,), {}),
    ):
        with pytest.raises(kind, match=match):
            mx.kv_cache_attention(*args, cache, table, lens, **kwargs)


def test_rotary_refusals_and_frequencies():
    f = mx.rotary_frequencies(32, 1.0e4, [8, 4, 4], device="cpu")
    assert f.axis.tolist() == [0] * 8 + [1] * 4 + [2] * 4 and f.rotary_dim == 32
    assert f.inv_freq[0] == 1.0 and math.isclose(float(f.inv_freq[8]), 1.0e-2)
    g = mx.rotary_frequencies(32, 1.0e4, [8, 4, 4], interleaved=True, device="cpu")
    assert g.axis.tolist() == [0, 1, 2] * 4 + [0] * 4
    with pytest.raises(ValueError, match="cannot be interleaved"):
        mx.rotary_frequencies(32, 1.0e4, [2, 12, 2], interleaved=True, device="cpu")
    with pytest.raises(ValueError, match="sum to 16"):
        mx.rotary_frequencies(32, 1.0e4, [8, 4], device="cpu")
    for bad in (24, 0, 512, -16):
        with pytest.raises(ValueError, match="rotary_dim"):
            mx.rotary_frequencies(bad, device="cpu")
    with pytest.raises(ValueError, match="theta"):
        mx.rotary_frequencies(32, 0.0, device="cpu")
    with pytest.raises(TypeError, match="float64"):
        mx.RotaryFrequencies(f.inv_freq.float(), f.axis)
    with pytest.raises(TypeError, match="int32"):
        mx.RotaryFrequencies(f.inv_freq, f.axis.long())
    q = torch.zeros((3, 4, 64), dtype=torch.float16)
    pos = torch.zeros((3, 3), dtype=torch.int64)
    for kind, match, args, kwargs in (
        (TypeError, "RotaryFrequencies", (q, q, pos, None), {}),
        (ValueError, "one token count", (q, q[:2], pos, f), {}),
        (ValueError, "k must be", (q, q[..., :32], pos, f), {}),
        (ValueError, "at least rotary_dim", (q[..., :16], q[..., :16], pos, f), {}),
        (TypeError, "positions", (q, q, pos.float(), f), {}),
        (ValueError, "positions must be", (q, q, pos[:, :2], f), {}),
        (ValueError, "positions must be", (q, q, pos[:0], f), {}),
        (ValueError, "match its input", (q, q.clone(), pos, f), dict(k_out=q.bfloat16())),
        (ValueError, "overlap itself", (q, q, pos, f), dict(q_out=q[:1].expand(3, 4, 64))),
        (ValueError, "CUDA device", (q, q.clone(), pos, f), {}),
    ):
        with pytest.raises(kind, match=match):
            mx.rotary_multi_axis(*args, **kwargs)


def test_c_entries_refuse_before_any_launch():
    from mxfp6_sm120_b200._loader import library

    lib = library()
    p = 4096  # a non-null, aligned address that nothing dereferences on these paths

    def write(cache=(p, p, p, p, 4, 2, 32, 64), batch=(p, p, None, 2, 2, 2, 2), k=p, dtype=1):
        return lib.mxfp6_kv_cache_write(*cache, *batch, k, p, dtype, 128, 64, 128, 64, None)

    for message, kwargs in (
        (b"null", dict(cache=(None, p, p, p, 4, 2, 32, 64))),
        (b"head_dim", dict(cache=(p, p, p, p, 4, 2, 32, 80))),
        (b"page_size", dict(cache=(p, p, p, p, 4, 2, 48, 64))),
        (b"pages and", dict(cache=(p, p, p, p, 0, 2, 32, 64))),
        (b"below 2^31", dict(cache=(p, p, p, p, 1 << 30, 2, 32, 64))),
        (b"aligned", dict(cache=(p + 8, p, p, p, 4, 2, 32, 64))),
        (b"batch must be positive", dict(batch=(p, p, None, 2, 0, 2, 0))),
        (b"block_table and seq_lens", dict(batch=(None, p, None, 2, 2, 2, 2))),
        (b"columns", dict(batch=(p, p, None, 2, 2, 0, 2))),
        (b"columns", dict(batch=(p, p, None, 2, 2, 1 << 27, 2))),
        (b"exactly one row", dict(batch=(p, p, None, 2, 3, 2, 2))),
        (b"float16 or bfloat16", dict(dtype=2)),
        (b"must not be null", dict(k=None)),
    ):
        assert write(**kwargs) == 1, message
        assert message in lib.mxfp6_b200_last_error(), message
    assert lib.mxfp6_kv_cache_attention_workspace(2, 2, 1, 3, 2, 64, 1, 64) in (-1, 0)


def test_c_attention_refuses_before_any_launch():
    from mxfp6_sm120_b200._loader import library

    lib = library()
    p = 4096

    def attend(batch=(p, p, None, 2, 2, 64, 2), q=p, dtype=1, heads=4, most=1, scale=0.125, workspace=(p, 1 << 40)):
        return lib.mxfp6_kv_cache_attention(p, p, p, p, 4, 2, 32, 64, *batch, q, p, dtype, heads, 256, 64, 256, 64,
                                            most, scale, 1, *workspace, None)

    for message, kwargs in (
        (b"float16 or bfloat16", dict(dtype=2)),
        (b"multiple of the cache", dict(heads=3)),
        (b"multiple of the cache", dict(heads=0)),
        (b"max_query_len", dict(most=0)),
        (b"scale must be finite", dict(scale=math.inf)),
        (b"scale must be finite", dict(scale=math.nan)),
        (b"scale must be finite", dict(scale=3.0e38)),
        (b"must not be null", dict(q=None)),
        (b"2^30 rows", dict(batch=(p, p, p, 2, 1 << 30, 64, 2))),
        (b"workspace must be", dict(workspace=(p, 16))),
        (b"workspace must be", dict(workspace=(p + 4, 1 << 40))),
        (b"workspace must be", dict(workspace=(None, 1 << 40))),
    ):
        assert attend(**kwargs) == 1, message
        assert message in lib.mxfp6_b200_last_error(), (message, lib.mxfp6_b200_last_error())
    # no rows: nothing to do
    assert attend(batch=(p, p, p, 2, 0, 64, 2)) == 0


def test_rotary_refuses_positions_with_too_few_axes():
    """Frequencies of three sections need three rows of positions, whichever way they are laid out;
    rows that no pair follows are not asked for."""
    q = torch.zeros((3, 4, 64), dtype=torch.float16)
    pos = torch.zeros((3, 3), dtype=torch.int64)
    for sections, interleaved, axes in (([8, 4, 4], False, 3), ([8, 4, 4], True, 3), ([8, 8], False, 2),
                                        ([8, 8, 0], False, 2), ([0, 16], False, 2), (None, False, 1)):
        f = mx.rotary_frequencies(32, 1.0e4, sections, interleaved=interleaved, device="cpu")
        assert f.axes == axes
        for rows in range(1, 4):
            match = "a row for each" if rows < axes else "CUDA device"
            with pytest.raises(ValueError, match=match):
                mx.rotary_multi_axis(q, q.clone(), pos[:rows], f)
        with pytest.raises(ValueError, match="a row for each" if axes > 1 else "CUDA device"):
            mx.rotary_multi_axis(q, q.clone(), pos[0], f)
    f = mx.rotary_frequencies(32, 1.0e4, [8, 8], device="cpu")
    for bad in (0, 9):
        with pytest.raises(ValueError, match="axes must be 1 to 8"):
            mx.RotaryFrequencies(f.inv_freq, f.axis, axes=bad)
    with pytest.raises(ValueError, match="a row for each"):
        mx.rotary_multi_axis(q, q.clone(), pos[:2], mx.RotaryFrequencies(f.inv_freq, f.axis, False, 3))
    assert mx.RotaryFrequencies(f.inv_freq, f.axis).axes is None      # nothing is read from the device


def test_workspace_query_refuses_what_the_call_refuses():
    """-1 for sizes that the call would refuse, 0 where it needs no scratch, else its bytes."""
    from mxfp6_sm120_b200._loader import library

    query = library().mxfp6_kv_cache_attention_workspace
    good = dict(batch=2, tokens=2, most=1, q_heads=4, kv_heads=2, dim=64, dtype=1, context=4096)

    def ask(**kwargs):
        return query(*{**good, **kwargs}.values())

    # 32 tiles of 128 tokens: 4 sequences x heads of 33 units cut into shares of 3 = 44 CTAs, each with two
    # ends of 8 rows x 64 values, a maximum and a sum; before them 148 borders of 32 bytes
    assert ask() == 148 * 32 + 44 * 2 * (8 * 64 + 2 * 8) * 4
    assert ask(context=1024) == 0 and ask(tokens=0) == 0
    for bad in (dict(batch=0), dict(batch=-1), dict(batch=1 << 31), dict(tokens=-1), dict(tokens=(1 << 30) + 1, q_heads=2),
                dict(tokens=(1 << 29) + 1), dict(tokens=1 << 62), dict(most=0), dict(q_heads=0), dict(q_heads=-2),
                dict(q_heads=3), dict(q_heads=65536), dict(kv_heads=0), dict(kv_heads=3), dict(dim=80),
                dict(dtype=2), dict(context=0), dict(context=(1 << 30) + 32)):
        assert ask(**bad) == -1, bad
        if "context" not in bad:
            assert ask(**bad, context=64) == -1, bad
    assert ask(tokens=1 << 29, most=1 << 29) > 0 and ask(context=1 << 30) > 0 and ask(q_heads=65534) > 0


@pytest.mark.parametrize("name,hundred", [("kv_attention_decode", 4), ("kv_attention_prefill", 5)])
def test_a_status_code_names_one_wait(name, hundred):
    """The code that a wait leaves when it runs out tells which barrier was waited for where: no two
    waits of a kernel share one, but for the two places of which a variant compiles one."""
    import re
    from pathlib import Path

    text = (Path(mx.__file__).parent / "csrc" / f"{name}.cu").read_text()
    calls = re.findall(rf"\b(bounded_wait|wait|wait_output|meet)\(((?:[^;{{}}]*?,)?\s*({hundred}\d\d))\)", text)
    places: dict[str, list[str]] = {}
    for _, arguments, code in calls:
        places.setdefault(code, []).append(re.sub(r"\s+", " ", arguments))
    assert len(places) >= 14
    for code, found in places.items():
        assert len(set(found)) == 1, (code, found)
        assert len(found) == 1 or all("sfull0" in f for f in found), (code, found)
