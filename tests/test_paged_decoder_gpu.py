"""The decoder step over the paged 8-bit cache: the operators run together as a server uses them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_oracle as kvo

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _model(mx, layers=2, head_dim=128):
    cfg = mx.DecoderConfig(hidden=512, q_heads=4, kv_heads=2, head_dim=head_dim, intermediate=1024,
                           layers=layers)
    gen = torch.Generator(device=DEV).manual_seed(5000)
    return cfg, mx.DenseDecoder(cfg, [mx.random_layer(cfg, DEV, gen) for _ in range(layers)])


def _rope(mx, cfg):
    return mx.rotary_frequencies(cfg.head_dim // 2, 1.0e6, [16, 8, 8] if cfg.head_dim == 128 else None,
                                 device=DEV)


def _positions(starts, news, axes=3):
    p = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, news)])
    return torch.stack([p * (a + 1) % 977 for a in range(axes)]).to(DEV)


def test_refusals(mx):
    cfg, model = _model(mx, layers=1)
    ws = model.workspace(2)
    caches = model.new_paged_cache(4)
    table, lens = torch.zeros((2, 1), dtype=torch.int32, device=DEV), _i32([1, 1])
    with pytest.raises(ValueError, match="one per layer"):
        model.paged_step(ws, [], table, lens)
    with pytest.raises(ValueError, match="go together"):
        model.paged_step(ws, caches, table, lens, rotary=_rope(mx, cfg))


def test_prompt_then_tokens_match_the_operators_definitions(mx):
    """One layer: its attention output (the operand of the output projection) against the
    definitions in 64 bits on the layer's own QKV rows, for a ragged prompt batch and for the
    token after it.  Off by the BF16 rounding of the output and of the turned rows; the cached
    values are those of the definition's own rounding, so they agree exactly."""
    cfg, model = _model(mx, layers=1)
    page = 64
    news, lens = [70, 1, 33], [70, 1, 33]
    caches = model.new_paged_cache(8, page)
    table = np.array([[5, 2, 7], [0, 7, 7], [3, 7, 7]], np.int32)
    dev_table = torch.from_numpy(table).to(DEV)
    rope = _rope(mx, cfg)
    shape = (8, cfg.kv_heads, page, cfg.head_dim)
    values = [np.zeros(shape, np.uint8) for _ in range(2)]
    scales = [np.full((8, cfg.kv_heads, page // 32), 127, np.uint8) for _ in range(2)]
    starts = [0, 0, 0]
    for step in range(2):
        tokens = sum(news)
        cu = np.concatenate([[0], np.cumsum(news)])
        positions = _positions(starts, news)
        ws = model.workspace(tokens)
        ws.x.copy_(torch.randn((tokens, cfg.hidden), generator=_gen(step)).to(torch.bfloat16))
        x0 = ws.x.clone()
        model.paged_step(ws, caches, dev_table, _i32(lens), _i32(cu.tolist()) if step == 0 else None,
                         max_query_len=max(news), rotary=rope, positions=positions)
        torch.cuda.synchronize()
        # the layer's QKV rows once more, not turned
        a = mx.rmsnorm_quantize_mxfp8(x0.clone(), model.layers[0].ln1, cfg.eps)
        qkv = mx.gemm_w6a8(a, model.layers[0].qkv, out_dtype=torch.bfloat16)
        hd = cfg.head_dim
        q = qkv[:, : 4 * hd].view(tokens, 4, hd)
        k = qkv[:, 4 * hd : 6 * hd].view(tokens, 2, hd)
        v = qkv[:, 6 * hd :].view(tokens, 2, hd)
        turned = [torch.from_numpy(kvo.rotary(kvo.to_numpy(t), positions.cpu().numpy(),
                                              rope.inv_freq.cpu().numpy(), rope.axis.cpu().numpy()))
                  for t in (q, k)]
        got_rows = ws.qkv[:, : 6 * hd].view(tokens, 6, hd)
        want_rows = torch.cat(turned, 1)
        size = want_rows.abs().amax(-1, keepdim=True)
        assert bool(((got_rows.cpu().double() - want_rows).abs()
                     <= want_rows.abs() * 2.0 ** -8 + size * 2.0 ** -20).all())
        for rows, val, sc in zip((ws.qkv[:, 4 * hd : 6 * hd], ws.qkv[:, 6 * hd :]), values, scales):
            kvo.write(val, sc, kvo.to_numpy(rows.reshape(tokens, 2, hd)), table, lens, cu, 8, page)
        assert np.array_equal(caches[0].k_values.cpu().numpy()[[5, 2, 0, 3]], values[0][[5, 2, 0, 3]])
        assert np.array_equal(caches[0].v_scales.cpu().numpy()[[5, 2, 0, 3]], scales[1][[5, 2, 0, 3]])
        want = kvo.attention(kvo.to_numpy(got_rows[:, :4]), *values, *scales, table, lens, cu, hd ** -0.5, True)
        weight = kvo.attention(kvo.to_numpy(got_rows[:, :4]), values[0], values[1] & 127, *scales, table, lens,
                               cu, hd ** -0.5, True)
        off = np.abs(kvo.to_numpy(ws.attn.view(tokens, 4, hd)) - want)
        assert np.all(off <= 2.0 ** -8 * np.abs(want) + 2.0 ** -8 * weight + 1e-7)
        starts, news = list(lens), [1, 1, 1]
        lens = [n + 1 for n in lens]
    assert mx.device_status() == 0


def test_chunks_reach_the_state_of_one_prompt(mx):
    """A prompt in one piece and in three gives the same cached values wherever the layer's input
    is the same (layer 0), and hidden states that agree to the 8-bit cache's rounding."""
    cfg, model = _model(mx)
    total, page = 150, 32
    x = torch.randn((total, cfg.hidden), generator=_gen(4)).to(torch.bfloat16).to(DEV)
    table = _i32([[4, 0, 3, 1, 2]])
    rope = _rope(mx, cfg)
    outs, states = [], []
    for chunks in ([150], [64, 53, 33]):
        caches = model.new_paged_cache(5, page)
        done, out = 0, []
        for n in chunks:
            ws = model.workspace(n)
            ws.x.copy_(x[done : done + n])
            model.paged_step(ws, caches, table, _i32([done + n]), _i32([0, n]), max_query_len=n,
                             rotary=rope, positions=_positions([done], [n]))
            out.append(ws.x.clone())
            done += n
        outs.append(torch.cat(out).float())
        states.append(caches)
    # layer 0 sees the same rows; the quantised linears may differ in a few roundings between sizes
    a, b = (mx.kv_cache_read(c[0], table, _i32([total]), _i32([0, total]), tokens=total) for c in states)
    for p, q in zip(a, b):
        assert float((p.float() - q.float()).norm() / p.float().norm()) <= 2.0 ** -4
    cos = torch.nn.functional.cosine_similarity(outs[0].flatten(), outs[1].flatten(), dim=0)
    assert float(cos) >= 0.998


@pytest.mark.parametrize("head_dim", [128, 256])
def test_captured_decode_step_follows_lengths_and_tables(mx, head_dim):
    """One graph of the whole step serves growing sequences: replays equal eager steps."""
    cfg, model = _model(mx, head_dim=head_dim)
    rope = mx.rotary_frequencies(64, 1.0e6, device=DEV)
    batch, page = 3, 32
    table = _i32([[0, 1, 2], [3, 4, 5], [6, 7, 8]])
    start = [31, 5, 64]
    xs = [torch.randn((batch, cfg.hidden), generator=_gen(i)).to(torch.bfloat16).to(DEV) for i in range(4)]

    def fresh():
        caches = model.new_paged_cache(9, page)
        n = sum(start)
        ws = model.workspace(n)
        ws.x.copy_(torch.randn((n, cfg.hidden), generator=_gen(99)).to(torch.bfloat16))
        model.paged_step(ws, caches, table, _i32(start), _i32([0, *np.cumsum(start).tolist()]),
                         max_query_len=max(start), rotary=rope,
                         positions=_positions([0] * 3, start, axes=1))
        return caches

    eager = []
    caches = fresh()
    ws = model.workspace(batch)
    for i, x in enumerate(xs):
        ws.x.copy_(x)
        lens = [n + i + 1 for n in start]
        model.paged_step(ws, caches, table, _i32(lens), rotary=rope, positions=_i32([n - 1 for n in lens]))
        eager.append(ws.x.clone())
    want_cache = [c.k_values.clone() for c in caches]

    caches = fresh()
    lens, pos = _i32([n + 1 for n in start]), _i32(start)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    keep = [t.clone() for c in caches for t in (c.k_values, c.v_values, c.k_scales, c.v_scales)]
    with torch.cuda.stream(side):
        ws.x.copy_(xs[0])
        model.paged_step(ws, caches, table, lens, rotary=rope, positions=pos)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            model.paged_step(ws, caches, table, lens, rotary=rope, positions=pos)
    torch.cuda.synchronize()
    for t, k in zip((t for c in caches for t in (c.k_values, c.v_values, c.k_scales, c.v_scales)), keep):
        t.copy_(k)
    for i, x in enumerate(xs):
        lens.copy_(_i32([n + i + 1 for n in start]))
        pos.copy_(_i32([n + i for n in start]))
        ws.x.copy_(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ws.x, eager[i])
    for c, k in zip(caches, want_cache):
        assert torch.equal(c.k_values, k)
    assert mx.device_status() == 0
