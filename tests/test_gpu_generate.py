"""Whole models token by token (gpt2.Gpt2Decoder, deepseek.MoeLayerDecoder)
against the graphs they stand for: with the weights of a graph quantised in
place, every row that the single-token path computes equals forward_ops' row
of the whole sequence, bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GPT2 = dict(m=64, d=64, d_real=48, heads=3, dh=16, ffn=128, ffn_real=96, vocab=512, vocab_real=500)
# an exp table of 2^20 entries: its first entry is zero, so masked columns do not count
MOE = dict(m=32, h=128, heads=2, qk_nope=16, qk_rope=8, v_head=16, kv_lora=32, n_routed=16, top_k=3, moe=64,
           moe_real=48, shared=128, shared_real=96, exp_bits=20, silu_bits=20, w_mod=1 << 8)


def _gpt2(zk, group, layers=2):
    s = zk.gpt2.LayerShape(**GPT2)
    store = zk.compose.Store()
    ops, tokens, out = zk.gpt2.gpt2_model(store, s, layers=layers)
    weights = zk.decode.quantise_weights(store, ops, ("Projection", "MatMul"), group)
    zk.compose.forward_ops(store, ops)
    masked = next(op for op in ops if op.kind == "Argmax").x
    return s, store, ops, weights, store.get_idx(tokens), store.get(masked).reshape(s.m, s.vocab), store.get_idx(out)


@pytest.mark.parametrize("group,prompt", [(32, 0), (64, 21), (128, 32)])
def test_gpt2_steps_equal_the_graph(zk, group, prompt):
    """From an empty cache, and from a prompt's keys and values: the logits and
    the choices of every later position, two sequences at different places."""
    import torch
    s, store, ops, weights, tokens, logits, argmax = _gpt2(zk, group)
    dec = zk.gpt2.Gpt2Decoder(store, ops, s, weights, batch=2)
    start = [prompt, prompt // 2]
    for b in range(2):
        dec.load(store, b, start[b])
    assert dec.lens.tolist() == start
    i64 = lambda t: t.view(torch.int64)  # noqa: E731
    for i in range(s.m - prompt):
        at = [start[0] + i, start[1] + i]
        dec.tokens.copy_(tokens.view(torch.int32)[at].view(torch.uint32))
        token, got = dec.step()
        assert torch.equal(i64(got), i64(logits)[at])
        assert torch.equal(token.view(torch.int32), argmax.view(torch.int32)[at])
    dec.check()


def test_gpt2_generates_what_the_graph_would(zk):
    """Its own choices fed back (a replayed CUDA graph): the graph run over the
    tokens that were generated chooses the same ones."""
    import torch
    s, store, ops, weights, tokens, _, argmax = _gpt2(zk, 64)
    n = 40
    dec = zk.gpt2.Gpt2Decoder(store, ops, s, weights, batch=1)
    dec.load(store, 0, n)
    dec.tokens.copy_(argmax[n - 1:n])
    graph, said = dec.capture(), [int(dec.tokens[0])]
    assert dec.lens.tolist() == [n] and int(dec.tokens[0]) == said[0]
    for _ in range(s.m - n - 1):
        graph.replay()
        said.append(int(dec.tokens[0]))
    dec.check()
    text = tokens.cpu().numpy().copy()
    text[n:] = said
    # the graph over the new text: its embedding indices are d vocab + token
    emb = ops[0].idx
    store.idx[emb].copy_(torch.from_numpy((np.arange(s.d)[None] * s.vocab + text[:, None]).astype(np.uint32).reshape(-1)).cuda())
    zk.compose.forward_ops(store, ops)
    again = store.get_idx(next(op for op in ops if op.kind == "Argmax").out).cpu().numpy()
    assert again[n - 1:s.m - 1].tolist() == said


def test_gpt2_refuses(zk):
    s, store, ops, weights, *_ = _gpt2(zk, 64, layers=1)
    dec = zk.gpt2.Gpt2Decoder(store, ops, s, weights)
    with pytest.raises(ValueError, match="positions"):
        dec.load(store, 0, s.m + 1)
    with pytest.raises(ValueError, match="sequence"):
        dec.load(store, 1, 3)
    with pytest.raises(ValueError, match="shape"):
        zk.gpt2.Gpt2Decoder(store, ops, zk.gpt2.LayerShape(**dict(GPT2, heads=2)), weights)
    dec.load(store, 0, s.m)  # full: the next step says so
    dec.step()
    with pytest.raises(ValueError, match="full"):
        dec.check()
    dec.check()


def test_gpt2_ends_with_the_graph_inside_a_block(zk):
    """A graph of 40 positions: the cache's blocks hold 64 tokens, the 41st is refused."""
    s = zk.gpt2.LayerShape(**dict(GPT2, m=40))
    store = zk.compose.Store()
    ops, _, _ = zk.gpt2.gpt2_model(store, s, layers=1)
    weights = zk.decode.quantise_weights(store, ops, ("Projection", "MatMul"))
    dec = zk.gpt2.Gpt2Decoder(store, ops, s, weights)
    for _ in range(40):
        dec.step()
    dec.check()
    dec.step()
    with pytest.raises(ValueError, match="full"):
        dec.check()


@pytest.mark.parametrize("batch", [1, 3])
def test_moe_layer_steps_equal_the_graph(zk, batch):
    import torch
    from zkie_b200 import deepseek as ds
    s = ds.MoeShape(**MOE)
    store = zk.compose.Store()
    ops, x, out = ds.moe_layer(store, s)
    weights = zk.decode.quantise_weights(store, ops)
    zk.compose.forward_ops(store, ops)
    rows = lambda t: store.get(t).view(torch.int64).reshape(s.m, s.h)  # noqa: E731
    # the experts alone, many rows at once
    soft = next(op for op in ops if op.kind == "Softmax")
    silu = [op for op in ops if op.kind == "Lookup" and any(o.kind == "GeluIndex" and o.out == op.idx for o in ops)][0]
    block = ds.moe_block(store, ops, weights, soft.table, silu.table)
    h2 = [op for op in ops if op.kind == "RmsNorm"][2].out
    total, gate = block.forward(store.get(h2).reshape(s.m, s.h))
    assert torch.equal(total.view(torch.int64), rows(ops[-1].b))
    top = next(op for op in ops if op.kind == "TopKSelect")
    assert torch.equal(gate.view(torch.int64).reshape(-1), store.get(top.gate).view(torch.int64))
    # the whole layer, token by token (every sequence the same text)
    dec = ds.MoeLayerDecoder(store, ops, s, weights, batch)
    for i in range(s.m):
        got = dec.step(rows(x)[i:i + 1].expand(batch, s.h).contiguous().view(torch.uint64))
        assert torch.equal(got.view(torch.int64), rows(out)[i:i + 1].expand(batch, s.h)), i
    dec.check()


def test_calls_on_two_streams_and_replays(zk):
    """The same handles used from two streams at once, and from two captured
    graphs replayed in turn and together: no call's workspace is another's."""
    import torch
    d = zk.decode
    g = torch.Generator(device="cuda").manual_seed(3)
    codes = lambda *shape: torch.randint(-8, 8, shape, generator=g, device="cuda", dtype=torch.int8)  # noqa: E731
    scales = lambda *shape: torch.randint(100, 400, shape, generator=g, device="cuda", dtype=torch.int32)  # noqa: E731
    h, e, f, sh = 256, 16, 96, 160
    w = [d.QuantWeight(codes(e, h, f), scales(e, 4, f)), d.QuantWeight(codes(e, h, f), scales(e, 4, f)),
         d.QuantWeight(codes(e, f, h), scales(e, 2, h)), d.QuantWeight(codes(h, sh), scales(4, sh)),
         d.QuantWeight(codes(h, sh), scales(4, sh)), d.QuantWeight(codes(sh, h), scales(3, h))]
    field = lambda t: torch.where(t < 0, t - 0xFFFFFFFF, t).view(torch.uint64)  # noqa: E731
    ints = lambda lim, *shape: torch.randint(-lim, lim, shape, generator=g, device="cuda", dtype=torch.int64)  # noqa: E731
    exp = torch.round(torch.exp(torch.arange(-(1 << 20), 0, device="cuda", dtype=torch.float64) / 65536) * 65536).to(torch.int64)
    block = d.MoeBlock(field(ints(1000, h, e)), *w, exp.view(torch.uint64), field(ints(60000, 1 << 16)), 4)
    lin = d.QuantWeight(codes(h, 4000), scales(4, 4000))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def work(x):
        out, gate = block.forward(x, err=err)
        y = d.project(out, lin, 16, err=err)
        token, adjusted = d.choose_token(y, repeat=(1 << 15, 1 << 17), err=err)
        return [t.view(torch.int64) if t.dtype == torch.uint64 else t.view(torch.int32) for t in (out, gate, y, token, adjusted)]

    xs = [field(ints(1 << 17, m, h)) for m in (1, 5, 16, 3)]
    want = [[t.clone() for t in work(x)] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = []
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append(work(x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for u, v in zip(want, got) for a, b in zip(u, v))
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work(x))
        graphs.append(graph)
    for _ in range(5):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for u, v in zip(want, outs) for a, b in zip(u, v))
    assert int(err.item()) == 0
