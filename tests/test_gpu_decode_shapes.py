"""The single-token decoders on the device at other shapes than the models'
own: bit for bit the graph's rows, or a refusal."""
import numpy as np
import pytest

from tests import decode_ref as ref, decode_shapes as ds_ref
from tests.test_gpu_decode import _moe_case, _quant, _s, _u

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", [0, 9, 14, 20])
@pytest.mark.parametrize("m,h,experts,top_k,f,shared,group", [
    (1, 64, 8, 2, 48, 96, 64), (3, 100, 17, 3, 40, 33, 32), (17, 64, 4, 4, 32, 16, 128)])
def test_moe_block_shared_shift(zk, m, h, experts, top_k, f, shared, group, shift):
    """The shift is the shared experts' Projections'; small numbers, so that a
    shift of none keeps them in range."""
    rng = np.random.default_rng(m + shift)
    router, w = _moe_case(rng, h, experts, f, shared, group)
    if shift < 12:  # |gate|, |up| of the shared experts below 2^22, silu(gate) up / 2^16 below 2^31
        w[3:] = [(c, np.minimum(s, 1)) for c, s in w[3:]]
    x = rng.integers(-(1 << (17 if shift >= 12 else 10)), 1 << (17 if shift >= 12 else 10), (m, h))
    exp, silu = ds_ref.exp_table(), ds_ref.silu_table()
    block = zk.decode.MoeBlock(_u(router), *[_quant(zk, t, group) for t in w], _u(exp), _u(silu), top_k, shift)
    out, gate = block.forward(_u(x))
    want, want_gate = ds_ref.moe(x, router, w, group, exp, silu, top_k, shift)
    assert np.array_equal(_s(gate), want_gate)
    assert np.array_equal(_s(out), want)


@pytest.mark.parametrize("shift", [13, 14, 18])
def test_moe_layer_steps_equal_the_graph_at_other_shifts(zk, shift):
    import torch
    from zkie_b200 import deepseek as ds
    s = ds.MoeShape(**ds_ref.MOE, shift=shift)
    store = zk.compose.Store()
    ops, x, out = ds.moe_layer(store, s)
    weights = zk.decode.quantise_weights(store, ops)
    zk.compose.forward_ops(store, ops)
    rows = lambda t: store.get(t).view(torch.int64).reshape(s.m, s.h)  # noqa: E731
    dec = ds.MoeLayerDecoder(store, ops, s, weights, 2)
    for i in range(s.m):
        got = dec.step(rows(x)[i:i + 1].expand(2, s.h).contiguous().view(torch.uint64))
        assert torch.equal(got.view(torch.int64), rows(out)[i:i + 1].expand(2, s.h)), i
    dec.check()


# ---- numbers at which attention, norms and experts count ------------------------------------------
@pytest.mark.parametrize("shift,group", [(16, 32), (16, 128), (14, 64), (17, 64)])
def test_gpt2_steps_equal_the_graph_where_attention_counts(zk, shift, group):
    """Every position's logits and choice, two sequences at different places."""
    import torch
    s = zk.gpt2.LayerShape(**ds_ref.GPT2, shift=shift)
    store = zk.compose.Store()
    ops, tok, out = zk.gpt2.gpt2_model(store, s, layers=2)
    ds_ref.liven(store, ops)
    weights = zk.decode.quantise_weights(store, ops, ("Projection", "MatMul"), group)
    zk.compose.forward_ops(store, ops)
    logits = store.get(next(op for op in ops if op.kind == "Argmax").x).view(torch.int64).reshape(s.m, s.vocab)
    tokens, argmax = store.get_idx(tok).view(torch.int32), store.get_idx(out).view(torch.int32)
    assert len(set(argmax.tolist())) > 20
    dec = zk.gpt2.Gpt2Decoder(store, ops, s, weights, batch=2)
    dec.load(store, 1, 13)
    for i in range(s.m - 13):
        at = [i, 13 + i]
        dec.tokens.copy_(tokens[at].view(torch.uint32))
        token, got = dec.step()
        assert torch.equal(got.view(torch.int64), logits[at]), i
        assert torch.equal(token.view(torch.int32), argmax[at]), i
    dec.check()


@pytest.mark.parametrize("shift", [14, 16])
def test_moe_layer_steps_equal_the_graph_where_attention_counts(zk, shift):
    """Three sequences over one text, begun at different steps."""
    import torch
    from zkie_b200 import deepseek as ds
    s = ds.MoeShape(**ds_ref.MOE, shift=shift)
    store = zk.compose.Store()
    ops, x, out = ds.moe_layer(store, s)
    ds_ref.liven(store, ops)
    weights = zk.decode.quantise_weights(store, ops)
    zk.compose.forward_ops(store, ops)
    rows = lambda t: store.get(t).view(torch.int64).reshape(s.m, s.h)  # noqa: E731
    dec = ds.MoeLayerDecoder(store, ops, s, weights, 3)
    first = [0, 3, 4]
    for i in range(s.m):
        at = [max(i - f, 0) for f in first]
        dec.cache.lens.copy_(torch.tensor(at))
        got = dec.step(rows(x)[at].view(torch.uint64))
        assert torch.equal(got.view(torch.int64), rows(out)[at]), i
    dec.check()


def test_gpt2_at_its_own_shape(zk):
    """Two layers of GPT-2's graph (1024 wide, 65536 logits, 512 positions):
    three sequences, from empty, within and at the end of the text."""
    import torch
    s, store = zk.gpt2.GPT2_SMALL, zk.compose.Store()
    ops, tok, out = zk.gpt2.gpt2_model(store, s, layers=2)
    ds_ref.liven(store, ops, 2500)
    weights = zk.decode.quantise_weights(store, ops, ("Projection", "MatMul"))
    zk.compose.forward_ops(store, ops)
    logits = store.get(next(op for op in ops if op.kind == "Argmax").x).view(torch.int64).reshape(s.m, s.vocab)
    tokens, argmax = store.get_idx(tok).view(torch.int32), store.get_idx(out).view(torch.int32)
    dec, start = zk.gpt2.Gpt2Decoder(store, ops, s, weights, batch=3), [0, 200, 502]
    for b in range(3):
        dec.load(store, b, start[b])
    for i in range(10):
        at = [a + i for a in start]
        dec.tokens.copy_(tokens[at].view(torch.uint32))
        token, got = dec.step()
        assert torch.equal(got.view(torch.int64), logits[at]) and torch.equal(token.view(torch.int32), argmax[at]), i
    dec.check()
    assert len(set(argmax.tolist())) > 400


def test_moe_layer_at_its_own_shape(zk):
    """DeepSeek-V2-Lite's layer (2048 wide, 64 experts, 512 positions), its
    first positions past a block of the cache."""
    import torch
    from zkie_b200 import deepseek as ds
    s, store = ds.DSV2_LITE, zk.compose.Store()
    ops, x, out = ds.moe_layer(store, s)
    ds_ref.liven(store, ops, 2500)
    weights = zk.decode.quantise_weights(store, ops)
    zk.compose.forward_ops(store, ops)
    rows = lambda t: store.get(t).view(torch.int64).reshape(s.m, s.h)  # noqa: E731
    dec = ds.MoeLayerDecoder(store, ops, s, weights, 2)
    for i in range(40):
        got = dec.step(rows(x)[[i, i]].view(torch.uint64))
        assert torch.equal(got.view(torch.int64), rows(out)[[i, i]]), i
    dec.check()


@pytest.mark.parametrize("token", [500, 512, 517, 1023, 512 * 63, 1 << 31, (1 << 32) - 1])
def test_gpt2_tokens_outside_the_vocabulary(zk, token):
    """Said at the step: the embedding's last dimension, or its first, lies
    outside the table.  (From vocab_real to vocab the graph's padding is a
    token like any other.)"""
    import torch
    s, store = zk.gpt2.LayerShape(**ds_ref.GPT2), zk.compose.Store()
    ops, _, _ = zk.gpt2.gpt2_model(store, s, layers=1)
    dec = zk.gpt2.Gpt2Decoder(store, ops, s, zk.decode.quantise_weights(store, ops, ("Projection", "MatMul")), batch=2)
    dec.tokens.copy_(torch.tensor([3, token], dtype=torch.int64).to(torch.uint32))
    dec.step()
    if token < s.vocab:
        dec.check()
    else:
        with pytest.raises(ValueError, match="index outside"):
            dec.check()
    dec.step()  # the next tokens are its own
    dec.check()


# ---- what the decoders refuse -----------------------------------------------------------------------
def test_decoders_refuse_a_table_that_does_not_begin_with_zero(zk):
    """A table of 2^19 entries begins with 22, which the graph counts for every masked column."""
    from zkie_b200 import deepseek as ds
    store = zk.compose.Store()
    s = zk.gpt2.LayerShape(**ds_ref.GPT2, exp_bits=19)
    ops, _, _ = zk.gpt2.gpt2_model(store, s, layers=1)
    with pytest.raises(ValueError, match="begins with zero"):
        zk.gpt2.Gpt2Decoder(store, ops, s, zk.decode.quantise_weights(store, ops, ("Projection", "MatMul")))
    store = zk.compose.Store()
    s = ds.MoeShape(**{**ds_ref.MOE, "exp_bits": 19})
    ops, _, _ = ds.moe_layer(store, s)
    with pytest.raises(ValueError, match="begins with zero"):
        ds.MoeLayerDecoder(store, ops, s, zk.decode.quantise_weights(store, ops))


# ---- one call after another over the same memory ---------------------------------------------------
@pytest.mark.parametrize("captured", [False, True])
def test_a_chain_over_reused_memory(zk, captured):
    """Projection -> attention -> projection onto the residual in place -> choice,
    every result written over memory that the call before last read: the same
    numbers as with memory of their own."""
    import torch
    d = zk.decode
    rng = np.random.default_rng(8)
    b, heads, dh, width, vocab, cap = 3, 4, 32, 128, 600, 96
    qkv, o, up, lm = (_quant(zk, ref.weight(rng, k, n, 32, seg, most=60), 32, seg) for k, n, seg in
                      ((width, 3 * heads * dh, 0), (heads * dh, width, dh), (width, width, 0), (width, vocab, 0)))
    table, bias = _u(ds_ref.exp_table()), _u(rng.integers(-9000, 9000, vocab))
    gelu, start = _u(rng.integers(-60000, 60000, 1 << 12)), _u(rng.integers(-(1 << 17), 1 << 17, (b, width)))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    steps, hd = 24, heads * dh
    pool = torch.zeros(4 * b * vocab, dtype=torch.int64, device="cuda").view(torch.uint64)
    at = lambda off, n: pool[off:off + b * n].reshape(b, n)  # noqa: E731

    def run(x, cache, reuse):
        place = (lambda off, n: at(off, n)) if reuse else (lambda off, n: None)
        said, x = [], x.clone()
        for i in range(steps):
            r = d.project(x, qkv, 12, out=place(0, 3 * hd), err=err)
            a = d.attend(r[:, :hd], cache, table, k=r[:, hd:2 * hd], v=r[:, 2 * hd:], score_scale=(11585, 32),
                         out=place(b * 3 * hd, hd), err=err)
            x = d.project(a, o, 12, residual=x, out=x if reuse else None, err=err)
            u = d.project(x, up, 12, table=gelu, out=place(0, width), err=err)  # over the queries
            x = d.project(u, up, 12, residual=x, out=x if reuse else None, err=err)
            l = d.project(x, lm, 0, out=place(b * width, vocab), err=err)       # over keys and attention
            token, y = d.choose_token(l, bias=bias, out=place(b * (width + vocab), vocab), err=err)
            cache.advance()
            said += [t.view(torch.int32 if t.dtype == torch.uint32 else torch.int64).clone() for t in (token, y, x)]
        return said

    new = lambda: d.KvCache.zeros(b, heads, dh, dh, cap)  # noqa: E731
    want = run(start, new(), False)
    if captured:
        cache = new()
        run(start, cache, True)
        cache.lens.zero_()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(start, cache, True)
        for _ in range(3):
            cache.lens.zero_()
            graph.replay()
            assert all(torch.equal(p, q) for p, q in zip(want, got))
    else:
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(want, run(start, new(), True)))
    assert int(err.item()) == 0 and len({int(t[0]) for t in want[::3]}) > 3
