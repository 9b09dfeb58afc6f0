"""CPU checks of the single-token decoders at other shapes than the models'
own: what they take from a graph, and what they refuse."""
import numpy as np
import pytest

from oracle import compose_oracle as co
from tests import decode_ref as ref, decode_shapes as ds_ref


@pytest.mark.parametrize("shift", [10, 14, 16, 18])
def test_plain_moe_with_the_graphs_shifts(zk, shift):
    """build_moe at another shift: the shared experts' Projections have it, everything else 2^16."""
    st = co.HostStore()
    s, ops, weights, top = ds_ref.moe_graph(zk, st, np.random.default_rng(6), m=4, h=32, heads=1, qk_nope=4, qk_rope=4, v_head=4,
                                            kv_lora=8, n_routed=8, top_k=2, moe=16, moe_real=12, shared=32, shared_real=24,
                                            silu_bits=14, w_mod=1 << 12, shift=shift)
    co.forward_ops(st, ops)
    norm = [op for op in ops if op.kind == "RmsNorm"][2]
    x = ref.signed(st.get(norm.out)).reshape(s.m, s.h)
    router = ref.signed(st.get(ops[top - 4].b)).reshape(s.h, s.n_routed)
    silu = next(op.table for op in ops if op.kind == "Lookup" and any(o.kind == "GeluIndex" and o.out == op.idx for o in ops))
    out, gate = ds_ref.moe(x, router, weights, 32, ref.signed(st.get(ops[top - 1].table)), ref.signed(st.get(silu)), s.top_k, shift)
    assert np.array_equal(gate.reshape(-1), ref.signed(st.get(ops[top].gate)))
    assert np.array_equal(out, ref.signed(st.get(ops[-1].b)).reshape(s.m, s.h))


def _block_of(zk, monkeypatch, **shape):
    """moe_block on a host store, the device's classes replaced: (graph's shape, call of moe_block)."""
    from zkie_b200 import deepseek as ds
    st = co.HostStore()
    s, ops, weights, top = ds_ref.moe_graph(zk, st, np.random.default_rng(1), **shape)
    read = [op for op in ops if op.kind == "GatherMatMul"] + [op for op in ops[top:] if op.kind == "Projection"]
    given = {op.w: (*w, 32) for op, w in zip(read, weights)}
    monkeypatch.setattr(zk.decode, "QuantWeight", lambda *a: a)
    monkeypatch.setattr(zk.decode, "MoeBlock", lambda *a: a)
    silu = next(op.table for op in ops if op.kind == "Lookup" and any(o.kind == "GeluIndex" and o.out == op.idx for o in ops))
    return s, ops, lambda *a: ds.moe_block(st, ops, given, ops[top - 1].table, silu, *a)


def test_moe_block_takes_the_graphs_shift(zk, monkeypatch):
    s, _, block = _block_of(zk, monkeypatch, m=4, shift=14)
    assert block()[-1] == 14 and block()[-2] == s.top_k and block(14)[-1] == 14
    with pytest.raises(ValueError, match="shift"):
        block(16)


@pytest.mark.parametrize("kind,field,value", [("Scale", "shift", 15), ("Scale", "factor", 2), ("ScaleVec", "shift", 14)])
def test_moe_block_refuses_other_scales(zk, monkeypatch, kind, field, value):
    """A graph whose router or experts divide by something else than the kernels do."""
    _, ops, block = _block_of(zk, monkeypatch, m=4)
    block()
    top = next(i for i, op in enumerate(ops) if op.kind == "TopKSelect")
    for op in [op for op in ops[top - 4:] if op.kind == kind]:
        was = getattr(op, field)
        setattr(op, field, value)
        with pytest.raises(ValueError, match="build_moe"):
            block()
        setattr(op, field, was)
    block()


# ---- tables with which a causal graph's masked columns would count ------------------------------------
def test_masked_columns_count_where_the_table_does_not_begin_with_zero(zk):
    """Why the decoders want a table that does: the graph's row counts table[0]
    for every later position, attention over a cache knows none of them."""
    rng, c, m = np.random.default_rng(2), zk.compose, 8
    rows = {}
    for bits in (19, 20, 21):
        table = ref.signed(zk.gpt2.exp_table(bits))
        st = co.HostStore()
        push = lambda a: st.push(ref.field(np.ascontiguousarray(a).reshape(-1)))  # noqa: E731
        z, idx, e, p = rng.integers(-(1 << 18), 1 << 18, (m, m)), st.push_idx(None), st.push(None), st.push(None)
        co.forward_ops(st, [c.StableSoftmaxIndex(push(z), st.push(zk.gpt2.causal_mask(m)), idx, table.size, table.size, m, m),
                            c.Softmax(idx, e, p, push(table), m, m)])
        got = ref.signed(st.get(p)).reshape(m, m)
        rows[bits] = all(np.array_equal(got[i, :i + 1], ref.softmax(z[i, :i + 1], table)) for i in range(m))
        assert (table[0] == 0) == rows[bits]
    assert rows == {19: False, 20: True, 21: True}


def _gpt2_ops(zk, **shape):
    s = zk.gpt2.LayerShape(**{**ds_ref.GPT2, **shape})
    st = co.HostStore()
    return st, zk.gpt2.gpt2_model(st, s, layers=1)[0], s


def _moe_ops(zk, **shape):
    from zkie_b200 import deepseek as ds
    s = ds.MoeShape(**{**ds_ref.MOE, **shape})
    st = co.HostStore()
    return st, ds.moe_layer(st, s)[0], s


def test_decoders_refuse_a_table_that_does_not_begin_with_zero(zk):
    """Before anything else: no device is needed."""
    from zkie_b200 import deepseek as ds
    for bits in (16, 19):
        with pytest.raises(ValueError, match="begins with zero"):
            zk.gpt2.Gpt2Decoder(*_gpt2_ops(zk, exp_bits=bits), {})
        with pytest.raises(ValueError, match="begins with zero"):
            ds.MoeLayerDecoder(*_moe_ops(zk, exp_bits=bits), {})


@pytest.mark.parametrize("change", [dict(shift=14), dict(exp_bits=21), dict(gelu_bits=20), dict(d_real=40), dict(vocab_real=499),
                                    dict(m=32), dict(d=32), dict(dh=8), dict(heads=2), dict(ffn=64), dict(vocab=256)])
def test_gpt2_decoder_refuses_another_shape(zk, change):
    """A shape that is not the graph's would compute other rows."""
    import dataclasses
    st, ops, s = _gpt2_ops(zk, exp_bits=20, gelu_bits=18)
    with pytest.raises(ValueError, match="shape"):
        zk.gpt2.Gpt2Decoder(st, ops, dataclasses.replace(s, **change), {})


@pytest.mark.parametrize("change", [dict(shift=14), dict(exp_bits=21), dict(m=16), dict(h=64), dict(heads=1), dict(qk_nope=8),
                                    dict(qk_rope=4), dict(v_head=8), dict(kv_lora=16)])
def test_moe_decoder_refuses_another_shape(zk, change):
    import dataclasses
    from zkie_b200 import deepseek as ds
    st, ops, s = _moe_ops(zk)
    with pytest.raises(ValueError, match="shape"):
        ds.MoeLayerDecoder(st, ops, dataclasses.replace(s, **change), {})


def test_decoders_know_their_shapes(zk):
    from zkie_b200 import deepseek as ds
    for change in (dict(), dict(vocab_real=512), dict(heads=1, dh=48), dict(shift=9, gelu_bits=12, exp_bits=20)):
        assert zk.gpt2.Gpt2Decoder._shaped(*_gpt2_ops(zk, **change))
    for change in (dict(), dict(heads=1), dict(shift=12, moe=48, top_k=1)):
        _, ops, s = _moe_ops(zk, **change)
        assert ds.MoeLayerDecoder._shaped(ops, s)


# ---- rows of a step -----------------------------------------------------------------------------------
def test_moe_decoder_refuses_other_rows(zk):
    """Fewer rows than sequences would be read past their end: refused before
    anything is enqueued (no device is needed)."""
    import torch
    from zkie_b200 import deepseek as ds
    dec = object.__new__(ds.MoeLayerDecoder)
    dec.s, dec.batch = ds.MoeShape(**ds_ref.MOE), 3
    for x in (torch.zeros((3, 128), dtype=torch.uint64), torch.zeros((2, 128), dtype=torch.uint64), torch.zeros(384, dtype=torch.uint64),
              torch.zeros((3, 128), dtype=torch.int64), torch.zeros((3, 64), dtype=torch.uint64), [0]):
        with pytest.raises(ValueError, match="MoeLayerDecoder: x"):
            dec.step(x)


# ---- quantising a store --------------------------------------------------------------------------------
class _TorchStore:
    def __init__(self):
        self.v = []

    def push(self, a):
        import torch
        self.v.append(torch.from_numpy(ref.field(np.asarray(a).reshape(-1))))
        return len(self.v) - 1

    def get(self, t):
        return self.v[t]


def test_quantise_weights_all_or_none(zk):
    """A weight that has no 4-bit form leaves the store as it was, with the
    weights before it as they were."""
    import torch
    c = zk.compose
    rng, st = np.random.default_rng(3), _TorchStore()
    a, b = st.push(rng.integers(-9000, 9000, (32, 8))), st.push(np.full((32, 8), 1 << 21))
    ops = [c.Projection(0, t, 0, 2, 3, 1, 32, 8, 16) for t in (a, b)]
    before = [t.clone() for t in st.v]
    with pytest.raises(ValueError, match="65535"):
        zk.decode.quantise_weights(st, ops, group=32)
    assert all(torch.equal(x.view(torch.int64), y.view(torch.int64)) for x, y in zip(st.v, before))
    done = zk.decode.quantise_weights(st, ops[:1], group=32)
    assert list(done) == [a] and np.array_equal(ref.signed(st.v[a].numpy()).reshape(32, 8),
                                                ref.dense(*[t.numpy() for t in done[a][:2]], 32))


def test_quantise_weights_in_the_stores_own_memory(zk):
    """A recorded forward or prover has the addresses of the Store's tensors:
    they stay, and hold the new numbers."""
    import torch
    c, rng, st = zk.compose, np.random.default_rng(4), _TorchStore()
    a, b = st.push(rng.integers(-9000, 9000, (32, 8))), st.push(rng.integers(-9000, 9000, (3, 40, 8)))
    ops = [c.Projection(9, a, 9, 7, 8, 1, 32, 8, 16), c.GatherMatMul(9, 0, b, 8, 1, 40, 8, 3)]
    held = list(st.v)
    done = zk.decode.quantise_weights(st, ops, group=32)
    for t in (a, b):
        assert st.v[t] is held[t]
        codes, scales = (x.numpy() for x in done[t][:2])
        want = ref.dense(codes, scales, 32) if t == a else np.stack([ref.dense(codes[e], scales[e], 32) for e in range(3)])
        assert np.array_equal(ref.signed(held[t].numpy()), want.reshape(-1))
    st.v.append(st.v[a][:64])  # another id for part of the same memory
    with pytest.raises(ValueError, match="share memory"):
        zk.decode.quantise_weights(st, [ops[0], c.Projection(9, 2, 9, 7, 8, 1, 8, 8, 16)], group=32)


def test_decoders_refuse_other_graphs(zk):
    """Graphs of other builders, and parts of their own."""
    from zkie_b200 import deepseek as ds
    st, ops, s = _gpt2_ops(zk)
    _, moe, ms = _moe_ops(zk)
    layer = zk.gpt2.gpt2_layer(co.HostStore(), s)[0]
    reference = zk.gpt2.reference_layer_roundtrip_case(co.HostStore(), zk.XorShift64)[0]
    kinds = sorted({op.kind for op in ops})
    for other in (layer, reference, moe, [], *[[op for op in ops if op.kind != k] for k in kinds if k not in ("Transpose", "MatMul", "Softmax")]):
        with pytest.raises(ValueError, match="shape"):
            zk.gpt2.Gpt2Decoder(st, other, s, {})
    for other in (ops, layer, [], *[[op for op in moe if op.kind != k] for k in ("Projection", "RmsNorm", "RoPE", "Scale")]):
        with pytest.raises(ValueError, match="shape"):
            ds.MoeLayerDecoder(st, other, ms, {})


def _changed(st, t, at):
    """The store with one word of a tensor changed; put back by calling what it returns."""
    old = st.v[t]
    st.v[t] = old.copy()
    st.v[t][at] = (int(old[at]) + 1) % ref.P
    return lambda: st.v.__setitem__(t, old)


def test_decoders_refuse_tensors_they_do_not_compute_with(zk, monkeypatch):
    """Norms and biases that differ from row to row, biases where a model has
    none, other masks than the causal one: the steps would leave them out."""
    from zkie_b200 import deepseek as ds
    st, ops, s = _gpt2_ops(zk)
    first = lambda ops, kind, i=0: [op for op in ops if op.kind == kind][i]  # noqa: E731
    assert zk.gpt2.Gpt2Decoder._filled(st, ops, s)
    for t, at in ((first(ops, "LayerNormCentered").w, s.d), (first(ops, "LayerNormCentered", 2).b, 3), (first(ops, "Projection").bias, 20),
                  (first(ops, "Projection", 3).bias, 0), (first(ops, "Projection", 7).bias, -1), (first(ops, "Projection", -1).bias, s.d + 1),
                  (first(ops, "StableSoftmaxIndex").mask, 0)):
        back = _changed(st, t, at)
        with pytest.raises(ValueError, match="biases or masks"):
            zk.gpt2.Gpt2Decoder(st, ops, s, {})
        back()
    assert zk.gpt2.Gpt2Decoder._filled(st, ops, s)
    st, ops, s = _moe_ops(zk)
    for t, at in ((first(ops, "RmsNorm").w, s.h), (first(ops, "RmsNorm", 2).w, 1), (first(ops, "Projection").bias, 5),
                  (first(ops, "Projection", 6).bias, 0), (first(ops, "Projection", -1).bias, 9), (first(ops, "StableSoftmaxIndex").mask, 1)):
        back = _changed(st, t, at)
        with pytest.raises(ValueError, match="biases or masks"):
            ds.MoeLayerDecoder(st, ops, s, {})
        back()
    monkeypatch.setattr(zk.decode, "QuantWeight", lambda *a: a)
    monkeypatch.setattr(zk.decode, "MoeBlock", lambda *a: a)
    top = next(i for i, op in enumerate(ops) if op.kind == "TopKSelect")
    given = {op.w: () for op in ops if op.kind in ("GatherMatMul", "Projection")}
    block = lambda: ds.moe_block(st, ops, given, ops[top - 1].table, ops[top - 1].table)  # noqa: E731
    block()
    for t, at in ((ops[top - 2].mask, 7), (first(ops, "Projection", -3).bias, 0), (first(ops, "Projection", -1).bias, -1)):
        back = _changed(st, t, at)
        with pytest.raises(ValueError, match="build_moe"):
            block()
        back()
    block()
