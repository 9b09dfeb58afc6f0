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
