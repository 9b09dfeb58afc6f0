"""CPU checks of the single-token operators: the plain forms the GPU tests
compare with (tests/decode_ref.py) against the op graph's CPU restatement, and
the refusals of the C entry points and of the Python calls, which come before
any device work."""
import ctypes as C

import numpy as np
import pytest

from oracle import compose_oracle as co
from tests import decode_ref as ref


def _table(bits=20):
    return np.round(np.exp(np.arange(-(1 << bits), 0) / 65536.0) * 65536).astype(np.int64)


@pytest.mark.parametrize("m,heads,k,n", [(3, 1, 40, 24), (2, 3, 16, 8)])
def test_plain_project_is_the_projection_arm(zk, m, heads, k, n):
    """One segment: Projection, GeluIndex, Lookup and Add; several: the sum of
    a Projection per head."""
    rng, c = np.random.default_rng(k), zk.compose
    w = ref.weight(rng, heads * k, n, 32, k if heads > 1 else 0)
    x, bias, res = rng.integers(-(1 << 20), 1 << 20, (m, heads * k)), rng.integers(-5000, 5000, n), \
        rng.integers(-9000, 9000, (m, n))
    table = rng.integers(-30000, 30000, 1 << 12)
    st, dense = co.HostStore(), ref.dense(*w, 32, k if heads > 1 else 0)
    push = lambda a: st.push(ref.field(np.ascontiguousarray(a).reshape(-1)))  # noqa: E731
    ops, parts = [], []
    for h in range(heads):
        out, rem = st.push(None), st.push(None)
        b = np.tile(bias if h == 0 else np.zeros(n, dtype=np.int64), m)
        ops.append(c.Projection(push(x[:, h * k:(h + 1) * k]), push(dense[h * k:(h + 1) * k]), push(b), out, rem, m, k, n, 8))
        parts.append(out)
    acc = parts[0]
    for p in parts[1:]:
        s = st.push(None)
        ops.append(c.Add(acc, p, s))
        acc = s
    idx, act, total = st.push_idx(None), st.push(None), st.push(None)
    ops += [c.GeluIndex(acc, idx, 100, table.size), c.Lookup(idx, act, push(table)), c.Add(act, push(res), total)]
    co.forward_ops(st, ops)
    seg = k if heads > 1 else 0
    assert np.array_equal(ref.project(x, *w, 32, seg, 8, bias), ref.signed(st.get(acc)).reshape(m, n))
    assert np.array_equal(ref.project(x, *w, 32, seg, 8, bias, table, 100, res), ref.signed(st.get(total)).reshape(m, n))


def test_plain_attend_is_the_causal_rows(zk):
    rng, c = np.random.default_rng(2), zk.compose
    m, dk, dv, table = 16, 8, 12, _table()
    q, k, v = (rng.integers(-(1 << 18), 1 << 18, (m, d)) for d in (dk, dk, dv))
    st = co.HostStore()
    push = lambda a: st.push(ref.field(np.ascontiguousarray(a).reshape(-1)))  # noqa: E731
    s, s16, e, p, a, a16 = (st.push(None) for _ in range(6))
    idx = st.push_idx(None)
    mask = st.push(zk.gpt2.causal_mask(m))
    ops = [c.MatMul(push(q), push(k.T), s, m, dk, m), c.Scale(s, s16, 7519, 32),
           c.StableSoftmaxIndex(s16, mask, idx, table.size, table.size, m, m), c.Softmax(idx, e, p, push(table), m, m),
           c.MatMul(p, push(v), a, m, m, dv), c.Scale(a, a16, 1, 16)]
    co.forward_ops(st, ops)
    got = np.stack([ref.attend(q[i], k[:i + 1], v[:i + 1], table, (7519, 32)) for i in range(m)])
    assert np.array_equal(got, ref.signed(st.get(a16)).reshape(m, dv))


def test_plain_moe_is_the_graphs_layer(zk):
    """build_moe's rows, the routed and shared weights being 4-bit ones."""
    from zkie_b200 import deepseek as ds
    s = ds.MoeShape(m=4, h=32, heads=1, qk_nope=4, qk_rope=4, v_head=4, kv_lora=8, n_routed=8, top_k=2, moe=16, moe_real=12,
                    shared=32, shared_real=24, exp_bits=20, silu_bits=14, w_mod=1 << 12)
    st = co.HostStore()
    ops, _, _ = ds.moe_layer(st, s)
    rng = np.random.default_rng(6)
    top = next(i for i, op in enumerate(ops) if op.kind == "TopKSelect")
    experts = [op for op in ops if op.kind == "GatherMatMul"]
    shared = [op for op in ops[top:] if op.kind == "Projection"]
    weights = []
    for op in experts + shared:
        n = s.n_routed if op.kind == "GatherMatMul" else 0
        w = ref.weight(rng, op.k, op.n, 32, experts=n)
        dense = np.stack([ref.dense(w[0][e], w[1][e], 32) for e in range(n)]) if n else ref.dense(*w, 32)
        st.v[op.w] = ref.field(dense.reshape(-1))
        weights.append(w)
    co.forward_ops(st, ops)
    norm = [op for op in ops if op.kind == "RmsNorm"][2]
    x = ref.signed(st.get(norm.out)).reshape(s.m, s.h)
    router = ref.signed(st.get(ops[top - 4].b)).reshape(s.h, s.n_routed)
    soft = ops[top - 1].table
    silu = next(op.table for op in ops if op.kind == "Lookup" and any(o.kind == "GeluIndex" and o.out == op.idx for o in ops))
    out, gate = ref.moe(x, router, weights, 32, ref.signed(st.get(soft)), ref.signed(st.get(silu)), s.top_k)
    assert np.array_equal(gate.reshape(-1), ref.signed(st.get(ops[top].gate)))
    assert np.array_equal(out, ref.signed(st.get(ops[-1].b)).reshape(s.m, s.h))


def test_plain_choose_is_the_masked_argmax(zk):
    rng, c = np.random.default_rng(3), zk.compose
    m, v = 5, 70
    logits = rng.integers(-(1 << 30), 1 << 30, (m, v))
    logits[0] = 7
    mask = np.where(np.arange(v) < 61, 0, -(1 << 41))
    st = co.HostStore()
    push = lambda a: st.push(ref.field(np.ascontiguousarray(a).reshape(-1)))  # noqa: E731
    sel, thr, gate, d1, d2, masked = (st.push(None) for _ in range(6))
    out = st.push_idx(None)
    co.forward_ops(st, [c.Add(push(logits), push(np.tile(mask, m)), masked), c.Argmax(masked, sel, thr, gate, d1, d2, out, m, v)])
    words = np.packbits(np.arange(96) < 61, bitorder="little").view(np.int32)
    token, got = ref.choose(logits, allowed=words)
    assert np.array_equal(token, st.idx[out]) and np.array_equal(got, ref.signed(st.get(masked)).reshape(m, v))


def test_cache_blocks_round_trip():
    keys = np.random.default_rng(1).integers(-99, 99, (2, 3, 64, 12))
    blocks = ref.blocks_of(keys)
    assert blocks.shape == (2, 3, 2, 3, 32, 4) and np.array_equal(ref.keys_of(blocks), keys)


# ---- refusals ---------------------------------------------------------------------------------------
A = 1 << 20  # an address: aligned, never used by a refused call


def test_packed_sizes(zk):
    words = zk.lib.zkie2_q4_words
    # tiles of 16 columns, blocks of 64 rows: 512 bytes of codes and 32 (two groups: 64) of scales
    assert words(1, 64, 16, 64, 0) == 136 and words(1, 64, 16, 32, 0) == 144 and words(1, 65, 17, 128, 0) == 4 * 136
    assert words(3, 60, 5, 64, 20) == 3 * 3 * 136 and words(1, 8192, 16, 64, 0) == 128 * 136
    for bad in ((0, 64, 16, 64, 0), (1, 0, 16, 64, 0), (1, 64, 0, 64, 0), (1, 64, 16, 48, 0), (1, 64, 16, 64, 60),
                (1, 64, 16, 64, 65), (1, 8193, 16, 64, 0), (1, 4096, 16, 64, 20), (4097, 64, 16, 64, 0)):
        assert words(*bad) == 0, bad
    assert zk.lib.zkie2_moe_router_words(100, 17) == 2 * 2 * 512
    assert zk.lib.zkie2_moe_router_words(100, 257) == 0 and zk.lib.zkie2_moe_router_words(8193, 8) == 0


def _refused(fn, good, changes):
    for change in changes:
        args = list(good)
        for i, v in change.items():
            args[i] = v
        assert fn(*args) != 0, change


def test_project_refusals(zk):
    good = (A, 64, 2, A, 64, 16, 64, 0, 16, None, None, 0, 0, None, 0, A, A, None)
    _refused(zk.lib.zkie2_q4_project, good, [
        {0: None}, {1: 63}, {2: 65536}, {3: None}, {3: A + 8}, {4: 0}, {4: 8193}, {5: 0}, {6: 16}, {7: 48}, {8: 63},
        {10: A, 11: 0}, {13: A, 14: 15}, {15: None}, {16: None}])
    assert zk.lib.zkie2_q4_project(A, 64, 0, A, 64, 16, 64, 0, 16, None, None, 0, 0, None, 0, A, A, None) == 0
    _refused(zk.lib.zkie2_q4_pack, (A, A, 1, 64, 16, 64, 0, A, A, None), [{0: None}, {2: 0}, {3: 0}, {5: 65}, {7: None}, {8: None}])
    _refused(zk.lib.zkie2_q4_pair, (A, A, 1, 64, 16, 64, A, None), [{0: None}, {1: A + 4}, {2: 0}, {6: None}])


def test_cache_refusals(zk):
    good = [A, 64, A, 64, 5, 1, 0, A, A, A, 2, 4, 16, 16, 64, A, None]
    _refused(zk.lib.zkie2_kv_append, good, [
        {0: None}, {1: 63}, {3: 63}, {4: (1 << 17) + 1}, {6: 63}, {7: None}, {8: None}, {9: None}, {10: 0}, {11: 0}, {12: 0},
        {12: 18}, {12: 260}, {13: 6}, {14: 0}, {14: 48 + 1}, {14: (1 << 17) + 32}, {15: None}])
    good = [A, 64, 4, 1, 0, A, 64, A, 64, 1, 0, A, A, A, 2, 4, 16, 16, 64, 1, 16, A, 256, 256, 16, A, A, None]
    _refused(zk.lib.zkie2_kv_attend, good, [
        {0: None}, {1: 63}, {2: 0}, {2: 6}, {4: 63}, {5: None}, {6: 63}, {7: None}, {8: 60}, {10: 63}, {11: None}, {11: A + 4},
        {12: None}, {12: A + 8}, {13: None}, {14: 0}, {15: 0}, {16: 6}, {16: 300}, {17: 2}, {18: 40}, {20: 63}, {21: None},
        {22: 0}, {24: 63}, {25: None}, {26: None}])


def test_moe_refusals(zk):
    w = (C.c_void_p * 4)(A, A, A, A)
    hole = (C.c_void_p * 4)(A, None, A, A)
    good = [A, 64, 2, 64, 8, 2, 32, 48, 64, A, w, A, 256, A, 256, 16, None, 0, A, A, A, A, None]
    _refused(zk.lib.zkie2_moe_rows, good, [
        {0: None}, {1: 63}, {2: 65536}, {3: 0}, {3: 8193}, {4: 0}, {4: 257}, {5: 0}, {5: 9}, {4: 64, 5: 17}, {6: 0}, {7: 8200},
        {8: 63}, {9: None}, {9: A + 4}, {10: hole}, {11: None}, {12: 0}, {13: None}, {14: 0}, {15: 63}, {16: A, 17: 63},
        {18: None}, {20: None}, {21: None}, {21: A + 8}])
    scratch = zk.lib.zkie2_moe_rows_scratch_elems
    assert scratch(1, 64, 8, 2, 32, 48, 64) > 0 and scratch(17, 64, 8, 2, 32, 48, 64) == scratch(16, 64, 8, 2, 32, 48, 64)
    assert scratch(1, 64, 8, 9, 32, 48, 64) == 0 and scratch(0, 64, 8, 2, 32, 48, 64) == 0
    _refused(zk.lib.zkie2_moe_router_pack, (A, 64, 8, A, A, None), [{0: None}, {1: 0}, {2: 0}, {3: None}, {4: None}])


def test_choose_refusals(zk):
    good = [A, 2, 100, A, 5, A, 1, 1, 0, 0, None, 0, None, 0, 0, A, A, A, None]
    _refused(zk.lib.zkie2_choose_token, good, [
        {0: None}, {1: 65536}, {2: 0}, {2: 1 << 31}, {3: None}, {4: 1 << 31}, {15: None}, {16: None}, {17: None}])


def test_python_refuses_host_tensors(zk):
    import torch
    d = zk.decode
    x, err = torch.zeros((2, 64), dtype=torch.uint64), torch.zeros(1, dtype=torch.int32)

    class Weight:  # stands for a QuantWeight: never reached
        call = (0, A, 64, 16, 64, 0, 1)
    for call in (lambda: d.project(x, Weight(), 16, err=err), lambda: d.choose_token(x, err=err),
                 lambda: d.project([1], Weight(), 16, err=err),
                 lambda: d.KvCache(torch.zeros((1, 1, 1, 1, 32, 4), dtype=torch.int32),
                                   torch.zeros((1, 1, 32, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError, match="CUDA device is wanted"):
            call()
