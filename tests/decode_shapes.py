"""What the tests of the single-token decoders at other shapes share: a small
MoE layer, and its plain form with the shifts that build_moe has -- 2^16 in the
router's Scale, the routed products' and every ScaleVec, the graph's own shift
in the shared experts' Projections."""
import numpy as np

from tests import decode_ref as ref

# an exp table of 2^20 entries: its first entry is zero, so masked columns do not count
MOE = dict(m=32, h=128, heads=2, qk_nope=16, qk_rope=8, v_head=16, kv_lora=32, n_routed=16, top_k=3, moe=64,
           moe_real=48, shared=128, shared_real=96, exp_bits=20, silu_bits=20, w_mod=1 << 8)
GPT2 = dict(m=64, d=64, d_real=48, heads=3, dh=16, ffn=128, ffn_real=96, vocab=512, vocab_real=500)


def exp_table(bits=20):
    return np.round(np.exp(np.arange(-(1 << bits), 0) / 65536.0) * 65536).astype(np.int64)


def silu_table(bits=20):
    x = (np.arange(1 << bits) - (1 << (bits - 1))) / 65536.0
    return np.round(x / (1 + np.exp(-x)) * 65536).astype(np.int64)


def moe(x, router, weights, group, exp, silu, top_k, shared_shift):
    """weights: six (codes, scales), the first three with a leading expert axis."""
    def feed(row, g, u, d, shift):
        half = silu.size // 2
        a = silu[np.clip(ref.round_shift(ref.product(row, ref.dense(*g, group)), shift) + half, 0, silu.size - 1)]
        act = ref.round_shift(a * ref.round_shift(ref.product(row, ref.dense(*u, group)), shift), 16)
        return ref.round_shift(ref.product(act, ref.dense(*d, group)), shift)

    m, experts = x.shape[0], router.shape[1]
    out, gate = feed(x, *weights[3:], shared_shift), np.zeros((m, experts), dtype=np.int64)
    logits = ref.round_shift(ref.product(x, router), 16)
    for r in range(m):
        p = ref.softmax(logits[r], exp)
        for e in sorted(range(experts), key=lambda i: (-p[i], i))[:top_k]:
            d = feed(x[r:r + 1], *[(c[e], s[e]) for c, s in weights[:3]], 16)[0]
            out[r] += ref.round_shift(d * p[e], 16)
            gate[r, e] = p[e]
    return out, gate


def moe_graph(zk, store, rng, group=32, **shape):
    """A layer graph with 4-bit expert weights drawn into its store:
    (shape, ops, expert and shared weights, TopKSelect's place)."""
    from zkie_b200 import deepseek as ds
    s = ds.MoeShape(**{**MOE, **shape})
    ops, _, _ = ds.moe_layer(store, s)
    top = next(i for i, op in enumerate(ops) if op.kind == "TopKSelect")
    weights = []
    for op in [op for op in ops if op.kind == "GatherMatMul"] + [op for op in ops[top:] if op.kind == "Projection"]:
        n = s.n_routed if op.kind == "GatherMatMul" else 0
        w = ref.weight(rng, op.k, op.n, group, experts=n)
        dense = np.stack([ref.dense(w[0][e], w[1][e], group) for e in range(n)]) if n else ref.dense(*w, group)
        store.v[op.w] = ref.field(dense.reshape(-1))
        weights.append(w)
    return s, ops, weights, top


def liven(store, ops, weight=12000):
    """Numbers at which every part of a layer counts, in place of a builder's
    (whose norms' scales of 1 to 5 in 2^16 leave little but the biases, and
    whose weights are all positive): norms' scales about 1, weights of both
    signs up to ``weight``, embeddings about 1.  Zeros stay, the padding among
    them."""
    import torch
    from zkie_b200 import decode

    def numbers(t):
        v = store.get(t)
        return decode._signed(torch.from_numpy(v) if isinstance(v, np.ndarray) else v)

    written, news = {t for op in ops for t in op.writes()}, {}
    for i, op in enumerate(ops):
        if op.kind == "LayerNormCentered":
            news[op.w], news[op.b] = (lambda v: 60000 + 2000 * v), (lambda v: 3000 * v)
        elif op.kind in ("Projection", "GatherMatMul") or (op.kind == "MatMul" and op.b not in written):
            t = op.b if op.kind == "MatMul" else op.w
            if int(numbers(t).min()) >= 0:
                news[t] = lambda v: torch.div((2 * v - v.max()) * weight, v.max(), rounding_mode="floor")
        elif i == 0 and op.kind == "Lookup":
            news[op.table] = lambda v: (v - 25) * 3000
        elif i == 1 and op.kind == "Add":
            news[op.b] = lambda v: (v - 25) * 2000
    for t, f in news.items():
        v = numbers(t)
        new = decode._field(torch.where(v != 0, f(v), torch.zeros_like(v)))
        store.v[t] = new.numpy() if isinstance(store.get(t), np.ndarray) else new
