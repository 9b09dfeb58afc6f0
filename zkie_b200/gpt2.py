"""GPT-2 op graphs for the shard prover, with synthetic weights.

- ``build_gpt2_layer``: the reference's random single-layer builder
  (crates/zkie-ops/src/compose.rs:4237-4470, Layernorm + SoftmaxIndex arms),
  drawing every weight from the caller's XorShift64 in the reference's order;
  ``reference_layer_roundtrip_case`` replays the store its test
  ``build_gpt2_layer_roundtrip`` (:6211-6259) builds.
- ``gpt2_layer``: one layer of the GPT-2 graph (models/gpt2/src/lib.rs
  build_layer, :48-319: LayerNormCentered, 12 heads of Projection / Scale /
  Transpose / MatMul / StableSoftmaxIndex / Softmax, the head sum, the FFN
  with GeluIndex + Lookup, 176 ops) over a store laid out as build_gpt2
  (:321-372) lays it out, minus the embedding: the layer input, then the exp,
  rsqrt and gelu tables and the causal mask.  The model's weight files are
  not in the tree; the weights are drawn from an XorShift64 with the value
  ranges of the random builder (weights in [0, 50), biases in [-5, 5), norm
  scales in [1, 6)) at the real extents (768 wide, FFN 3072) and zero-padded
  to the graph's powers of two (1024, 4096), as the model's export pads them.
- the lookup tables, from the formulas of the reference's table scripts
  (scripts/extract_exp_table.py, extract_rsqrt_piecewise.py,
  extract_gpt2.py:136-144): exp of [-32, 0] and gelu at scale 2^16, the
  piecewise rsqrt table, and ``causal_mask`` (compose.rs:834-846).

Builders take any store with ``push`` / ``push_idx`` taking numpy arrays (the
device Store, or a host store for the CPU checker).

``Gpt2Decoder`` answers one token at a time with the weights of such a graph
in 4 bits (``decode.quantise_weights``): its logits are the graph's rows, bit
for bit.
"""
import ctypes as C
from collections import defaultdict
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib, decode
from ._lib import check, lib
from .device import device, ptr, stream_handle
from .gkr import XorShift64
from .compose import (Add, Argmax, GeluIndex, Layernorm, LayerNormCentered, Lookup, MatMul, Projection, Scale, Softmax,
                      SoftmaxIndex, StableSoftmaxIndex, Transpose, layer_norm_centered_columns)

P = 0xFFFFFFFF00000001
SCALE = 65536.0


def xorshift_fill(rng, n: int, mod: int, offset: int = 0) -> np.ndarray:
    """n draws ``from_i64((rng.next_u64() % mod) + offset)`` from a product
    XorShift64 (advanced in place)."""
    out = np.zeros(max(n, 1), dtype=np.uint64)
    st = _lib.u64(rng.c.xorshift_state)
    lib.zkie2_xorshift_fill(C.byref(st), n, mod, offset, out.ctypes.data_as(_lib.pu64))
    rng.c.xorshift_state = st.value
    return out[:n]


def from_i64(a) -> np.ndarray:
    a = np.asarray(a, dtype=np.int64)
    u = a.astype(np.uint64)
    neg = a < 0
    u[neg] = np.uint64(P) - (np.uint64(0) - u[neg])
    return u


# ---- tables ----------------------------------------------------------------------------------
def exp_table(bits: int = 21) -> np.ndarray:
    """exp(x) at scale 2^16 for x = (j - 2^bits) / 2^16, j < 2^bits (the
    reference's table: bits = 21, x in [-32, 0))."""
    j = np.arange(1 << bits, dtype=np.float64)
    t = np.clip(np.round(np.exp((j - (1 << bits)) / SCALE) * SCALE), 0, 2 ** 31 - 1).astype(np.int64)
    return from_i64(t)


def gelu_table(bits: int = 24) -> np.ndarray:
    """gelu_new(x) at scale 2^16 for x = (j - 2^(bits-1)) / 2^16."""
    x = (np.arange(1 << bits, dtype=np.float64) - (1 << (bits - 1))) / SCALE
    g = 0.5 * x * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (x + 0.044715 * x ** 3)))
    return from_i64(np.clip(np.round(g * SCALE), -(2 ** 31), 2 ** 31 - 1).astype(np.int64))


RSQRT_TABLE_LEN = (1 << 20) + (1 << 22) + (1 << 21)


def rsqrt_table(length: int = RSQRT_TABLE_LEN) -> np.ndarray:
    """The piecewise rsqrt table (2^20 entries at index scale 2^14, then 2^22
    at step 2^8, then 2^21 at step 2^16), 1/sqrt(var + 1e-6) at scale 2^16;
    its first ``length`` entries."""
    fine, coarse, coarse2 = 1 << 20, 1 << 22, 1 << 21
    raw = np.concatenate([np.arange(fine, dtype=np.float64),
                          fine + np.arange(coarse, dtype=np.float64) * (1 << 8),
                          fine + coarse * (1 << 8) + np.arange(coarse2, dtype=np.float64) * (1 << 16)])[:length]
    t = np.clip(np.round(1.0 / np.sqrt(raw / (1 << 14) + 1e-6) * SCALE), 0, 2 ** 31 - 1).astype(np.int64)
    return from_i64(t)


def causal_mask(m: int) -> np.ndarray:
    """-(2^30) above the diagonal, 0 elsewhere (compose.rs:834-846)."""
    i, j = np.meshgrid(np.arange(m), np.arange(m), indexing="ij")
    return from_i64(np.where(j > i, -(1 << 30), 0).reshape(-1))


# ---- the reference's random builder (compose.rs:4237-4470) -------------------------------------
def build_gpt2_layer(store, x, heads, m, d, ffn, shift, exp_t, gelu_t, rsqrt_t, rng):
    """-> (ops, out): Layernorm, per head three Projections, Transpose,
    MatMul, SoftmaxIndex (256), Softmax, MatMul, Projection; the head sum and
    the residual; Layernorm, the FFN with SoftmaxIndex (64) + Lookup."""
    dh = d // heads
    ops = []
    draw = lambda n, mod, off=0: xorshift_fill(rng, n, mod, off)  # noqa: E731
    ln1_w = store.push(draw(m * d, 5, 1))
    ln1_b = store.push(draw(m * d, 10, -5))
    h = store.push(None)
    ops.append(Layernorm(x, ln1_w, ln1_b, h, rsqrt_t, m, d))
    head_outs = []
    for _ in range(heads):
        wq, wk, wv = (store.push(draw(d * dh, 50)) for _ in range(3))
        wo = store.push(draw(dh * d, 50))
        bq, bk, bv = (store.push(draw(m * dh, 10, -5)) for _ in range(3))
        bo = store.push(draw(m * d, 10, -5))
        q, k, v, qr, kr, vr, kt, scores = (store.push(None) for _ in range(8))
        idx = store.push_idx(None)
        e, probs, attn, out_h, out_h_rem = (store.push(None) for _ in range(5))
        ops += [Projection(h, wq, bq, q, qr, m, d, dh, shift), Projection(h, wk, bk, k, kr, m, d, dh, shift),
                Projection(h, wv, bv, v, vr, m, d, dh, shift), Transpose(k, kt, m, dh),
                MatMul(q, kt, scores, m, dh, m), SoftmaxIndex(scores, idx, 1 << 8),
                Softmax(idx, e, probs, exp_t, m, m), MatMul(probs, v, attn, m, m, dh),
                Projection(attn, wo, bo, out_h, out_h_rem, m, dh, d, shift)]
        head_outs.append(out_h)
    acc = head_outs[0]
    for ho in head_outs[1:]:
        s = store.push(None)
        ops.append(Add(acc, ho, s))
        acc = s
    x2 = store.push(None)
    ops.append(Add(x, acc, x2))
    ln2_w = store.push(draw(m * d, 5, 1))
    ln2_b = store.push(draw(m * d, 10, -5))
    h2 = store.push(None)
    ops.append(Layernorm(x2, ln2_w, ln2_b, h2, rsqrt_t, m, d))
    fc_w = store.push(draw(d * ffn, 50))
    fc_b = store.push(draw(m * ffn, 10, -5))
    proj_w = store.push(draw(ffn * d, 50))
    proj_b = store.push(draw(m * d, 10, -5))
    fc, fc_rem = store.push(None), store.push(None)
    gelu_idx = store.push_idx(None)
    act, proj2, proj2_rem = (store.push(None) for _ in range(3))
    ops += [Projection(h2, fc_w, fc_b, fc, fc_rem, m, d, ffn, shift), SoftmaxIndex(fc, gelu_idx, 64),
            Lookup(gelu_idx, act, gelu_t), Projection(act, proj_w, proj_b, proj2, proj2_rem, m, ffn, d, shift)]
    out = store.push(None)
    ops.append(Add(x2, proj2, out))
    return ops, out


def reference_layer_roundtrip_case(store, rng_cls):
    """The store and ops of build_gpt2_layer_roundtrip (compose.rs:6211-6259):
    XorShift64(0x1D1D), (m, d, ffn, heads, shift) = (4, 8, 16, 2, 8), tables
    of 256 / 64 / 256 entries.  Returns (ops, out, rng) with rng positioned
    where the test's prove_shard draws from it."""
    rng = rng_cls(0x1D1D)
    m, d, ffn, heads, shift = 4, 8, 16, 2, 8
    x = store.push(xorshift_fill(rng, m * d, 50))
    exp_t = store.push(from_i64(np.arange(256) % 255 + 1))
    gelu_t = store.push(from_i64(np.arange(64) ** 2 % 1000))
    rsqrt_t = store.push(from_i64(np.arange(256) % 255 + 1))
    ops, out = build_gpt2_layer(store, x, heads, m, d, ffn, shift, exp_t, gelu_t, rsqrt_t, rng)
    return ops, out, rng


# ---- one layer of the GPT-2 graph (models/gpt2/src/lib.rs:48-319) --------------------------
@dataclass
class LayerShape:
    m: int = 512            # sequence length
    d: int = 1024           # D (768 real)
    d_real: int = 768
    heads: int = 12
    dh: int = 64
    ffn: int = 4096         # FFN (3072 real)
    ffn_real: int = 3072
    shift: int = 16
    exp_bits: int = 21      # StableSoftmaxIndex offset / table length 2^21
    gelu_bits: int = 24     # GeluIndex offset 2^23, table 2^24
    rsqrt_len: int = RSQRT_TABLE_LEN
    vocab: int = 65536      # the padded vocabulary of the tied embedding / lm_head (50257 real)
    vocab_real: int = 50257


GPT2_SMALL = LayerShape()


def _pad2(a, rows, cols):
    out = np.zeros((rows, cols), dtype=np.uint64)
    out[:a.shape[0], :a.shape[1]] = a
    return out


def _pad1(a, n):
    out = np.zeros(n, dtype=np.uint64)
    out[:a.size] = a
    return out


def synthetic_layer_weights(rng, s: LayerShape):
    """Weights of one layer at the real extents, zero-padded: q/k/v/o
    (d_real x d_real), their biases, ln1/ln2 scale and shift, fc (d_real x
    ffn_real), proj (ffn_real x d_real) and their biases, in that order."""
    dr, fr = s.d_real, s.ffn_real
    w = {}
    for name in ("q_w", "k_w", "v_w", "o_w"):
        w[name] = _pad2(xorshift_fill(rng, dr * dr, 50).reshape(dr, dr), s.d, s.d)
    for name in ("q_b", "k_b", "v_b", "o_b"):
        w[name] = _pad1(xorshift_fill(rng, dr, 10, -5), s.d)
    for name in ("ln1", "ln2"):
        w[name + "_w"] = _pad1(xorshift_fill(rng, dr, 5, 1), s.d)
        w[name + "_b"] = _pad1(xorshift_fill(rng, dr, 10, -5), s.d)
    w["fc_w"] = _pad2(xorshift_fill(rng, dr * fr, 50).reshape(dr, fr), s.d, s.ffn)
    w["fc_b"] = _pad1(xorshift_fill(rng, fr, 10, -5), s.ffn)
    w["proj_w"] = _pad2(xorshift_fill(rng, fr * dr, 50).reshape(fr, dr), s.ffn, s.d)
    w["proj_b"] = _pad1(xorshift_fill(rng, dr, 10, -5), s.d)
    return w


def gpt2_layer(store, s: LayerShape, seed: int = 0x6B2):
    """A store holding one GPT-2 layer's inputs and the layer's ops:
    (ops, x, out).  The layer input x is drawn in [0, 50) on the real
    columns (zero padding), then the weights (synthetic_layer_weights)."""
    return gpt2_layers(store, s, 1, seed)


def gpt2_layers(store, s: LayerShape, layers: int, seed: int = 0x6B2):
    """``layers`` GPT-2 layers chained as build_gpt2 chains them (the output
    of layer l is the input of layer l + 1; models/gpt2/src/lib.rs:367-372),
    sharing the tables and the mask: (ops, x, out).  The input x is drawn
    first, then each layer's weights as the layer is built."""
    rng = XorShift64(seed)
    m = s.m
    x_host = _pad2(xorshift_fill(rng, m * s.d_real, 50).reshape(m, s.d_real), m, s.d).reshape(-1)
    x = store.push(x_host)
    exp_t = store.push(exp_table(s.exp_bits))
    rsqrt_t = store.push(rsqrt_table(s.rsqrt_len))
    gelu_t = store.push(gelu_table(s.gelu_bits))
    mask_t = store.push(causal_mask(m))
    ops, cur = [], x
    for _ in range(layers):
        layer_ops, cur = build_layer(store, s, cur, synthetic_layer_weights(rng, s), exp_t, rsqrt_t, gelu_t, mask_t)
        ops += layer_ops
    return ops, x, cur


def build_layer(store, s: LayerShape, x, w, exp_t, rsqrt_t, gelu_t, mask_t):
    """models/gpt2/src/lib.rs build_layer (:48-319) over weights w
    (synthetic_layer_weights): -> (ops, out)."""
    m, D, DH = s.m, s.d, s.dh
    bc = lambda v: np.tile(v, m)  # noqa: E731  broadcast a row vector over m rows
    ops = []
    ln1_w, ln1_b = store.push(bc(w["ln1_w"])), store.push(bc(w["ln1_b"]))
    h = store.push(None)
    ops.append(LayerNormCentered(x, ln1_w, ln1_b, h, rsqrt_t, m, D, s.d_real))
    head_outs = []
    for head in range(s.heads):
        cols = slice(head * DH, (head + 1) * DH)
        qh = store.push(np.ascontiguousarray(w["q_w"][:, cols]).reshape(-1))
        kh = store.push(np.ascontiguousarray(w["k_w"][:, cols]).reshape(-1))
        vh = store.push(np.ascontiguousarray(w["v_w"][:, cols]).reshape(-1))
        oh = store.push(np.ascontiguousarray(w["o_w"][cols, :]).reshape(-1))
        qb, kb, vb = (store.push(bc(w[n][cols])) for n in ("q_b", "k_b", "v_b"))
        ob = store.push(np.zeros(m * D, dtype=np.uint64))
        q, k, v, q_s, k_s, qr, kr, vr, kt, scores, scores_16 = (store.push(None) for _ in range(11))
        idx = store.push_idx(None)
        e, probs, attn, attn_16, out_h, out_rem = (store.push(None) for _ in range(6))
        ops += [Projection(h, qh, qb, q, qr, m, D, DH, s.shift), Projection(h, kh, kb, k, kr, m, D, DH, s.shift),
                Projection(h, vh, vb, v, vr, m, D, DH, s.shift), Scale(q, q_s, 23170, 16),
                Scale(k, k_s, 23170, 16), Transpose(k_s, kt, m, DH), MatMul(q_s, kt, scores, m, DH, m),
                Scale(scores, scores_16, 1, 16),
                StableSoftmaxIndex(scores_16, mask_t, idx, 1 << s.exp_bits, 1 << s.exp_bits, m, m),
                Softmax(idx, e, probs, exp_t, m, m), MatMul(probs, v, attn, m, m, DH), Scale(attn, attn_16, 1, 16),
                Projection(attn_16, oh, ob, out_h, out_rem, m, DH, D, s.shift)]
        head_outs.append(out_h)
    acc = head_outs[0]
    for ho in head_outs[1:]:
        t = store.push(None)
        ops.append(Add(acc, ho, t))
        acc = t
    o_b = store.push(bc(w["o_b"]))
    attn_biased = store.push(None)
    ops.append(Add(acc, o_b, attn_biased))
    x2 = store.push(None)
    ops.append(Add(x, attn_biased, x2))
    ln2_w, ln2_b = store.push(bc(w["ln2_w"])), store.push(bc(w["ln2_b"]))
    h2 = store.push(None)
    ops.append(LayerNormCentered(x2, ln2_w, ln2_b, h2, rsqrt_t, m, D, s.d_real))
    fc_w, fc_b = store.push(w["fc_w"].reshape(-1)), store.push(bc(w["fc_b"]))
    proj_w, proj_b = store.push(w["proj_w"].reshape(-1)), store.push(bc(w["proj_b"]))
    fc, fc_rem = store.push(None), store.push(None)
    gelu_idx = store.push_idx(None)
    act, proj2, proj2_rem = (store.push(None) for _ in range(3))
    ops += [Projection(h2, fc_w, fc_b, fc, fc_rem, m, D, s.ffn, s.shift),
            GeluIndex(fc, gelu_idx, 1 << (s.gelu_bits - 1), 1 << s.gelu_bits), Lookup(gelu_idx, act, gelu_t),
            Projection(act, proj_w, proj_b, proj2, proj2_rem, m, s.ffn, D, s.shift)]
    out = store.push(None)
    ops.append(Add(x2, proj2, out))
    return ops, out


def gpt2_model(store, s: LayerShape, layers: int = 12, seed: int = 0x6B2):
    """The GPT-2 graph of build_gpt2 (models/gpt2/src/lib.rs:321-436): the
    token embedding as a Lookup into the tied lm_head table (emb_idx[i D + d]
    = d vocab + token_i) plus the position embedding, ``layers`` layers, the
    final LayerNormCentered, the lm_head MatMul, the vocabulary mask Add and
    the Argmax over the masked logits (the next token of every position, a
    public index tensor).  Synthetic inputs: the tokens (below vocab_real),
    the position embedding, the lm_head weights (d_real x vocab_real,
    zero-padded) and the final norm's scale and shift, drawn after the
    layers' weights.  Returns (ops, tokens index id, argmax index id)."""
    rng = XorShift64(seed)
    m, D, V = s.m, s.d, s.vocab
    tokens = np.array([int(t) % s.vocab_real for t in xorshift_fill(rng, m, 1 << 30)], dtype=np.uint32)
    lm_w = _pad2(xorshift_fill(rng, s.d_real * s.vocab_real, 50).reshape(s.d_real, s.vocab_real), D, V)
    pos = _pad2(xorshift_fill(rng, m * s.d_real, 50).reshape(m, s.d_real), m, D).reshape(-1)
    tok_t = store.push_idx(tokens)
    emb_idx = (np.arange(D, dtype=np.uint64)[None, :] * V + tokens.astype(np.uint64)[:, None]).reshape(-1)
    emb_t = store.push_idx(emb_idx.astype(np.uint32))
    wte = store.push(lm_w.reshape(-1))
    token_emb = store.push(None)
    ops = [Lookup(emb_t, token_emb, wte)]
    pos_t = store.push(pos)
    x0 = store.push(None)
    ops.append(Add(token_emb, pos_t, x0))
    exp_t = store.push(exp_table(s.exp_bits))
    rsqrt_t = store.push(rsqrt_table(s.rsqrt_len))
    gelu_t = store.push(gelu_table(s.gelu_bits))
    mask_t = store.push(causal_mask(m))
    cur = x0
    for _ in range(layers):
        layer_ops, cur = build_layer(store, s, cur, synthetic_layer_weights(rng, s), exp_t, rsqrt_t, gelu_t, mask_t)
        ops += layer_ops
    bc = lambda v: np.tile(v, m)  # noqa: E731
    lnf_w = store.push(bc(_pad1(xorshift_fill(rng, s.d_real, 5, 1), D)))
    lnf_b = store.push(bc(_pad1(xorshift_fill(rng, s.d_real, 10, -5), D)))
    h_final = store.push(None)
    ops.append(LayerNormCentered(cur, lnf_w, lnf_b, h_final, rsqrt_t, m, D, s.d_real))
    lm_t = store.push(lm_w.reshape(-1))
    logits = store.push(None)
    ops.append(MatMul(h_final, lm_t, logits, m, D, V))
    vmask = from_i64(np.where(np.arange(V) < s.vocab_real, 0, -(1 << 41)))
    mask_v = store.push(np.tile(vmask, m))
    logits_masked = store.push(None)
    ops.append(Add(logits, mask_v, logits_masked))
    sel, thr, gate, d1, d2 = (store.push(None) for _ in range(5))
    out = store.push_idx(None)
    ops.append(Argmax(logits_masked, sel, thr, gate, d1, d2, out, m, V))
    return ops, tok_t, out


# ---- token by token ---------------------------------------------------------------------------
class CapturedStep(torch.cuda.CUDAGraph):
    """A step of a Gpt2Decoder as a CUDA graph: ``replay()`` takes the
    decoder's next tokens and leaves the choice in ``tokens`` (the decoder's
    own) and the adjusted logits in ``logits`` (batch x vocab), until the next
    replay.  The graph keeps the decoder and the tensors of ``choice``, whose
    addresses it has recorded."""

    decoder = choice = tokens = logits = None


class Gpt2Decoder:
    """The graph of ``gpt2_model`` one token at a time, for ``batch`` sequences
    side by side: the tied embedding and its position row, per layer
    LayerNormCentered, the heads' q, k and v as one projection, attention over
    the layer's cache, the output projection summed over the heads onto the
    residual, LayerNormCentered, the feed-forward with the gelu table; the
    final norm, the lm_head and the choice of the token.

    ``weights`` is what ``decode.quantise_weights(store, ops, ("Projection",
    "MatMul"))`` returned for the graph: the Store then holds the same numbers,
    and a step's adjusted logits (without penalties) are the row that
    ``forward_ops`` leaves in the Argmax arm's input, so the tokens generated
    are the ones the graph proves.  The graph's exp table begins with zero
    (exp_bits from 20 on).  Sequences hold at most the graph's m
    tokens.  ``tokens`` (uint32, batch) is each sequence's next token to take;
    a step replaces it by its choice."""

    def __init__(self, store, ops, s: LayerShape, weights: dict, batch: int = 1):
        if not self._shaped(store, ops, s):
            raise ValueError("Gpt2Decoder: not a graph of gpt2_model with this shape")
        if not self._filled(store, ops, s):
            raise ValueError("Gpt2Decoder: biases or masks that the steps do not compute with")
        tables = {op.kind: op for op in ops}
        decode.masked_counts_nothing(store.get(tables["Softmax"].table), "Gpt2Decoder")
        self.s, self.batch, self.err = s, batch, torch.zeros(1, dtype=torch.int32, device=device())
        rows = lambda t, n: store.get(t).reshape(-1, n)[0]  # noqa: E731  a row vector broadcast over m rows
        wide = lambda t, n: rows(t, n).view(torch.int64).repeat(batch).view(torch.uint64)  # noqa: E731

        def quant(ids, dim, segment=0):
            parts = [weights[t] for t in ids]
            return decode.QuantWeight(torch.cat([p[0] for p in parts], dim), torch.cat([p[1] for p in parts], dim),
                                      parts[0][2], segment)

        norms = [op for op in ops if op.kind == "LayerNormCentered"]
        projections = [op for op in ops if op.kind == "Projection"]
        per = 4 * s.heads + 2  # a layer's projections: q, k, v, o per head, then fc and proj
        if s.d * s.vocab > 0x7FFFFFFF:
            raise ValueError("Gpt2Decoder: an embedding table of at most 2^31 - 1 entries is wanted")
        self.exp = store.get(tables["Softmax"].table)
        lookups = [op for op in ops if op.kind == "Lookup"]
        self.gelu, self.rsqrt = store.get(lookups[1].table), store.get(norms[0].rsqrt_table)
        self._lens = torch.zeros(batch, dtype=torch.int32, device=device())
        self.layers, self.witness = [], []
        for i in range(0, len(projections), per):
            layer = projections[i:i + per]
            heads, fc, proj = layer[:4 * s.heads], layer[-2], layer[-1]
            kinds = [[heads[4 * h + j] for h in range(s.heads)] for j in range(4)]
            n = 2 * (i // per)
            cat = lambda ids: torch.cat([rows(t, s.dh).view(torch.int64) for t in ids]).view(torch.uint64)  # noqa: E731
            # the output bias is added after the heads' sum: Add(acc, o_b)
            o_b = next(op.b for op in ops if op.kind == "Add" and op.a == self._sum_of(ops, [o.out for o in kinds[3]]))
            if not decode.same_rows(store.get(o_b), s.d):
                raise ValueError("Gpt2Decoder: biases or masks that the steps do not compute with")
            self.layers.append(dict(
                ln1=(wide(norms[n].w, s.d), wide(norms[n].b, s.d)), ln2=(wide(norms[n + 1].w, s.d), wide(norms[n + 1].b, s.d)),
                qkv=quant([o.w for j in range(3) for o in kinds[j]], 1), qkv_b=cat([o.bias for j in range(3) for o in kinds[j]]),
                o=quant([o.w for o in kinds[3]], 0, s.dh), o_b=rows(o_b, s.d).clone(),
                fc=quant([fc.w], 1), fc_b=rows(fc.bias, s.ffn).clone(),
                proj=quant([proj.w], 1), proj_b=rows(proj.bias, s.d).clone(),
                cache=decode.KvCache.zeros(batch, s.heads, s.dh, s.dh, s.m, self.lens)))
            scaled = {op.x: op.out for op in ops if op.kind == "Scale"}
            self.witness.append(([scaled[o.out] for o in kinds[1]], [o.out for o in kinds[2]]))
        self.lnf = (wide(norms[-1].w, s.d), wide(norms[-1].b, s.d))
        lm = next(op for op in ops if op.kind == "MatMul" and op.a == norms[-1].out)
        self.lm = quant([lm.b], 1)
        self.wte, self.pos = store.get(lookups[0].table), store.get(ops[1].b).reshape(s.m, s.d)
        self.columns = torch.arange(s.d, dtype=torch.int32, device=device()) * s.vocab
        bits = np.arange(-(-s.vocab // 32) * 32) < s.vocab_real
        self.allowed = torch.from_numpy(np.packbits(bits, bitorder="little").view(np.int32).copy()).to(device())
        self._tokens = torch.zeros(batch, dtype=torch.uint32, device=device())

    # read, and written in place, but not replaced: the caches count in lens
    lens, tokens = decode._kept("_lens"), decode._kept("_tokens")

    @staticmethod
    def _shaped(store, ops, s: LayerShape) -> bool:
        """Whether the graph is gpt2_model's of this shape: sizes, shifts, the
        Scales' factors, the tables' offsets and the vocabulary's mask."""
        of = defaultdict(list)
        for op in ops:
            of[op.kind].append(op)
        proj, norms, per = of["Projection"], of["LayerNormCentered"], 4 * s.heads + 2
        layers = len(proj) // per
        if not layers or len(proj) % per or len(norms) != 2 * layers + 1 or not of["Argmax"] or len(of["Lookup"]) != 1 + layers:
            return False
        sizes = [(s.d, s.dh)] * 3 + [(s.dh, s.d)]
        sizes = sizes * s.heads + [(s.d, s.ffn), (s.ffn, s.d)]
        if any((op.m, op.k, op.n, op.shift) != (s.m, *sizes[i % per], s.shift) for i, op in enumerate(proj)) or \
                any((op.m, op.d, op.n_real) != (s.m, s.d, s.d_real) for op in norms):
            return False
        scales = [(23170, 16)] * 2 + [(1, 16)] * 2  # queries, keys, scores, outputs
        if [(op.factor, op.shift) for op in of["Scale"]] != scales * (layers * s.heads) or \
                [(op.offset, op.table_len) for op in of["StableSoftmaxIndex"]] != [(1 << s.exp_bits,) * 2] * (layers * s.heads) or \
                [(op.offset, op.table_len) for op in of["GeluIndex"]] != [(1 << s.gelu_bits >> 1, 1 << s.gelu_bits)] * layers:
            return False
        last = of["Argmax"][-1]
        mask = next((store.get(op.b)[:s.vocab] for op in of["Add"] if op.c == last.x), None)
        if mask is None or (last.m, last.n) != (s.m, s.vocab):
            return False
        return decode.masks(mask, from_i64(np.where(np.arange(s.vocab) < s.vocab_real, 0, decode.MASKED)))

    @staticmethod
    def _filled(store, ops, s: LayerShape) -> bool:
        """Whether the graph's tensors are what the steps compute with: norms'
        scales and biases one row over and over, no bias of a head's output
        projection, the causal mask."""
        proj, per = [op for op in ops if op.kind == "Projection"], 4 * s.heads + 2
        row = [(t, s.d) for op in ops if op.kind == "LayerNormCentered" for t in (op.w, op.b)]
        none = [op.bias for i, op in enumerate(proj) if i % per < 4 * s.heads and i % per % 4 == 3]
        row += [(op.bias, op.n) for op in proj if op.bias not in none]
        causal = causal_mask(s.m)
        return all(decode.same_rows(store.get(t), n) for t, n in row) and all(decode.all_zero(store.get(t)) for t in none) and \
            all(decode.masks(store.get(t), causal) for t in {op.mask for op in ops if op.kind == "StableSoftmaxIndex"})

    @staticmethod
    def _sum_of(ops, heads):
        """The tensor that adds up the heads' outputs."""
        acc = heads[0]
        for h in heads[1:]:
            acc = next(op.c for op in ops if op.kind == "Add" and op.a == acc and op.b == h)
        return acc

    def load(self, store, sequence: int, tokens: int):
        """Take the first ``tokens`` positions of a forward pass of the graph as
        the past of one sequence: its scaled keys and values, from the Store."""
        s = self.s
        if not 0 <= sequence < self.batch or not 0 <= tokens <= s.m:
            raise ValueError("load: a sequence of the batch and at most the graph's positions are wanted")
        self.lens[sequence] = 0
        for layer, (ks, vs) in zip(self.layers, self.witness):
            c = layer["cache"]
            one = decode.KvCache(c.k[sequence:sequence + 1], c.v[sequence:sequence + 1], self.lens[sequence:sequence + 1])
            side = lambda ids: torch.stack([store.get(t).view(torch.int64).reshape(s.m, s.dh)[:tokens] for t in ids],  # noqa: E731
                                           dim=1).reshape(1, tokens, -1).contiguous().view(torch.uint64)
            if tokens:
                one.append(side(ks), side(vs), err=self.err)
        self.lens[sequence] = tokens

    def _norm(self, x, w):
        return layer_norm_centered_columns(x.reshape(-1), w[0], w[1], self.rsqrt, self.batch, self.s.d, self.s.d_real,
                                           self.err)["out"].reshape(self.batch, self.s.d)

    def _embed(self):
        s, n = self.s, self.batch * self.s.d
        idx = (self.columns + self.tokens.view(torch.int32)[:, None]).contiguous()
        rows, x = torch.empty(n, dtype=torch.uint64, device=idx.device), torch.empty(n, dtype=torch.uint64, device=idx.device)
        sh = stream_handle()
        check(lib.zkie2_op_lookup(idx.data_ptr(), n, ptr(self.wte), self.wte.numel(), ptr(rows), self.err.data_ptr(), sh),
              "zkie2_op_lookup")
        at = self.lens.clamp(0, s.m - 1).to(torch.int64)
        pos = self.pos.view(torch.int64)[at].reshape(-1).view(torch.uint64)
        check(lib.zkie2_op_add(ptr(rows), ptr(pos), n, ptr(x), sh), "zkie2_op_add")
        return x.reshape(self.batch, s.d)

    def logits(self) -> torch.Tensor:
        """One step up to the lm_head: the logits (batch x vocab) after the
        present tokens, whose keys and values go into the caches at position
        lens (``lens`` stays)."""
        s = self.s
        self.layers[0]["cache"].room(s.m, self.err)  # the graph's positions, not the cache's whole blocks
        x = self._embed()
        hd = s.heads * s.dh
        for w in self.layers:
            r = decode.project(self._norm(x, w["ln1"]), w["qkv"], s.shift, bias=w["qkv_b"], err=self.err)
            a = decode.attend(r[:, :hd], w["cache"], self.exp, k=r[:, hd:2 * hd], v=r[:, 2 * hd:], q_scale=(23170, 16),
                              k_scale=(23170, 16), score_scale=(1, 16), offset=1 << s.exp_bits, err=self.err)
            x = decode.project(a, w["o"], s.shift, bias=w["o_b"], residual=x, err=self.err)
            f = decode.project(self._norm(x, w["ln2"]), w["fc"], s.shift, bias=w["fc_b"], table=self.gelu,
                               offset=1 << (s.gelu_bits - 1), err=self.err)
            x = decode.project(f, w["proj"], s.shift, bias=w["proj_b"], residual=x, err=self.err)
        return decode.project(self._norm(x, self.lnf), self.lm, 0, err=self.err)

    def step(self, **choice):
        """Take ``tokens``, choose the next ones (``choice``: what
        ``decode.choose_token`` takes; the vocabulary's padding is masked as in
        the graph unless ``allowed`` is given) and count the position.  Returns
        (tokens, adjusted logits).  Nothing is read back: ``check`` does."""
        choice.setdefault("allowed", self.allowed)
        tokens, logits = decode.choose_token(self.logits(), err=self.err, **choice)
        layer = self.layers[0]["cache"]
        layer.advance()
        self.tokens.copy_(tokens)
        return self.tokens, logits

    def capture(self, **choice) -> "CapturedStep":
        """A step recorded as a CUDA graph, to be replayed once per token; the
        position, the tokens and the error word of the step that it ran for
        warm-up are put back.  What ``choice`` gives is read from the same
        memory at every replay."""
        lens, tokens, err = self.lens.clone(), self.tokens.clone(), self.err.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.step(**choice)
            self.lens.copy_(lens)
            self.tokens.copy_(tokens)
            self.err.copy_(err)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = CapturedStep()
        graph.decoder, graph.choice = self, choice
        with torch.cuda.graph(graph):
            graph.tokens, graph.logits = self.step(**choice)
        return graph

    def check(self):
        """Raise if a step since the last check met data its kernels do not take."""
        try:
            decode.check_err(self.err, "Gpt2Decoder")
        finally:
            self.err.zero_()
