"""A DeepSeek-V2-Lite-shaped MoE layer as an op graph (models/deepseek-v2-lite/
src/lib.rs: build_attention :57-250, build_moe :252-470 and one layer of the
loop in build_deepseek :620-672), with synthetic weights in place of the
reference's weight files.

Shapes follow the reference: hidden 2048, MLA with 16 heads (q/k nope 128,
rope 64, v 128, kv_lora 512), 64 routed experts (top 6, expert FFN padded to
2048 with 1408 real columns) plus the shared experts (4096 padded, 2816 real),
sequence 512, shift 16.  The routed experts run expert-major as in the
reference: TopKSelect over the router's softmax, Scatter into expert order,
per-expert GatherMatMul for gate / up / down, SiLU by lookup, the gate
values gathered back by (token, expert), and Gather (scatter-add) into token
order.  The tables are the reference's kinds: exp (2^21), the piecewise rsqrt,
the 2^16 limb range, SiLU at scale 2^16 over 2^24 points, the causal mask and
RoPE's cos / sin at scale 2^16.

``moe_block`` and ``MoeLayerDecoder`` compute the experts and the whole layer
for a few rows, one token at a time, with the weights of such a graph in 4
bits (``decode.quantise_weights``), bit for bit the graph's rows.
"""
from collections import defaultdict
from dataclasses import dataclass
from typing import Optional

import numpy as np
import torch

from . import decode
from .compose import (Add, BroadcastScale, CombineIdx, Gather, GatherMatMul, GeluIndex, IdxBroadcast, Lookup,
                      MatMul, PadIdx, Projection, RmsNorm, RoPE, Scale, ScaleVec, Scatter, Softmax, StableSoftmaxIndex,
                      TopKSelect, Transpose, rms_norm_columns)
from ._lib import check, lib
from .device import device, ptr, stream_handle
from .gkr import XorShift64
from .gpt2 import RSQRT_TABLE_LEN, SCALE, _pad2, causal_mask, exp_table, from_i64, rsqrt_table, xorshift_fill


@dataclass(frozen=True)
class MoeShape:
    m: int = 512            # sequence length
    h: int = 2048           # hidden
    heads: int = 16
    qk_nope: int = 128
    qk_rope: int = 64
    v_head: int = 128
    kv_lora: int = 512
    n_routed: int = 64
    top_k: int = 6
    moe: int = 2048         # routed expert FFN, padded (1408 real)
    moe_real: int = 1408
    shared: int = 4096      # shared experts' FFN, padded (2816 real)
    shared_real: int = 2816
    shift: int = 16
    exp_bits: int = 21
    silu_bits: int = 24
    rsqrt_len: int = RSQRT_TABLE_LEN
    w_mod: int = 50          # weights drawn in [0, w_mod)
    router_mod: int = 1 << 10  # router weights in [-router_mod / 2, router_mod / 2): routing spread over the experts


DSV2_LITE = MoeShape()


def silu_table(bits: int = 24) -> np.ndarray:
    """silu(x) = x sigmoid(x) at scale 2^16 for x = (j - 2^(bits-1)) / 2^16."""
    x = (np.arange(1 << bits, dtype=np.float64) - (1 << (bits - 1))) / SCALE
    y = x / (1.0 + np.exp(-np.clip(x, -700, 700)))
    return from_i64(np.clip(np.round(y * SCALE), -(2 ** 31), 2 ** 31 - 1).astype(np.int64))


def rope_tables(m: int, rope: int, base: float = 10000.0):
    """cos / sin (m x rope/2) of p theta_i, theta_i = base^(-2 i / rope), at scale 2^16."""
    half = rope // 2
    ang = np.arange(m, dtype=np.float64)[:, None] * base ** (-2.0 * np.arange(half) / rope)[None, :]
    q = lambda a: from_i64(np.round(a * SCALE).astype(np.int64).reshape(-1))  # noqa: E731
    return q(np.cos(ang)), q(np.sin(ang))


def _draw(rng, n, mod, off=0):
    return xorshift_fill(rng, n, mod, off)


def _norm_weights(rng, n):
    """RMSNorm scales near 1.0 at scale 2^16 (1 +- 2^-5), so the normalised
    activations keep the 2^16 scale the projections' shift assumes."""
    return _draw(rng, n, 1 << 12, (1 << 16) - (1 << 11))


def _cols(mat, cols, c0, c1):
    return np.ascontiguousarray(mat.reshape(-1, cols)[:, c0:c1]).reshape(-1)


def _rows(mat, cols, r0, r1):
    return np.ascontiguousarray(mat.reshape(-1, cols)[r0:r1]).reshape(-1)


def build_attention(store, ops, x, s: MoeShape, t, rng):
    """build_attention (lib.rs:57-250): the shared kv latent (Projection to
    kv_lora, RmsNorm) and the MQA rope key (Projection, RoPE, Transpose), then
    per head the q nope / rope, k nope and v Projections, RoPE on q rope, the
    two score MatMuls, Scale (7519 / 2^32), StableSoftmaxIndex, Softmax, the
    value MatMul, Scale (2^-16) and the output Projection; the head sum."""
    m, H, nope, rp, vh, kvl = s.m, s.h, s.qk_nope, s.qk_rope, s.v_head, s.kv_lora
    zeros = lambda n: np.zeros(n, dtype=np.uint64)  # noqa: E731
    wm = s.w_mod
    qnope_w = _draw(rng, H * s.heads * nope, wm)
    qpe_w = _draw(rng, H * s.heads * rp, wm)
    kvlora_w = _draw(rng, H * kvl, wm)
    kpe_w = _draw(rng, H * rp, wm)
    kva_ln = _norm_weights(rng, kvl)
    knope_w = _draw(rng, kvl * s.heads * nope, wm)
    v_w = _draw(rng, kvl * s.heads * vh, wm)
    o_w = _draw(rng, s.heads * vh * H, wm)
    kvlora_w_t, kpe_w_t = store.push(kvlora_w), store.push(kpe_w)
    kv_b, kpe_b = store.push(zeros(m * kvl)), store.push(zeros(m * rp))
    kvlora, kvlora_rem, kpe, kpe_rem = (store.push(None) for _ in range(4))
    ops.append(Projection(x, kvlora_w_t, kv_b, kvlora, kvlora_rem, m, H, kvl, s.shift))
    ops.append(Projection(x, kpe_w_t, kpe_b, kpe, kpe_rem, m, H, rp, s.shift))
    kva_ln_t = store.push(np.tile(kva_ln, m))
    kvlora_n = store.push(None)
    ops.append(RmsNorm(kvlora, kva_ln_t, kvlora_n, t["rsqrt"], t["limb"], m, kvl, kvl))
    kpe_rot = store.push(None)
    ops.append(RoPE(kpe, t["cos"], t["sin"], kpe_rot, t["limb"], m, rp, s.shift))
    kt = store.push(None)
    ops.append(Transpose(kpe_rot, kt, m, rp))
    head_outs = []
    for hd in range(s.heads):
        qn_w = store.push(_cols(qnope_w, s.heads * nope, hd * nope, (hd + 1) * nope))
        qp_w = store.push(_cols(qpe_w, s.heads * rp, hd * rp, (hd + 1) * rp))
        kn_w = store.push(_cols(knope_w, s.heads * nope, hd * nope, (hd + 1) * nope))
        vh_w = store.push(_cols(v_w, s.heads * vh, hd * vh, (hd + 1) * vh))
        oh = store.push(_rows(o_w, H, hd * vh, (hd + 1) * vh))
        qn, qn_rem, qp, qp_rem, kn, kn_rem, vv, vv_rem = (store.push(None) for _ in range(8))
        ops.append(Projection(x, qn_w, store.push(zeros(m * nope)), qn, qn_rem, m, H, nope, s.shift))
        ops.append(Projection(x, qp_w, store.push(zeros(m * rp)), qp, qp_rem, m, H, rp, s.shift))
        ops.append(Projection(kvlora_n, kn_w, store.push(zeros(m * nope)), kn, kn_rem, m, kvl, nope, s.shift))
        ops.append(Projection(kvlora_n, vh_w, store.push(zeros(m * vh)), vv, vv_rem, m, kvl, vh, s.shift))
        qp_rot = store.push(None)
        ops.append(RoPE(qp, t["cos"], t["sin"], qp_rot, t["limb"], m, rp, s.shift))
        knt = store.push(None)
        ops.append(Transpose(kn, knt, m, nope))
        s_nope, s_rope, sc, s16 = (store.push(None) for _ in range(4))
        idx = store.push_idx(None)
        e, probs, attn, attn16, out_h, out_rem = (store.push(None) for _ in range(6))
        ops += [MatMul(qn, knt, s_nope, m, nope, m), MatMul(qp_rot, kt, s_rope, m, rp, m), Add(s_nope, s_rope, sc),
                Scale(sc, s16, 7519, 32),
                StableSoftmaxIndex(s16, t["mask"], idx, 1 << s.exp_bits, 1 << s.exp_bits, m, m),
                Softmax(idx, e, probs, t["exp"], m, m), MatMul(probs, vv, attn, m, m, vh), Scale(attn, attn16, 1, 16)]
        ops.append(Projection(attn16, oh, store.push(zeros(m * H)), out_h, out_rem, m, vh, H, s.shift))
        head_outs.append(out_h)
    acc = head_outs[0]
    for ho in head_outs[1:]:
        nxt = store.push(None)
        ops.append(Add(acc, ho, nxt))
        acc = nxt
    return acc


def build_moe(store, ops, x, s: MoeShape, t, rng):
    """build_moe (lib.rs:252-470): router MatMul, Scale, StableSoftmaxIndex,
    Softmax, TopKSelect (6 of 64); Scatter into expert order, PadIdx to a
    power of two, the token rows gathered by Lookup and zeroed past the real
    positions (BroadcastScale); gate / up GatherMatMuls with Scale, SiLU by
    GeluIndex + Lookup, ScaleVec, the down GatherMatMul with Scale; the gate
    values by CombineIdx + Lookup, BroadcastScale, Scale and Gather back to
    token order; the shared experts as Projections with SiLU; the sum."""
    m, H, E, F, wm = s.m, s.h, s.n_routed, s.moe, s.w_mod
    zeros = lambda n: np.zeros(n, dtype=np.uint64)  # noqa: E731
    router_t = store.push(_draw(rng, H * E, s.router_mod, -(s.router_mod // 2)))
    logits, logits_16 = store.push(None), store.push(None)
    ops += [MatMul(x, router_t, logits, m, H, E), Scale(logits, logits_16, 1, 16)]
    zero_mask = store.push(zeros(m * E))
    scores_idx = store.push_idx(None)
    ops.append(StableSoftmaxIndex(logits_16, zero_mask, scores_idx, 1 << s.exp_bits, 1 << s.exp_bits, m, E))
    scores_e, scores = store.push(None), store.push(None)
    ops.append(Softmax(scores_idx, scores_e, scores, t["exp"], m, E))
    sel, thr, gate, d1, d2 = (store.push(None) for _ in range(5))
    ops.append(TopKSelect(scores, sel, thr, gate, d1, d2, m, E, s.top_k))
    shared_g = _pad2(_draw(rng, H * s.shared_real, wm).reshape(H, s.shared_real), H, s.shared).reshape(-1)
    shared_u = _pad2(_draw(rng, H * s.shared_real, wm).reshape(H, s.shared_real), H, s.shared).reshape(-1)
    shared_d = _pad2(_draw(rng, s.shared_real * H, wm).reshape(s.shared_real, H), s.shared, H).reshape(-1)
    experts = lambda k, n, kr, nr: np.stack([_pad2(_draw(rng, kr * nr, wm).reshape(kr, nr), k, n)  # noqa: E731
                                             for _ in range(E)]).reshape(-1)
    eg, eu = experts(H, F, H, s.moe_real), experts(H, F, H, s.moe_real)
    ed = experts(F, H, s.moe_real, H)
    n_pos = s.top_k * m
    s_pad = 1 << max(n_pos - 1, 0).bit_length()
    token_id, expert_of = store.push_idx(None), store.push_idx(None)
    ops.append(Scatter(sel, token_id, expert_of, m, E))
    token_id_pad, expert_of_pad = store.push_idx(None), store.push_idx(None)
    ops += [PadIdx(token_id, token_id_pad, s_pad), PadIdx(expert_of, expert_of_pad, s_pad)]
    idx_seg = store.push_idx(None)
    ops.append(IdxBroadcast(token_id_pad, idx_seg, H))
    seg = store.push(None)
    ops.append(Lookup(idx_seg, seg, x))
    pos_mask = zeros(s_pad)
    pos_mask[:n_pos] = 1
    mask_t = store.push(pos_mask)
    seg_z = store.push(None)
    ops.append(BroadcastScale(seg, mask_t, seg_z, H))
    eg_full, eu_full, ed_full = store.push(eg), store.push(eu), store.push(ed)
    g_raw, g = store.push(None), store.push(None)
    ops += [GatherMatMul(seg_z, expert_of_pad, eg_full, g_raw, s_pad, H, F, E), Scale(g_raw, g, 1, 16)]
    u_raw, u = store.push(None), store.push(None)
    ops += [GatherMatMul(seg_z, expert_of_pad, eu_full, u_raw, s_pad, H, F, E), Scale(u_raw, u, 1, 16)]
    silu_idx = store.push_idx(None)
    silu, act = store.push(None), store.push(None)
    ops += [GeluIndex(g, silu_idx, 1 << (s.silu_bits - 1), 1 << s.silu_bits), Lookup(silu_idx, silu, t["silu"]),
            ScaleVec(silu, u, act, 16)]
    d_raw, dd = store.push(None), store.push(None)
    ops += [GatherMatMul(act, expert_of_pad, ed_full, d_raw, s_pad, F, H, E), Scale(d_raw, dd, 1, 16)]
    idx_gate = store.push_idx(None)
    ops.append(CombineIdx(token_id_pad, expert_of_pad, idx_gate, E))
    gate_pos = store.push(None)
    ops.append(Lookup(idx_gate, gate_pos, gate))
    weighted_raw, weighted = store.push(None), store.push(None)
    ops += [BroadcastScale(dd, gate_pos, weighted_raw, H), Scale(weighted_raw, weighted, 1, 16)]
    gate_ones = store.push(np.ones(s_pad, dtype=np.uint64))
    out = store.push(None)
    ops.append(Gather(weighted, token_id_pad, gate_ones, out, m, H))
    sg_w, su_w, sd_w = store.push(shared_g), store.push(shared_u), store.push(shared_d)
    sg, sg_rem, su, su_rem = (store.push(None) for _ in range(4))
    ss_idx = store.push_idx(None)
    ss, sa, sd, sd_rem = (store.push(None) for _ in range(4))
    ops += [Projection(x, sg_w, store.push(zeros(m * s.shared)), sg, sg_rem, m, H, s.shared, s.shift),
            Projection(x, su_w, store.push(zeros(m * s.shared)), su, su_rem, m, H, s.shared, s.shift),
            GeluIndex(sg, ss_idx, 1 << (s.silu_bits - 1), 1 << s.silu_bits), Lookup(ss_idx, ss, t["silu"]),
            ScaleVec(ss, su, sa, 16),
            Projection(sa, sd_w, store.push(zeros(m * H)), sd, sd_rem, m, s.shared, H, s.shift)]
    total = store.push(None)
    ops.append(Add(out, sd, total))
    return total


def moe_layer(store, s: MoeShape = DSV2_LITE, seed: int = 0xD5E):
    """One MoE layer (a layer >= 1 of build_deepseek, lib.rs:620-672) over a
    synthetic input: (ops, x, out).  The input x (m x hidden, drawn in [0,
    2^12)) comes first, then the tables, then the weights as the layer is
    built."""
    rng = XorShift64(seed)
    m, H = s.m, s.h
    x = store.push(_draw(rng, m * H, 1 << 12))
    cos, sin = rope_tables(m, s.qk_rope)
    t = {"exp": store.push(exp_table(s.exp_bits)), "rsqrt": store.push(rsqrt_table(s.rsqrt_len)),
         "limb": store.push(np.arange(1 << 16, dtype=np.uint64)), "silu": store.push(silu_table(s.silu_bits)),
         "mask": store.push(causal_mask(m)), "cos": store.push(cos), "sin": store.push(sin)}
    ops = []
    in_norm = store.push(np.tile(_norm_weights(rng, H), m))
    hn = store.push(None)
    ops.append(RmsNorm(x, in_norm, hn, t["rsqrt"], t["limb"], m, H, H))
    attn = build_attention(store, ops, hn, s, t, rng)
    x2 = store.push(None)
    ops.append(Add(x, attn, x2))
    post_norm = store.push(np.tile(_norm_weights(rng, H), m))
    h2 = store.push(None)
    ops.append(RmsNorm(x2, post_norm, h2, t["rsqrt"], t["limb"], m, H, H))
    ff = build_moe(store, ops, h2, s, t, rng)
    x3 = store.push(None)
    ops.append(Add(x2, ff, x3))
    return ops, x, x3



# ---- token by token ---------------------------------------------------------------------------
def moe_block(store, ops, weights: dict, exp_table: int, silu_table: int, shift: Optional[int] = None) -> decode.MoeBlock:
    """The experts of a graph that ``build_moe`` built, for a few rows: the
    router as it is, the routed and the shared experts' weights from what
    ``decode.quantise_weights(store, ops)`` returned, the shift of the shared
    experts' Projections from the graph (one that is given has to be it)."""
    at = next(i for i, op in enumerate(ops) if op.kind == "TopKSelect")
    route, router = ops[at], ops[at - 4]  # MatMul, Scale, StableSoftmaxIndex, Softmax, TopKSelect
    experts = [op for op in ops[at:] if op.kind == "GatherMatMul"]
    shared = [op for op in ops[at:] if op.kind == "Projection"]
    scales = [op for op in ops[at - 3:] if op.kind in ("Scale", "ScaleVec")]
    if router.kind != "MatMul" or ops[at - 2].kind != "StableSoftmaxIndex" or len(experts) != 3 or len(shared) != 3:
        raise ValueError("moe_block: not a graph of build_moe")
    if any((op.factor, op.shift) != (1, 16) for op in scales if op.kind == "Scale") or \
            any(op.shift != 16 for op in scales if op.kind == "ScaleVec") or len({op.shift for op in shared}) != 1:
        raise ValueError("moe_block: not a graph of build_moe: Scales by 2^16 and one shift of the shared experts are wanted")
    if not all(decode.all_zero(store.get(t)) for t in (ops[at - 2].mask, *[op.bias for op in shared])):
        raise ValueError("moe_block: not a graph of build_moe: a mask of the experts or biases that the kernels do not have")
    if shift not in (None, shared[0].shift):
        raise ValueError(f"moe_block: shift {shift}, the graph's shared experts have {shared[0].shift}")
    quant = lambda op: decode.QuantWeight(*weights[op.w])  # noqa: E731
    return decode.MoeBlock(store.get(router.b).reshape(router.k, router.n), *[quant(op) for op in experts + shared],
                           store.get(exp_table), store.get(silu_table), route.k, shared[0].shift)


class MoeLayerDecoder:
    """One layer of ``moe_layer`` one token at a time, for ``batch`` sequences
    side by side: RmsNorm, the kv latent with its norm and the rotated key that
    all heads share, the heads' q, k and v as wide projections, RoPE, attention
    over the cache (keys of nope + rope dimensions), the output projection
    summed over the heads onto the residual, RmsNorm and ``moe_block``.  The
    graph's exp table begins with zero (exp_bits from 20 on)."""

    def __init__(self, store, ops, s: MoeShape, weights: dict, batch: int = 1):
        if not self._shaped(ops, s):
            raise ValueError("MoeLayerDecoder: not a graph of moe_layer with this shape")
        causal = {op.mask for op in [op for op in ops if op.kind == "StableSoftmaxIndex"][:s.heads]}
        if not all(decode.all_zero(store.get(op.bias)) for op in ops if op.kind == "Projection") or \
                not all(decode.same_rows(store.get(op.w), op.d) for op in ops if op.kind == "RmsNorm") or \
                not all(decode.masks(store.get(t), causal_mask(s.m)) for t in causal):
            raise ValueError("MoeLayerDecoder: biases or masks that the steps do not compute with")
        soft = next(op for op in ops if op.kind == "Softmax")
        decode.masked_counts_nothing(store.get(soft.table), "MoeLayerDecoder")
        self.s, self.batch, self.err = s, batch, torch.zeros(1, dtype=torch.int32, device=device())
        wide = lambda t, n: store.get(t).view(torch.int64).reshape(-1, n)[0].repeat(batch).view(torch.uint64)  # noqa: E731
        norms = [op for op in ops if op.kind == "RmsNorm"]
        proj = [op for op in ops if op.kind == "Projection"]
        ropes = [op for op in ops if op.kind == "RoPE"]
        silu = next(op for op in ops if op.kind == "Lookup" and op.table != norms[0].rsqrt_table and
                    any(o.kind == "GeluIndex" and o.out == op.idx for o in ops))

        def quant(ids, dim, segment=0):
            parts = [weights[o.w] for o in ids]
            return decode.QuantWeight(torch.cat([p[0] for p in parts], dim), torch.cat([p[1] for p in parts], dim),
                                      parts[0][2], segment)

        kinds = [[proj[2 + 5 * h + j] for h in range(s.heads)] for j in range(5)]  # q nope, q rope, k nope, v, o
        self.latent = quant([proj[0], proj[1]], 1)          # kv latent | shared rope key
        self.q, self.kv = quant(kinds[0] + kinds[1], 1), quant(kinds[2] + kinds[3], 1)
        self.o = quant(kinds[4], 0, s.v_head)
        self.norms = [(wide(op.w, op.d), op.d) for op in norms]  # input, latent, after attention
        self.rsqrt, self.exp = store.get(norms[0].rsqrt_table), store.get(soft.table)
        half = s.qk_rope // 2
        self.cos, self.sin = (store.get(t).view(torch.int64).reshape(s.m, half) for t in (ropes[0].cos, ropes[0].sin))
        self.block = moe_block(store, ops, weights, soft.table, silu.table, s.shift)
        self.cache = decode.KvCache.zeros(batch, s.heads, s.qk_nope + s.qk_rope, s.v_head, s.m)

    @staticmethod
    def _shaped(ops, s: MoeShape) -> bool:
        """Whether the graph is moe_layer's of this shape: the attention's sizes,
        shifts, Scales and tables (the experts are read from the graph)."""
        of = defaultdict(list)
        for op in ops:
            of[op.kind].append(op)
        proj, norms = of["Projection"], of["RmsNorm"]
        if len(proj) != 2 + 5 * s.heads + 3 or len(norms) != 3:
            return False
        sizes = [(s.h, s.kv_lora), (s.h, s.qk_rope)] + [
            (s.h, s.qk_nope), (s.h, s.qk_rope), (s.kv_lora, s.qk_nope), (s.kv_lora, s.v_head), (s.v_head, s.h)] * s.heads
        return [(op.m, op.k, op.n, op.shift) for op in proj[:-3]] == [(s.m, k, n, s.shift) for k, n in sizes] and \
            [(op.m, op.d, op.n_real) for op in norms] == [(s.m, d, d) for d in (s.h, s.kv_lora, s.h)] and \
            [(op.m, op.d, op.shift) for op in of["RoPE"]] == [(s.m, s.qk_rope, s.shift)] * (1 + s.heads) and \
            [(op.factor, op.shift) for op in of["Scale"][:2 * s.heads]] == [(7519, 32), (1, 16)] * s.heads and \
            [(op.offset, op.table_len) for op in of["StableSoftmaxIndex"]] == [(1 << s.exp_bits,) * 2] * (s.heads + 1)

    def _norm(self, x, i):
        w, d = self.norms[i]
        return rms_norm_columns(x.reshape(-1), w, self.rsqrt, self.batch, d, d, self.err)["out"].reshape(self.batch, d)

    def _rotate(self, x, heads):
        """RoPE of batch x (heads rope) at each sequence's position."""
        s = self.s
        at = self.cache.lens.clamp(0, s.m - 1).to(torch.int64)
        cos, sin = (t[at].reshape(-1).view(torch.uint64) for t in (self.cos, self.sin))
        x = x.contiguous().reshape(-1)
        out = torch.empty_like(x)
        check(lib.zkie2_op_rope(ptr(x), x.numel(), ptr(cos), ptr(sin), self.batch, s.qk_rope, s.shift, ptr(out),
                                stream_handle()), "zkie2_op_rope")
        return out.reshape(self.batch, heads * s.qk_rope)

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """The layer's output rows (batch x hidden) for the next token of every
        sequence (x: batch x hidden on the current device); its key and value go
        into the cache, the position is counted."""
        s, b = self.s, self.batch
        if not isinstance(x, torch.Tensor) or x.dtype != torch.uint64 or tuple(x.shape) != (b, s.h) or not x.is_cuda or \
                x.get_device() != torch.cuda.current_device():
            raise ValueError(f"MoeLayerDecoder: x of uint64 ({b}, {s.h}) on the current device is wanted")
        if self.cache.batch != b:
            raise ValueError("MoeLayerDecoder: a cache of as many sequences is wanted")
        x = x.contiguous()
        i64 = lambda t: t.view(torch.int64)  # noqa: E731
        self.cache.room(s.m, self.err)  # the graph's positions, not the cache's whole blocks
        h = self._norm(x, 0)
        lat = decode.project(h, self.latent, s.shift, err=self.err)
        kv = decode.project(self._norm(lat[:, :s.kv_lora].contiguous(), 1), self.kv, s.shift, err=self.err)
        q = decode.project(h, self.q, s.shift, err=self.err)
        nope, rope, n = s.heads * s.qk_nope, s.qk_rope, s.heads
        side = lambda a, r: torch.cat([i64(a).reshape(b, n, -1), r], 2).reshape(b, -1).view(torch.uint64)  # noqa: E731
        key = i64(self._rotate(lat[:, s.kv_lora:], 1)).reshape(b, 1, rope).expand(b, n, rope)
        query = i64(self._rotate(q[:, nope:], n)).reshape(b, n, rope)
        a = decode.attend(side(q[:, :nope], query), self.cache, self.exp, k=side(kv[:, :nope], key), v=kv[:, nope:],
                          score_scale=(7519, 32), offset=1 << s.exp_bits, err=self.err)
        x = decode.project(a, self.o, s.shift, residual=x, err=self.err)
        out, _ = self.block.forward(self._norm(x, 2), residual=x, err=self.err)
        self.cache.advance()
        return out

    def check(self):
        """Raise if a step since the last check met data its kernels do not take."""
        try:
            decode.check_err(self.err, "MoeLayerDecoder")
        finally:
            self.err.zero_()
