"""The fixed-point operators that answer one token at a time, and what they are measured on.

Four operators: a projection of a few rows by a 4-bit weight with group scales, attention of one new
token per sequence over a cache, a mixture-of-experts layer for a few tokens, and the choice of the next
token from adjusted logits.  Every value is signed fixed point embedded in the Goldilocks field (a 64-bit
word v stands for v below 2^63 and for v - p above) and every result is a whole number, so the plain forms
and the kernels have to agree in every bit.
"""
import math

import torch

own = False

WRAP = 0xFFFFFFFF          # 2^64 - p: what a negative number's word lies below its two's complement
BLOCK = 32                 # tokens in a block of the key cache
LOG_MASK = -(1 << 41)      # added to a logit that may not be chosen

# ---- the cases ----------------------------------------------------------------------------------


def listed():
    return [
        # one head's query, key and value of a 1024-wide layer for one token: the smallest call of a step
        dict(name="project_head", op="project", m=1, k=1024, n=192, group=64, segment=0, gelu=False, residual=False,
             shift=16),
        # the output projection summed over 12 heads, each rounded by itself, onto the residual, four sequences
        dict(name="project_heads_out", op="project", m=4, k=768, n=1024, group=64, segment=64, gelu=False,
             residual=True, shift=16),
        # the first half of the feed-forward with its activation table, two sequences
        dict(name="project_gelu", op="project", m=2, k=1024, n=4096, group=32, segment=0, gelu=True, residual=False,
             shift=16),
        # the logits of eight sequences over the padded vocabulary
        dict(name="project_logits", op="project", m=8, k=1024, n=65536, group=128, segment=0, gelu=False,
             residual=False, shift=0),
        # one short sequence of a 12-head layer
        dict(name="attend_short", op="attend", b=1, heads=12, kv_heads=12, dk=64, dv=64, cap=512, least=0.9),
        # 16 heads with keys of 128 + 64 (rotated) and values of 128, one long sequence
        dict(name="attend_wide_keys", op="attend", b=1, heads=16, kv_heads=16, dk=192, dv=128, cap=4096, least=0.95),
        # eight sequences of very different lengths, four query heads to each key head
        dict(name="attend_shared_ragged", op="attend", b=8, heads=16, kv_heads=4, dk=128, dv=128, cap=8192,
             least=0.02),
        # a small layer for an odd number of tokens
        dict(name="moe_small", op="moe", m=3, h=256, experts=16, top_k=3, f=48, shared=96, group=32),
        # 64 experts of 1408, top 6, with the shared ones: one token
        dict(name="moe_one_token", op="moe", m=1, h=2048, experts=64, top_k=6, f=1408, shared=2816, group=64),
        # the same layer for sixteen sequences at once
        dict(name="moe_sixteen", op="moe", m=16, h=2048, experts=64, top_k=6, f=1408, shared=2816, group=64),
        # one sequence's next token after a prompt of 512
        dict(name="choose_one", op="choose", b=1, v=65536, history=512, bias="vocabulary", mask="none"),
        # sixteen sequences, each with a grammar's mask and a bias of its own, over an odd vocabulary
        dict(name="choose_masked", op="choose", b=16, v=50257, history=4096, bias="row", mask="row"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["project", "attend", "moe", "choose"])
    if op == "project":
        segment = rng.choice([0, 0, 0, 20, 64, 128])
        heads = rng.randint(1, 16)
        group = rng.choice([32, 64, 128] if segment in (0, 128) else [32, 64])
        k = segment * heads if segment else _log(rng, 16, 4096)
        n = _log(rng, 16, 65536 if k <= 1024 else 16384)
        return dict(op=op, m=rng.randint(1, 8), k=k, n=n, group=group, segment=segment,
                    gelu=rng.random() < 0.3, residual=rng.random() < 0.5, shift=rng.choice([0, 8, 16, 16]))
    if op == "attend":
        kv_heads, each = rng.choice([1, 2, 4, 12, 16]), rng.choice([1, 1, 2, 3, 4])
        dk, dv = rng.choice([(16, 16), (40, 40), (64, 64), (128, 128), (192, 128)])
        b = rng.randint(1, 8)
        most = max(2, min(1024, (8 * 4 * 256 * 4096) // (b * kv_heads * (dk + dv) * BLOCK * each)))
        return dict(op=op, b=b, heads=kv_heads * each, kv_heads=kv_heads, dk=dk, dv=dv,
                    cap=BLOCK * _log(rng, 1, most), least=round(rng.uniform(0.0, 1.0), 3))
    if op == "moe":
        experts = rng.choice([4, 8, 16, 33, 64])
        return dict(op=op, m=rng.randint(1, 16), h=_log(rng, 64, 2048), experts=experts,
                    top_k=rng.randint(1, min(6, experts)), f=_log(rng, 16, 1408), shared=_log(rng, 16, 2816),
                    group=rng.choice([32, 64, 128]))
    return dict(op=op, b=rng.randint(1, 16), v=_log(rng, 32, 65536), history=_log(rng, 1, 4096),
                bias=rng.choice(["none", "vocabulary", "row"]), mask=rng.choice(["none", "vocabulary", "row"]))


def _weight_bytes(k, n, group, segment=0):
    rows = (k // segment) * -(-segment // group) if segment else -(-k // group)
    return k * n / 2 + 2 * rows * n


def work(case):
    c = case
    if c["op"] == "project":
        words = c["m"] * (c["k"] + c["n"] * (2 if c["residual"] else 1) + (c["n"] if c["gelu"] else 0)) + c["n"]
        return {"bytes": _weight_bytes(c["k"], c["n"], c["group"], c["segment"]) + 8 * words,
                "flops": 2 * c["m"] * c["k"] * c["n"]}
    if c["op"] == "attend":
        tokens = c["b"] * c["cap"] * (1 + c["least"]) / 2
        rows = 8 * c["b"] * (c["heads"] * (c["dk"] + c["dv"]) + c["kv_heads"] * (c["dk"] + c["dv"]))
        return {"bytes": 4 * tokens * c["kv_heads"] * (c["dk"] + c["dv"]) + rows,
                "flops": 2 * tokens * c["heads"] * (c["dk"] + c["dv"])}
    if c["op"] == "moe":
        m, h, f, s, g = c["m"], c["h"], c["f"], c["shared"], c["group"]
        hit = c["experts"] * (1 - (1 - c["top_k"] / c["experts"]) ** m)
        expert = 2 * _weight_bytes(h, f, g) + _weight_bytes(f, h, g)
        common = 2 * _weight_bytes(h, s, g) + _weight_bytes(s, h, g)
        return {"bytes": hit * expert + common + 2 * h * c["experts"] + 8 * m * (2 * h + c["experts"]),
                "flops": 6 * m * h * (f * c["top_k"] + s) + 2 * m * h * c["experts"]}
    row = c["b"] * c["v"]
    extra = {"none": 0, "vocabulary": c["v"], "row": row}
    return {"bytes": 16 * row + 8 * extra[c["bias"]] + extra[c["mask"]] / 8 + 4 * c["b"] * c["history"],
            "flops": 6 * row}


# ---- inputs --------------------------------------------------------------------------------------


def _field(x):
    """Signed numbers as the field's 64-bit words (held in int64)."""
    return torch.where(x < 0, x - WRAP, x)


def _signed(w):
    return torch.where(w < 0, w + WRAP, w)


def _normal(g, shape, std):
    return torch.round(torch.randn(shape, generator=g, device="cuda", dtype=torch.float64) * std).to(torch.int64)


def _weight(g, experts, k, n, group, segment=0):
    """Codes in [-8, 7] and one scale for each group of a column: weights of about 0.02 at scale 2^16."""
    rows = (k // segment) * -(-segment // group) if segment else -(-k // group)
    lead = (experts,) if experts else ()
    codes = torch.randint(-8, 8, lead + (k, n), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.randint(150, 450, lead + (rows, n), generator=g, device="cuda", dtype=torch.int32)
    return codes, scales


def _exp_table(bits=21):
    x = torch.arange(-(1 << bits), 0, device="cuda", dtype=torch.float64) / 65536
    return torch.round(torch.exp(x) * 65536).to(torch.int64)


def _act_table(silu, bits=24):
    x = torch.arange(-(1 << (bits - 1)), 1 << (bits - 1), device="cuda", dtype=torch.float64) / 65536
    if silu:
        y = x / (1 + torch.exp(-x))
    else:
        y = 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    return _field(torch.round(y * 65536).to(torch.int64))


def _quant(decode, w, group, segment=0):
    return decode.QuantWeight(w[0], w[1], group=group, segment=segment)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "project":
        s["x"] = _field(_normal(g, (c["m"], c["k"]), 65536.0))
        s["w"] = _weight(g, 0, c["k"], c["n"], c["group"], c["segment"])
        s["bias"] = _field(_normal(g, (c["n"],), 6000.0))
        s["table"] = _act_table(silu=False) if c["gelu"] else None
        s["residual"] = _field(_normal(g, (c["m"], c["n"]), 65536.0)) if c["residual"] else None
    elif c["op"] == "attend":
        b, cap, hk, dk, dv = c["b"], c["cap"], c["kv_heads"], c["dk"], c["dv"]
        # the query, key and value of the new token side by side, as one wide projection leaves them
        s["rows"] = _field(_normal(g, (b, c["heads"] * dk + hk * (dk + dv)), 65536.0))
        s["k"] = _normal(g, (b, hk, cap // BLOCK, dk // 4, BLOCK, 4), 40000.0).to(torch.int32)
        s["v"] = _normal(g, (b, hk, cap, dv), 65536.0).to(torch.int32)
        least = min(int(c["least"] * cap), cap - 1)
        s["lens"] = torch.randint(least, cap, (b,), generator=g, device="cuda", dtype=torch.int32)
        s["table"] = _exp_table()
        # 1 / sqrt(dk) at scale 2^32, so that one shift by 32 leaves the scores at scale 2^16
        s["factor"] = round(2 ** 16 / math.sqrt(dk))
    elif c["op"] == "moe":
        m, h, e, f, sh, gr = c["m"], c["h"], c["experts"], c["f"], c["shared"], c["group"]
        s["x"] = _field(_normal(g, (m, h), 65536.0))
        s["router"] = _field(_normal(g, (h, e), 1500.0).clamp(-32767, 32767))
        s["gate"], s["up"], s["down"] = _weight(g, e, h, f, gr), _weight(g, e, h, f, gr), _weight(g, e, f, h, gr)
        s["sgate"], s["sup"], s["sdown"] = _weight(g, 0, h, sh, gr), _weight(g, 0, h, sh, gr), _weight(g, 0, sh, h, gr)
        s["exp"], s["silu"] = _exp_table(), _act_table(silu=True)
    else:
        b, v, t = c["b"], c["v"], c["history"]
        s["logits"] = _field(_normal(g, (b, v), 3.0 * 2 ** 32))
        # a text's tokens: few of them often, most of them rarely
        often = torch.rand((b, t), generator=g, device="cuda", dtype=torch.float64) ** 4
        s["history"] = (often * v).to(torch.int32).clamp(max=v - 1)
        s["lens"] = torch.randint(t // 2, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        shape = {"none": None, "vocabulary": (v,), "row": (b, v)}
        s["bias"] = None if c["bias"] == "none" else _field(_normal(g, shape[c["bias"]], 0.5 * 2 ** 32))
        words = {"none": None, "vocabulary": (-(-v // 32),), "row": (b, -(-v // 32))}
        s["allowed"] = None if c["mask"] == "none" else torch.randint(
            -(1 << 31), 1 << 31, words[c["mask"]], generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    if own:
        _prepare_own(s)
    return s


def _prepare_own(s):
    from zkie_b200 import decode
    c = s["case"]
    u = lambda t: None if t is None else t.view(torch.uint64)  # noqa: E731
    s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if c["op"] == "project":
        s["weight"] = _quant(decode, s["w"], c["group"], c["segment"])
        for t in ("x", "bias", "table", "residual"):
            s[t] = u(s[t])
        del s["w"]
    elif c["op"] == "attend":
        s["cache"] = decode.KvCache(s["k"], s["v"], s["lens"])
        s["rows"], s["table"] = u(s["rows"]), u(s["table"])
    elif c["op"] == "moe":
        w = {t: _quant(decode, s.pop(t), c["group"]) for t in ("gate", "up", "down", "sgate", "sup", "sdown")}
        s["block"] = decode.MoeBlock(u(s["router"]), w["gate"], w["up"], w["down"], w["sgate"], w["sup"], w["sdown"],
                                     u(s["exp"]), u(s["silu"]), c["top_k"])
        s["x"] = u(s["x"])
    else:
        s["logits"], s["bias"] = u(s["logits"]), u(s["bias"])


# ---- the plain forms --------------------------------------------------------------------------------


def _round_shift(x, shift):
    return x if shift == 0 else (x + (1 << (shift - 1))) >> shift


def _round_div(a, b):
    return torch.div(2 * a + b, 2 * b, rounding_mode="floor")


def _products(x, w):
    """x @ w of whole numbers: 64-bit floats hold both halves' sums without rounding."""
    hi = x >> 16
    lo = x - (hi << 16)
    return ((hi.double() @ w).to(torch.int64) << 16) + (lo.double() @ w).to(torch.int64)


def _dense(w, group, segment, k):
    """The weights that codes and scales stand for, as 64-bit floats (whole numbers below 2^19)."""
    codes, scales = w
    at = torch.arange(k, device=codes.device)
    row = (at // segment) * -(-segment // group) + (at % segment) // group if segment else at // group
    return codes.double() * scales.double()[..., row, :]


def _plain_project(s):
    c = s["case"]
    x, w = _signed(s["x"]), _dense(s["w"], c["group"], c["segment"], c["k"])
    part = c["segment"] or c["k"]
    x = x.reshape(c["m"], -1, part).transpose(0, 1)
    y = _round_shift(_products(x, w.reshape(-1, part, c["n"])), c["shift"]).sum(0) + _signed(s["bias"])
    if c["gelu"]:
        t = s["table"]
        y = _signed(t[(y + t.numel() // 2).clamp(0, t.numel() - 1)])
    if c["residual"]:
        y = y + _signed(s["residual"])
    return _field(y)


def _plain_attend(s):
    c = s["case"]
    b, hk, dk, dv, cap = c["b"], c["kv_heads"], c["dk"], c["dv"], c["cap"]
    each = c["heads"] // hk
    q, k_new, v_new = _signed(s["rows"]).split([c["heads"] * dk, hk * dk, hk * dv], dim=1)
    k, v, at = s["k"], s["v"], s["lens"].long()
    seq = torch.arange(b, device=k.device)
    k[seq, :, at // BLOCK, :, at % BLOCK, :] = k_new.reshape(b, hk, dk // 4, 4).to(torch.int32)
    v[seq, :, at, :] = v_new.reshape(b, hk, dv).to(torch.int32)
    keys = k.permute(0, 1, 2, 4, 3, 5).reshape(b, hk, cap, dk)
    scores = (q.reshape(b, hk, each, dk).double() @ keys.double().transpose(2, 3)).to(torch.int64)
    scores = _round_shift(scores * s["factor"], 32)
    live = (torch.arange(cap, device=k.device) <= at[:, None])[:, None, None, :]
    top = torch.where(live, scores, torch.iinfo(torch.int64).min).amax(-1, keepdim=True)
    t = s["table"]
    e = torch.where(live, t[(scores - top + t.numel()).clamp(0, t.numel() - 1)], 0)
    p = _round_div(e << 16, e.sum(-1, keepdim=True))
    y = _round_shift((p.double() @ v.double()).to(torch.int64), 16)
    return [_field(y.reshape(b, c["heads"] * dv)), k, v]


def _plain_half(x, w, group):
    """One product of a feed-forward: rounded back to scale 2^16."""
    return _round_shift(_products(x, _dense(w, group, 0, x.shape[-1])), 16)


def _plain_act(x, gate, up, silu, group):
    g, u = _plain_half(x, gate, group), _plain_half(x, up, group)
    half = silu.numel() // 2
    return _round_shift(_signed(silu[(g + half).clamp(0, silu.numel() - 1)]) * u, 16)


def _plain_moe(s):
    c = s["case"]
    m, h, e, top, gr = c["m"], c["h"], c["experts"], c["top_k"], c["group"]
    x = _signed(s["x"])
    logits = _round_shift(_products(x, _signed(s["router"]).double()), 16)
    t = s["exp"]
    ex = t[(logits - logits.amax(1, keepdim=True) + t.numel()).clamp(0, t.numel() - 1)]
    score = _round_div(ex << 16, ex.sum(1, keepdim=True))
    key = score * e + torch.arange(e - 1, -1, -1, device=x.device)  # ties: the lowest expert first
    rank = (key[:, None, :] > key[:, :, None]).sum(2)
    gate = torch.where(rank < top, score, 0)
    pick = torch.argsort(rank, dim=1)[:, :top].reshape(-1)
    xs = x.repeat_interleave(top, 0)[:, None, :]
    take = lambda w: (w[0][pick], w[1][pick])  # noqa: E731
    act = _plain_act(xs, take(s["gate"]), take(s["up"]), s["silu"], gr)
    d = _plain_half(act, take(s["down"]), gr).reshape(m, top, h)
    y = _round_shift(d * torch.gather(score, 1, pick.reshape(m, top))[:, :, None], 16).sum(1)
    y = y + _plain_half(_plain_act(x, s["sgate"], s["sup"], s["silu"], gr), s["sdown"], gr)
    return [_field(y), _field(gate)]


#: a penalty of 1.25 for a token that was there: positive logits by 1 / 1.25, others by 1.25, at scale 2^16
REPEAT = (52429, 81920)
PRESENCE, FREQUENCY = 1 << 30, 1 << 28


def _plain_choose(s):
    c = s["case"]
    b, v = c["b"], c["v"]
    x = _signed(s["logits"])
    there = (torch.arange(c["history"], device=x.device) < s["lens"][:, None]).to(torch.int64)
    count = torch.zeros_like(x).scatter_add_(1, s["history"].long(), there)
    y = _round_shift(x * torch.where(x > 0, REPEAT[0], REPEAT[1]), 16)
    y = torch.where(count > 0, y - PRESENCE - count * FREQUENCY, x)
    if s["bias"] is not None:
        y = y + _signed(s["bias"])
    if s["allowed"] is not None:
        at = torch.arange(v, device=x.device)
        ok = (s["allowed"][..., at // 32] >> (at % 32)) & 1
        y = y + torch.where(ok == 1, 0, LOG_MASK)
    first = torch.where(y == y.amax(1, keepdim=True), torch.arange(v, device=x.device), v).amin(1)
    return [first.to(torch.int32), _field(y)]


# ---- one pass -----------------------------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    return {"project": _plain_project, "attend": _plain_attend, "moe": _plain_moe,
            "choose": _plain_choose}[s["case"]["op"]](s)


def _run_own(s):
    from zkie_b200 import decode
    c = s["case"]
    if c["op"] == "project":
        return decode.project(s["x"], s["weight"], c["shift"], bias=s["bias"], table=s["table"],
                              residual=s["residual"], err=s["err"]).view(torch.int64)
    if c["op"] == "attend":
        nq, nk = c["heads"] * c["dk"], c["kv_heads"] * c["dk"]
        r = s["rows"]
        out = decode.attend(r[:, :nq], s["cache"], s["table"], k=r[:, nq:nq + nk], v=r[:, nq + nk:],
                            score_scale=(s["factor"], 32), err=s["err"])
        return [out.view(torch.int64), s["cache"].k, s["cache"].v]
    if c["op"] == "moe":
        out, gate = s["block"].forward(s["x"], err=s["err"])
        return [out.view(torch.int64), gate.view(torch.int64)]
    token, logits = decode.choose_token(s["logits"], s["history"], s["lens"], repeat=REPEAT, presence=PRESENCE,
                                        frequency=FREQUENCY, bias=s["bias"], allowed=s["allowed"],
                                        mask_value=LOG_MASK, err=s["err"])
    return [token.view(torch.int32), logits.view(torch.int64)]


# ---- the definitions in 64-bit whole numbers, on the host ------------------------------------------------


def _div_exact(a, b):
    """round(a / b), halves up: the quotient rounded down, and one more when twice the remainder reaches b."""
    q = torch.div(a, b, rounding_mode="floor")
    return q + (2 * (a - q * b) >= b).to(torch.int64)


def _whole(w, group):
    codes, scales = (t.cpu().to(torch.int64) for t in w)
    return codes * scales.repeat_interleave(group, 0)[: codes.shape[0]]


def _exact_project(s):
    c, x = s["case"], _signed(s["x"].cpu())
    seg, per = c["segment"] or c["k"], -(-(c["segment"] or c["k"]) // c["group"])
    y = _signed(s["bias"].cpu()).repeat(c["m"], 1)
    for i in range(c["k"] // seg):
        w = _whole((s["w"][0][i * seg:(i + 1) * seg], s["w"][1][i * per:(i + 1) * per]), c["group"])
        y = y + _div_exact(x[:, i * seg:(i + 1) * seg] @ w, torch.tensor(1 << c["shift"]))
    if c["gelu"]:
        t = s["table"].cpu()
        y = _signed(t[torch.clamp(y + t.numel() // 2, 0, t.numel() - 1)])
    return _field(y + _signed(s["residual"].cpu()) if c["residual"] else y)


def _exact_attend(s):
    c = s["case"]
    b, hk, dk, dv, each = c["b"], c["kv_heads"], c["dk"], c["dv"], c["heads"] // c["kv_heads"]
    rows, k, v, t = _signed(s["rows"].cpu()), s["k"].cpu(), s["v"].cpu(), s["table"].cpu()
    out = torch.zeros(b, c["heads"], dv, dtype=torch.int64)
    for i, n in enumerate(s["lens"].tolist()):
        new_k = rows[i, c["heads"] * dk:][: hk * dk].reshape(hk, dk).to(torch.int32)
        v[i, :, n] = rows[i, (c["heads"] + hk) * dk:].reshape(hk, dv).to(torch.int32)
        k[i, :, n // BLOCK, :, n % BLOCK] = new_k.reshape(hk, dk // 4, 4)
        for h in range(c["heads"]):
            keys = k[i, h // each].transpose(1, 2).reshape(-1, dk)[: n + 1].to(torch.int64)
            z = _div_exact((keys @ rows[i, h * dk:(h + 1) * dk]) * s["factor"], torch.tensor(1 << 32))
            e = t[torch.clamp(z - z.max() + t.numel(), 0, t.numel() - 1)]
            p = _div_exact(e * 65536, e.sum())
            out[i, h] = _div_exact(p @ v[i, h // each, : n + 1].to(torch.int64), torch.tensor(65536))
    return [_field(out.reshape(b, -1)), k, v]


def _exact_moe(s):
    c, x = s["case"], _signed(s["x"].cpu())
    one, silu, t = torch.tensor(65536), s["silu"].cpu(), s["exp"].cpu()

    def feed(row, gate, up, down):
        g = _div_exact(row @ _whole(gate, c["group"]), one)
        u = _div_exact(row @ _whole(up, c["group"]), one)
        a = _signed(silu[torch.clamp(g + silu.numel() // 2, 0, silu.numel() - 1)])
        return _div_exact(_div_exact(a * u, one) @ _whole(down, c["group"]), one)

    out, gates = feed(x, s["sgate"], s["sup"], s["sdown"]), torch.zeros(c["m"], c["experts"], dtype=torch.int64)
    logits = _div_exact(x @ _signed(s["router"].cpu()), one)
    pairs = lambda w, i: (w[0][i], w[1][i])  # noqa: E731
    for r in range(c["m"]):
        e = t[torch.clamp(logits[r] - logits[r].max() + t.numel(), 0, t.numel() - 1)]
        p = _div_exact(e * 65536, e.sum()).tolist()
        for i in sorted(range(c["experts"]), key=lambda i: (-p[i], i))[: c["top_k"]]:
            d = feed(x[r], pairs(s["gate"], i), pairs(s["up"], i), pairs(s["down"], i))
            out[r] += _div_exact(d * p[i], one)
            gates[r, i] = p[i]
    return [_field(out), gates]


def _exact_choose(s):
    c, x = s["case"], _signed(s["logits"].cpu())
    b, v = c["b"], c["v"]
    count = torch.stack([torch.bincount(s["history"][i, : s["lens"][i]].cpu().long(), minlength=v) for i in range(b)])
    pen = torch.where(x > 0, _div_exact(x * REPEAT[0], torch.tensor(65536)), _div_exact(x * REPEAT[1], torch.tensor(65536)))
    y = torch.where(count > 0, pen - PRESENCE - FREQUENCY * count, x)
    if s["bias"] is not None:
        y = y + _signed(s["bias"].cpu())
    if s["allowed"] is not None:
        words = s["allowed"].cpu().to(torch.int64) & WRAP
        bits = ((words[..., None] >> torch.arange(32)) & 1).reshape(*words.shape[:-1], -1)[..., :v]
        y = y + (1 - bits) * LOG_MASK
    best = [int((row == row.max()).nonzero()[0, 0]) for row in y]
    return [torch.tensor(best, dtype=torch.int32), _field(y)]


def exact(case, seed):
    if work(case)["flops"] > 2.5e9:  # whole-number products on the host: about a tenth of that a second
        return None
    s = prepare(case, seed)
    return {"project": _exact_project, "attend": _exact_attend, "moe": _exact_moe,
            "choose": _exact_choose}[case["op"]](s)
