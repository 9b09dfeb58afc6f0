"""Plain forms of the single-token operators (zkie_b200/decode.py) in Python
integers and numpy int64, from their definitions.  Field elements come and go
as signed int64 here; ``field`` / ``signed`` convert."""
import numpy as np

P = 0xFFFFFFFF00000001


def field(x):
    x = np.asarray(x, dtype=np.int64)
    return np.where(x < 0, x - np.int64(0xFFFFFFFF), x).view(np.uint64)


def signed(u):
    v = np.asarray(u, dtype=np.uint64).view(np.int64)
    return np.where(v < 0, v + np.int64(0xFFFFFFFF), v)


def round_shift(x, s):
    """round_div(x, 2^s): floor, plus one when twice the remainder reaches 2^s."""
    x = np.asarray(x, dtype=np.int64)
    return (x >> s) + (((x & ((1 << s) - 1)) * 2 >= (1 << s)) if s else 0)


def round_div(a, b):
    q = np.floor_divide(a, b)
    return q + (2 * (a - q * b) >= b)


def dense(codes, scales, group, segment=0):
    """k x n weights of codes (k x n) and scales (rows x n)."""
    k = codes.shape[0]
    at = np.arange(k)
    row = at // segment * -(-segment // group) + at % segment // group if segment else at // group
    return codes.astype(np.int64) * scales.astype(np.int64)[row]


def scale_rows(k, group, segment=0):
    return k // segment * -(-segment // group) if segment else -(-k // group)


def weight(rng, k, n, group, segment=0, experts=0, most=450):
    lead = (experts,) if experts else ()
    return (rng.integers(-8, 8, lead + (k, n), dtype=np.int8),
            rng.integers(0, most, lead + (scale_rows(k, group, segment), n), dtype=np.int32))


def product(x, w):
    """x @ w in Python integers (any size), as int64."""
    return np.array(x.astype(object) @ w.astype(object), dtype=object).astype(np.int64)


def project(x, codes, scales, group, segment, shift, bias=None, table=None, offset=0, residual=None):
    w, part = dense(codes, scales, group, segment), segment or codes.shape[0]
    y = np.zeros((x.shape[0], codes.shape[1]), dtype=np.int64)
    for s in range(0, codes.shape[0], part):
        y += round_shift(product(x[:, s:s + part], w[s:s + part]), shift)
    if bias is not None:
        y = y + bias
    if table is not None:
        y = table[np.clip(y + offset, 0, table.size - 1)]
    return y if residual is None else y + residual


def softmax(z, table, offset=None):
    e = table[np.clip(z - z.max() + (table.size if offset is None else offset), 0, table.size - 1)]
    return round_div(e << 16, e.sum())


def attend(q, keys, values, table, score_scale, out_shift=16, offset=None):
    """One head: q (dk), keys (n x dk), values (n x dv)."""
    z = round_shift(product(keys, q[:, None])[:, 0] * score_scale[0], score_scale[1])
    return round_shift(product(softmax(z, table, offset)[None], values)[0], out_shift)


def blocks_of(keys):
    """(.., cap, dk) -> the cache's (.., cap / 32, dk / 4, 32, 4)."""
    *lead, cap, dk = keys.shape
    return np.ascontiguousarray(np.moveaxis(keys.reshape(*lead, cap // 32, 32, dk // 4, 4), -2, -3))


def keys_of(blocks):
    *lead, nb, d4, _, _ = blocks.shape
    return np.moveaxis(blocks, -3, -2).reshape(*lead, nb * 32, d4 * 4)


def moe(x, router, weights, group, exp_table, silu, top_k, shift=16):
    """weights: six (codes, scales), the first three with a leading expert axis."""
    def feed(row, g, u, d):
        half = silu.size // 2
        a = silu[np.clip(round_shift(product(row, dense(*g, group)), shift) + half, 0, silu.size - 1)]
        act = round_shift(a * round_shift(product(row, dense(*u, group)), shift), shift)
        return round_shift(product(act, dense(*d, group)), shift)

    m, experts = x.shape[0], router.shape[1]
    out, gate = feed(x, *weights[3:]), np.zeros((m, experts), dtype=np.int64)
    logits = round_shift(product(x, router), shift)
    for r in range(m):
        p = softmax(logits[r], exp_table)
        for e in sorted(range(experts), key=lambda i: (-p[i], i))[:top_k]:
            d = feed(x[r:r + 1], *[(c[e], s[e]) for c, s in weights[:3]])[0]
            out[r] += round_shift(d * p[e], 16)
            gate[r, e] = p[e]
    return out, gate


def choose(logits, history=None, lens=None, repeat=(1 << 16, 1 << 16), presence=0, frequency=0, bias=None,
           allowed=None, mask_value=-(1 << 41)):
    b, v = logits.shape
    y = logits.copy()
    for r in range(b):
        if history is not None:
            row = history[r] if lens is None else history[r, :max(0, lens[r])]
            count = np.bincount(row[(row >= 0) & (row < v)], minlength=v)
            pen = np.where(y[r] > 0, round_shift(y[r] * repeat[0], 16), round_shift(y[r] * repeat[1], 16))
            y[r] = np.where(count > 0, pen - presence - count * frequency, y[r])
        if bias is not None:
            y[r] += bias if bias.ndim == 1 else bias[r]
        if allowed is not None:
            words = (allowed if allowed.ndim == 1 else allowed[r]).view(np.uint32)
            ok = (words[np.arange(v) // 32] >> (np.arange(v) % 32).astype(np.uint32)) & 1
            y[r] += np.where(ok == 1, 0, mask_value)
    return y.argmax(axis=1), y  # numpy's argmax: the first of equals
