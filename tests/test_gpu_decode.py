"""The single-token operators on the device (zkie_b200/csrc/decode.cu,
decode_moe.cu, zkie_b200/decode.py) against their plain forms in 64-bit whole
numbers (tests/decode_ref.py).  Every result is a whole number: equality, no
tolerance."""
import numpy as np
import pytest

from tests import decode_ref as ref

pytestmark = pytest.mark.gpu


def _u(x):
    import torch
    return torch.from_numpy(ref.field(x)).cuda()


def _i32(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _s(t):
    return ref.signed(t.cpu().numpy())


def _quant(zk, w, group, segment=0):
    import torch
    return zk.decode.QuantWeight(torch.from_numpy(w[0]), torch.from_numpy(w[1]), group=group, segment=segment)


def _exp_table(bits=21):
    return np.round(np.exp(np.arange(-(1 << bits), 0) / 65536.0) * 65536).astype(np.int64)


def _silu_table(bits=20):
    x = (np.arange(1 << bits) - (1 << (bits - 1))) / 65536.0
    return np.round(x / (1 + np.exp(-x)) * 65536).astype(np.int64)


# ---- 4-bit weights -----------------------------------------------------------------------------------
@pytest.mark.parametrize("k,n,group,segment,experts", [
    (1, 1, 32, 0, 0), (64, 16, 64, 0, 0), (100, 17, 32, 0, 0), (130, 33, 128, 0, 2), (60, 5, 64, 20, 0),
    (256, 40, 128, 128, 0), (8192, 16, 64, 0, 0), (96, 24, 32, 48, 3)])
def test_weight_layout_round_trip(zk, k, n, group, segment, experts):
    rng = np.random.default_rng(k + n)
    w = ref.weight(rng, k, n, group, segment, experts, most=65536)
    q = _quant(zk, w, group, segment)
    c, s = w if experts else (w[0][None], w[1][None])
    assert np.array_equal(q.codes().cpu().numpy(), c)
    assert np.array_equal(q.scales().cpu().numpy(), s)
    want = np.stack([ref.dense(c[e], s[e], group, segment) for e in range(c.shape[0])]).reshape(-1)
    assert np.array_equal(_s(q.dense()), want)


def test_quantise_is_nearest(zk):
    import torch
    rng = np.random.default_rng(5)
    w = rng.integers(-3000, 3000, (100, 40))
    w[:32, 0] = 0
    codes, scales = zk.decode.quantise(_u(w), group=32)
    d = ref.dense(codes.cpu().numpy(), scales.cpu().numpy(), 32)
    assert np.all(2 * np.abs(d - w) <= scales.cpu().numpy()[np.arange(100) // 32])
    again = zk.decode.quantise(torch.from_numpy(d).cuda(), group=32)  # numbers, not field elements
    assert np.array_equal(ref.dense(*[t.cpu().numpy() for t in again], 32), d)
    with pytest.raises(ValueError, match="65535"):
        zk.decode.quantise(torch.full((4, 4), 1 << 20, device="cuda", dtype=torch.int64))


@pytest.mark.parametrize("m,k,n,group,segment,shift", [
    (1, 1, 1, 32, 0, 0), (1, 64, 16, 64, 0, 16), (2, 100, 17, 32, 0, 8), (3, 130, 300, 128, 0, 16),
    (4, 768, 64, 64, 64, 16), (5, 60, 33, 64, 20, 7), (8, 1024, 192, 128, 128, 16), (9, 200, 40, 32, 0, 1),
    (17, 96, 50, 64, 32, 16), (8, 4100, 20, 64, 0, 16), (3, 8192, 31, 128, 0, 0), (1, 2048, 5000, 32, 0, 16),
    (2, 40, 45000, 64, 0, 3), (5, 260, 4000, 128, 0, 16), (3, 512, 2400, 128, 256, 9)])
def test_project(zk, m, k, n, group, segment, shift):
    rng = np.random.default_rng(m * k + n)
    w = ref.weight(rng, k, n, group, segment)
    x = rng.integers(-(1 << 22), 1 << 22, (m, k))
    bias = rng.integers(-(1 << 20), 1 << 20, n)
    got = zk.decode.project(_u(x), _quant(zk, w, group, segment), shift, bias=_u(bias))
    assert np.array_equal(_s(got), ref.project(x, *w, group, segment, shift, bias))
    plain = zk.decode.project(_u(x), _quant(zk, w, group, segment), shift)
    assert np.array_equal(_s(plain), ref.project(x, *w, group, segment, shift))


@pytest.mark.parametrize("offset", [None, 100])
def test_project_epilogue_and_strides(zk, offset):
    """Table and residual, x and residual as columns of wider matrices, an output given."""
    import torch
    rng = np.random.default_rng(3)
    m, k, n = 3, 96, 37
    w = ref.weight(rng, k, n, 32)
    x, res, table = rng.integers(-(1 << 20), 1 << 20, (m, k)), rng.integers(-9000, 9000, (m, n)), \
        rng.integers(-70000, 70000, 1001)
    wide_x = _u(np.concatenate([x + 1, x, x - 1], axis=1))
    wide_r = _u(np.concatenate([res, res + 5], axis=1))
    out = torch.zeros((m, n), dtype=torch.uint64, device="cuda")
    got = zk.decode.project(wide_x[:, k:2 * k], _quant(zk, w, 32), 20, table=_u(table), offset=offset,
                            residual=wide_r[:, :n], out=out)
    assert got is out
    want = ref.project(x, *w, 32, 0, 20, table=table, offset=500 if offset is None else offset, residual=res)
    assert np.array_equal(_s(got), want)


def test_project_odd_rows(zk):
    """Rows that start at odd places (8-byte aligned only) and none at all."""
    import torch
    rng = np.random.default_rng(12)
    w, wide = ref.weight(rng, 130, 40, 64), rng.integers(-(1 << 20), 1 << 20, (6, 133))
    q, u = _quant(zk, w, 64), _u(wide)
    for off in (0, 1, 2, 3):
        got = zk.decode.project(u[:, off:off + 130], q, 12)
        assert np.array_equal(_s(got), ref.project(wide[:, off:off + 130], *w, 64, 0, 12))
    got = zk.decode.project(u[1::2, 1:131], q, 12)
    assert np.array_equal(_s(got), ref.project(wide[1::2, 1:131], *w, 64, 0, 12))
    assert zk.decode.project(u[:0, :130], q, 12).shape == (0, 40)
    with pytest.raises(ValueError, match="unit stride"):
        zk.decode.project(torch.as_strided(u, (3, 130), (133, 2)), q, 12)
    with pytest.raises(ValueError, match="unit stride"):
        zk.decode.project(torch.as_strided(u, (3, 130), (7, 1)), q, 12)


def test_project_extremes(zk):
    """The largest numbers and weights over the longest sum: |h| just below 2^63."""
    for sign in (1, -1):
        for code in (-8, 7):
            x = np.full((2, 8192), sign * 0x7F7F7F7F)
            w = (np.full((8192, 3), code, dtype=np.int8), np.full((64, 3), 65535, dtype=np.int32))
            for shift in (0, 16):
                got = zk.decode.project(_u(x), _quant(zk, w, 128), shift)
                assert np.array_equal(_s(got), ref.project(x, *w, 128, 0, shift))


@pytest.mark.parametrize("value", [0x7F7F7F80, -0x7F7F7F80, 1 << 40, -(1 << 62)])
def test_project_refuses_values_out_of_range(zk, value):
    import torch
    rng = np.random.default_rng(1)
    w, x = ref.weight(rng, 64, 16, 64), rng.integers(-1000, 1000, (2, 64))
    x[1, 7] = value
    with pytest.raises(ValueError, match="range"):
        zk.decode.project(_u(x), _quant(zk, w, 64), 4)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = zk.decode.project(_u(x), _quant(zk, w, 64), 4, err=err)
    x[1, 7] = 0
    assert int(err.item()) == 8 and np.array_equal(_s(got), ref.project(x, *w, 64, 0, 4))


# ---- attention over a cache ----------------------------------------------------------------------------
def _cache(zk, rng, b, hk, dk, dv, cap, lens, big=False):
    lim = 1 << (27 if big else 19)
    keys = rng.integers(-lim, lim, (b, hk, cap, dk))
    values = rng.integers(-(1 << 31) if big else -(1 << 19), (1 << 31) if big else 1 << 19, (b, hk, cap, dv))
    return keys, values, zk.decode.KvCache(_i32(ref.blocks_of(keys)), _i32(values), _i32(lens))


@pytest.mark.parametrize("b,hk,each,dk,dv,cap,lens", [
    (1, 1, 1, 4, 4, 32, [0]), (1, 2, 1, 64, 64, 64, [31]), (3, 2, 1, 64, 64, 96, [32, 0, 95]),
    (2, 3, 2, 40, 24, 320, [33, 300]), (2, 1, 3, 16, 100, 64, [5, 63]), (1, 2, 4, 128, 128, 2048, [2000]),
    (1, 1, 9, 8, 12, 160, [129]), (2, 2, 1, 192, 128, 512, [511, 256]), (1, 1, 1, 256, 256, 992, [700]),
    (1, 1, 2, 36, 132, 128, [70]), (1, 2, 5, 4, 200, 96, [65]), (1, 1, 4, 8, 8, 131072, [131071]),
    (1, 1, 1, 16, 4, 131072, [100003]),
    (40, 5, 1, 16, 16, 64, list(range(40)))])
def test_attend(zk, b, hk, each, dk, dv, cap, lens):
    rng = np.random.default_rng(dk + cap + b)
    keys, values, cache = _cache(zk, rng, b, hk, dk, dv, cap, lens)
    heads, table = hk * each, _exp_table()
    q = rng.integers(-(1 << 18), 1 << 18, (b, heads * dk))
    nk, nv = rng.integers(-(1 << 18), 1 << 18, (b, hk * dk)), rng.integers(-(1 << 18), 1 << 18, (b, hk * dv))
    rows = _u(np.concatenate([q, nk, nv], axis=1))  # as one wide projection leaves them
    scale = (round(2 ** 16 / dk ** 0.5), 34)
    got = zk.decode.attend(rows[:, :heads * dk], cache, _u(table), k=rows[:, heads * dk:(heads + hk) * dk],
                           v=rows[:, (heads + hk) * dk:], q_scale=(23170, 16), k_scale=(50000, 16), score_scale=scale)
    qs, ks = ref.round_shift(q * 23170, 16), ref.round_shift(nk * 50000, 16)
    for i, n in enumerate(lens):
        keys[i, :, n], values[i, :, n] = ks[i].reshape(hk, dk), nv[i].reshape(hk, dv)
    want = np.stack([np.concatenate([
        ref.attend(qs[i, h * dk:(h + 1) * dk], keys[i, h // each, :n + 1], values[i, h // each, :n + 1], table, scale)
        for h in range(heads)]) for i, n in enumerate(lens)])
    assert np.array_equal(_s(got), want)
    # the cache holds the new token and nothing else has changed
    assert np.array_equal(ref.keys_of(cache.k.cpu().numpy()), keys) and np.array_equal(cache.v.cpu().numpy(), values)
    cache.advance()
    again = zk.decode.attend(rows[:, :heads * dk], cache, _u(table), q_scale=(23170, 16), score_scale=scale)
    assert np.array_equal(_s(again), want)  # the same tokens, now from the cache alone


def test_attend_far_into_a_large_cache(zk):
    """A cache of more than 2^32 numbers: the last heads' keys and values."""
    import torch
    rng = np.random.default_rng(14)
    hk, dk, dv, cap, n = 130, 256, 4, 131072, 40
    cache = zk.decode.KvCache.zeros(1, hk, dk, dv, cap)
    assert cache.k.numel() > 1 << 32
    keys, values = rng.integers(-(1 << 19), 1 << 19, (hk, 64, dk)), rng.integers(-(1 << 19), 1 << 19, (hk, 64, dv))
    cache.k[0, :, cap // 32 - 2:] = _i32(ref.blocks_of(keys))
    cache.v[0, :, cap - 64:] = _i32(values)
    cache.lens.fill_(cap - 1)
    q, nk, nv = (rng.integers(-(1 << 18), 1 << 18, (1, hk * d)) for d in (dk, dk, dv))
    table = _exp_table()
    got = _s(zk.decode.attend(_u(q), cache, _u(table), k=_u(nk), v=_u(nv), score_scale=(4096, 32))).reshape(hk, dv)
    for h in (0, 63, hk - 1):
        full_k, full_v = np.zeros((cap, dk), dtype=np.int64), np.zeros((cap, dv), dtype=np.int64)
        full_k[-64:], full_v[-64:] = keys[h], values[h]
        full_k[-1], full_v[-1] = nk.reshape(hk, dk)[h], nv.reshape(hk, dv)[h]
        z = ref.round_shift((full_k @ q.reshape(hk, dk)[h]) * 4096, 32)
        want = ref.round_shift(ref.softmax(z, table) @ full_v, 16)
        assert np.array_equal(got[h], want), h
    assert torch.equal(cache.v[0, :, cap - 1].cpu(), torch.from_numpy(nv.reshape(hk, dv).astype(np.int32)))


def test_attend_inactive_empty_and_full(zk):
    """A sequence of negative length and one without tokens answer zeros, a
    full cache takes no new token and says so."""
    import torch
    rng = np.random.default_rng(8)
    keys, values, cache = _cache(zk, rng, 4, 1, 8, 8, 32, [-1, 0, 32, 31])
    table = _exp_table()
    q, nk, nv = (rng.integers(-(1 << 17), 1 << 17, (4, 8)) for _ in range(3))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = _s(zk.decode.attend(_u(q), cache, _u(table), err=err))
    assert int(err.item()) == 0 and not got[:2].any() and got[2:].any(axis=1).all()
    got = _s(zk.decode.attend(_u(q), cache, _u(table), k=_u(nk), v=_u(nv), err=err))
    assert int(err.item()) == 16 and not got[0].any()
    assert np.array_equal(got[1], ref.round_shift(nv[1] << 16, 16))
    assert np.array_equal(got[2], ref.attend(q[2], keys[2, 0], values[2, 0], table, (1, 16)))
    keys[1, 0, 0], keys[3, 0, 31], values[1, 0, 0], values[3, 0, 31] = nk[1], nk[3], nv[1], nv[3]
    assert np.array_equal(ref.keys_of(cache.k.cpu().numpy()), keys) and np.array_equal(cache.v.cpu().numpy(), values)
    with pytest.raises(ValueError, match="full"):
        zk.decode.attend(_u(q), cache, _u(table), k=_u(nk), v=_u(nv))
    cache.advance()
    assert cache.lens.tolist() == [-1, 1, 33, 32]


def test_attend_extremes(zk):
    """Keys and queries of 2^27 over 256 dimensions, values of the whole 32
    bits, and a row whose scores are all equal."""
    rng = np.random.default_rng(9)
    dk = 256
    keys, values, cache = _cache(zk, rng, 1, 1, dk, 8, 64, [64], big=True)
    keys[0, 0, 3], keys[0, 0, 9] = 1 << 27, -(1 << 27)
    cache.k.copy_(_i32(ref.blocks_of(keys)))
    table = _exp_table()
    for q in (np.full(dk, 1 << 27), np.full(dk, -(1 << 27)), np.zeros(dk, dtype=np.int64)):
        got = zk.decode.attend(_u(q[None]), cache, _u(table), score_scale=(1, 40))
        assert np.array_equal(_s(got)[0], ref.attend(q, keys[0, 0], values[0, 0], table, (1, 40)))


def test_attend_refuses_values_out_of_range(zk):
    import torch
    rng = np.random.default_rng(10)
    _, _, cache = _cache(zk, rng, 1, 1, 4, 4, 32, [3])
    table = _exp_table(8)
    ok, bad = _u(np.ones((1, 4), dtype=np.int64)), _u(np.array([[1, (1 << 27) + 1, 0, 0]]))
    wide = _u(np.array([[1, 1 << 31, 0, 0]]))
    for args in ((bad, ok, ok), (ok, bad, ok), (ok, ok, wide)):
        with pytest.raises(ValueError, match="range"):
            zk.decode.attend(args[0], cache, _u(table), k=args[1], v=args[2])
    with pytest.raises(ValueError, match="range"):  # a negative table entry
        zk.decode.attend(ok, cache, _u(np.full(4, -1)))
    with pytest.raises(ValueError, match="row sum of zero"):
        zk.decode.attend(ok, cache, _u(np.zeros(4, dtype=np.int64)))
    torch.cuda.synchronize()


@pytest.mark.parametrize("tokens,lens", [(1, [0, 31]), (33, [0, 40]), (64, [-1, 0])])
def test_append(zk, tokens, lens):
    rng = np.random.default_rng(tokens)
    b, hk, dk, dv, cap = 2, 3, 12, 20, 96
    keys, values, cache = _cache(zk, rng, b, hk, dk, dv, cap, lens)
    k = rng.integers(-(1 << 20), 1 << 20, (b, tokens, hk, dk))
    v = rng.integers(-(1 << 31), 1 << 31, (b, tokens, hk, dv))
    cache.append(_u(k.reshape(b, tokens, -1)), _u(v.reshape(b, tokens, -1)), k_scale=(23170, 16))
    for i, n in enumerate(lens):
        if n >= 0:
            keys[i, :, n:n + tokens] = np.moveaxis(ref.round_shift(k[i] * 23170, 16), 0, 1)
            values[i, :, n:n + tokens] = np.moveaxis(v[i], 0, 1)
    assert np.array_equal(ref.keys_of(cache.k.cpu().numpy()), keys) and np.array_equal(cache.v.cpu().numpy(), values)
    with pytest.raises(ValueError, match="full"):
        cache.append(_u(np.zeros((b, 97, hk * dk), dtype=np.int64)), _u(np.zeros((b, 97, hk * dv), dtype=np.int64)))


# ---- a mixture-of-experts layer -----------------------------------------------------------------------
def _moe_case(rng, h, experts, f, shared, group):
    w = [ref.weight(rng, h, f, group, experts=experts), ref.weight(rng, h, f, group, experts=experts),
         ref.weight(rng, f, h, group, experts=experts), ref.weight(rng, h, shared, group),
         ref.weight(rng, h, shared, group), ref.weight(rng, shared, h, group)]
    return rng.integers(-32639, 32640, (h, experts)), w


def _moe_block(zk, router, w, group, top_k, exp_table, silu):
    q = [_quant(zk, t, group) for t in w]
    return zk.decode.MoeBlock(_u(router), *q, _u(exp_table), _u(silu), top_k)


@pytest.mark.parametrize("m,h,experts,top_k,f,shared,group", [
    (1, 16, 1, 1, 8, 8, 32), (1, 64, 8, 2, 48, 96, 64), (3, 100, 17, 3, 40, 33, 32), (8, 256, 33, 6, 64, 128, 128),
    (16, 130, 64, 6, 70, 50, 64), (17, 64, 4, 4, 32, 16, 32), (40, 48, 20, 5, 20, 24, 64), (5, 1000, 200, 16, 24, 40, 128),
    (16, 70, 40, 16, 24, 20, 32), (3, 8192, 5, 2, 16, 20, 64), (2, 64, 4, 2, 8192, 8190, 128), (7, 40, 256, 9, 600, 5, 64)])
def test_moe_block(zk, m, h, experts, top_k, f, shared, group):
    rng = np.random.default_rng(m + h)
    router, w = _moe_case(rng, h, experts, f, shared, group)
    x, exp_table, silu = rng.integers(-(1 << 17), 1 << 17, (m, h)), _exp_table(), _silu_table()
    block = _moe_block(zk, router, w, group, top_k, exp_table, silu)
    res = rng.integers(-(1 << 20), 1 << 20, (m, h))
    out, gate = block.forward(_u(x), residual=_u(res))
    want, want_gate = ref.moe(x, router, w, group, exp_table, silu, top_k)
    assert np.array_equal(_s(gate), want_gate)
    assert np.array_equal(_s(out), want + res)
    assert np.array_equal(_s(block.forward(_u(x))[0]), want)


def test_moe_ties_and_one_expert_for_all(zk):
    """Equal scores go to the lowest expert; every token to the same experts
    (more than eight tokens to an expert)."""
    rng = np.random.default_rng(4)
    h, experts, f, shared, group, m = 64, 12, 40, 24, 32, 16
    router, w = _moe_case(rng, h, experts, f, shared, group)
    router[:] = router[:, :1]
    x, exp_table, silu = rng.integers(-(1 << 17), 1 << 17, (m, h)), _exp_table(), _silu_table()
    out, gate = _moe_block(zk, router, w, group, 5, exp_table, silu).forward(_u(x))
    want, want_gate = ref.moe(x, router, w, group, exp_table, silu, 5)
    assert np.array_equal(_s(gate), want_gate) and np.array_equal(_s(out), want)
    assert (np.flatnonzero(want_gate.any(axis=0)) == np.arange(5)).all()


def test_moe_refuses_values_out_of_range(zk):
    rng = np.random.default_rng(6)
    router, w = _moe_case(rng, 32, 4, 16, 16, 32)
    block = _moe_block(zk, router, w, 32, 2, _exp_table(12), _silu_table(12))
    x = rng.integers(-1000, 1000, (2, 32))
    x[1, 3] = 1 << 33
    with pytest.raises(ValueError, match="range"):
        block.forward(_u(x))
    router[0, 0] = 40000
    with pytest.raises(ValueError, match="range"):
        _moe_block(zk, router, w, 32, 2, _exp_table(12), _silu_table(12))


# ---- the next token -----------------------------------------------------------------------------------
@pytest.mark.parametrize("b,v,t,bias,allowed", [
    (1, 1, 0, None, None), (1, 31, 5, "shared", "shared"), (3, 1000, 200, "row", "row"), (2, 50257, 600, None, "row"),
    (5, 65536, 64, "shared", None), (2, 70001, 900, "row", "shared"), (17, 2049, 1, None, None)])
def test_choose_token(zk, b, v, t, bias, allowed):
    rng = np.random.default_rng(v + t)
    logits = rng.integers(-(1 << 35), 1 << 35, (b, v))
    history = rng.integers(0, v, (b, t)).astype(np.int32) if t else None
    if t:
        history[:, :t // 2] = rng.integers(0, max(1, v // 50), (b, t // 2))
    lens = rng.integers(0, t + 1, b).astype(np.int32) if t else None
    bs = None if bias is None else rng.integers(-(1 << 33), 1 << 33, (v,) if bias == "shared" else (b, v))
    words = -(-v // 32)
    al = None if allowed is None else rng.integers(-(1 << 31), 1 << 31, (words,) if allowed == "shared" else (b, words))
    al = None if al is None else al.astype(np.int32)
    kw = dict(repeat=(52429, 81920), presence=1 << 30, frequency=12345678)
    tok, out = zk.decode.choose_token(_u(logits), None if history is None else _i32(history),
                                      None if lens is None else _i32(lens), bias=None if bs is None else _u(bs),
                                      allowed=None if al is None else _i32(al), **kw)
    want_tok, want = ref.choose(logits, history, lens, bias=bs, allowed=al, **kw)
    assert np.array_equal(_s(out), want) and np.array_equal(tok.cpu().numpy(), want_tok)


def test_choose_token_ties_empty_masks_and_bad_history(zk):
    import torch
    v = 5000
    logits = np.zeros((2, v), dtype=np.int64)
    logits[1, [17, 4096, 4999]] = 5
    tok, _ = zk.decode.choose_token(_u(logits))
    assert tok.tolist() == [0, 17]
    nothing = _i32(np.zeros(-(-v // 32)))
    tok, out = zk.decode.choose_token(_u(logits), allowed=nothing)
    assert tok.tolist() == [0, 17] and np.array_equal(_s(out), logits - (1 << 41))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    hist = np.array([[3, -1, v], [17, 17, 4096]], dtype=np.int32)
    tok, out = zk.decode.choose_token(_u(logits), _i32(hist), repeat=(1 << 15, 1 << 17), err=err)
    want_tok, want = ref.choose(logits, hist, repeat=(1 << 15, 1 << 17))
    assert int(err.item()) == 1 and np.array_equal(_s(out), want) and tok.tolist() == want_tok.tolist() == [0, 4999]
    with pytest.raises(ValueError, match="index"):
        zk.decode.choose_token(_u(logits), _i32(hist))
    # no history, and rows that are none
    empty = zk.decode.choose_token(_u(logits), _i32(np.zeros((2, 0))), _i32([0, 0]), presence=5)[1]
    assert np.array_equal(_s(empty), logits)
    assert zk.decode.choose_token(_u(logits)[:0])[0].shape == (0,)
    # a length past the row is the whole row, a negative one none of it
    got = zk.decode.choose_token(_u(logits), _i32(hist), _i32([-4, 9]), presence=1, err=err)[1]
    assert np.array_equal(_s(got), ref.choose(logits, hist, [0, 3], presence=1)[1])


# ---- outputs that are given --------------------------------------------------------------------------
def test_outputs_apart_from_inputs(zk):
    """An output may be the residual, and shares memory with nothing else that a call reads."""
    import torch
    rng = np.random.default_rng(77)
    m, k = 3, 64
    w = ref.weight(rng, k, k, 32)
    q = _quant(zk, w, 32)
    x, r = rng.integers(-1 << 18, 1 << 18, (m, k)), rng.integers(-1 << 18, 1 << 18, (m, k))
    want = ref.project(x, *w, 32, 0, 16, residual=r)
    both = torch.cat([_u(x), _u(r)])
    out = zk.decode.project(both[:m], q, 16, residual=both[m:], out=both[m:])
    assert out.data_ptr() == both[m:].data_ptr() and np.array_equal(_s(both[m:]), want)
    for to in (both[:m], both[1:m + 1]):
        with pytest.raises(ValueError, match="shares memory"):
            zk.decode.project(both[:m], q, 16, out=to)
    with pytest.raises(ValueError, match="shares memory"):
        zk.decode.project(_u(x), q, 16, residual=both[:m], out=both[1:m + 1])
    table = _u(_exp_table(10))
    cache = zk.decode.KvCache.zeros(m, 1, k, k, 32)
    with pytest.raises(ValueError, match="shares memory"):
        zk.decode.attend(both[:m], cache, table, out=both[:m])
    with pytest.raises(ValueError, match="shares memory"):
        zk.decode.attend(_u(x), cache, table, k=_u(x), v=both[m:], out=both[m:])
    logits, bias = both[:m], both[m]
    with pytest.raises(ValueError, match="shares memory"):
        zk.decode.choose_token(logits, out=logits)
    with pytest.raises(ValueError, match="shares memory"):
        zk.decode.choose_token(_u(x), bias=bias, out=both[m:])
    with pytest.raises(AttributeError):
        cache.lens = cache.lens + 1


def test_moe_output_apart_from_input(zk):
    rng = np.random.default_rng(78)
    m, h = 2, 64
    router, w = _moe_case(rng, h, 4, 32, 32, 32)
    block = _moe_block(zk, router, w, 32, 2, _exp_table(), _silu_table())
    x, r = rng.integers(-1 << 17, 1 << 17, (m, h)), rng.integers(-1 << 17, 1 << 17, (m, h))
    to = _u(r)
    plain, gate = block.forward(_u(x), residual=_u(r))
    got, gate2 = block.forward(_u(x), residual=to, out=to)
    assert np.array_equal(_s(got), _s(plain)) and np.array_equal(_s(gate), _s(gate2))
    xs = _u(x)
    with pytest.raises(ValueError, match="shares memory"):
        block.forward(xs, out=xs)


@pytest.mark.parametrize("b,v", [(15, 4097), (22, 20000), (40, 8193), (70, 33000), (300, 12345), (1000, 40)])
def test_choose_token_many_rows(zk, b, v):
    """More rows than find room as clusters of one step's blocks: fewer blocks
    to a row, more steps, down to one block."""
    rng = np.random.default_rng(b)
    logits, history = rng.integers(-(1 << 35), 1 << 35, (b, v)), rng.integers(0, v, (b, 50)).astype(np.int32)
    bias = rng.integers(-(1 << 33), 1 << 33, v)
    tok, out = zk.decode.choose_token(_u(logits), _i32(history), presence=1 << 34, bias=_u(bias))
    want_tok, want = ref.choose(logits, history, presence=1 << 34, bias=bias)
    assert np.array_equal(_s(out), want) and np.array_equal(tok.cpu().numpy(), want_tok)


def test_moe_no_rows(zk):
    rng = np.random.default_rng(9)
    router, w = _moe_case(rng, 32, 4, 16, 16, 32)
    out, gate = _moe_block(zk, router, w, 32, 2, _exp_table(12), _silu_table(12)).forward(_u(np.zeros((0, 32), dtype=np.int64)))
    assert out.shape == (0, 32) and gate.shape == (0, 4)


def test_numbers_beyond_the_field(zk):
    """Words from p on stand for what they are modulo p, as in the op layer."""
    import torch
    rng = np.random.default_rng(10)
    k, n = 70, 33
    w = ref.weight(rng, k, n, 64)
    x = rng.integers(0, 1 << 30, (2, k))
    q = _quant(zk, w, 64)
    beyond = torch.from_numpy((x.astype(np.uint64) + np.uint64(0xFFFFFFFF00000001))).cuda()
    assert np.array_equal(_s(zk.decode.project(beyond, q, 10)), ref.project(x, *w, 64, 0, 10))


@pytest.mark.parametrize("m,h,experts,top_k,f,shared,group", [
    (16, 2048, 20, 3, 32, 40, 64), (16, 2048, 20, 3, 33, 500, 32), (15, 2048, 256, 4, 20, 24, 128),
    (12, 2048, 10, 4, 100, 300, 64)])
def test_moe_block_of_many_wide_tokens(zk, m, h, experts, top_k, f, shared, group):
    """Tokens whose digits leave less room for rings and sums."""
    rng = np.random.default_rng(h + experts)
    router, w = _moe_case(rng, h, experts, f, shared, group)
    x, exp_table, silu = rng.integers(-(1 << 17), 1 << 17, (m, h)), _exp_table(), _silu_table()
    out, gate = _moe_block(zk, router, w, group, top_k, exp_table, silu).forward(_u(x))
    want, want_gate = ref.moe(x, router, w, group, exp_table, silu, top_k)
    assert np.array_equal(_s(gate), want_gate) and np.array_equal(_s(out), want)
