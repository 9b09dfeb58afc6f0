"""Weights, caches, expert blocks and decoders that are copied, restored or
changed: each works on its own memory."""
import copy
import io

import numpy as np
import pytest

from tests import decode_ref as ref, decode_shapes as ds_ref
from tests.test_gpu_decode import _cache, _exp_table, _i32, _moe_block, _moe_case, _quant, _s, _silu_table, _u

pytestmark = pytest.mark.gpu



def _saved(handle):
    import torch
    file = io.BytesIO()
    torch.save(handle, file)  # (plain pickle does not read torch's uint64 tensors back)
    file.seek(0)
    return torch.load(file, weights_only=False)


COPIES = {"deepcopy": copy.deepcopy, "saved": _saved}


@pytest.mark.parametrize("how", COPIES)
def test_a_forked_cache_steps_apart(zk, how):
    """Two continuations of one sequence: each sees the common past and its own
    tokens, the other's cache stays as it was."""
    rng = np.random.default_rng(1)
    hk, dk, dv, cap, n = 2, 16, 12, 64, 20
    keys, values, cache = _cache(zk, rng, 1, hk, dk, dv, cap, [n])
    table, q = _exp_table(), rng.integers(-(1 << 18), 1 << 18, (1, hk * dk))
    fork = COPIES[how](cache)
    for a, b in ((fork.k, cache.k), (fork.v, cache.v), (fork.lens, cache.lens)):
        assert a.data_ptr() != b.data_ptr()
    before = [t.clone() for t in (cache.k, cache.v, cache.lens)]
    sides = [(cache, keys, values), (fork, keys.copy(), values.copy())]
    for step in range(3):
        for c, ks, vs in reversed(sides):
            nk, nv = rng.integers(-(1 << 18), 1 << 18, (1, hk * dk)), rng.integers(-(1 << 18), 1 << 18, (1, hk * dv))
            ks[0, :, n + step], vs[0, :, n + step] = nk.reshape(hk, dk), nv.reshape(hk, dv)
            got = zk.decode.attend(_u(q), c, _u(table), k=_u(nk), v=_u(nv))
            c.advance()
            want = np.concatenate([ref.attend(q[0, h * dk:(h + 1) * dk], ks[0, h, :n + step + 1], vs[0, h, :n + step + 1], table, (1, 16))
                                   for h in range(hk)])
            assert np.array_equal(_s(got)[0], want)
            if c is fork and step == 0:
                assert all(bool((a == b).all()) for a, b in zip(before, (cache.k, cache.v, cache.lens)))
    for c, ks, vs in sides:
        assert c.lens.tolist() == [n + 3]
        assert np.array_equal(ref.keys_of(c.k.cpu().numpy()), ks) and np.array_equal(c.v.cpu().numpy(), vs)
    # and a prompt's rows
    tail = rng.integers(-99, 99, (1, 2, hk * dk)), rng.integers(-99, 99, (1, 2, hk * dv))
    fork.append(_u(tail[0]), _u(tail[1]))
    assert np.array_equal(fork.v[0, :, n + 3:n + 5].cpu().numpy(), np.moveaxis(tail[1].reshape(2, hk, dv), 0, 1))
    assert np.array_equal(cache.v.cpu().numpy(), sides[0][2])


@pytest.mark.parametrize("how", COPIES)
def test_a_copied_weight_has_its_own_memory(zk, how):
    rng = np.random.default_rng(2)
    w, x = ref.weight(rng, 96, 40, 32), rng.integers(-(1 << 18), 1 << 18, (3, 96))
    q = _quant(zk, w, 32)
    other = COPIES[how](q)
    import torch
    q.packed.zero_()  # codes and scales of zero
    torch.cuda.synchronize()
    assert not _s(zk.decode.project(_u(x), q, 9)).any()
    del q
    _i32(np.full(1 << 16, -1))  # whoever takes the memory that is free now
    assert np.array_equal(_s(zk.decode.project(_u(x), other, 9)), ref.project(x, *w, 32, 0, 9))
    assert np.array_equal(other.codes()[0].cpu().numpy(), w[0])


@pytest.mark.parametrize("how", COPIES)
def test_a_copied_block_has_its_own_memory(zk, how):
    import torch
    rng = np.random.default_rng(3)
    router, w = _moe_case(rng, 64, 8, 48, 40, 32)
    x, exp, silu = rng.integers(-(1 << 17), 1 << 17, (3, 64)), _exp_table(), _silu_table()
    block = _moe_block(zk, router, w, 32, 3, exp, silu)
    other = COPIES[how](block)
    for t in (block.router, *block.packed, block.exp_table, block.silu_table):
        t.zero_()
    torch.cuda.synchronize()
    del block
    out, gate = other.forward(_u(x))
    want, want_gate = ref.moe(x, router, w, 32, exp, silu, 3)
    assert np.array_equal(_s(out), want) and np.array_equal(_s(gate), want_gate)


def test_tensors_of_handles_are_not_replaced(zk):
    import torch
    rng = np.random.default_rng(4)
    q = _quant(zk, ref.weight(rng, 64, 16, 32), 32)
    router, w = _moe_case(rng, 32, 4, 16, 16, 32)
    block = _moe_block(zk, router, w, 32, 2, _exp_table(12), _silu_table(12))
    cache = zk.decode.KvCache.zeros(1, 1, 4, 4, 32)
    for handle, names in ((q, ("packed",)), (block, ("router", "packed", "exp_table", "silu_table")), (cache, ("k", "v", "lens"))):
        for name in names:
            with pytest.raises(AttributeError):
                setattr(handle, name, getattr(handle, name))
    # memory that has become less is refused, not read past its end
    x = _u(np.ones((1, 64), dtype=np.int64))
    q.packed.resize_(16)
    with pytest.raises(ValueError, match="QuantWeight: packed"):
        zk.decode.project(x, q, 4)
    block.packed[1].resize_(16)
    with pytest.raises(ValueError, match="MoeBlock: packed"):
        block.forward(x[:, :32])
    k = _u(np.ones((1, 4), dtype=np.int64))
    cache.v.resize_(4)
    with pytest.raises(ValueError, match="KvCache: v"):
        zk.decode.attend(k, cache, _u(_exp_table(8)), k=k, v=k)
    with pytest.raises(ValueError, match="sizes"):
        cache.append(k[None], k[None])
    with pytest.raises(ValueError, match="handle"):
        zk.decode._calls.project(x, (1, 2), 4, None, None, None, None, None, torch.zeros(1, dtype=torch.int32, device="cuda"))


def test_a_forked_decoder_steps_apart(zk):
    """A GPT-2 decoder copied in the middle of a text: both go on, each with
    other tokens, as two decoders that had the same past from the start."""
    import torch
    s = zk.gpt2.LayerShape(**ds_ref.GPT2)
    store = zk.compose.Store()
    ops, tokens, _ = zk.gpt2.gpt2_model(store, s, layers=2)
    ds_ref.liven(store, ops)
    weights = zk.decode.quantise_weights(store, ops, ("Projection", "MatMul"))
    text = store.get_idx(tokens).view(torch.int32)
    new = lambda: zk.gpt2.Gpt2Decoder(store, ops, s, weights, batch=1)  # noqa: E731

    def run(dec, ids):
        out = []
        for t in ids:
            dec.tokens.copy_(t.reshape(1).view(torch.uint32))
            out.append(dec.step()[1].view(torch.int64).clone())
        return torch.cat(out)

    past, left, right = text[:10], text[10:20], text.flip(0)[:10]
    want, apart = [], []
    for rest in (left, right):
        dec = new()
        run(dec, past)
        want.append(run(dec, rest))
        apart.append(dec)
    dec = new()
    run(dec, past)
    fork = copy.deepcopy(dec)
    assert all(layer["cache"].lens.data_ptr() == fork.lens.data_ptr() for layer in fork.layers)
    got_right = run(fork, right[:5])
    got_left = run(dec, left)
    assert torch.equal(got_left, want[0])
    assert torch.equal(torch.cat([got_right, run(fork, right[5:])]), want[1])
    for one, other in zip((dec, fork), apart):
        one.check()
        for a, b in zip(one.layers, other.layers):
            assert torch.equal(a["cache"].k, b["cache"].k) and torch.equal(a["cache"].v, b["cache"].v)
        assert one.lens.tolist() == [20]
    assert not torch.equal(dec.layers[0]["cache"].v, fork.layers[0]["cache"].v)
    with pytest.raises(AttributeError):
        dec.lens = dec.lens.clone()
    with pytest.raises(AttributeError):
        dec.tokens = dec.tokens.clone()


# ---- captured steps -----------------------------------------------------------------------------------
def _lively(zk, batch, prompt):
    import torch
    s = zk.gpt2.LayerShape(**ds_ref.GPT2)
    store = zk.compose.Store()
    ops, tokens, _ = zk.gpt2.gpt2_model(store, s, layers=2)
    ds_ref.liven(store, ops)
    weights = zk.decode.quantise_weights(store, ops, ("Projection", "MatMul"))
    zk.compose.forward_ops(store, ops)
    text = store.get_idx(tokens).view(torch.int32)

    def new():
        dec = zk.gpt2.Gpt2Decoder(store, ops, s, weights, batch)
        for b in range(batch):
            dec.load(store, b, prompt + b)
        dec.tokens.copy_(text[[prompt + b for b in range(batch)]].view(torch.uint32))
        return dec
    return s, new


def test_a_captured_step_keeps_what_it_reads(zk):
    """The penalties' history, a bias and a mask that nobody else holds, and a
    decoder that is dropped: a replay reads them as they were, and its logits
    can be read."""
    import gc

    import torch
    s, new = _lively(zk, 2, 9)
    rng = np.random.default_rng(5)
    history, bias = rng.integers(0, s.vocab_real, (2, 30)), rng.integers(-(1 << 33), 1 << 33, (2, s.vocab))
    allowed = rng.integers(-(1 << 31), 1 << 31, (2, s.vocab // 32))
    choice = lambda: dict(history=_i32(history), history_lens=_i32([30, 17]), bias=_u(bias), allowed=_i32(allowed),  # noqa: E731
                          repeat=(52429, 81920), presence=1 << 30, frequency=1 << 29)
    dec, kept, want = new(), choice(), []
    for _ in range(12):
        tokens, logits = dec.step(**kept)
        want.append((tokens.view(torch.int32).clone(), logits.view(torch.int64).clone()))
    graph = new().capture(**choice())
    gc.collect()
    rubbish = [torch.full((n,), 0x5A5A5A5A, dtype=torch.int32, device="cuda") for n in (2, 17, 32, 60, 64, 1024, 2048, 2048) for _ in range(20)]
    for tokens, logits in want:
        graph.replay()
        assert torch.equal(graph.tokens.view(torch.int32), tokens) and torch.equal(graph.logits.view(torch.int64), logits)
    assert graph.decoder.lens.tolist() == [21, 22] and graph.tokens.data_ptr() == graph.decoder.tokens.data_ptr()
    graph.decoder.check()
    assert len(rubbish) == 160


def test_capture_leaves_no_error_of_its_own(zk):
    """A full sequence: recording a step says nothing, replaying it does."""
    s, new = _lively(zk, 1, 5)
    dec = new()
    dec.lens.fill_(s.m)
    graph = dec.capture()
    dec.check()
    graph.replay()
    with pytest.raises(ValueError, match="full"):
        dec.check()


# ---- outputs that are given ----------------------------------------------------------------------------
def test_outputs_apart_from_everything_else(zk):
    """Biases, tables, masks, histories, weights, caches and the error word:
    an output over one of them is refused before anything is enqueued."""
    import torch
    d, rng = zk.decode, np.random.default_rng(6)
    m, k, v = 4, 64, 96
    u64 = lambda t: t.reshape(-1)[:t.numel() // 2 * 2].view(torch.uint64)  # noqa: E731  any tensor's memory
    err = torch.zeros(2 * m * v, dtype=torch.int32, device="cuda")
    cells = lambda t, n, off=0: u64(t)[off:off + m * n].reshape(m, n)  # noqa: E731
    q, x = _quant(zk, ref.weight(rng, k, k, 32), 32), _u(rng.integers(-99, 99, (m, k)))
    out, table = torch.zeros((m, k), dtype=torch.uint64, device="cuda"), torch.zeros(2 * m * k, dtype=torch.uint64, device="cuda")
    assert q.packed.numel() >= 2 * m * k

    def refused(call):
        with pytest.raises(ValueError, match="shares memory"):
            call()
    for row in range(m):
        refused(lambda: d.project(x, q, 16, bias=out[row], out=out))
    refused(lambda: d.project(x, q, 16, table=table, out=cells(table, k, 5)))
    refused(lambda: d.project(x, q, 16, table=table[m * k - 1:], out=cells(table, k)))
    refused(lambda: d.project(x, q, 16, out=cells(q.packed, k)))
    refused(lambda: d.project(x, q, 16, out=cells(err, k), err=err[8:9]))
    d.project(x, q, 16, bias=table[:k], table=table[k:], out=out, err=err[:1])

    cache = d.KvCache.zeros(m, 1, k, k, 32)
    big = d.KvCache(cache.k, cache.v, err[:m])
    refused(lambda: d.attend(x, cache, table, out=cells(table, k, 7)))
    refused(lambda: d.attend(x, cache, table, out=cells(cache.k, k)))
    refused(lambda: d.attend(x, cache, table, out=cells(cache.v, k, 3)))
    refused(lambda: d.attend(x, big, table, out=cells(err, k), err=err[-1:]))
    refused(lambda: d.attend(x, cache, table, out=cells(err, k), err=err[3:4]))

    router, w = _moe_case(rng, k, 4, 32, 32, 32)
    block = _moe_block(zk, router, w, 32, 2, _exp_table(), _silu_table())
    for t in (block.packed[0], block.packed[2], block.exp_table, block.silu_table):
        refused(lambda: block.forward(x, out=cells(t, k, 1)))
    refused(lambda: block.forward(x, out=cells(err, k), err=err[1:2]))

    logits = _u(rng.integers(-99, 99, (m, v)))
    words = torch.zeros(2 * m * v + 16, dtype=torch.int32, device="cuda")
    refused(lambda: d.choose_token(logits, allowed=words[:3], out=cells(words, v)))
    refused(lambda: d.choose_token(logits, allowed=words[:3 * m].reshape(m, 3), out=cells(words, v, 1)))
    refused(lambda: d.choose_token(logits, words[-5 * m:].reshape(m, 5), out=cells(words, v)))
    refused(lambda: d.choose_token(logits, _i32(np.zeros((m, 2))), words[40:40 + m], out=cells(words, v)))
    refused(lambda: d.choose_token(logits, out=cells(words, v), err=words[9:10]))
    assert not err[1:].any()


def test_caches_apart_from_their_rows(zk):
    """A cache is written while its rows are read: they share no memory, nor do
    its own tensors."""
    import torch
    d = zk.decode
    mem = torch.zeros(32 * 8 * 4, dtype=torch.int32, device="cuda")
    k, v, lens = mem[:256].reshape(1, 1, 1, 2, 32, 4), mem[256:512].reshape(1, 1, 32, 8), mem[512:513]
    cache, table = d.KvCache(k, v, lens), _u(_exp_table(8))
    u64 = lambda a: mem[a:a + 16].view(torch.uint64).reshape(1, 8)  # noqa: E731
    free = u64(600)
    for args in ((u64(0), free, free), (free, u64(100), free), (free, free, u64(248)), (free, u64(500), free)):
        with pytest.raises(ValueError, match="shares memory"):
            d.attend(args[0], cache, table, k=args[1], v=args[2])
    for args in ((u64(100), free), (free, u64(240)), (free, u64(512))):
        with pytest.raises(ValueError, match="share memory"):
            cache.append(args[0][None], args[1][None])
    for bad in ((k, mem[252:508].reshape(1, 1, 32, 8), lens), (k, v, mem[3:4]), (k, v, mem[511:512])):
        with pytest.raises(ValueError, match="share memory"):
            d.KvCache(*bad)
    assert not mem.any()
    d.attend(free, cache, table, k=free, v=free)  # side by side they may lie
    d.attend(u64(0), cache, table)  # and what is only read may be read twice


def test_a_length_beyond_the_capacity_is_said(zk):
    """Tokens that the cache does not hold were counted: the answer over those
    it holds is not the row's."""
    import torch
    rng = np.random.default_rng(7)
    _, _, cache = _cache(zk, rng, 3, 1, 8, 8, 32, [32, 5, 20])
    q, table, err = _u(rng.integers(-99, 99, (3, 8))), _u(_exp_table()), torch.zeros(1, dtype=torch.int32, device="cuda")
    zk.decode.attend(q, cache, table, err=err)
    assert int(err.item()) == 0
    cache.lens[2] = 33
    zk.decode.attend(q, cache, table, err=err)
    assert int(err.item()) == 16
    with pytest.raises(ValueError, match="full"):
        zk.decode.attend(q, cache, table)


def test_a_recorded_forward_runs_the_quantised_weights(zk):
    """Recorded before the weights were quantised, replayed after."""
    import torch
    s = zk.gpt2.LayerShape(**ds_ref.GPT2)
    store = zk.compose.Store()
    ops, _, out = zk.gpt2.gpt2_layer(store, s)
    ds_ref.liven(store, ops)
    recorded = zk.compose.GraphForward(store, ops)
    plain = store.get(out).view(torch.int64).clone()
    zk.decode.quantise_weights(store, ops, ("Projection",), 32)
    recorded.run()
    got = store.get(out).view(torch.int64).clone()
    zk.compose.forward_ops(store, ops)
    assert torch.equal(got, store.get(out).view(torch.int64)) and not torch.equal(got, plain)


def test_append_refuses_factors_beyond_64_bits(zk):
    """As attend does; they were cut to 64 bits."""
    cache = zk.decode.KvCache.zeros(1, 1, 4, 4, 32)
    rows = _u(np.ones((1, 1, 4), dtype=np.int64))
    for factor in ((1 << 64) + 1, 1 << 63, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="64 bits"):
            cache.append(rows, rows, k_scale=(factor, 0))
    assert not cache.k.any()
    with pytest.raises(OverflowError):
        zk.decode.attend(rows[0], cache, _u(_exp_table(8)), k=rows[0], v=rows[0], k_scale=(1 << 64, 0))


def test_a_copy_of_weights_is_complete(zk):
    """Calls start to read weights while earlier kernels still run, so a copy's
    are there when copying returns, whatever the stream had to do."""
    import torch
    rng = np.random.default_rng(9)
    router, w = _moe_case(rng, 32, 4, 16, 16, 32)
    for handle in (_quant(zk, w[3], 32), _moe_block(zk, router, w, 32, 2, _exp_table(12), _silu_table(12))):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            torch.cuda._sleep(50_000_000)  # 25 ms
            copy.deepcopy(handle)
            assert side.query()
        torch.cuda.synchronize()


def test_an_output_without_memory(zk):
    """Raised as torch raises it, and nothing is left behind."""
    import torch
    n = 1 << 22
    q = zk.decode.QuantWeight(torch.ones((1, n), dtype=torch.int8), torch.ones((1, n), dtype=torch.int32), group=32)
    x = torch.ones((65535, 1), dtype=torch.int64, device="cuda").view(torch.uint64)
    with pytest.raises(torch.OutOfMemoryError):
        zk.decode.project(x, q, 0)
    assert _s(zk.decode.project(x[:2], q, 0)).sum() == 2 * n
