"""The forward of single tokens on the device: what a step of generation needs
of the op layer, for a few rows instead of a whole, fixed-length sequence.

``compose.forward_ops`` computes the witness of a whole sequence, ending in
the Argmax arm (models/gpt2/src/lib.rs:321-436).  Answering token by token
needs one row at a time; these operators compute it, and since every value is
a whole number the row is the graph's own row, bit for bit: the answer that is
generated is the answer the proof is about.

- ``QuantWeight`` and ``project``: Projection / MatMul of a few rows by a
  weight held in 4 bits with group scales.  Its numbers codes x scales are the
  model's weights; ``QuantWeight.dense()`` is the tensor the Store gets.
- ``KvCache`` and ``attend``: one new token per sequence over the keys and
  values of the earlier ones, held exactly in 32 bits.
- ``MoeBlock``: build_moe (models/deepseek-v2-lite/src/lib.rs:252-470) for a
  few tokens in two kernels.
- ``choose_token``: penalties for repeated tokens, biases and masks on the
  logits, and the Argmax arm.

Every call takes rows of field elements (torch.uint64, unit stride within a
row) on the current device and enqueues on the current stream.  ``err`` is the
device error word of ``forward_ops``: given, the caller reads it when it
likes (``check_err``); not given, the call reads its own, which synchronises,
and raises ValueError.  Besides the op layer's bits, 8 is a value outside the
32-bit range the kernels take (computed on as zero) and 16 a full cache.
"""
from importlib import import_module
from typing import Optional, Tuple

import numpy as np
import torch

from ._lib import check, lib
from .compose import _INDEX_WRITERS, _check_err, _err_word
from .device import P, device

GROUPS = (32, 64, 128)
KV_BLOCK = 32
MASKED = -(1 << 41)  # the graph's vocabulary mask (models/gpt2/src/lib.rs:410-418)


def check_err(err: torch.Tensor, what: str = "decode"):
    """Read an error word (synchronises) and raise ValueError if a bit is set."""
    _check_err(err, what)


class _Calls:
    """The extension zkie_b200._calls, loaded with the first per-token call:
    one built for another torch fails here and leaves the rest of the package
    alone."""

    def __getattr__(self, name: str):
        try:
            module = import_module(__package__ + "._calls")
        except ImportError as e:
            raise ImportError("zkie_b200/_calls.so is missing or does not load: build it with `python -m zkie_b200.build` "
                              "(there is no fallback)") from e
        for call in ("project", "attend", "moe", "choose"):
            setattr(self, call, getattr(module, call))
        return getattr(module, name)


_calls = _Calls()
_U64, _I32 = torch.uint64, torch.int32


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _device_of(t, name: str) -> int:
    """The index of the device that ``t`` and the call are on."""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() == torch.cuda.current_device():
        return t.get_device()
    what = f"{t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
    raise ValueError(f"{name}: a tensor on the current CUDA device is wanted, not {what}")


def _flat(t, name: str, dtype, dev: int, shape=None) -> torch.Tensor:
    if isinstance(t, torch.Tensor) and t.dtype == dtype and t.get_device() == dev and t.is_contiguous() and \
            (shape is None or tuple(t.shape) == tuple(shape)):
        return t
    what = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
    raise ValueError(f"{name}: a contiguous {dtype} tensor{'' if shape is None else f' of shape {tuple(shape)}'} on the "
                     f"call's device is wanted, not {what}")


def _signed(t: torch.Tensor) -> torch.Tensor:
    """Field elements (or whole numbers) as int64: fixed_point.rs to_i64."""
    if t.dtype == torch.uint64:
        t = t.view(torch.int64)
        return torch.where(t < 0, t + ((1 << 64) - P), t)
    return t.to(torch.int64)


def _field(t: torch.Tensor) -> torch.Tensor:
    """int64 as field elements: fixed_point.rs from_i64."""
    return torch.where(t < 0, t - ((1 << 64) - P), t).view(torch.uint64)


# ---- 4-bit weights ------------------------------------------------------------------------------
def _scale_rows(k: int, group: int, segment: int) -> int:
    return k // segment * -(-segment // group) if segment else -(-k // group)


def _group_of(k: int, group: int, segment: int, dev) -> torch.Tensor:
    """The row of scales that each of the k rows of codes has."""
    at = torch.arange(k, device=dev)
    return at // segment * -(-segment // group) + at % segment // group if segment else at // group


def quantise(w: torch.Tensor, group: int = 64, segment: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The nearest 4-bit form of a weight (k x n or experts x k x n, field
    elements or whole numbers): codes (int8, in [-8, 7]) and scales (int32),
    the smallest whole scale that covers each group of ``group`` rows of a
    column.  Raises where a weight needs a scale above 65535."""
    if group not in GROUPS or segment < 0 or w.dim() not in (2, 3) or (segment and w.shape[-2] % segment):
        raise ValueError("quantise: group 32, 64 or 128, and segments that divide the rows, are wanted")
    w = _signed(w)
    k, n = w.shape[-2:]
    row = _group_of(k, group, segment, w.device)
    at = row[:, None].expand(k, n).expand(w.shape)
    lo = torch.zeros(w.shape[:-2] + (_scale_rows(k, group, segment), n), dtype=torch.int64, device=w.device)
    hi = lo.clone().scatter_reduce_(-2, at, w, "amax")
    lo = lo.scatter_reduce_(-2, at, w, "amin")
    scales = torch.maximum(torch.maximum((hi + 6) // 7, (7 - lo) // 8), torch.ones_like(lo))
    if int(scales.max()) > 65535:
        raise ValueError("quantise: a weight needs a scale above 65535")
    s = scales[..., row, :]
    codes = torch.div(2 * w + s, 2 * s, rounding_mode="floor").clamp(-8, 7)
    return codes.to(torch.int8), scales.to(torch.int32)


def quantise_weights(store, ops, kinds=("Projection", "GatherMatMul"), group: int = 64) -> dict:
    """Quantise the weights that the ops of these kinds read (Projection w,
    GatherMatMul w, MatMul b where no op writes it), in the Store's own tensors: they hold the
    dense numbers that the codes stand for (all of them, or none where one
    raises), so the model that is run and proven is the quantised one, by a
    forward or a prover that was recorded before, too.  Returns {tensor id:
    (codes, scales, group)}, what QuantWeight takes."""
    written = {t for op in ops if op.kind not in _INDEX_WRITERS for t in op.writes()}
    done = {}
    for op in ops:
        t = op.b if op.kind == "MatMul" else getattr(op, "w", None)
        if op.kind not in kinds or t is None or t in done or t in written:
            continue
        shape = (op.n_experts, op.k, op.n) if op.kind == "GatherMatMul" else (op.k, op.n)
        done[t] = (*quantise(store.get(t).reshape(shape), group), group)
    spans = sorted((store.get(t).data_ptr(), store.get(t).data_ptr() + 8 * store.get(t).numel()) for t in done)
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError("quantise_weights: weights that share memory")
    for t, (codes, scales, _) in done.items():  # all of them have a 4-bit form
        row = _group_of(codes.shape[-2], group, 0, codes.device)
        dense = _field(codes.to(torch.int64) * scales.to(torch.int64)[..., row, :]).reshape(-1)
        store.get(t).view(torch.int64).copy_(dense.view(torch.int64))
    return done


def _kept(name: str) -> property:
    """A handle's tensor: not replaced -- calls take it from ``call``, which a
    copy or a pickle of the handle has its own of.  A cache's may be written
    in place; a weight's are only read, unless the host waits before the next
    call (calls start to read weights while earlier kernels still run)."""
    return property(lambda self: getattr(self, name))


class _Weights:
    """Handles of weights: those of a copy are complete before a call too."""

    def __setstate__(self, state: dict):
        self.__dict__.update(state)
        torch.cuda.current_stream(self.device).synchronize()


class QuantWeight(_Weights):
    """A weight w[k][n] = codes[k][n] scales[row of k][n] in 4 bits, laid out
    once for the kernels (``packed``).

    codes: int8, k x n or experts x k x n, in [-8, 7]; scales: whole numbers in
    [0, 65535], one for each ``group`` (32, 64 or 128) rows of a column, as
    many rows of them as groups begin.  ``segment`` splits the rows into runs
    (the heads of an output projection) that the product rounds one by one and
    adds, as the graph's Projection per head and its Adds do; groups begin
    anew in each run.  At most 8192 rows, each run counted as a multiple of
    64."""

    def __init__(self, codes, scales, group: int = 64, segment: int = 0):
        codes, scales = torch.as_tensor(codes).to(device()), torch.as_tensor(scales).to(device())
        if codes.dtype != torch.int8 or codes.dim() not in (2, 3) or scales.is_floating_point():
            raise ValueError("QuantWeight: codes int8 (k x n or experts x k x n) and whole scales are wanted")
        if group not in GROUPS or segment < 0:
            raise ValueError("QuantWeight: group 32, 64 or 128 is wanted")
        self.experts = codes.shape[0] if codes.dim() == 3 else 1
        self.k, self.n = int(codes.shape[-2]), int(codes.shape[-1])
        self.group, self.segment = group, segment
        words = lib.zkie2_q4_words(self.experts, self.k, self.n, group, segment)
        if words == 0:
            raise ValueError(f"QuantWeight: {self.experts} x {self.k} x {self.n} with group {group} and segment "
                             f"{segment} is not taken (at most 8192 padded rows, segments that divide them)")
        want = tuple(codes.shape[:-2]) + (_scale_rows(self.k, group, segment), self.n)
        if tuple(scales.shape) != want:
            raise ValueError(f"QuantWeight: scales of shape {tuple(scales.shape)}, {want} is wanted")
        if int(codes.min()) < -8 or int(codes.max()) > 7 or int(scales.min()) < 0 or int(scales.max()) > 65535:
            raise ValueError("QuantWeight: a code outside [-8, 7] or a scale outside [0, 65535]")
        codes, scales = codes.contiguous(), scales.to(torch.int32).contiguous()
        dev = codes.device
        self._packed = torch.empty(words, dtype=torch.int32, device=dev)
        self.call = (self._packed, self.k, self.n, group, segment, self.experts)
        err = _err_word()
        check(lib.zkie2_q4_pack(codes.data_ptr(), scales.data_ptr(), self.experts, self.k, self.n, group, segment,
                                self.packed.data_ptr(), err.data_ptr(), _stream()), "zkie2_q4_pack")
        _check_err(err, "QuantWeight")

    packed = _kept("_packed")
    device = property(lambda self: self._packed.get_device())

    def _blocks(self) -> torch.Tensor:
        return self.packed.reshape(self.experts, -(-self.n // 16), -1, 144 if self.group == 32 else 136)

    def codes(self) -> torch.Tensor:
        """The codes back (experts x k x n)."""
        tiles, seg = -(-self.n // 16), self.segment or self.k
        b = self._blocks()[..., :128].contiguous().view(torch.uint8).reshape(self.experts, tiles, -1, 8, 4, 2, 2, 4)
        both = torch.stack([b & 15, b >> 4], dim=-1).to(torch.int8)  # expert tile block g t q/2 q%2 j half
        both = torch.where(both > 7, both - 16, both)
        full = both.permute(0, 2, 8, 4, 5, 7, 1, 6, 3).reshape(self.experts, self.k // seg, -(-seg // 64) * 64, tiles * 16)
        return full[:, :, :seg, :self.n].reshape(self.experts, self.k, self.n)

    def scales(self) -> torch.Tensor:
        """The scales back (experts x rows x n)."""
        tiles, seg = -(-self.n // 16), self.segment or self.k
        w = self._blocks()[..., 128:].reshape(self.experts, tiles, -1, 8)
        both = torch.stack([w & 0xFFFF, (w >> 16) & 0xFFFF], dim=-1)  # expert tile group g half
        full = both.permute(0, 2, 1, 4, 3).reshape(self.experts, self.k // seg, -1, tiles * 16)
        full = full[:, :, ::2 if self.group == 128 else 1]  # two blocks repeat a group of 128
        return full[:, :, :-(-seg // self.group), :self.n].reshape(self.experts, -1, self.n)

    def dense(self) -> torch.Tensor:
        """The weights as field elements, flat and row-major (experts one after
        another): the tensor of a Store."""
        row = _group_of(self.k, self.group, self.segment, self.packed.device)
        return _field(self.codes().to(torch.int64) * self.scales().to(torch.int64)[:, row]).reshape(-1)


def project(x: torch.Tensor, weight: QuantWeight, shift: int, *, bias: Optional[torch.Tensor] = None,
            table: Optional[torch.Tensor] = None, offset: Optional[int] = None,
            residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
            err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The Projection arm's out for the rows of x (m x k -> m x n):
    round_div(x w, 2^shift), one rounding per segment of the weight, + bias (n);
    then ``table[clamp(y + offset, 0, len - 1)]`` (GeluIndex and Lookup; offset
    defaults to the table's middle) and ``+ residual`` (m x n; Add) where
    given.  shift 0 without a bias is the MatMul arm.  |x| <= 0x7F7F7F7F."""
    word = _err_word() if err is None else err
    out = _calls.project(x, weight.call, shift, bias, table, offset, residual, out, word)
    if err is None:
        _check_err(word, "project")
    return out


# ---- attention over a cache -----------------------------------------------------------------------
class KvCache:
    """The keys and values of ``batch`` sequences, exact in 32 bits.

    k: int32 (batch, heads, capacity / 32, dk / 4, 32, 4) -- blocks of 32
    tokens, four dimensions of a token side by side; v: int32 (batch, heads,
    capacity, dv); lens: int32 (batch), tokens held (negative: an inactive
    sequence).  The layers of a model may share one ``lens``.  dk and dv are
    multiples of 4 up to 256, the capacity a multiple of 32 up to 131072."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor):
        dev = _device_of(k, "k")
        _flat(k, "k", _I32, dev)
        _flat(v, "v", _I32, dev)
        _flat(lens, "lens", _I32, dev)
        if k.dim() != 6 or v.dim() != 4 or k.shape[4:] != (KV_BLOCK, 4):
            raise ValueError("KvCache: k (batch, heads, capacity / 32, dk / 4, 32, 4) and v (batch, heads, capacity, "
                             "dv) are wanted")
        self.batch, self.heads, self.capacity, self.dv = v.shape
        self.dk = k.shape[3] * 4
        if tuple(k.shape[:3]) != (self.batch, self.heads, self.capacity // KV_BLOCK) or \
                tuple(lens.shape) != (self.batch,):
            raise ValueError("KvCache: k, v and lens do not match")
        if self.capacity % KV_BLOCK or not 0 < self.capacity <= 1 << 17 or not 0 < self.dk <= 256 or self.dv % 4 or \
                not 0 < self.dv <= 256 or not 0 < self.batch <= 65535 or not 0 < self.heads <= 65535:
            raise ValueError("KvCache: head sizes in multiples of 4 up to 256 and a capacity in multiples of 32 up to "
                             "131072 are wanted")
        if (k.data_ptr() | v.data_ptr()) & 15:
            raise ValueError("KvCache: 16-byte aligned buffers are wanted")
        spans = sorted((t.data_ptr(), t.data_ptr() + 4 * t.numel()) for t in (k, v, lens))
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("KvCache: k, v and lens share memory")
        self._k, self._v, self._lens = k, v, lens
        self._numels = (k.numel(), v.numel(), lens.numel())
        self.call = (k, v, lens, self.batch, self.heads, self.dk, self.dv, self.capacity)

    k, v, lens = _kept("_k"), _kept("_v"), _kept("_lens")
    device = property(lambda self: self._k.get_device())

    @classmethod
    def zeros(cls, batch: int, heads: int, dk: int, dv: int, capacity: int,
              lens: Optional[torch.Tensor] = None) -> "KvCache":
        """An empty cache; the capacity is rounded up to whole blocks."""
        blocks, dev = -(-capacity // KV_BLOCK), device()
        if dk % 4:
            raise ValueError("KvCache: head sizes in multiples of 4 are wanted")
        return cls(torch.zeros((batch, heads, blocks, dk // 4, KV_BLOCK, 4), dtype=torch.int32, device=dev),
                   torch.zeros((batch, heads, blocks * KV_BLOCK, dv), dtype=torch.int32, device=dev),
                   torch.zeros(batch, dtype=torch.int32, device=dev) if lens is None else lens)

    def append(self, k: torch.Tensor, v: torch.Tensor, k_scale: Tuple[int, int] = (1, 0),
               err: Optional[torch.Tensor] = None):
        """Store rows of a prompt from position lens on (lens stays: see
        ``advance``): k (batch, tokens, heads dk) and v (batch, tokens, heads
        dv) field elements, the keys through Scale by k_scale = (factor,
        shift).  |key| <= 2^27, values in 32 bits."""
        dev = _device_of(k, "k")
        for name, t, cols in (("k", k, self.heads * self.dk), ("v", v, self.heads * self.dv)):
            if not isinstance(t, torch.Tensor) or t.dtype != _U64 or t.get_device() != dev or t.dim() != 3 or \
                    tuple(t.shape) != (self.batch, k.shape[1], cols):
                raise ValueError(f"{name}: uint64 ({self.batch}, tokens, {cols}), as many tokens of k and v, is wanted")
        if self.device != dev or k.shape[1] > 1 << 17 or not 0 <= k_scale[1] <= 62:
            raise ValueError("append: the cache's device, at most 131072 tokens and a shift 0 .. 62 are wanted")
        if not -(1 << 63) <= k_scale[0] < 1 << 63:
            raise ValueError("append: a factor of 64 bits is wanted")
        k, v, word = k.contiguous(), v.contiguous(), _err_word() if err is None else _flat(err, "err", _I32, dev)
        mine, sizes = self.call[:3], self.call[3:]
        if any(t.numel() != n for t, n in zip(mine, self._numels)):
            raise ValueError("append: the cache's tensors have other sizes than they had")
        if any(a.data_ptr() < b.data_ptr() + 8 * b.numel() and b.data_ptr() < a.data_ptr() + 4 * a.numel()
               for a in mine for b in (k, v)):
            raise ValueError("append: the rows share memory with the cache")
        check(lib.zkie2_kv_append(k.data_ptr(), k.shape[2], v.data_ptr(), v.shape[2], k.shape[1], *k_scale,
                                  *[t.data_ptr() for t in mine], *sizes, word.data_ptr(), _stream()), "zkie2_kv_append")
        if err is None:
            _check_err(word, "append")

    def room(self, limit: int, err: torch.Tensor):
        """Set the error word's bit for a full cache where a sequence has
        reached ``limit`` tokens: for a limit within the last block."""
        if limit < self.capacity:
            err.bitwise_or_((self.lens >= limit).any().to(torch.int32) * 16)

    def advance(self, tokens: int = 1):
        """Count ``tokens`` more in every active sequence."""
        self.lens.add_((self.lens >= 0).to(torch.int32), alpha=tokens)


def attend(q: torch.Tensor, cache: KvCache, table: torch.Tensor, *, k: Optional[torch.Tensor] = None,
           v: Optional[torch.Tensor] = None, q_scale: Tuple[int, int] = (1, 0), k_scale: Tuple[int, int] = (1, 0),
           score_scale: Tuple[int, int] = (1, 16), offset: Optional[int] = None, out_shift: int = 16,
           out: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One query row per sequence (batch x heads dk, as many query heads as a
    multiple of the cache's) over its cache -> batch x (query heads dv): the
    row of Scale (q_scale), MatMul, Scale (score_scale), StableSoftmaxIndex
    (offset, the table's length if not given), Softmax over ``table``, MatMul
    and Scale (1, out_shift) in a causal graph.  With k (batch x heads dk) and
    v (batch x heads dv) the new token is stored at position lens first, its
    key through Scale (k_scale), and attended to; ``cache.advance`` then counts
    it.  Rows may be columns of a wider matrix.  A graph's masked columns count
    table[0] each in its softmax's sum: the rows agree where that is zero, as
    in the models' tables from 2^20 entries on, and where no masked score is
    2^30 - len(table) above the row's largest (the graph's mask takes off 2^30).
    A sequence without tokens answers zeros.  Scaled
    queries and keys |q|, |k| <= 2^27; table values in [0, 2^31)."""
    word = _err_word() if err is None else err
    out = _calls.attend(q, cache.call, table, k, v, q_scale, k_scale, score_scale, offset, out_shift, out, word)
    if err is None:
        _check_err(word, "attend")
    return out


def _numbers(t):
    """A store's tensor (of the device's or a host store) to compare words of."""
    return t.view(torch.int64) if isinstance(t, torch.Tensor) else t


def same_rows(t, n: int) -> bool:
    """Whether a matrix of n columns is one row over and over."""
    rows = _numbers(t).reshape(-1, n)
    return bool((rows == rows[:1]).all())


def all_zero(t) -> bool:
    return not bool((_numbers(t) != 0).any())


def masks(t, mask) -> bool:
    """Whether a store's tensor holds the words of ``mask`` (numpy)."""
    t = t.cpu().numpy() if isinstance(t, torch.Tensor) else t
    return np.array_equal(t, mask)


def masked_counts_nothing(table, what: str):
    """Refuse a causal graph's exp table that does not begin with zero: the
    graph counts the first entry for every masked column of a softmax row, and
    attention over a cache, which has no such columns, would answer other rows
    (exp at scale 2^16 rounds to zero from 2^20 entries on)."""
    first = int(_signed(table[:1])[0]) if isinstance(table, torch.Tensor) else int(table[0]) % P
    if first:
        raise ValueError(f"{what}: an exp table that begins with zero is wanted, this one with {first}: the graph's masked "
                         "columns would count")


# ---- a mixture-of-experts layer -----------------------------------------------------------------------
class MoeBlock(_Weights):
    """build_moe's layer for a few tokens: router (h x experts, field elements
    of at most 32639 in size), the routed experts' gate, up (experts x h x f)
    and down (experts x f x h) and the shared experts' gate, up (h x shared f)
    and down weights, all of one group without segments, the exp and silu
    tables (field elements; silu's middle is zero) and how many experts a token
    takes.  ``shift`` is the shared experts' Projections', as in the graph,
    whose other products are all divided by 2^16.  The block keeps copies of
    its own of the weights."""

    def __init__(self, router: torch.Tensor, gate: QuantWeight, up: QuantWeight, down: QuantWeight,
                 shared_gate: QuantWeight, shared_up: QuantWeight, shared_down: QuantWeight, exp_table: torch.Tensor,
                 silu_table: torch.Tensor, top_k: int, shift: int = 16):
        self.h, self.f, self.shared_f = gate.k, gate.n, shared_gate.n
        self.experts, self.group, self.top_k, self.shift = gate.experts, gate.group, top_k, shift
        h, f, s, e = self.h, self.f, self.shared_f, self.experts
        weights = (gate, up, down, shared_gate, shared_up, shared_down)
        want = ((e, h, f), (e, h, f), (e, f, h), (1, h, s), (1, h, s), (1, s, h))
        for w, shape in zip(weights, want):
            if (w.experts, w.k, w.n) != shape or w.group != self.group or w.segment:
                raise ValueError(f"MoeBlock: weight {w.experts} x {w.k} x {w.n}, group {w.group}, segment {w.segment}: "
                                 f"{shape} with group {self.group} and no segments is wanted")
        dev = _device_of(router, "router")
        if any(w.device != dev for w in weights):
            raise ValueError("MoeBlock: weights on the current device are wanted")
        router = _flat(router, "router", _U64, dev, (h, e))
        self._exp, self._silu = _flat(exp_table, "exp_table", _U64, dev), _flat(silu_table, "silu_table", _U64, dev)
        if exp_table.numel() == 0 or silu_table.numel() == 0:
            raise ValueError("MoeBlock: an empty table")
        if not 1 <= top_k <= min(e, 16) or e > 256 or not 0 <= shift <= 62:
            raise ValueError("MoeBlock: at most 256 experts, 1 .. 16 of them to a token, and a shift 0 .. 62 are wanted")
        self._router = torch.empty(lib.zkie2_moe_router_words(h, e), dtype=torch.int32,
                                   device=router.device)
        err = _err_word()
        check(lib.zkie2_moe_router_pack(router.data_ptr(), h, e, self._router.data_ptr(), err.data_ptr(), _stream()), "zkie2_moe_router_pack")
        _check_err(err, "MoeBlock: router")
        self._packed = (self._pair(gate, up), self._pair(down), self._pair(shared_gate, shared_up), self._pair(shared_down))
        torch.cuda.current_stream().synchronize()  # weights are complete before a call: it reads them at once
        self.call = (h, e, top_k, f, s, self.group, shift, self._router, *self._packed, self._exp, self._silu)

    router, packed, exp_table, silu_table = _kept("_router"), _kept("_packed"), _kept("_exp"), _kept("_silu")
    device = property(lambda self: self._router.get_device())

    @staticmethod
    def _pair(a: QuantWeight, b: Optional[QuantWeight] = None) -> torch.Tensor:
        """Gate and up, or the tiles of down two by two, block by block side by
        side: one copy brings both."""
        tiles = -(-a.n // 16)
        words = a.packed.numel() // tiles * (2 * tiles if b is not None else tiles + tiles % 2)
        out = torch.empty(words, dtype=torch.int32, device=a.packed.device)
        check(lib.zkie2_q4_pair(a.packed.data_ptr(), b.packed.data_ptr() if b is not None else None, a.experts, a.k, a.n, a.group, out.data_ptr(),
                                _stream()), "zkie2_q4_pair")
        return out

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(out, gate) of the rows of x (m x h, m <= 65535; two launches to 16
        rows): the layer's output (+ residual where given) and TopKSelect's
        gate (m x experts).  |x| and |silu(gate) up| <= 0x7F7F7F7F."""
        word = _err_word() if err is None else err
        both = _calls.moe(x, self.call, residual, out, word)
        if err is None:
            _check_err(word, "MoeBlock")
        return both


# ---- the next token -----------------------------------------------------------------------------------
def choose_token(logits: torch.Tensor, history: Optional[torch.Tensor] = None,
                 history_lens: Optional[torch.Tensor] = None, *, repeat: Tuple[int, int] = (1 << 16, 1 << 16),
                 presence: int = 0, frequency: int = 0, bias: Optional[torch.Tensor] = None,
                 allowed: Optional[torch.Tensor] = None, mask_value: int = MASKED,
                 out: Optional[torch.Tensor] = None,
                 err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(token, adjusted logits) of each row of logits (batch x vocab field
    elements): the Argmax arm (the lowest index among equals) after, in
    wrapping i64,

    - for a token that occurs c > 0 times in its row of ``history`` (batch x
      tokens, int32; the first ``history_lens`` of a row where given):
      round_div(y repeat[0], 2^16) where y > 0, else round_div(y repeat[1],
      2^16), then - presence - c frequency;
    - ``+ bias`` (vocab, or batch x vocab, field elements);
    - ``+ mask_value`` where bit v % 32 of word v / 32 of ``allowed`` (int32
      words, ceil(vocab / 32), or batch x that) is clear.  With the graph's
      mask value a row that allows nothing still has a maximum."""
    word = _err_word() if err is None else err
    both = _calls.choose(logits, history, history_lens, repeat, presence, frequency, bias, allowed, mask_value, out, word)
    if err is None:
        _check_err(word, "choose_token")
    return both
