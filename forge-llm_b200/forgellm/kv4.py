"""Generation over a 4-bit KV cache: quantized writes and values, attention,
eviction by accumulated attention weight, beam-search selection and the
reordering of caches after it (libforgecu's fcu_kv4_*, fcu_beam_step and
fcu_cache_reorder; the layouts and the arithmetic are in include/forgecu.h).

The functions take the arrays of one cache layer: codes `k`, `v` uint8
[blocks, nKV, blockSize, rowBytes], grids `kg`, `vg` bf16 [blocks, nKV,
blockSize, 2] (step, base) and, where they are kept, `weight` fp32 and `pos`
int32 [blocks, nKV, blockSize].  `table` (int32 [B, maxBlocks]) maps a
sequence's blocks to the arrays'; without one, sequence b owns the b-th equal
share of them.  `QuantKVCache` holds such arrays for every layer.  The forge-llm
reference has no counterpart: its caches are fp32 and it samples one sequence.

All tensors are on the current CUDA device and every call runs on its current
stream.  A call that finds them anywhere else, or of another type, shape or
stride than it takes, raises ValueError before anything is launched, and one
that the library refuses (head counts, overlapping tensors, sizes past its
limits) ForgeCUError.  Host threads may call these functions at the same time,
each on streams of its own; a Transformer's steps are one thread's at a time.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
import threading

import numpy as np
import torch

from ._lib import CacheArray, Context, Kv4, check, lib
from .autograd import device
from .infer import KVCache, _dev_f32

_U8, _BF, _F32, _I32, _BOOL = torch.uint8, torch.bfloat16, torch.float32, torch.int32, torch.bool
_ROW_BYTES: dict = {}

# A decode step makes these calls once per layer, and the kernels take a few
# microseconds, so the common path of every function is one test per tensor (what
# fails it is looked at again for the message), structures are packed bytes (a
# ctypes structure takes three times as long to fill and pass), and results of
# one shape are made like one another (torch.empty_like takes half of what
# new_empty takes).


def _need(ok, what: str) -> None:
    if not ok:
        raise ValueError(what)


class _Contexts(threading.local):
    """This thread's contexts by device.  (The package's own is one per device: a
    thread that binds it to its stream would take along a call that another has
    begun, and the kernels of one call would run on two streams.)  A thread that
    ends leaves them to the next one that needs some, so there are as many as
    threads have been in these calls at once."""

    __slots__ = ("free",)               # (one for all threads, as slots of a threading.local are)

    def __init__(self):
        if not hasattr(self, "free"):
            self.free = {}              # contexts of no thread, by device
        self.of = _Held(self.free)


class _Held(dict):
    def __init__(self, free):
        super().__init__()
        self.free = free

    def __del__(self):
        for dev, c in self.items():
            self.free.setdefault(dev, []).append(c)


_CONTEXTS = _Contexts()


def _context(dev: int):
    """A context of device `dev` that no thread holds.  (No lock: a collection that
    ends another thread's dict may run inside any of these operations, and each of
    them is one step to other threads.)"""
    try:
        return _CONTEXTS.free[dev].pop()
    except (KeyError, IndexError):
        return Context(dev)


def _on(dev: int):
    """This thread's fcu_ctx of the current device `dev`, bound to its current stream."""
    c = _CONTEXTS.of.get(dev)
    if c is None:
        c = _CONTEXTS.of[dev] = _context(dev)
    c.bind_stream(torch._C._cuda_getCurrentRawStream(dev))
    return c.handle


def _device() -> int:
    try:
        return torch.cuda.current_device()
    except Exception:
        device()                        # no CUDA device: the package's error
        raise


class _Functions(dict):
    """The library's functions by name, taking structures as their bytes."""

    def __missing__(self, name):
        declared, fn = getattr(lib(), name), lib()[name]
        fn.restype = declared.restype
        fn.argtypes = [C.c_void_p if t in (C.POINTER(Kv4), C.POINTER(CacheArray)) else t for t in declared.argtypes]
        self[name] = fn
        return fn


_FN = _Functions()
_KV4 = struct.Struct("@7P2q4i")
_ARRAYS = [struct.Struct("@" + "P2q" * n) for n in range(9)]
assert _KV4.size == C.sizeof(Kv4) and _ARRAYS[8].size == C.sizeof(CacheArray * 8)


def _check(name: str, t, dtype, dev: int, shape=None) -> None:
    """t is a contiguous tensor of `dtype` (and `shape`) on device `dev`."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev and t.is_contiguous() and (
            shape is None or t.shape == shape):
        return
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype:
        raise ValueError(f"{name}: a {dtype} tensor is needed, got "
                         f"{t.dtype if isinstance(t, torch.Tensor) else type(t).__name__}")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, not on the current CUDA device")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, {tuple(shape)} is needed")
    raise ValueError(f"{name} is not contiguous")


def _row_bytes(dHead: int) -> int:
    rb = _ROW_BYTES.get(dHead)
    if rb is None:
        rb = _FN["fcu_kv4_row_bytes"](int(dHead))
        if rb <= 0:
            raise ValueError(f"head dim {dHead}: even, 2 to 256")
        _ROW_BYTES[dHead] = rb
    return rb


def _cache(dev, k, kg, v, vg, dHead, B, table, weight=None, pos=None, layers=False) -> bytes:
    """The C-ABI's view (fcu_kv4) of one layer's arrays (five dimensions: of all layers)."""
    rb = _ROW_BYTES.get(dHead) or _row_bytes(dHead)
    try:
        shape = k.shape
        if layers:
            L, blocks, nKV, bs, row = shape
            grid = (L, blocks, nKV, bs, 2)
        else:
            blocks, nKV, bs, row = shape
            grid, L = (blocks, nKV, bs, 2), 1
        ok = (row == rb and v.shape == shape and kg.shape == grid and vg.shape == grid
              and k.dtype is _U8 and v.dtype is _U8 and kg.dtype is _BF and vg.dtype is _BF
              and k.get_device() == dev and v.get_device() == dev and kg.get_device() == dev and vg.get_device() == dev
              and k.is_contiguous() and v.is_contiguous() and kg.is_contiguous() and vg.is_contiguous())
    except (AttributeError, TypeError, ValueError):
        ok = False
    if not ok:
        _check("k", k, _U8, dev)
        if k.ndim != (5 if layers else 4):
            raise ValueError(f"k: {k.ndim} dimensions")
        if k.shape[-1] != rb:
            raise ValueError(f"k: rows of {k.shape[-1]} bytes, head dim {dHead} has {rb}")
        _check("v", v, _U8, dev, k.shape)
        _check("kg", kg, _BF, dev, (*k.shape[:-1], 2))
        _check("vg", vg, _BF, dev, (*k.shape[:-1], 2))
        raise ValueError("k, kg, v, vg: not the arrays of a cache")
    if weight is not None:
        _check("weight", weight, _F32, dev, grid[:-1])
    if pos is not None:
        _check("pos", pos, _I32, dev, grid[:-1])
    if table is not None:
        _check("table", table, _I32, dev)
        if table.ndim != 2 or table.shape[0] != B:
            raise ValueError(f"table: shape {tuple(table.shape)} for {B} sequences")
        mb = table.shape[1]
    else:
        mb, rest = divmod(blocks, B or 1)
        if rest:
            raise ValueError(f"{blocks} blocks do not divide among {B} sequences")
    if max(nKV, bs, mb) >= 2 ** 31:
        raise ValueError(f"k: shape {tuple(shape)}")
    return _KV4.pack(k.data_ptr(), v.data_ptr(), kg.data_ptr(), vg.data_ptr(),
                     weight.data_ptr() if weight is not None else 0, pos.data_ptr() if pos is not None else 0,
                     table.data_ptr() if table is not None else 0, L, blocks, nKV, dHead, bs, mb)


def _rows(name: str, t, dev: int) -> int:
    """Row stride of a two-dimensional fp32 tensor with unit column stride."""
    if not isinstance(t, torch.Tensor) or t.dtype is not _F32 or t.ndim != 2:
        raise ValueError(f"{name}: a two-dimensional float32 tensor is needed")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, not on the current CUDA device")
    rows, cols = t.shape
    ld = t.stride(0)
    if cols < 1 or (cols > 1 and t.stride(1) != 1) or (rows > 1 and ld < cols):
        raise ValueError(f"{name}: shape {tuple(t.shape)} with strides {t.stride()}")
    return ld if rows > 1 else cols


# A call's workspace comes from torch's allocator, which hands it out again only
# to work queued behind the call on the same stream (in a capture: from the
# graph's own pool), so calls on two streams and captured graphs share none.


def kv4Put(qkv, nHeads: int, positions, slots, k, kg, v, vg, T: int = 1, theta: float = 10000.0, table=None,
           weight=None, pos=None) -> None:
    """T new tokens of each of B sequences: qkv [B * T, (nHeads + 2 nKV) dHead]
    fp32 (rows may be strided), token t of sequence b at position positions[b] + t
    and slot slots[b] + t (int32 [B]).  The q heads are rotated in place, k and v
    go to the cache in 4 bits; their columns of qkv stay as they are.  theta 0:
    the rows carry their rotation already.  A token whose slot is outside the
    cache, or whose position is negative or past int32, changes nothing.  No two
    tokens of a call may go to the same place."""
    dev = _device()
    _check("positions", positions, _I32, dev)
    B = positions.numel()
    _check("slots", slots, _I32, dev)
    if slots.numel() != B:
        raise ValueError(f"{slots.numel()} slots for {B} sequences")
    if T < 1 or nHeads < 0 or not theta >= 0:
        raise ValueError(f"T={T}, nHeads={nHeads}, theta={theta}")
    if not isinstance(k, torch.Tensor) or k.ndim != 4:
        raise ValueError("k: an array of four dimensions is needed")
    heads = nHeads + 2 * k.shape[1]
    ld = _rows("qkv", qkv, dev)
    if qkv.shape[0] != B * T or qkv.shape[1] % heads:
        raise ValueError(f"qkv: shape {tuple(qkv.shape)} for {B} x {T} tokens of {heads} heads")
    c = _cache(dev, k, kg, v, vg, qkv.shape[1] // heads, B, table, weight, pos)
    rc = _FN["fcu_kv4_put"](_on(dev), qkv.data_ptr(), ld, B, T, nHeads, float(theta), positions.data_ptr(),
                            slots.data_ptr(), c)
    if rc:
        check(rc, "fcu_kv4_put")


def kv4Values(k, kg, v, vg, dHead: int, start, T: int, table=None):
    """(K, V) fp32 [B, T, nKV, dHead]: the values of slots start[b] .. start[b] + T
    (start int32 [B]).  A slot outside the cache gives NaN."""
    dev = _device()
    _check("start", start, _I32, dev)
    B = start.numel()
    if T < 0:
        raise ValueError(f"T={T}")
    c = _cache(dev, k, kg, v, vg, dHead, B, table)
    K = k.new_empty((B, T, k.shape[1], dHead), dtype=_F32)
    V = torch.empty_like(K)
    rc = _FN["fcu_kv4_values"](_on(dev), c, start.data_ptr(), B, T, K.data_ptr(), V.data_ptr())
    if rc:
        check(rc, "fcu_kv4_values")
    return K, V


def kv4Attention(q, k, kg, v, vg, lens, scale: float | None = None, table=None, weight=None, out=None):
    """[B, nHeads, dHead]: attention of q [B, nHeads, dHead] fp32 (the sequences
    may be strided) over the first lens[b] slots of each sequence (int32 [B];
    0 gives zeros), grouped heads as in attentionDecode.  scale: 1 / sqrt(dHead)
    unless given.  With `weight`, every slot's attention weight, summed over its
    kv head's q heads, is added to it; the sequences may then share no block among
    those slots, and the call takes 4 B nHeads (slots of a sequence's blocks) bytes of
    workspace.  `out` may not overlap q."""
    dev = _device()
    if not (isinstance(q, torch.Tensor) and q.dtype is _F32 and q.ndim == 3):
        raise ValueError("q: a float32 [B, nHeads, dHead] is needed")
    B, nH, dH = q.shape
    if q.get_device() != dev:
        raise ValueError("q is not on the current CUDA device")
    ld, plain = nH * dH, q.is_contiguous()
    if not plain:
        s = q.stride()
        if not ((dH == 1 or s[2] == 1) and (nH == 1 or s[1] == dH) and (B == 1 or s[0] >= ld)):
            raise ValueError(f"q: strides {s}")
        ld = s[0] if B > 1 else ld
    _check("lens", lens, _I32, dev, (B,))
    c = _cache(dev, k, kg, v, vg, dH, B, table, weight)
    if out is None:
        out = torch.empty_like(q) if plain else q.new_empty((B, nH, dH))
    else:
        _check("out", out, _F32, dev)
        if out.numel() != B * nH * dH:
            raise ValueError(f"out: shape {tuple(out.shape)}")
    h = _on(dev)
    nbytes = _FN["fcu_kv4_attn_work"](h, c, B, nH)
    work = k.new_empty((nbytes,)) if nbytes > 0 else None
    rc = _FN["fcu_kv4_attn"](h, q.data_ptr(), ld, c, lens.data_ptr(), B, nH,
                             dH ** -0.5 if scale is None else float(scale), out.data_ptr(),
                             work.data_ptr() if work is not None else None, nbytes)
    if rc:
        check(rc, "fcu_kv4_attn")
    return out


def kv4Evict(k, kg, v, vg, weight, pos, lens, budget: int, recent: int, table=None, newLens=None):
    """Cuts every head of every layer (arrays with a leading layer dimension)
    of sequences longer than `budget` down to it: the slots of the `recent`
    newest positions and those of largest weight stay (ties: the lowest slot),
    moved into the freed slots.  No two sequences may share a block.  Returns the
    new lengths, min(lens, budget)."""
    dev = _device()
    _check("lens", lens, _I32, dev)
    B = lens.numel()
    if weight is None or pos is None:
        raise ValueError("eviction goes by `weight` and `pos`")
    if not 1 <= budget < 2 ** 31 or not 0 <= recent <= budget:
        raise ValueError(f"budget {budget}, recent {recent}")
    if not isinstance(k, torch.Tensor) or k.ndim != 5:
        raise ValueError("k: an array of five dimensions is needed")
    c = _cache(dev, k, kg, v, vg, 2 * k.shape[-1], B, table, weight, pos, layers=True)
    if newLens is None:
        newLens = torch.empty_like(lens)
    else:
        _check("newLens", newLens, _I32, dev, tuple(lens.shape))
    h = _on(dev)
    nbytes = _FN["fcu_kv4_evict_work"](h, c, B, budget)
    work = k.new_empty((nbytes,)) if nbytes > 0 else None
    rc = _FN["fcu_kv4_evict"](h, c, lens.data_ptr(), B, budget, recent, newLens.data_ptr(),
                              work.data_ptr() if work is not None else None, nbytes)
    if rc:
        check(rc, "fcu_kv4_evict")
    return newLens


def beamStep(logits, scores, done, beams: int, eos: int):
    """One beam-search selection: logits [B * beams, V] fp32 (rows may be
    strided), scores fp32 and done bool [B * beams].  Returns (scores, tokens,
    parents, done), [B, beams] each, best first: score + log softmax(logits) over
    all beams and tokens of a sequence, ties to the lowest (beam, token); a beam
    that is done goes on as (eos, its score)."""
    dev = _device()
    ld = _rows("logits", logits, dev)
    R, V = logits.shape
    if not 1 <= beams <= 32 or R % beams:
        raise ValueError(f"{R} rows for searches of {beams} beams (1 to 32)")
    if not 0 <= eos < V:
        raise ValueError(f"eos {eos} outside the vocabulary of {V}")
    _check("scores", scores, _F32, dev)
    _check("done", done, _BOOL, dev)
    if scores.numel() != R or done.numel() != R:
        raise ValueError(f"{scores.numel()} scores, {done.numel()} done for {R} rows")
    B = R // beams
    outScores = scores.new_empty((B, beams))
    tokens = torch.empty_like(outScores, dtype=_I32)
    parents = torch.empty_like(tokens)
    outDone = torch.empty_like(outScores, dtype=_BOOL)
    h = _on(dev)
    nbytes = _FN["fcu_beam_work"](h, B, beams, V)
    work = scores.new_empty((nbytes // 4 + 1,))
    rc = _FN["fcu_beam_step"](h, logits.data_ptr(), ld, scores.data_ptr(), done.data_ptr(), B, beams, V, eos,
                              outScores.data_ptr(), tokens.data_ptr(), parents.data_ptr(), outDone.data_ptr(),
                              work.data_ptr(), nbytes)
    if rc:
        check(rc, "fcu_beam_step")
    return outScores, tokens, parents, outDone


def cacheReorder(arrays, parents, lens, table=None) -> None:
    """The caches of B searches of W beams follow a selection, in place: beam w
    of sequence b (cache sequence b * W + w) takes over slots [0, lens[source])
    of its source b * W + parents[b, w].  arrays: up to 8 tensors [layers, blocks,
    heads, blockSize, ...] whose slots hold a multiple of 4 bytes (an fp32 cache
    has one head: its rows); parents int32 [B, W]; lens int32 [B * W].  No two
    beams may share a block, and no two arrays memory."""
    dev = _device()
    _check("parents", parents, _I32, dev)
    if parents.ndim != 2 or not 1 <= parents.shape[1] <= 32:
        raise ValueError(f"parents: shape {tuple(parents.shape)} (1 to 32 beams)")
    B, W = parents.shape
    _check("lens", lens, _I32, dev)
    if lens.numel() != B * W:
        raise ValueError(f"{lens.numel()} lengths for {B} x {W} beams")
    n = len(arrays)
    if not 1 <= n <= 8:
        raise ValueError(f"{n} arrays (1 to 8)")
    spec = []
    for i, t in enumerate(arrays):
        if not isinstance(t, torch.Tensor) or t.ndim < 4:
            raise ValueError(f"arrays[{i}]: a tensor of at least four dimensions is needed")
        l, m, heads, slots, *rest = t.shape
        if i == 0:
            L, blocks, bs = l, m, slots
        if not (t.get_device() == dev and t.is_contiguous() and l == L and m == blocks and slots == bs):
            _check(f"arrays[{i}]", t, t.dtype, dev)
            raise ValueError(f"arrays[{i}]: shape {tuple(t.shape)} beside {tuple(arrays[0].shape)}")
        spec += t.data_ptr(), heads, math.prod(rest) * t.element_size()
    if table is not None:
        _check("table", table, _I32, dev)
        if table.ndim != 2 or table.shape[0] != B * W:
            raise ValueError(f"table: shape {tuple(table.shape)} for {B * W} beams")
        mb = table.shape[1]
    else:
        if blocks % max(B * W, 1):
            raise ValueError(f"{blocks} blocks do not divide among {B * W} beams")
        mb = blocks // max(B * W, 1)
    rc = _FN["fcu_cache_reorder"](_on(dev), _ARRAYS[n].pack(*spec), n, L, blocks,
                                  table.data_ptr() if table is not None else None, bs, mb, parents.data_ptr(),
                                  lens.data_ptr(), B, W)
    if rc:
        check(rc, "fcu_cache_reorder")


class QuantKVCache(KVCache):
    """KVCache / PagedKVCache holding 4-bit rows (blockSize given: paged, with
    `table` and `physBlocks` as in PagedKVCache).  Transformer.forward and
    forwardBatch take it in their place.  track=True keeps every slot's attention
    weight and position, which evict() goes by; after an eviction a position no
    longer names its slot: sequence b's next token goes to slot lens[b], and only
    tokens that came after it may be written again."""

    def __init__(self, nLayers: int, maxSeq: int, nKvHeads: int, dHead: int, batch: int = 1,
                 blockSize: int | None = None, table=None, physBlocks: int | None = None, track: bool = False):
        rb = _row_bytes(dHead)
        self.nLayers, self.maxSeq, self.batch = nLayers, maxSeq, batch
        self.nKvHeads, self.dHead, self.kvDim = nKvHeads, dHead, nKvHeads * dHead
        self.block_size = maxSeq if blockSize is None else blockSize
        self.max_blocks = -(-maxSeq // self.block_size)
        phys = physBlocks if physBlocks is not None else batch * self.max_blocks
        dev = device()
        lead = (nLayers, phys, nKvHeads, self.block_size)
        self.k = torch.zeros(*lead, rb, dtype=_U8, device=dev)
        self.v = torch.zeros_like(self.k)
        self.kg = torch.zeros(*lead, 2, dtype=_BF, device=dev)
        self.vg = torch.zeros_like(self.kg)
        self.weight = torch.zeros(lead, dtype=_F32, device=dev) if track else None
        self.pos = torch.zeros(lead, dtype=_I32, device=dev) if track else None
        self.table, self._table_host = None, None
        if table is not None:
            t = np.ascontiguousarray(table, np.int32).reshape(batch, self.max_blocks)
            if t.min() < 0 or t.max() >= phys:
                raise ValueError("QuantKVCache: block table entry outside the physical blocks")
            if track and np.unique(t).size < t.size:
                raise ValueError("QuantKVCache: sequences that share blocks cannot keep their weights apart")
            self._table_host, self.table = t, torch.from_numpy(t).to(dev)
        elif phys != batch * self.max_blocks:
            raise ValueError(f"QuantKVCache: {phys} physical blocks need a block table")
        self.reset()

    def reset(self) -> None:
        self.len = 0
        self.lens = np.zeros(self.batch, np.int32)       # slots in use
        self.dropped = np.zeros(self.batch, np.int32)    # tokens evicted so far
        self.kept = np.zeros(self.batch, np.int32)       # slots that the last eviction left, in no order of position

    def slotOf(self, pos: int, seq: int = 0) -> int:
        """The slot that position `pos` of a sequence is written to: its next one, one
        written since the last eviction or, while nothing was evicted, any."""
        s = int(pos) - int(self.dropped[seq])
        if s < 0 or s >= self.max_blocks * self.block_size:
            raise ValueError(f"QuantKVCache: no slot for position {pos} ({self.dropped[seq]} tokens evicted, "
                             f"{self.max_blocks * self.block_size} slots)")
        if self.dropped[seq] and s < self.kept[seq]:
            raise ValueError(f"QuantKVCache: position {pos} may have been evicted")
        if self.dropped[seq] and s > self.lens[seq]:
            raise ValueError(f"QuantKVCache: position {pos} is not next ({self.lens[seq] + self.dropped[seq]} is), and "
                             "the slots between hold evicted tokens")
        return s

    def _used(self, seq: int, slot: int) -> None:
        self.lens[seq] = max(self.lens[seq], slot + 1)
        self.len = max(self.len, int(self.lens[seq]))

    def _layer(self, l: int, seq: int | None = None):
        """Arrays and table of layer l (of one sequence: its own table row)."""
        if seq is None:
            return (self.k[l], self.kg[l], self.v[l], self.vg[l]), self.table
        if self.table is not None:
            return (self.k[l], self.kg[l], self.v[l], self.vg[l]), self.table[seq:seq + 1]
        a, b = seq * self.max_blocks, (seq + 1) * self.max_blocks
        return (self.k[l, a:b], self.kg[l, a:b], self.v[l, a:b], self.vg[l, a:b]), None

    def rows_per_layer(self) -> int:
        return self.k.shape[1] * self.block_size

    def put(self, layer: int, pos: int, k, v, seq: int = 0) -> None:
        slot = self.slotOf(pos, seq)
        row = torch.cat([_dev_f32(k).reshape(1, -1), _dev_f32(v).reshape(1, -1)], 1)
        at = torch.tensor([[pos], [slot]], dtype=_I32, device=row.device)
        arrays, table = self._layer(layer, seq)
        w = p = None
        if self.weight is not None:
            a, b = (seq * self.max_blocks, (seq + 1) * self.max_blocks) if table is None else (0, self.k.shape[1])
            w, p = self.weight[layer, a:b], self.pos[layer, a:b]
        kv4Put(row, 0, at[0], at[1], *arrays, theta=0.0, table=table, weight=w, pos=p)
        self._used(seq, slot)

    def _view(self, layer: int, start: int, n: int, seq: int):
        arrays, table = self._layer(layer, seq)
        K, V = kv4Values(*arrays, self.dHead, torch.tensor([start], dtype=_I32, device=self.k.device), n, table=table)
        return K.reshape(n, self.kvDim), V.reshape(n, self.kvDim)

    def kView(self, layer: int, upto: int, seq: int = 0) -> torch.Tensor:
        """The values of the first `upto` slots (a copy)."""
        return self._view(layer, 0, upto, seq)[0]

    def vView(self, layer: int, upto: int, seq: int = 0) -> torch.Tensor:
        return self._view(layer, 0, upto, seq)[1]

    def sliceK(self, layer: int, pos: int, seq: int = 0) -> torch.Tensor:
        return self._view(layer, pos, 1, seq)[0][0]

    def sliceV(self, layer: int, pos: int, seq: int = 0) -> torch.Tensor:
        return self._view(layer, pos, 1, seq)[1][0]

    def _own_blocks(self) -> None:
        t = self._table_host
        if t is not None and np.unique(t).size < t.size:
            raise ValueError("QuantKVCache: sequences that share blocks cannot be evicted from or reordered")

    def evict(self, budget: int, recent: int) -> None:
        """kv4Evict of every layer and sequence."""
        _need(self.weight is not None, "QuantKVCache: made without track=True")
        _need(budget >= 1 and 0 <= recent <= budget, f"budget {budget}, recent {recent}")
        self._own_blocks()
        if self.lens.max(initial=0) <= budget:
            return
        lens = torch.from_numpy(self.lens.copy()).to(self.k.device)
        kv4Evict(self.k, self.kg, self.v, self.vg, self.weight, self.pos, lens, budget, recent, table=self.table)
        new = np.minimum(self.lens, budget).astype(np.int32)
        self.kept = np.where(new < self.lens, new, self.kept)
        self.dropped += self.lens - new
        self.lens, self.len = new, int(new.max())

    def reorder(self, parents) -> None:
        """cacheReorder for searches of parents.shape[1] beams over all `batch`
        sequences (parents: a host or device int array [B, W])."""
        self._own_blocks()
        p = np.asarray(parents.cpu() if isinstance(parents, torch.Tensor) else parents)
        _reorder(self, [t for t in (self.k, self.kg, self.v, self.vg, self.weight, self.pos) if t is not None], p,
                 self.lens)
        src = (np.arange(p.shape[0])[:, None] * p.shape[1] + p).reshape(-1)
        self.lens, self.dropped, self.kept = self.lens[src].copy(), self.dropped[src].copy(), self.kept[src].copy()
        self.len = int(self.lens.max(initial=0))

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.kg, self.vg, self.weight, self.pos)
                   if t is not None)


def _reorder(cache, arrays, parents, lens) -> None:
    p = parents if isinstance(parents, torch.Tensor) else torch.as_tensor(np.asarray(parents))
    _need(p.ndim == 2 and p.numel() == cache.batch and not p.is_floating_point(),
          f"parents: {p.dtype} of shape {tuple(p.shape)} for a cache of {cache.batch}")
    if not p.is_cuda and p.numel():
        _need(int(p.min()) >= 0 and int(p.max()) < p.shape[1], "parents outside their search's beams")
    lens = torch.from_numpy(np.ascontiguousarray(lens, np.int32)).to(cache.k.device)
    table = cache.table
    if table is None and arrays[0].shape[1] != cache.batch * cache.max_blocks:      # more blocks than it uses
        table = torch.arange(cache.batch * cache.max_blocks, dtype=_I32, device=cache.k.device).view(cache.batch, -1)
    cacheReorder(arrays, p.to(device=cache.k.device, dtype=_I32).contiguous(), lens, table=table)
