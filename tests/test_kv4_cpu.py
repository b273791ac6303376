"""Refusals of the 4-bit cache's, beam search's and reordering's entry points
(CPU: they return before any CUDA call, so a zeroed block stands for the
context), and the 64-bit restatements the GPU tests compare with."""
import ctypes as C
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "forge-llm_b200"))

import kv4_ref as R  # noqa: E402
from forgellm import _lib  # noqa: E402

ARG = _lib.FCU_ERR_ARG


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


@pytest.fixture(scope="module")
def ctx():
    return C.create_string_buffer(4096)


def cache(**kw):
    """A cache of made-up addresses: 4 sequences of 2 blocks of 16 slots."""
    d = dict(k=4096, v=8192, kg=4096, vg=4096, weight=None, pos=None, table=None, layers=1, blocks=8, n_kv=2, dH=64,
             block_size=16, max_blocks=2)
    d.update(kw)
    return _lib.Kv4(**d)


BAD_CACHES = [dict(dH=63), dict(dH=0), dict(dH=258), dict(n_kv=0), dict(blocks=-1), dict(block_size=0),
              dict(max_blocks=0), dict(layers=0), dict(k=4097), dict(v=8), dict(kg=2), dict(vg=None), dict(k=None),
              dict(blocks=7), dict(block_size=1 << 20, max_blocks=1 << 20), dict(table=6)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda d: "-".join(map(str, d)))
def test_bad_caches_are_refused_everywhere(L, ctx, bad):
    c = cache(weight=4096, pos=4096, **bad)
    assert L.fcu_kv4_put(ctx, 4096, 4096, 4, 1, 4, 1e4, 4096, 4096, c) == ARG
    assert L.fcu_kv4_values(ctx, c, 4096, 4, 1, 4096, 4096) == ARG
    assert L.fcu_kv4_attn(ctx, 4096, 4096, c, 4096, 4, 4, 1.0, 4096, 4096, 1 << 40) == ARG
    assert L.fcu_kv4_evict(ctx, c, 4096, 4, 8, 4, 8192, 4096, 1 << 40) == ARG
    assert b"fcu_kv4_evict" in L.fcu_last_error()


def test_bad_arguments_are_refused(L, ctx):
    ok = cache()
    put = lambda **k: L.fcu_kv4_put(*{**dict(ctx=ctx, qkv=4096, ld=512, B=4, T=1, nH=4, theta=1e4, pos=4096,  # noqa: E731
                                             slots=4096, c=ok), **k}.values())
    for bad in (dict(ctx=None), dict(qkv=None), dict(ld=511), dict(B=-1), dict(T=-1), dict(nH=-1), dict(theta=-1.0),
                dict(theta=float("nan")), dict(theta=float("inf")), dict(pos=None), dict(slots=None), dict(c=None)):
        assert put(**bad) == ARG, bad
    val = lambda **k: L.fcu_kv4_values(*{**dict(ctx=ctx, c=ok, start=4096, B=4, T=1, K=4096, V=4096), **k}.values())  # noqa: E731
    for bad in (dict(ctx=None), dict(c=None), dict(start=None), dict(B=5), dict(B=-1), dict(T=-1)):
        assert val(**bad) == ARG, bad
    att = lambda **k: L.fcu_kv4_attn(*{**dict(ctx=ctx, q=4096, ld=256, c=ok, lens=4096, B=4, nH=4, scale=1.0,  # noqa: E731
                                              out=1 << 20, work=4096, n=1 << 40), **k}.values())
    for bad in (dict(ctx=None), dict(q=None), dict(ld=255), dict(c=None), dict(lens=None), dict(B=-1), dict(B=70000),
                dict(nH=3), dict(nH=0), dict(nH=34), dict(out=None), dict(out=4096), dict(out=4096 + 4 * 1016),
                dict(ld=1000, out=4096 + 4 * 3000), dict(q=1 << 20), dict(q=(1 << 20) + 4 * 1020)):
        assert att(**bad) == ARG, bad
    tracked = cache(weight=4096, pos=4096)
    for bad in (dict(work=None), dict(n=16), dict(work=4100)):
        assert att(c=tracked, **bad) == ARG, bad
    ev = lambda **k: L.fcu_kv4_evict(*{**dict(ctx=ctx, c=tracked, lens=4096, B=4, budget=8, recent=4, new=8192,  # noqa: E731
                                              work=None, n=0), **k}.values())
    for bad in (dict(ctx=None), dict(c=ok), dict(c=None), dict(lens=None), dict(B=-1), dict(budget=0), dict(recent=-1),
                dict(recent=9), dict(new=None), dict(new=4096), dict(new=4104)):
        assert ev(**bad) == ARG, bad
    long = cache(weight=4096, pos=4096, block_size=1 << 17, max_blocks=1, blocks=4)
    assert L.fcu_kv4_evict_work(ctx, long, 4, 8) == 4 * 2 * ((1 << 17) + (1 << 12)) * 4
    assert L.fcu_kv4_evict_work(ctx, long, 4, 1000) == 4 * 2 * ((1 << 17) + (1 << 12) + 2 * 1000 + 1) * 4
    assert ev(c=long) == ARG and ev(c=long, work=4096, n=100) == ARG
    beam = lambda **k: L.fcu_beam_step(*{**dict(ctx=ctx, x=4096, ld=100, s=8192, d=8256, B=2, W=4, V=100, eos=2,  # noqa: E731
                                                os=8320, t=8352, p=8384, od=8416, work=16384, n=1 << 40), **k}.values())
    for bad in (dict(ctx=None), dict(x=None), dict(ld=99), dict(s=None), dict(d=None), dict(B=-1), dict(B=20000),
                dict(W=0), dict(W=33), dict(V=0), dict(V=1 << 31, ld=1 << 32), dict(eos=-1), dict(eos=100),
                dict(os=None), dict(t=None), dict(work=None), dict(n=8), dict(work=16388),
                # outputs that overlap an input or one another
                dict(os=8192), dict(od=8256), dict(os=8196), dict(od=8249), dict(t=8220), dict(p=8352), dict(od=8340),
                dict(t=4096), dict(p=4096 + 3196)):
        assert beam(**bad) == ARG, bad

    def reorder(arrays=((4096, 2, 32),), **k):
        spec = (_lib.CacheArray * max(len(arrays), 1))(*[_lib.CacheArray(*a) for a in arrays])
        a = dict(ctx=ctx, spec=spec, n=len(arrays), layers=2, blocks=16, table=None, bs=16, mb=2, parents=4096,
                 lens=4096, B=2, W=4)
        return L.fcu_cache_reorder(*{**a, **k}.values())

    for bad in (dict(ctx=None), dict(n=9), dict(n=-1), dict(spec=None), dict(layers=-1), dict(blocks=15), dict(bs=0),
                dict(mb=0), dict(parents=None), dict(lens=None), dict(B=-1), dict(W=0), dict(W=33),
                dict(arrays=((None, 2, 32),)), dict(arrays=((4100, 2, 32),)), dict(arrays=((4096, 0, 32),)),
                dict(arrays=((4096, 2, 30),)), dict(arrays=((4096, 2, 0),)),
                # 32 blocks of 16 slots: 32768 and 2048 bytes
                dict(arrays=((4096, 2, 32), (4096, 2, 32))), dict(arrays=((4096, 2, 32), (4096 + 32752, 1, 4))),
                dict(arrays=((4096 + 2032, 2, 32), (4096, 1, 4)))):
        assert reorder(**bad) == ARG, bad


def test_empty_calls_do_nothing(L, ctx):
    c = cache(weight=4096, pos=4096)
    assert L.fcu_kv4_put(ctx, None, 512, 0, 1, 4, 1e4, None, None, c) == 0
    assert L.fcu_kv4_put(ctx, None, 512, 4, 0, 4, 1e4, None, None, c) == 0
    assert L.fcu_kv4_values(ctx, c, None, 4, 0, None, None) == 0
    assert L.fcu_kv4_attn(ctx, None, 256, c, None, 0, 4, 1.0, None, None, 0) == 0
    assert L.fcu_kv4_evict(ctx, c, None, 0, 8, 4, None, None, 0) == 0
    assert L.fcu_beam_step(ctx, None, 100, None, None, 0, 4, 100, 2, None, None, None, None, None, 0) == 0


def test_row_bytes(L):
    for d in range(-2, 300):
        assert L.fcu_kv4_row_bytes(d) == (R.row_bytes(d) if 2 <= d <= 256 and d % 2 == 0 else -1)


def test_work_sizes_are_refused_for_bad_arguments(L, ctx):
    assert L.fcu_kv4_attn_work(None, cache(), 4, 4) == -1
    assert L.fcu_kv4_attn_work(ctx, cache(dH=3), 4, 4) == -1
    assert L.fcu_kv4_attn_work(ctx, cache(), 4, 3) == -1
    assert L.fcu_kv4_evict_work(ctx, cache(), -1, 8) == -1
    assert L.fcu_kv4_evict_work(ctx, cache(), 4, 0) == -1
    assert L.fcu_beam_work(ctx, 1, 33, 100) == -1
    assert L.fcu_beam_work(ctx, 1, 4, 0) == -1


def test_python_refuses_tensors_off_the_device():
    torch = pytest.importorskip("torch")
    import forgellm as F
    z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t)  # noqa: E731
    k, kg = z(4, 2, 16, 32, t=torch.uint8), z(4, 2, 16, 2, t=torch.bfloat16)
    i = z(4, t=torch.int32)
    for f in (lambda: F.kv4Attention(z(4, 4, 64), k, kg, k, kg, i), lambda: F.kv4Put(z(4, 512), 4, i, i, k, kg, k, kg),
              lambda: F.kv4Values(k, kg, k, kg, 64, i, 1), lambda: F.beamStep(z(4, 9), z(4), z(4, t=torch.bool), 2, 1),
              lambda: F.kv4Evict(k[None], kg[None], k[None], kg[None], z(1, 4, 2, 16), z(1, 4, 2, 16), i, 4, 2),
              lambda: F.cacheReorder([k[None]], z(2, 2, t=torch.int32), i)):
        with pytest.raises((ValueError, F.ForgeCUError)):      # the latter where there is no device at all
            f()


def test_every_thread_has_a_context_of_its_own(monkeypatch):
    """A thread that binds its stream leaves the calls of others where they are."""
    torch = pytest.importorskip("torch")
    import threading
    from forgellm import kv4

    class Fake:
        def __init__(self, device):
            self.handle, self.stream = object(), None

        def bind_stream(self, s):
            self.stream = s

    streams = threading.local()
    monkeypatch.setattr(kv4, "Context", Fake)
    monkeypatch.setattr(kv4, "_CONTEXTS", kv4._Contexts())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: streams.now, raising=False)
    seen, gate = {}, threading.Barrier(3)

    def work(i):
        streams.now = i
        first = kv4._on(0)
        gate.wait(10)
        c = kv4._CONTEXTS.of[0]
        seen[i] = (first, kv4._on(0), kv4._on(1), c.stream)
        gate.wait(10)

    threads = [threading.Thread(target=work, args=(i,)) for i in (1, 2)]
    for t in threads:
        t.start()
    work(0)
    for t in threads:
        t.join()
    for i in range(3):
        assert seen[i][0] is seen[i][1] and seen[i][3] == i
    assert len({id(h) for s in seen.values() for h in s[:3]}) == 6


def test_a_finished_threads_contexts_are_used_again(monkeypatch):
    """Many short threads make as many contexts as are held at once, each bound to its
    holder's stream."""
    torch = pytest.importorskip("torch")
    import gc
    import threading
    from forgellm import kv4

    class Fake:
        made = []

        def __init__(self, device):
            self.handle, self.stream, self.device = object(), None, device
            self.made.append(self)

        def bind_stream(self, s):
            self.stream = s

    streams = threading.local()
    monkeypatch.setattr(kv4, "Context", Fake)
    monkeypatch.setattr(kv4, "_CONTEXTS", kv4._Contexts())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: streams.now, raising=False)
    wrong = []

    def work(i, gate=None):
        streams.now = i
        for dev in (0, 1, 0):
            h = kv4._on(dev)
            c = kv4._CONTEXTS.of[dev]
            if c.handle is not h or c.stream != i or c.device != dev:
                wrong.append(i)
            if gate:
                gate.wait(10)
                if c.stream != i:
                    wrong.append(i)

    def run(n, gate=None):
        threads = [threading.Thread(target=work, args=(i, gate)) for i in range(n)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        gc.collect()

    for _ in range(20):
        run(1)
    assert len(Fake.made) == 2 and not wrong
    run(5, threading.Barrier(5))
    assert len(Fake.made) == 10 and not wrong
    for _ in range(10):
        run(5)
    assert len(Fake.made) == 10 and not wrong
    # they are this _Contexts' alone
    monkeypatch.undo()
    assert not any(isinstance(c, Fake) for cs in kv4._CONTEXTS.free.values() for c in cs)


# ------------------------------------------------------------------ the restatements themselves
def test_reference_quantizer_bound():
    """|x - x^| <= step / 2 inside the grid; the ends add the roundings of base and
    step to bf16 (2^-9 of |base|, 15 * 2^-9 of step) and the value its fp32 one."""
    rng = np.random.default_rng(0)
    for off in (0.0, 5.0, -300.0):
        x = (rng.standard_normal((500, 96)) + off).astype(np.float32)
        c, s, b = R.quantize(x)
        err = np.abs(R.values(c, s, b).astype(np.float64) - x)
        assert (err <= s / 2 + np.abs(b) * 2.0 ** -8 + 15 * s * 2.0 ** -8 + np.abs(x) * 2.0 ** -23).all()


def test_reference_eviction_keeps_the_right_slots():
    w = np.array([5, 1, 9, 1, 7, np.nan, 2, 3], np.float32)
    pos = np.arange(8)
    dst, src = R.evict(w, pos, 8, 4, 2)     # 6 and 7 are recent, 2 and 4 are heavy
    assert dst.tolist() == [0, 1, 3] and src.tolist() == [4, 6, 7]
    dst, src = R.evict(np.ones(6, np.float32), pos, 6, 3, 0)   # all equal: the lowest slots
    assert len(dst) == 0 and len(src) == 0


def test_reference_beam_ties_and_finished_beams():
    x = np.zeros((1, 2, 5))
    s, t, p, d = R.beam(x, np.array([[0.0, -1.0]]), np.array([[False, True]]), 2, 4)
    assert t.tolist() == [[4, 0]] and p.tolist() == [[1, 0]] and d.tolist() == [[True, False]]
