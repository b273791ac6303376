"""The 4-bit KV cache on the GPU against 64-bit restatements (kv4_ref.py).

Tolerances, from the arithmetic:
- put / values: codes, grids and the values read back equal the restatement's
  bit for bit (its border cases are decided in double by both); q within
  2^-24 relative of the double rotation's rounding, i.e. 1e-7 of the row's
  largest value.
- attention: the operator runs in fp32, each product q_e * x^_e held to 2^-23
  relative.  A score sums dH of them, |x^_e| <= b_j = |base_j| + 15 step_j; with
  roundings independent of one another its error is of the size 2^-23 * A,
  A = |scale| * |q|_2 * max_j b_j, and twice that, d = 2^-22 * A, is taken for
  the whole (|s| itself is below A, so its own rounding is in there).  A weight p
  then has the relative error 2 d plus 2^-20 (the exponential, its argument, the
  sums), and an output is a mean of values below C = max_j b_j:
  |error| <= C * (4 d + 2^-19).  Over a whole sequence the errors of the weights
  are as many as the outputs: the relative error of its output in the 2-norm is
  held to 2 d + 2^-20.  An accumulated weight adds g such p.
- eviction moves bytes: everything equal.
"""
import math

import numpy as np
import pytest

import kv4_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

I32, F32, U8, BF = torch.int32, torch.float32, torch.uint8, torch.bfloat16


def F():
    import forgellm
    return forgellm


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


class Cache:
    """A filled cache of B sequences, on the host (values) and the device."""

    def __init__(self, B, cap, nKV, dH, block=0, seed=0, shuffle=True, scale=1.0, rows=None):
        rng = np.random.default_rng(seed)
        self.B, self.nKV, self.dH = B, nKV, dH
        self.bs = block or cap
        self.mb = -(-cap // self.bs)
        self.phys = B * self.mb
        self.table = (rng.permutation(self.phys) if shuffle and block else np.arange(self.phys)).astype(np.int32)
        self.table = self.table.reshape(B, self.mb)
        shape = (self.phys, nKV, self.bs, dH)
        self.x = [(rng.standard_normal(shape) * scale).astype(np.float32) for _ in range(2)]
        if rows is not None:
            for x in self.x:
                rows(x, rng)
        rb = R.row_bytes(dH)
        self.code, self.step, self.base = zip(*[R.quantize(x) for x in self.x])
        self.k, self.v = [dev(R.pack(c, rb)) for c in self.code]
        self.kg, self.vg = [dev(np.concatenate([s, b], -1).astype(np.float32), BF) for s, b in zip(self.step, self.base)]
        self.dtable = dev(self.table) if block else None

    def args(self):
        return self.k, self.kg, self.v, self.vg

    def places(self, b, n):
        j = np.arange(n)
        return self.table[b, j // self.bs], j % self.bs

    def rows(self, which, b, h, n):
        """Values [n, dH] in 64 bits (the fp32 values' exact counterparts)."""
        blk, off = self.places(b, n)
        return (self.base[which][blk, h, off] + self.step[which][blk, h, off] * self.code[which][blk, h, off])

    def bound(self, which):
        return np.abs(self.base[which]) + 15 * self.step[which]


def score_error(c, q, scale):
    return 2.0 ** -22 * abs(scale) * np.sqrt((q.astype(np.float64) ** 2).sum(-1)).max() * np.nanmax(c.bound(0))


def tolerance(c, q, scale):
    return np.nanmax(c.bound(1)) * (4 * score_error(c, q, scale) + 2.0 ** -19)


def check_attention(c, q, lens, scale=None, weight=None, got=None):
    B, nH, dH = q.shape
    g = nH // c.nKV
    sc = 1 / math.sqrt(dH) if scale is None else scale
    w = dev(weight) if weight is not None else None
    if got is None:
        got = F().kv4Attention(dev(q), *c.args(), dev(np.array(lens, np.int32)), scale=scale, table=c.dtable, weight=w)
    got = got.cpu().numpy()
    tol = tolerance(c, q, sc)
    want_w = weight.astype(np.float64).copy() if weight is not None else None
    for b, n in enumerate(lens):
        n = max(0, min(n, c.mb * c.bs))
        blk, off = c.places(b, n)
        off2 = norm2 = 0.0
        for h in range(c.nKV):
            K, V = c.rows(0, b, h, n), c.rows(1, b, h, n)
            for hg in range(g):
                want, p = R.attention(q[b, h * g + hg], K, V, sc)
                err = np.abs(want - got[b, h * g + hg])
                assert not np.isnan(got[b, h * g + hg]).any(), (b, n, h, hg)
                assert err.max(initial=0) <= tol, (b, n, h, hg, err.max(), tol)
                off2, norm2 = off2 + float((err ** 2).sum()), norm2 + float((want ** 2).sum())
                if want_w is not None:
                    want_w[blk, h, off] += p
        assert math.sqrt(off2) <= math.sqrt(norm2) * (2 * score_error(c, q, sc) + 2.0 ** -20), (b, n, math.sqrt(off2 / norm2))
    if want_w is not None:
        # every p within its relative error; adding it to the slot rounds once (2^-24 of the sum)
        err = np.abs(w.cpu().numpy() - want_w)
        assert (err <= (want_w - weight) * (2 * score_error(c, q, sc) + 2.0 ** -19) + want_w * 2.0 ** -23 + 1e-30).all()
    return got


LENS = [0, 1, 5, 31, 63, 64, 65, 256, 257, 1000]


@pytest.mark.parametrize("nH,nKV,dH", [(12, 4, 64), (4, 4, 16), (16, 1, 128), (4, 2, 256), (6, 2, 96), (5, 5, 80),
                                       (24, 3, 48), (9, 3, 34), (12, 1, 160), (16, 2, 32), (8, 8, 2), (26, 2, 192)])
@pytest.mark.parametrize("block", [0, 48, 7])
def test_attention(nH, nKV, dH, block):
    c = Cache(len(LENS), 1008, nKV, dH, block, seed=dH + block)
    q = np.random.default_rng(1).standard_normal((len(LENS), nH, dH)).astype(np.float32)
    check_attention(c, q, LENS)


@pytest.mark.parametrize("nH,nKV,dH,block", [(12, 4, 64, 0), (16, 2, 96, 48), (32, 2, 80, 16), (3, 3, 128, 100),
                                             (8, 1, 256, 1)])
def test_attention_accumulates_weights(nH, nKV, dH, block):
    lens = [0, 1, 63, 300, 517]
    c = Cache(len(lens), 600, nKV, dH, block, seed=3)
    rng = np.random.default_rng(2)
    q = rng.standard_normal((len(lens), nH, dH)).astype(np.float32) * 2
    weight = rng.random((c.phys, nKV, c.bs)).astype(np.float32)
    out = check_attention(c, q, lens, weight=weight)
    assert np.array_equal(out, check_attention(c, q, lens, weight=weight))    # run to run the same bits


def test_attention_with_sharp_and_flat_scores():
    """Scores tens of units apart (one slot takes all) and all alike."""
    c = Cache(3, 700, 2, 64, 64, seed=9)
    q = np.random.default_rng(5).standard_normal((3, 8, 64)).astype(np.float32)
    check_attention(c, q * 30, [700, 699, 2])
    check_attention(c, q * 0, [700, 699, 2])
    check_attention(c, q, [700, 0, 130], scale=0.0)
    check_attention(c, q, [700, 64, 130], scale=-0.3)


@pytest.mark.parametrize("nH,nKV,dH,n,size", [(12, 4, 72, 333, 0.05), (8, 2, 128, 3000, 0.05), (16, 2, 64, 3000, 0.01),
                                              (4, 1, 64, 30000, 0.3)])
@pytest.mark.parametrize("seed", range(3))
def test_attention_with_nearly_equal_weights(nH, nKV, dH, n, size, seed):
    """The mean of many rows is far smaller than the rows and than their grids' bases."""
    c = Cache(2, n, nKV, dH, 0, seed=seed)
    q = np.random.default_rng(seed + 50).standard_normal((2, nH, dH)).astype(np.float32) * np.float32(size)
    check_attention(c, q, [n, n // 3])


def test_attention_over_unequal_rows():
    """Constant rows (step 0), rows far from zero, tiny and large rows."""
    def rows(x, rng):
        x[:, :, 3] = 0.75
        x[:, :, 5] = 0
        x[:, :, 10:20] += 40
        x[:, :, 30:40] *= 1e-20
        x[:, :, 50] *= 100
    c = Cache(2, 333, 4, 72, 0, seed=2, rows=rows)
    q = np.random.default_rng(6).standard_normal((2, 12, 72)).astype(np.float32) * 0.05
    check_attention(c, q, [333, 60])
    c = Cache(2, 333, 4, 72, 0, seed=2, scale=1e-18)
    check_attention(c, q * 1e18, [333, 60])


@pytest.mark.parametrize("nH,dH", [(4, 64), (8, 64), (3, 128), (10, 96), (2, 24)])
def test_attention_with_large_values_of_little_weight(nH, dH):
    """Every 32nd slot holds values 2^18 times the others' with weights of about
    e^-19: what is kept of the others' must not go by either alone."""
    seen = []

    def rows(x, rng):
        if seen:
            x[:, :, 7::32] *= 2.0 ** 18
        else:
            x[:, :, 7::32] = -3 * np.sqrt(64 / dH)
        seen.append(1)
    c = Cache(2, 512, 1, dH, 0, seed=13, rows=rows)
    q = np.abs(np.random.default_rng(14).standard_normal((2, nH, dH))).astype(np.float32)
    check_attention(c, q, [512, 75])


@pytest.mark.parametrize("nH", [8, 16])
def test_attention_with_extreme_queries(nH):
    """Queries and scales whose product is ordinary, heads that are not finite
    beside ones that are, and grids that run downwards."""
    c = Cache(2, 200, 2, 64, 64, seed=15)
    q = np.random.default_rng(16).standard_normal((2, nH, 64)).astype(np.float32)
    for big in (1e30, 1e-30, 2.0 ** 90):
        check_attention(c, (q * np.float32(big)), [200, 77], scale=0.125 / big)
    check_attention(c, q * np.float32(1e-36), [200, 77])
    bad = q.copy()
    bad[0, 1, 5] = np.nan
    bad[1, nH - 1, 63] = np.inf
    bad[1, 2, 0] = -np.inf
    out = F().kv4Attention(dev(bad), *c.args(), dev(np.array([200, 77], np.int32)), table=c.dtable).cpu().numpy()
    hit = np.isnan(out).all(-1)
    assert hit[0, 1] and hit[1, nH - 1] and hit[1, 2] and hit.sum() == 3
    good = check_attention(c, q, [200, 77])
    assert np.array_equal(out[~hit], good[~hit])
    c.step = tuple(-x for x in c.step)
    c.kg, c.vg = [dev(np.concatenate([x, b], -1).astype(np.float32), BF) for x, b in zip(c.step, c.base)]
    c.bound = lambda w: np.abs(c.base[w]) + 15 * np.abs(c.step[w])
    check_attention(c, q, [200, 77])


@pytest.mark.parametrize("nH,dH", [(4, 128), (16, 64), (6, 256)])
@pytest.mark.parametrize("size", [2.0 ** 92, 2.0 ** 100, 2.0 ** 115, 2.0 ** 120])
def test_attention_over_keys_of_any_size(nH, dH, size):
    """Keys up to what the cache holds as finite: with queries that make the scores
    ordinary, and with ones that make them large (one slot takes all, or equal
    rows share)."""
    def rows(x, rng):
        if not seen:
            x *= np.float32(size)
        seen.append(1)
    seen = []
    c = Cache(2, 200, 2, dH, 64, seed=17, rows=rows)
    q = np.random.default_rng(18).standard_normal((2, nH, dH)).astype(np.float32)
    check_attention(c, q * np.float32(1 / size), [200, 77])
    check_attention(c, q, [200, 77], scale=0.125 / size)
    check_attention(c, q * np.float32(2.0 ** 14), [200, 77], scale=2.0 ** -17 / size)
    # scores of the keys' own size: a query along the unit vector e picks the slot of the
    # largest element e, and the largest two are further apart than any rounding
    K = [np.concatenate([c.rows(0, b, h, n) for h in range(2)], 1).reshape(n, 2, dH) for b, n in ((0, 200), (1, 77))]
    one = np.zeros((2, nH, dH), np.float32)
    want = np.zeros((2, nH, dH))
    for b in range(2):
        for h in range(nH):
            kv = h // (nH // 2)
            col = K[b][:, kv]
            top = np.sort(col, 0)
            e = int(np.argmax(top[-1] - top[-2]))
            assert top[-1, e] - top[-2, e] > size * 2.0 ** -10
            one[b, h, e] = 1
            want[b, h] = c.rows(1, b, kv, len(col))[int(np.argmax(col[:, e]))]
    got = F().kv4Attention(dev(one), *c.args(), dev(np.array([200, 77], np.int32)), scale=1.0, table=c.dtable)
    assert np.abs(got.cpu().numpy() - want).max() <= 2.0 ** -19 * np.abs(want).max()


def test_attention_with_queries_whose_sum_leaves_fp32():
    """Finite queries of one sign: their sum, which meets the rows' base, passes
    2^128, their scaled sum does not; and queries so large that only tiny keys
    make ordinary scores of them."""
    c = Cache(2, 200, 2, 64, 64, seed=19)
    q = np.abs(np.random.default_rng(20).standard_normal((2, 8, 64))).astype(np.float32) + 1
    check_attention(c, q * np.float32(2.0 ** 124), [200, 77], scale=2.0 ** -128)
    tiny = []

    def rows(x, rng):
        if not tiny:
            x *= np.float32(2.0 ** -112)      # the keys
        tiny.append(1)
    c = Cache(2, 200, 2, 64, 64, seed=19, rows=rows)
    check_attention(c, q * np.float32(2.0 ** 109), [200, 77])
    check_attention(c, q * np.float32(2.0 ** 100), [200, 77], scale=2.0 ** 8)


@pytest.mark.parametrize("nH,dH,n", [(4, 64, 200), (8, 128, 3000), (1, 16, 70001)])
def test_attention_over_values_near_the_largest(nH, dH, n):
    """Values near 2^122 under weights that are nearly equal: their mean is in the type,
    their sum is not; with small ones beside them."""
    seen = []

    def rows(x, rng):
        if seen:
            x[:] = 2.0 ** 122 * (0.8 + 0.19 * rng.random(x.shape))
            x[:, :, 3::5] *= -0.5
            x[:, :, 4::7] *= 2.0 ** -110
        else:
            x *= 0.05
        seen.append(1)
    c = Cache(2, n, 1, dH, 0, seed=22, rows=rows)
    q = np.random.default_rng(23).standard_normal((2, nH, dH)).astype(np.float32)
    check_attention(c, q, [n, n // 3], weight=np.zeros((2, 1, n), np.float32))
    check_attention(c, q, [n, 1])


def test_slots_past_the_length_are_not_read():
    c = Cache(3, 256, 2, 64, 32, seed=4)
    lens = [100, 0, 33]
    q = np.random.default_rng(7).standard_normal((3, 4, 64)).astype(np.float32)
    want = check_attention(c, q, lens)
    weight = np.full((c.phys, 2, 32), 0.5, np.float32)
    for b, n in enumerate(lens):
        blk, off = c.places(b, 256)
        blk, off = torch.from_numpy(blk[n:].astype(np.int64)).cuda(), torch.from_numpy(off[n:]).cuda()
        for g, x in ((c.kg, c.k), (c.vg, c.v)):
            g[blk, :, off] = float("nan")
            x[blk, :, off] = 255
    assert np.array_equal(want, check_attention(c, q, lens))
    w = dev(weight)
    out = F().kv4Attention(dev(q), *c.args(), dev(np.array(lens, np.int32)), table=c.dtable, weight=w)
    assert np.isfinite(out.cpu().numpy()).all()
    w = w.cpu().numpy()
    for b, n in enumerate(lens):
        blk, off = c.places(b, 256)
        assert (w[blk[n:], :, off[n:]] == 0.5).all()
        assert (w[blk[:n], :, off[:n]] > 0.5).all()


def test_lengths_outside_the_capacity_are_clamped():
    c = Cache(2, 96, 2, 64, 32)
    q = np.random.default_rng(8).standard_normal((2, 2, 64)).astype(np.float32)
    got = F().kv4Attention(dev(q), *c.args(), dev(np.array([1000, -5], np.int32)), table=c.dtable)
    check_attention(c, q, [96, 0], got=got)


def test_a_bad_row_and_a_bad_page_give_nan_where_they_are_read():
    c = Cache(3, 128, 2, 64, 32, seed=5)
    q = np.random.default_rng(9).standard_normal((3, 4, 64)).astype(np.float32)
    lens = dev(np.array([128, 128, 90], np.int32))
    c.kg[c.table[0, 1], 0, 3] = float("nan")          # one row of kv head 0 of sequence 0
    c.vg[c.table[2, 0], 1, 7] = float("nan")          # one of kv head 1 of sequence 2
    t = c.dtable.clone()
    t[1, 2] = c.phys                                   # a page that does not exist
    w = torch.zeros(c.phys, 2, 32, device="cuda")
    out = F().kv4Attention(dev(q), *c.args(), lens, table=t, weight=w).cpu().numpy()
    nan = np.isnan(out)
    assert nan[0, :2].all() and not nan[0, 2:].any()
    assert nan[1].all()
    assert nan[2, 2:].all() and not nan[2, :2].any()
    t[1, 2] = -7
    assert np.isnan(F().kv4Attention(dev(q), *c.args(), lens, table=t).cpu().numpy()[1]).all()
    # the page past the length is never looked at
    short = dev(np.array([10, 64, 10], np.int32))
    assert np.isfinite(F().kv4Attention(dev(q), *c.args(), short, table=t).cpu().numpy()[1]).all()


def test_attention_reads_strided_queries_and_writes_into_out():
    c = Cache(3, 300, 4, 64, 0, seed=6)
    rng = np.random.default_rng(3)
    wide = rng.standard_normal((3, 20 * 64 + 3)).astype(np.float32)
    d = dev(wide)
    q = torch.as_strided(d, (3, 12, 64), (wide.shape[1], 64, 1))
    out = torch.full((3, 12 * 64), 7.0, device="cuda")
    lens = [300, 17, 0]
    got = F().kv4Attention(q, *c.args(), dev(np.array(lens, np.int32)), out=out)
    assert got is out
    check_attention(c, wide[:, :12 * 64].reshape(3, 12, 64), lens, got=out.view(3, 12, 64))


def test_attention_past_four_gigabytes_of_codes():
    """The last block of a cache whose codes pass 2^32 bytes (and 2^31 rows' bytes)."""
    nKV, dH, bs = 8, 256, 1024
    blocks = (1 << 32) // (nKV * bs * 128) + 2
    c = Cache(1, bs, nKV, dH, bs, seed=7, shuffle=False)
    k = torch.empty(blocks, nKV, bs, 128, dtype=U8, device="cuda")
    v = torch.empty_like(k)
    kg = torch.empty(blocks, nKV, bs, 2, dtype=BF, device="cuda")
    vg = torch.empty_like(kg)
    for big, small in ((k, c.k), (v, c.v), (kg, c.kg), (vg, c.vg)):
        big[-1] = small[0]
    q = np.random.default_rng(4).standard_normal((1, 8, dH)).astype(np.float32)
    table = torch.tensor([[blocks - 1]], dtype=I32, device="cuda")
    got = F().kv4Attention(dev(q), k, kg, v, vg, dev(np.array([1000], np.int32)), table=table)
    check_attention(c, q, [1000], got=got)


def test_attention_of_more_heads_than_an_int_counts():
    """65535 sequences of 32784 q heads of 2 (2^31 of them and more, 17 GB of q), all
    but the first empty, whose segments the runs' ends cut."""
    B, nKV, dH, n = 65535, 2049, 2, 13 * 128
    c = Cache(1, n, nKV, dH, n, seed=24, shuffle=False)
    nH = 16 * nKV
    q = torch.zeros(B, nH, dH, device="cuda")
    q0 = np.random.default_rng(25).standard_normal((nH, dH)).astype(np.float32)
    q[0] = dev(q0)
    lens = torch.zeros(B, dtype=I32, device="cuda")
    lens[0] = n
    out = torch.full((B, nH, dH), float("nan"), device="cuda")
    F().kv4Attention(q, *c.args(), lens, table=torch.zeros(B, 1, dtype=I32, device="cuda"), out=out)
    got = out[0].cpu().numpy()
    assert float(out[1:].abs().max()) == 0
    K, V = [np.stack([c.rows(w, 0, h, n) for h in range(nKV)]) for w in range(2)]
    s = np.einsum("hgd,hnd->hgn", q0.reshape(nKV, 16, dH).astype(np.float64), K) / math.sqrt(dH)
    p = np.exp(s - s.max(-1, keepdims=True))
    want = np.einsum("hgn,hnd->hgd", p / p.sum(-1, keepdims=True), V).reshape(nH, dH)
    assert np.abs(got - want).max() <= tolerance(c, q0[None], 1 / math.sqrt(dH))
    del q, out
    torch.cuda.empty_cache()


def test_a_long_sequence():
    c = Cache(1, 70001, 1, 32, 0, seed=8)
    q = np.random.default_rng(10).standard_normal((1, 4, 32)).astype(np.float32)
    weight = np.zeros((1, 1, 70001), np.float32)
    check_attention(c, q, [70001], weight=weight)


def test_graphs_and_streams():
    """Two captured calls replayed on two streams at once, each with its own
    workspace, give the eager bits; so does a call on another stream."""
    fw = F()
    c = Cache(4, 2000, 2, 64, 0, seed=11)
    rng = np.random.default_rng(12)
    qs = [dev(rng.standard_normal((4, 8, 64)).astype(np.float32)) for _ in range(2)]
    lens = dev(np.array([2000, 1500, 3, 0], np.int32))
    want = [fw.kv4Attention(q, *c.args(), lens).clone() for q in qs]
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q, s in zip(qs, side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(fw.kv4Attention(q, *c.args(), lens))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
            o.zero_()
        torch.cuda.synchronize()
    with torch.cuda.stream(side[0]):
        got = fw.kv4Attention(qs[1], *c.args(), lens)
    torch.cuda.synchronize()
    assert torch.equal(got, want[1])


# ------------------------------------------------------------------ put, values
def put_case(B, T, nH, nKV, dH, block, theta, seed=0, x=None, ld_extra=0, cap=64):
    rng = np.random.default_rng(seed)
    heads = nH + 2 * nKV
    x = rng.standard_normal((B * T, heads * dH)).astype(np.float32) if x is None else x
    c = Cache(B, cap, nKV, dH, block, seed=seed + 1)
    slots = rng.integers(0, cap - T + 1, B).astype(np.int32)
    pos = (slots + rng.integers(0, 5000, B)).astype(np.int32)
    wide = np.full((B * T, heads * dH + ld_extra), 3.5, np.float32)
    wide[:, :heads * dH] = x
    d = dev(wide)
    return x, c, slots, pos, d


@pytest.mark.parametrize("B,T,nH,nKV,dH,block", [(3, 1, 4, 2, 64, 16), (2, 9, 12, 4, 64, 0), (1, 40, 3, 3, 80, 7),
                                                 (2, 17, 2, 1, 256, 8), (5, 1, 1, 1, 2, 3), (2, 8, 6, 2, 34, 0),
                                                 (2, 3, 0, 5, 128, 64), (1, 5, 4, 4, 96, 5), (2, 2, 2, 2, 160, 16)])
@pytest.mark.parametrize("theta,extra", [(10000.0, 0), (0.0, 4), (500000.0, 3)])
def test_put_and_values(B, T, nH, nKV, dH, block, theta, extra):
    fw = F()
    x, c, slots, pos, d = put_case(B, T, nH, nKV, dH, block, theta, seed=dH + T, ld_extra=extra)
    heads = nH + 2 * nKV
    weight = torch.full((c.phys, nKV, c.bs), 9.0, device="cuda")
    at = torch.full((c.phys, nKV, c.bs), -3, dtype=I32, device="cuda")
    before = [t.clone() for t in (*c.args(), weight, at)]
    fw.kv4Put(d[:, :heads * dH], nH, dev(pos), dev(slots), *c.args(), T=T, theta=theta, table=c.dtable, weight=weight,
              pos=at)
    K, V = fw.kv4Values(*c.args(), dH, dev(slots), T, table=c.dtable)
    got = d.cpu().numpy()
    K, V = K.cpu().numpy(), V.cpu().numpy()
    rb = R.row_bytes(dH)
    touched = np.zeros((c.phys, c.bs), bool)
    for b in range(B):
        for t in range(T):
            r = x[b * T + t].reshape(heads, dH)
            turned = R.rope(r[:nH + nKV], int(pos[b]) + t, theta) if theta else r[:nH + nKV]
            q = got[b * T + t, :nH * dH].reshape(nH, dH)
            assert np.abs(q - turned[:nH]).max(initial=0) <= 1e-7 * np.abs(r).max()
            assert np.array_equal(got[b * T + t, nH * dH:heads * dH], x[b * T + t, nH * dH:])
            j = int(slots[b]) + t
            blk, off = c.table[b, j // c.bs], j % c.bs
            touched[blk, off] = True
            for rows, codes, grid, read in ((turned[nH:], c.k, c.kg, K), (r[nH + nKV:], c.v, c.vg, V)):
                code, step, base = R.quantize(rows)
                assert np.array_equal(codes[blk, :, off].cpu().numpy(), R.pack(code, rb)), (b, t)
                gr = grid[blk, :, off].float().cpu().numpy()
                assert np.array_equal(gr[:, :1], step.astype(np.float32)) and np.array_equal(gr[:, 1:], base.astype(np.float32))
                assert np.array_equal(read[b, t], R.values(code, step, base))
            assert (weight[blk, :, off] == 0).all() and (at[blk, :, off] == int(pos[b]) + t).all()
    if extra:
        assert (got[:, heads * dH:] == 3.5).all()
    keep = torch.from_numpy(~touched).cuda()[:, None].expand(-1, nKV, -1)
    for a, b_ in zip((*c.args(), weight, at), before):
        assert torch.equal(a[keep].view(torch.int8), b_[keep].view(torch.int8))


def test_put_of_unusual_rows():
    """Constant, zero, huge, subnormal, tied and non-finite rows."""
    fw = F()
    dH = 32
    rows = np.random.default_rng(1).standard_normal((14, dH)).astype(np.float32)
    rows[0] = 0.1
    rows[1] = 0
    rows[2] *= 1e37
    rows[3] *= 1e-39
    rows[4] = np.arange(dH) * 0.5            # quotients on halves
    rows[5] = -np.arange(dH) * 1.5
    rows[6, 3] = np.inf
    rows[7, 5] = np.nan
    rows[8, 1] = -np.inf
    rows[9, 0] = 2.0 ** 127
    rows[10, 0] = -np.nextafter(np.float32(2.0 ** 127), np.float32(0))
    rows[11] = 1000 + rows[11] * 1e-3
    rows[12] = np.where(np.arange(dH) % 2, 3.0, -0.0)
    rows[13] *= 1e-30
    n = len(rows)
    x = np.concatenate([rows, rows[::-1]], 1)
    k = torch.zeros(n, 1, 1, 16, dtype=U8, device="cuda")
    kg = torch.zeros(n, 1, 1, 2, dtype=BF, device="cuda")
    v, vg = torch.zeros_like(k), torch.zeros_like(kg)
    z = torch.zeros(n, dtype=I32, device="cuda")
    fw.kv4Put(dev(x), 0, z, z, k, kg, v, vg, theta=0.0)
    K, V = fw.kv4Values(k, kg, v, vg, dH, z, 1)
    code, step, base = R.quantize(rows)
    want = R.values(code, step, base)
    bad = ~np.isfinite(want)
    assert bad.all(1).tolist() == [i in (6, 7, 8, 9) for i in range(n)] and (bad.any(1) == bad.all(1)).all()
    assert np.array_equal(k.cpu().numpy()[:, 0, 0][~bad[:, 0]], R.pack(code, 16)[~bad[:, 0]])
    assert np.array_equal(K.cpu().numpy()[:, 0, 0], want, equal_nan=True)
    assert np.array_equal(V.cpu().numpy()[:, 0, 0], want[::-1], equal_nan=True)


def test_put_of_rows_as_wide_as_the_cache_takes():
    """From just above -2^127 to just below 2^127: the difference of the ends rounds to
    2^128 in fp32, the grid's step is finite."""
    fw = F()
    dH, top = 32, np.nextafter(np.float32(2.0 ** 127), np.float32(0))
    rows = (np.random.default_rng(3).uniform(-1, 1, (6, dH)) * 2.0 ** 126).astype(np.float32)
    for i, (lo, hi) in enumerate(((-top, top), (-top, 0), (0, top), (-top * 0.99, top), (-top, top * 0.99), (-2.0 ** 126, top))):
        rows[i, 5], rows[i, 9] = lo, hi
    n = len(rows)
    k = torch.zeros(n, 1, 1, 16, dtype=U8, device="cuda")
    kg = torch.zeros(n, 1, 1, 2, dtype=BF, device="cuda")
    v, vg = torch.zeros_like(k), torch.zeros_like(kg)
    z = torch.zeros(n, dtype=I32, device="cuda")
    fw.kv4Put(dev(np.concatenate([rows, rows], 1)), 0, z, z, k, kg, v, vg, theta=0.0)
    K, _ = fw.kv4Values(k, kg, v, vg, dH, z, 1)
    code, step, base = R.quantize(rows)
    assert np.isfinite(step).all()
    assert np.array_equal(k.cpu().numpy()[:, 0, 0], R.pack(code, 16))
    with np.errstate(over="ignore"):
        assert np.array_equal(K.cpu().numpy()[:, 0, 0], R.values(code, step, base))


def test_put_outside_the_cache_changes_nothing():
    fw = F()
    x, c, _, _, d = put_case(5, 2, 2, 2, 64, 16, 1e4, seed=4)
    slots = np.array([63, -2, 70, 4, 2 ** 31 - 1], np.int32)      # only slot 63 of the first, 4 and 5 of the fourth
    pos = np.array([5, 5, 5, -1, 5], np.int32)                    # the fourth's first token has position -1
    t = c.dtable.clone()
    before, q0 = [a.clone() for a in c.args()], d.clone()
    fw.kv4Put(d, 2, dev(pos), dev(slots), *c.args(), T=2, table=t)
    hit = {(c.table[0, 3], 15), (c.table[3, 0], 5)}
    for a, b in zip(c.args(), before):
        for blk in range(c.phys):
            for off in range(16):
                assert torch.equal(a[blk, :, off].view(torch.int8), b[blk, :, off].view(torch.int8)) != ((blk, off) in hit)
    same = [torch.equal(d[i], q0[i]) for i in range(10)]
    # (the fourth's second token stands at position 0, whose rotation is the identity)
    assert same == [False, True, True, True, True, True, True, True, True, True]
    # the last position of int32 is one, the next is none
    before, q0 = [a.clone() for a in c.args()], d.clone()
    pos = np.full(5, 2 ** 31 - 1, np.int32)
    fw.kv4Put(d, 2, dev(pos), dev(np.full(5, 8, np.int32)), *c.args(), T=2, table=t)
    hit = {(c.table[b, 0], 8) for b in range(5)}
    for a, b in zip(c.args(), before):
        for blk in range(c.phys):
            for off in range(16):
                assert torch.equal(a[blk, :, off].view(torch.int8), b[blk, :, off].view(torch.int8)) != ((blk, off) in hit)
    assert [torch.equal(d[i], q0[i]) for i in range(10)] == [False, True] * 5
    t.fill_(c.phys + 3)
    before, q0 = [a.clone() for a in c.args()], d.clone()
    fw.kv4Put(d, 2, dev(np.full(5, 3, np.int32)), dev(np.zeros(5, np.int32)), *c.args(), T=2, table=t)
    assert torch.equal(d, q0) and all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(c.args(), before))
    K, V = fw.kv4Values(*c.args(), 64, dev(np.array([0, 62, 63, -1, 5], np.int32)), 2, table=c.dtable)
    nan = torch.isnan(K).all(-1).all(-1).cpu().numpy()
    assert nan.tolist() == [[False, False], [False, False], [False, True], [True, False], [False, False]]
    assert torch.equal(torch.isnan(V), torch.isnan(K))


# ------------------------------------------------------------------ evict
def check_evict(L, B, nKV, dH, cap, block, lens, budget, recent, weight=None, pos=None, seed=0):
    fw = F()
    rng = np.random.default_rng(seed)
    cs = [Cache(B, cap, nKV, dH, block, seed=seed) for _ in range(1)]
    c = cs[0]
    shape = (L, c.phys, nKV, c.bs)
    rb = R.row_bytes(dH)
    host = [rng.integers(0, 256, (*shape, rb)).astype(np.uint8) for _ in range(2)]
    grid = [rng.integers(0, 1 << 15, (*shape, 2)).astype(np.int16) for _ in range(2)]
    w = rng.exponential(1, shape).astype(np.float32) if weight is None else weight(shape, rng)
    p = rng.permutation(int(np.prod(shape))).reshape(shape).astype(np.int32) if pos is None else pos(shape, rng)
    d = [dev(host[0]), dev(grid[0]).view(BF), dev(host[1]), dev(grid[1]).view(BF), dev(w), dev(p)]
    dl = dev(np.array(lens, np.int32))
    new = fw.kv4Evict(*d, dl, budget, recent, table=c.dtable)
    assert new.cpu().tolist() == [min(max(n, 0), cap, budget) if n > budget or n < 0 else n for n in lens]
    want = [host[0].copy(), grid[0].copy(), host[1].copy(), grid[1].copy(), w.copy(), p.copy()]
    for l in range(L):
        for b, n in enumerate(lens):
            n = max(0, min(n, c.mb * c.bs))
            blk, off = c.places(b, n)
            for h in range(nKV):
                dst, src = R.evict(w[l, blk, h, off], p[l, blk, h, off], n, budget, recent)
                for x in want:
                    x[l, blk[dst], h, off[dst]] = x[l, blk[src], h, off[src]].copy()
    for got, x in zip(d, want):
        g = got.view(torch.int16) if got.dtype == BF else got
        assert np.array_equal(g.cpu().numpy(), x, equal_nan=x.dtype.kind == "f")
    return d, new


@pytest.mark.parametrize("L,B,nKV,dH,cap,block,lens,budget,recent", [
    (2, 3, 2, 64, 128, 16, [128, 100, 20], 30, 8),
    (1, 2, 1, 96, 50, 7, [50, 11], 10, 10),
    (3, 1, 4, 16, 300, 0, [257], 256, 0),
    (1, 4, 2, 256, 64, 64, [64, 1, 0, 33], 1, 0),
    (1, 2, 2, 128, 64, 0, [64, 60], 1, 1),
    (2, 2, 3, 48, 2100, 100, [2100, 2099], 1500, 333),
    (1, 1, 2, 32, 5000, 0, [4999], 1023, 1023),
    (1, 2, 1, 64, 64, 16, [64, 40], 100, 50),
])
def test_evict(L, B, nKV, dH, cap, block, lens, budget, recent):
    check_evict(L, B, nKV, dH, cap, block, lens, budget, recent, seed=cap + budget)


def test_evict_ties_nan_infinite_and_negative_weights():
    def ties(shape, rng):
        return rng.integers(0, 3, shape).astype(np.float32)

    def odd(shape, rng):
        w = rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.0, 1e-45, 3.0], np.float32), shape)
        return w

    for weight in (ties, odd, lambda s, r: np.zeros(s, np.float32)):
        check_evict(1, 2, 3, 32, 1200, 50, [1200, 77], 64, 5, weight=weight, seed=3)
    # positions that repeat: more protected slots than the budget
    check_evict(1, 1, 2, 32, 300, 0, [300], 20, 20, pos=lambda s, r: r.integers(0, 3, s).astype(np.int32))
    # positions at the ends of their type
    check_evict(1, 1, 1, 32, 300, 0, [300], 20, 20,
                pos=lambda s, r: r.choice(np.array([-2 ** 31, 2 ** 31 - 1, 0], np.int32), s))


def test_evict_longer_than_shared_memory_holds():
    from forgellm import _lib
    assert _lib.lib().fcu_kv4_evict_work is not None
    check_evict(1, 2, 1, 32, 60000, 0, [60000, 41000], 30001, 1000, seed=5)


def test_evict_leaves_a_sequence_with_a_bad_page():
    fw = F()
    c = Cache(2, 64, 2, 64, 16, seed=1)
    shape = (1, c.phys, 2, 16)
    w, p = torch.rand(shape, device="cuda"), torch.arange(int(np.prod(shape)), device="cuda", dtype=I32).view(shape)
    t = c.dtable.clone()
    t[0, 1] = 99
    a = [x[None].clone() for x in c.args()]
    before = [x.clone() for x in (*a, w, p)]
    new = fw.kv4Evict(*a, w, p, dev(np.array([64, 64], np.int32)), 8, 4, table=t)
    assert new.cpu().tolist() == [64, 8]
    for x, y in zip((*a, w, p), before):
        for i in range(4):
            blk = int(c.table[0, i])
            assert torch.equal(x[0, blk].view(torch.int8), y[0, blk].view(torch.int8))


def test_python_refusals():
    fw = F()
    c = Cache(2, 64, 2, 64, 16)
    q = torch.zeros(2, 4, 64, device="cuda")
    lens = torch.zeros(2, dtype=I32, device="cuda")
    k, kg, v, vg = c.args()
    ok = dict(table=c.dtable)
    bad = [
        lambda: fw.kv4Attention(q.half(), k, kg, v, vg, lens, **ok),
        lambda: fw.kv4Attention(q.transpose(1, 2), k, kg, v, vg, lens, **ok),
        lambda: fw.kv4Attention(q, k, kg, v, vg, lens.long(), **ok),
        lambda: fw.kv4Attention(q, k, kg, v, vg, lens[:1], **ok),
        lambda: fw.kv4Attention(q, k.transpose(0, 1), kg, v, vg, lens, **ok),
        lambda: fw.kv4Attention(q, k, kg.half(), v, vg, lens, **ok),
        lambda: fw.kv4Attention(q, k, kg, v[:-1], vg, lens, **ok),
        lambda: fw.kv4Attention(q, k, kg, v, vg, lens, table=c.dtable[:1]),
        lambda: fw.kv4Attention(q, k, kg, v, vg, lens, table=c.dtable.long()),
        lambda: fw.kv4Attention(q, k, kg, v, vg, lens, weight=torch.zeros(1, device="cuda"), **ok),
        lambda: fw.kv4Attention(q.cpu(), k, kg, v, vg, lens, **ok),
        lambda: fw.kv4Attention(q, k, kg, v, vg, lens.cpu(), **ok),
        lambda: fw.kv4Attention(torch.zeros(2, 4, 96, device="cuda"), k, kg, v, vg, lens, **ok),
        lambda: fw.kv4Attention(torch.zeros(3, 4, 64, device="cuda"), k, kg, v, vg, torch.zeros(3, dtype=I32, device="cuda")),
        lambda: fw.kv4Attention(q, k, kg, v, vg, lens, out=torch.zeros(3, device="cuda"), **ok),
        lambda: fw.kv4Put(torch.zeros(2, 100, device="cuda"), 4, lens, lens, k, kg, v, vg, **ok),
        lambda: fw.kv4Put(torch.zeros(1, 512, device="cuda").expand(2, -1), 4, lens, lens, k, kg, v, vg, **ok),
        lambda: fw.kv4Put(torch.zeros(2, 512, device="cuda"), 4, lens, lens[:1], k, kg, v, vg, **ok),
        lambda: fw.kv4Put(torch.zeros(2, 512, device="cuda"), 4, lens, lens, k, kg, v, vg, theta=-1.0, **ok),
        lambda: fw.kv4Values(k, kg, v, vg, 63, lens, 1, **ok),
        lambda: fw.kv4Evict(k[None], kg[None], v[None], vg[None], None, None, lens, 4, 2, **ok),
        lambda: fw.kv4Attention(q, None, kg, v, vg, lens, **ok),
        lambda: fw.kv4Values(k, kg, v, None, 64, lens, 1, **ok),
        lambda: fw.kv4Put(torch.zeros(2, 512, device="cuda"), 4, lens, lens, k.cpu().numpy(), kg, v, vg, **ok),
        lambda: fw.kv4Evict(k, kg, v, vg, torch.zeros(1, device="cuda"), lens, lens, 4, 2, **ok),
        lambda: fw.kv4Evict(None, kg, v, vg, torch.zeros(1, device="cuda"), lens, lens, 4, 2, **ok),
        lambda: fw.kv4Evict(k[None], kg[None], v[None], vg[None], k, k, lens, 2 ** 32 + 4, 2, **ok),
        lambda: fw.cacheReorder([None], lens.view(1, 2), lens),
        lambda: fw.cacheReorder([lens], lens.view(1, 2), lens),
        lambda: fw.QuantKVCache(1, 16, 1, 8, batch=2, blockSize=16, table=[[0], [0]], physBlocks=1, track=True),
        lambda: fw.QuantKVCache(1, 16, 1, 8, batch=2).reorder([[0.0, 1.0]]),
        lambda: fw.QuantKVCache(1, 16, 1, 8, batch=2).reorder(torch.tensor([[0, 2]], device="cuda")),
        lambda: fw.QuantKVCache(1, 16, 1, 7),
        lambda: fw.QuantKVCache(1, 16, 1, 8, blockSize=4, table=[[0, 1, 2, 9]], physBlocks=4),
        lambda: fw.QuantKVCache(1, 16, 1, 8).evict(4, 2),
        lambda: fw.QuantKVCache(1, 16, 1, 8, batch=2, blockSize=16, table=[[0], [0]], physBlocks=1).reorder([[0, 0]]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")
    with pytest.raises(fw.ForgeCUError):
        fw.kv4Attention(torch.zeros(2, 3, 64, device="cuda"), k, kg, v, vg, lens, **ok)
    with pytest.raises(fw.ForgeCUError):
        fw.kv4Attention(q, k, kg, v, vg, lens, out=q, **ok)
    with pytest.raises(fw.ForgeCUError):
        x = torch.zeros(1, 2, 4, 8, device="cuda")
        fw.cacheReorder([x, x], lens.view(1, 2), lens)


def test_two_host_threads():
    """Calls of two kernels each from two threads, each on a stream of its own."""
    import threading
    fw = F()
    rng = np.random.default_rng(31)
    lens = dev(np.array([900, 0, 130, 1024], np.int32))
    cs = [Cache(4, 1024, 2, 64, 64, seed=i) for i in range(2)]
    qs = [dev(rng.standard_normal((4, 6, 64)).astype(np.float32)) for _ in cs]
    want = [fw.kv4Attention(q, *c.args(), lens, table=c.dtable) for q, c in zip(qs, cs)]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(100):
                out = fw.kv4Attention(qs[i], *cs[i].args(), lens, table=cs[i].dtable)
                got[i].append(out.clone())
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, w in zip(got, want):
        assert len(g) == 100 and all(torch.equal(x, w) for x in g)


def test_attention_of_more_sequences_than_a_block_has_threads():
    """300 sequences, most of them short or empty, and one long."""
    rng = np.random.default_rng(20)
    lens = rng.choice([0, 1, 2, 30, 70], 300)
    lens[170] = 700
    lens[299] = 65
    c = Cache(300, 704, 1, 16, 64, seed=12)
    q = rng.standard_normal((300, 3, 16)).astype(np.float32)
    check_attention(c, q, lens.tolist(), weight=np.zeros((c.phys, 1, 64), np.float32))
    check_attention(c, q, [0] * 300)
