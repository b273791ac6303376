"""Beam search on the GPU, and generation over the 4-bit cache as a whole.

Tolerances: selections (tokens, parents, done) are equal to the 64-bit
restatement's: the inputs are fixed and none of their candidates is closer to
another than 1e-6 unless they are equal.  Scores: each is a double rounded to
fp32 over a log-sum-exp summed in fp32, whose relative error over V terms summed
per thread, warp and slice is below 2^-18: 2^-23 * |score| + 2^-18."""
import numpy as np
import pytest

import kv4_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

I32 = torch.int32


def F():
    import forgellm
    return forgellm


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def check_beam(x, scores, done, eos, pad=0):
    """x [B, W, V]."""
    B, W, V = x.shape
    wide = np.full((B * W, V + pad), np.nan, np.float32)
    wide[:, :V] = x.reshape(B * W, V)
    got = F().beamStep(dev(wide)[:, :V], dev(scores.astype(np.float32)).view(-1), dev(done).view(-1), W, eos)
    s, t, p, d = [g.cpu().numpy() for g in got]
    ws, wt, wp, wd = R.beam(x, scores.astype(np.float32), done, W, eos)
    assert np.array_equal(t, wt) and np.array_equal(p, wp), (t, wt, p, wp)
    assert np.array_equal(d, wd)
    fin = np.isfinite(ws)
    assert np.array_equal(fin, np.isfinite(s)) and (s[~fin] == -np.inf).all()
    assert (np.abs(s[fin] - ws[fin]) <= 2.0 ** -23 * np.abs(ws[fin]) + 2.0 ** -18).all()


@pytest.mark.parametrize("B,W,V", [(1, 1, 1), (1, 4, 2), (2, 3, 5), (3, 4, 64), (2, 8, 1000), (1, 32, 4097),
                                   (5, 5, 2048), (2, 16, 9001), (1, 4, 32000), (40, 8, 700), (1, 32, 70001)])
def test_beam_step(B, W, V):
    rng = np.random.default_rng(B * 1000 + W + V)
    x = (rng.standard_normal((B, W, V)) * 3).astype(np.float32)
    scores = -rng.random((B, W)) * 5
    done = np.zeros((B, W), bool)
    eos = min(2, V - 1)
    check_beam(x, scores, done, eos)
    check_beam(x, scores, rng.random((B, W)) < 0.5, eos, pad=3)
    check_beam(x, scores, np.ones((B, W), bool), eos)
    first = np.where(np.arange(W) > 0, -np.inf, 0.0) * np.ones((B, 1))
    check_beam(x, first, done, eos)


def test_beam_step_ties_go_to_the_lowest_beam_and_token():
    for V in (7, 3000, 9000):
        x = np.zeros((2, 4, V), np.float32)
        check_beam(x, np.zeros((2, 4)), np.zeros((2, 4), bool), 1)
        x[:, :, V // 2:] = 1.5
        x[:, 1, V - 1] = -0.0
        check_beam(x, np.zeros((2, 4)), np.zeros((2, 4), bool), 1)
        x = np.random.default_rng(V).integers(0, 3, (2, 4, V)).astype(np.float32)
        # log-sum-exps differ between beams, so only a beam's own tokens tie
        check_beam(x, np.array([[0.0, -1.0, -2.0, -3.0]] * 2), np.zeros((2, 4), bool), 1)


def test_beam_step_ties_among_many_tiles():
    """Warps that run ahead of one another meet equal logits again and again."""
    rng = np.random.default_rng(8)
    x = rng.integers(0, 6, (6, 16, 70001)).astype(np.float32)
    x[1] = np.where(x[1] == 5, 0, 1)           # two values
    x[2, :, 40000:] = 6                        # the largest all come late
    x[3, :, :69990] = -np.inf                  # few are allowed at all
    x[4] = 0
    scores = -np.arange(16.0) * np.ones((6, 1))
    done = np.zeros((6, 16), bool)
    for _ in range(3):
        check_beam(x, scores, done, 2)
    done[:, ::3] = True
    check_beam(x, scores, done, 2)


def test_beam_step_ascending_logits():
    """The worst order for a running selection: every tile beats the last."""
    x = np.tile(np.arange(20000, dtype=np.float32) / 1000, (1, 32, 1)) + np.arange(32, dtype=np.float32)[None, :, None] * 0
    check_beam(x, -np.arange(32.0)[None] * 0.01, np.zeros((1, 32), bool), 2)
    check_beam(x[:, :, ::-1].copy(), -np.arange(32.0)[None] * 0.01, np.zeros((1, 32), bool), 2)


def test_beam_step_banned_and_unusable_rows():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((4, 4, 500)).astype(np.float32)
    x[0, :, :] = -np.inf                      # nothing allowed at all
    x[0, 2, [7, 400]] = 1.0                   # but two tokens of one beam
    x[1, 0, 33] = np.nan
    x[1, 1, 44] = np.inf
    x[1, 2, :] = -np.inf
    x[2, :, 3:] = -np.inf
    x[3, 0, :499] = -np.inf
    scores = np.zeros((4, 4)) - rng.random((4, 4))
    scores[3, 1:] = -np.inf
    check_beam(x, scores, np.zeros((4, 4), bool), 2)
    done = np.zeros((4, 4), bool)
    done[:, 1] = True
    check_beam(x, scores, done, 2)
    scores[2, 1] = np.nan
    check_beam(x, scores, done, 2)
    x[:] = np.nan
    check_beam(x, scores, np.zeros((4, 4), bool), 2)


@pytest.mark.parametrize("V", [64, 65, 513, 2049, 9001])
def test_beam_step_a_nan_wherever_it_lies(V):
    """One NaN makes its beam unusable, whatever the logits beside it are: alone at
    the end, with its whole 16-byte piece, beside banned tokens only, in a run of
    NaN at the start, on rows that start at any 4 bytes."""
    rng = np.random.default_rng(V)
    none = np.zeros((4, 4), bool)
    for pad in (0, 1, 2, 3):
        x = rng.standard_normal((4, 4, V)).astype(np.float32)
        x[0, 0, V - 1] = np.nan
        x[0, 2, :4] = np.nan
        x[1, 0, :] = -np.inf
        x[1, 0, V // 2] = np.nan
        x[1, 1, :64] = -np.inf
        x[1, 1, 17] = np.nan
        x[2, 1, :min(512, V - 1)] = np.nan
        x[2, 3, 60] = np.nan
        x[2, 3, 61:] = -np.inf
        x[3, 0, V // 2:] = np.nan
        x[3, 1, ::2] = -np.inf
        x[3, 1, 1::2] = np.where(np.arange(1, V, 2) < V // 2, np.nan, 1.0)
        check_beam(x, -rng.random((4, 4)), none, 2, pad=pad)


def test_beam_step_logits_at_the_ends_of_their_type():
    """Tokens and whole rows masked with the type's lowest value, and rows of its
    largest: all of them finite, so their log-softmax is (a row of equal logits
    offers each token at its score - log V)."""
    top = float(np.finfo(np.float32).max)
    rng = np.random.default_rng(3)
    for V in (4, 70, 5000):
        x = rng.standard_normal((5, 4, V)).astype(np.float32)
        x[0, :, 3:] = -top                      # tokens of every beam
        x[1, :3] = -top                         # whole beams
        x[2] = -top                             # all of them
        x[3, 0] = top
        x[3, 1] = np.float32(-3e38)
        x[3, 2, 1:] = -top
        x[4, 0] = np.where(np.arange(V) == 2, np.float32(2.5e38), np.float32(1e38))
        x[4, 1] = np.where(np.arange(V) % 3 == 1, -np.float32(top), -np.inf)
        done = np.zeros((5, 4), bool)
        for order in (1, -1):
            scores = -np.arange(4.0)[::order] * np.ones((5, 1)) / 8
            got = F().beamStep(dev(x.reshape(20, V)), dev(scores.astype(np.float32)).view(-1), dev(done).view(-1), 4, 2)
            s, t, p, d = [g.cpu().numpy() for g in got]
            # a log-softmax does not change with the row's offset; in 64 bits it is lost beside one of 2^128
            y = x.astype(np.float64)
            y -= y.max(-1, keepdims=True)
            ws, wt, wp, wd = R.beam(y, scores, done, 4, 2)
            assert np.array_equal(t, wt) and np.array_equal(p, wp) and np.array_equal(d, wd), (V, order)
            assert (np.abs(s - ws) <= 2.0 ** -23 * np.abs(ws) + 2.0 ** -18).all(), (V, order)


def test_beam_step_ties_that_doubles_make():
    """Logits that differ where their scores do not: below a score of -1e30, and
    tiny ones beside a log-sum-exp of about 8.  The lowest tokens are first, those
    that are not among the largest logits too."""
    rng = np.random.default_rng(21)
    done = np.zeros((4, 4), bool)
    for V in (3, 40, 3000):
        x = rng.standard_normal((4, 4, V)).astype(np.float32)
        x[1] = rng.random((4, V)).astype(np.float32) * np.float32(1e-20)
        x[2] = np.where(rng.random((4, V)) < 0.2, 1.0, x[1])
        x[2, 0, 0] = -np.inf
        x[3, 1] = -np.arange(V, dtype=np.float32)[::-1]
        scores = np.array([[-1e30] * 4, [0, -1, -2, -3], [-0.5, 0, -1, -2], [-1e25, -1e20, -1e30, -1e30]])
        check_beam(x, scores, done, 2)
        x[0, :, 0] = np.nan
        x[0, 2] = -np.inf
        x[0, 2, 1:] = 0
        check_beam(x, scores, done, 2, pad=2)
        d = done.copy()
        d[:, 0] = True
        check_beam(x, scores, d, 1)


@pytest.mark.parametrize("W", [1, 4, 9])
@pytest.mark.parametrize("V", [40, 3001, 20000])
def test_beam_step_ties_spread_over_a_row(W, V):
    """A few tokens that tie in double lie anywhere in a row, the largest of them last;
    some larger ones are before them; other beams take all or a part of the places."""
    rng = np.random.default_rng(100 * W + V)
    B = 12
    x = (-4 - rng.random((B, W, V))).astype(np.float32)
    for b in range(B):
        for w in range(W):
            at = np.sort(rng.choice(V, 14, replace=False))
            x[b, w, at] = np.arange(1, 15, dtype=np.float32) * np.float32(1e-21)      # rises with the token
            larger = b % 4
            x[b, w, rng.choice(at, larger, replace=False)] = 1 + np.arange(larger)
    x[7] -= x[7].max(-1, keepdims=True)
    scores = np.where(np.arange(B)[:, None] % 3 == 0, -np.arange(W) * 0.01, -np.arange(W) * 3.0)
    done = np.zeros((B, W), bool)
    check_beam(x, scores, done, 2)
    check_beam(x, scores[:, ::-1].copy(), done, 2, pad=3)


@pytest.mark.parametrize("L,B,W,heads,bs,mb,unit,table", [
    (2, 2, 4, 2, 16, 4, 32, True), (1, 3, 2, 1, 100, 1, 768, False), (3, 1, 5, 3, 7, 5, 4, True),
    (1, 2, 32, 2, 5, 3, 12, False), (2, 1, 3, 1, 1, 40, 20, True), (1, 4, 8, 4, 64, 2, 16, True)])
def test_reorder(L, B, W, heads, bs, mb, unit, table):
    rng = np.random.default_rng(W * bs)
    R_, cap = B * W, bs * mb
    blocks = R_ * mb + 2
    tab = rng.permutation(blocks)[:R_ * mb].reshape(R_, mb) if table else np.arange(R_ * mb).reshape(R_, mb)
    blocks = blocks if table else R_ * mb
    host = [rng.integers(0, 256, (L, blocks, heads, bs, unit)).astype(np.uint8),
            rng.integers(-2 ** 31, 2 ** 31, (L, blocks, 1, bs)).astype(np.int32)]
    cycle = (np.arange(W) + 1) % W
    for parents, lens in ((rng.integers(0, W, (B, W)), rng.integers(0, cap + 1, R_)), (np.tile(cycle, (B, 1)), np.full(R_, cap)),
                          (np.zeros((B, W), int), np.full(R_, cap - 1)), (np.tile(np.arange(W), (B, 1)), np.full(R_, cap)),
                          (rng.integers(-1, W + 1, (B, W)), rng.integers(-3, 2 * cap, R_))):
        d = [dev(h) for h in host]
        F().cacheReorder(d, dev(parents.astype(np.int32)), dev(lens.astype(np.int32)),
                         table=dev(tab.astype(np.int32)) if table else None)
        for got, h in zip(d, host):
            want = h.copy()
            for b in range(B):
                for w in range(W):
                    p = int(parents[b, w])
                    if not 0 <= p < W:
                        continue
                    src, dst = b * W + p, b * W + w
                    j = np.arange(max(0, min(int(lens[src]), cap)))
                    want[:, tab[dst, j // bs], :, j % bs] = h[:, tab[src, j // bs], :, j % bs]
            assert np.array_equal(got.cpu().numpy(), want)


def test_reorder_skips_bad_blocks():
    x = torch.arange(4 * 2 * 4, dtype=I32, device="cuda").view(1, 4, 2, 4).contiguous()
    t = torch.tensor([[0, 1], [2, 9]], dtype=I32, device="cuda")
    want = x.clone()
    want[0, 2] = x[0, 0]                       # beam 1's second block does not exist
    F().cacheReorder([x], torch.tensor([[0, 0]], dtype=I32, device="cuda"), torch.tensor([8, 8], dtype=I32, device="cuda"),
                     table=t)
    assert torch.equal(x, want)


# ------------------------------------------------------------------ together
CFG = dict(dim=256, hidden=512, nLayers=2, nHeads=4, nKvHeads=2, vocabSize=128, maxSeq=64)


@pytest.fixture(scope="module")
def model():
    from forgellm.train import Config, init_weights_flat
    import oracle as O
    cfg = Config(**CFG)
    ocfg = O.Config(**{k: v for k, v in CFG.items() if k != "maxSeq"})
    w = O.unflatten_weights(ocfg, init_weights_flat(cfg, 11))
    # larger embeddings than initWeights draws, so that the logits tell the beams apart
    w["tok_emb"] = (np.asarray(w["tok_emb"]) * 20).astype(np.float32)
    return cfg, F().Transformer(cfg).loadWeights(w)


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / np.linalg.norm(a))


def values_step(tr, cfg, token, pos, fp):
    """One decode step of one sequence on an fp32 cache whose new rows are
    replaced by what the 4-bit cache would hold of them."""
    from forgellm._lib import call
    from forgellm.autograd import ctx
    call_ = lambda name, *a: call(name, ctx().handle, *a)  # noqa: E731
    z = lambda n: torch.empty(n, device="cuda")  # noqa: E731
    x = tr.tokEmb.rows(torch.tensor([token], dtype=I32, device="cuda"))[0].clone()
    inv, att = z(1), z(cfg.dim)
    at, ln = torch.tensor([pos], dtype=I32, device="cuda"), torch.tensor([pos + 1], dtype=I32, device="cuda")

    def norm(w):
        out = z(cfg.dim)
        call_("fcu_rmsnorm_fwd", x.data_ptr(), w.data_ptr(), 1, cfg.dim, float(cfg.normEps), out.data_ptr(), inv.data_ptr())
        return out

    for l, Ly in enumerate(tr.layers):
        q = Ly["wqkv"].forward(norm(Ly["ln1"]))
        k, v = fp.k[l], fp.v[l]
        call_("fcu_decode_rope_kv", q.data_ptr(), cfg.qkvOut, 1, cfg.nHeads, cfg.nKvHeads, cfg.dHead, float(cfg.ropeTheta),
              at.data_ptr(), k.data_ptr(), v.data_ptr(), cfg.kvDim, None, 1, cfg.maxSeq)
        for t in (k, v):
            t[pos] = dev(R.values(*R.quantize(t[pos].cpu().numpy().reshape(cfg.nKvHeads, cfg.dHead)))).view(-1)
        call_("fcu_attn_decode", q.data_ptr(), cfg.qkvOut, k.data_ptr(), v.data_ptr(), cfg.kvDim, None, 1, cfg.maxSeq,
              ln.data_ptr(), 1, cfg.nHeads, cfg.nKvHeads, cfg.dHead, cfg.dHead ** -0.5, att.data_ptr())
        x = x + Ly["wo"].forward(att)
        h = norm(Ly["ln2"])
        g, u, act = Ly["gate"].forward(h), Ly["up"].forward(h), z(cfg.hidden)
        call_("fcu_swiglu_fwd", g.data_ptr(), u.data_ptr(), cfg.hidden, act.data_ptr())
        x = x + Ly["down"].forward(act)
    return tr.wcls.forward(norm(tr.lnF))


@pytest.mark.parametrize("block", [None, 8])
def test_decode_over_the_4bit_cache(model, block):
    """Every step's logits are those of fp32 attention over the values the cache
    holds (1e-5, as the fp32 decode path is held to); eager and graph agree bit
    for bit."""
    cfg, tr = model
    fw = F()
    mk = lambda: fw.QuantKVCache(cfg.nLayers, cfg.maxSeq, cfg.nKvHeads, cfg.dHead, blockSize=block)  # noqa: E731
    q4, graphed, fp = mk(), mk(), fw.KVCache(cfg.nLayers, cfg.maxSeq, cfg.kvDim)
    ids = np.random.default_rng(3).integers(0, cfg.vocabSize, 14)
    for p, t in enumerate(ids):
        got = tr.forward(int(t), p, q4).cpu().numpy().copy()
        assert rel(values_step(tr, cfg, int(t), p, fp).cpu().numpy(), got) <= 1e-5, p
        assert np.array_equal(got, tr.forward(int(t), p, graphed, graph=True).cpu().numpy()), p
    assert q4.len == 14 and q4.bytes() * 6 < fp.bytes()
    for l in range(cfg.nLayers):
        assert rel(fp.k[l, :14].cpu().numpy(), q4.kView(l, 14).cpu().numpy()) <= 1e-5
        assert rel(fp.v[l, 13].cpu().numpy(), q4.sliceV(l, 13).cpu().numpy()) <= 1e-5


def test_put_writes_a_row_of_one_sequence(model):
    cfg, _ = model
    c = F().QuantKVCache(2, 32, 2, 64, batch=3, blockSize=8, track=True)
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((2, 128)).astype(np.float32)
    c.put(1, 9, k, v, seq=2)
    assert c.lens.tolist() == [0, 0, 10] and c.len == 10
    assert np.array_equal(c.sliceK(1, 9, 2).cpu().numpy(), R.values(*R.quantize(k.reshape(2, 64))).ravel())
    assert np.array_equal(c.vView(1, 10, 2)[9].cpu().numpy(), R.values(*R.quantize(v.reshape(2, 64))).ravel())
    assert int(c.pos[1, 2 * 4 + 1, 0, 1]) == 9 and int((c.pos != 0).sum()) == 2


def test_put_after_an_eviction():
    """Rows put layer by layer go on after an eviction: every layer's row of a new
    position goes to one slot, a position since then may be put again, an evicted
    one and one that would leave stale slots between may not."""
    c = F().QuantKVCache(3, 32, 2, 64, batch=2, blockSize=8, track=True)
    rng = np.random.default_rng(2)
    rows = rng.standard_normal((30, 3, 2, 128)).astype(np.float32)
    put = lambda p: [c.put(l, p, *rows[p, l], seq=1) for l in range(3)]  # noqa: E731
    for p in range(20):
        put(p)
    c.evict(6, 6)                             # the newest six stay
    assert c.lens.tolist() == [0, 6] and c.dropped.tolist() == [0, 14]
    for p in (20, 21, 21, 20, 22):
        put(p)
    assert c.lens.tolist() == [0, 9] and c.len == 9
    blk = torch.arange(4, 8, device="cuda")
    pos = c.pos[:, blk].movedim(2, 1).flatten(2)[:, :, :9].cpu().numpy()      # [layers, heads, slots]
    assert (np.sort(pos, -1) == np.arange(14, 23)).all() and (pos[:, :, 6:] == [20, 21, 22]).all()
    for l in range(3):
        for p, slot in ((20, 6), (21, 7), (22, 8)):
            want = R.values(*R.quantize(rows[p, l, 0].reshape(2, 64))).ravel()
            assert np.array_equal(c.sliceK(l, slot, 1).cpu().numpy(), want)
    for p in (0, 13, 19, 24, 29):
        with pytest.raises(ValueError):
            c.put(0, p, *rows[p, 0], seq=1)
    c.reorder([[1, 1]])
    put(23)
    c.put(0, 22, *rows[22, 0], seq=0)
    for p in (19, 24):
        with pytest.raises(ValueError):
            c.put(0, p, *rows[p, 0], seq=0)
    assert c.lens.tolist() == [9, 10]
    c.reset()
    put(3)
    assert c.lens.tolist() == [0, 4]


def reference_search(tr, cfg, prompt, W, n, eos, cache_of):
    """Beam search that recomputes every hypothesis from its tokens."""
    def logits_of(text):
        c = cache_of()
        for p, t in enumerate(list(prompt) + text):
            out = tr.forward(int(t), p, c)
        return out.cpu().numpy().astype(np.float64)

    texts, scores, done = [[] for _ in range(W)], np.array([0.0] + [-np.inf] * (W - 1)), np.zeros(W, bool)
    for _ in range(n):
        x = np.stack([logits_of([t for t in tx]) for tx in texts])
        s, t, p, d = R.beam(x[None], scores[None], done[None], W, eos)
        texts = [texts[p[0, i]] + ([] if done[p[0, i]] else [int(t[0, i])]) for i in range(W)]
        scores, done = s[0], d[0]
        if done.all():
            break
    return texts, scores


@pytest.mark.parametrize("kind", ["fp32", "paged", "4bit", "4bit paged"])
def test_beam_search(model, kind):
    """The search over reordered caches finds what recomputing every hypothesis
    from its tokens finds; scores to 1e-4 (the logits' 1e-5 over 10 tokens)."""
    cfg, tr = model
    fw = F()
    W, n = 4, 7

    def mk(batch):
        if kind == "fp32":
            return fw.KVCache(cfg.nLayers, cfg.maxSeq, cfg.kvDim, batch=batch)
        if kind == "paged":
            return fw.PagedKVCache(cfg.nLayers, cfg.maxSeq, cfg.kvDim, blockSize=8, batch=batch,
                                   table=np.random.default_rng(2).permutation(batch * 8).reshape(batch, 8))
        return fw.QuantKVCache(cfg.nLayers, cfg.maxSeq, cfg.nKvHeads, cfg.dHead, batch=batch,
                               blockSize=8 if "paged" in kind else None)

    prompt = [5, 77, 31]
    for eos in (2, None):
        if eos is None:      # an ending that the search does reach
            eos = [t for t, _ in found][0][2]
        found = tr.beamSearch(prompt, W, n, mk(W), eosId=eos)
        texts, scores = reference_search(tr, cfg, prompt, W, n, eos, lambda: mk(1))
        assert [t for t, _ in found] == texts
        assert np.abs(np.array([s for _, s in found]) - scores).max() <= 1e-4
    assert any(t[-1] == eos and len(t) < n for t, _ in found)


def test_search_with_eviction(model):
    """Search, 4-bit cache and eviction together: the caches stay at the budget,
    hold the newest positions and no position twice, and graph replay finds the
    same tokens and scores as eager steps."""
    cfg, tr = model
    fw = F()
    W, budget, recent = 3, 9, 4
    runs = []
    for graph in (False, True):
        c = fw.QuantKVCache(cfg.nLayers, 16, cfg.nKvHeads, cfg.dHead, batch=W, blockSize=4, track=True,
                            table=np.random.default_rng(4).permutation(W * 4).reshape(W, 4))
        prompt = np.random.default_rng(6).integers(3, cfg.vocabSize, 12)
        runs.append((tr.beamSearch(prompt, W, 12, c, eosId=0, budget=budget, recent=recent, graph=graph), c))
    assert runs[0][0] == runs[1][0]
    found, c = runs[0]
    assert len(found) == W and all(np.isfinite(s) for _, s in found)
    n = c.lens
    assert (n == budget).all() and (c.dropped > 0).all()
    for b in range(W):
        pos = c.pos[:, torch.from_numpy(c._table_host[b].astype(np.int64)).cuda()].movedim(2, 1).flatten(2)[:, :, :budget]
        last = int(c.lens[b] + c.dropped[b]) - 1
        for row in pos.reshape(-1, budget).cpu().numpy():
            assert np.unique(row).size == budget and set(range(last - recent + 1, last + 1)) <= set(row.tolist())
    with pytest.raises(ValueError):
        c.slotOf(0)
    w = c.weight.sum().item()
    assert np.isfinite(w) and w > 0


def test_weights_loaded_again(model):
    """Graphs of a step go with the weights that they were captured with."""
    from forgellm.train import init_weights_flat
    import oracle as O
    cfg, _ = model
    fw = F()
    ocfg = O.Config(**{k: v for k, v in CFG.items() if k != "maxSeq"})
    tr = fw.Transformer(cfg)
    c = fw.QuantKVCache(cfg.nLayers, 32, cfg.nKvHeads, cfg.dHead, batch=2)
    for seed in (11, 12):
        tr.loadWeights(O.unflatten_weights(ocfg, init_weights_flat(cfg, seed)))
        out = []
        for graph in (True, False):
            c.reset()
            out.append(torch.stack([tr.forwardBatch([3 + p, 40 - p], [p, p], c, graph=graph).clone() for p in range(4)]))
        assert torch.equal(*out), seed


def test_reorder_of_a_paged_cache_with_spare_blocks():
    """Without a table the beams' blocks are the first of a larger pool."""
    fw = F()
    c = fw.PagedKVCache(2, 24, 8, blockSize=8, batch=3, physBlocks=18)
    c.k.copy_(torch.arange(c.k.numel(), device="cuda").view_as(c.k))
    c.v.copy_(-c.k)
    c.len = 20
    want = c.k.clone()
    for w, p in enumerate([2, 2, 0]):
        want[:, 24 * w:24 * w + 20] = c.k[:, 24 * p:24 * p + 20]
    c.reorder([[2, 2, 0]])
    assert torch.equal(c.k, want) and torch.equal(c.v, -want)


def test_search_refusals(model):
    """Refused before the first step, so that the cache stays unused."""
    cfg, tr = model
    fw = F()
    fp = fw.KVCache(cfg.nLayers, 16, cfg.kvDim, batch=2)
    q4 = fw.QuantKVCache(cfg.nLayers, 16, cfg.nKvHeads, cfg.dHead, batch=2, track=True)
    other = fw.QuantKVCache(cfg.nLayers, 16, cfg.nKvHeads, cfg.dHead - 4, batch=2)
    ids = list(range(3, 13))
    for f in (lambda: tr.beamSearch(ids, 2, 8, fp), lambda: tr.beamSearch(ids, 2, 8, q4),
              lambda: tr.beamSearch(ids, 2, 8, q4, budget=16), lambda: tr.beamSearch(ids, 2, 4, fp, budget=8),
              lambda: tr.beamSearch(ids, 2, 4, q4, budget=8, recent=9), lambda: tr.beamSearch(ids, 2, 4, q4, budget=0),
              lambda: tr.beamSearch(ids, 2, 4, q4, eosId=cfg.vocabSize), lambda: tr.beamSearch(ids, 3, 4, q4),
              lambda: tr.beamSearch(ids, 33, 4, fw.QuantKVCache(1, 16, 1, 8, batch=33)),
              lambda: tr.beamSearch([], 2, 4, q4), lambda: tr.beamSearch(ids, 2, 0, q4),
              lambda: tr.beamSearch(ids, 2, 4, other), lambda: tr.forward(3, 16, q4), lambda: tr.forward(3, -1, q4)):
        with pytest.raises(ValueError):
            f()
    assert fp.len == q4.len == other.len == 0
    for n, c in ((7, fp), (7, q4)):            # the last new token is never written
        assert len(tr.beamSearch(ids, 2, n, c)) == 2 and c.len == 16
    assert len(tr.beamSearch(ids, 1, 1, fw.QuantKVCache(cfg.nLayers, 16, cfg.nKvHeads, cfg.dHead))[0][0]) == 1
