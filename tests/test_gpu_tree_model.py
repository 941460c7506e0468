"""The model's calls on trees, windows and scores, the operators as they are
used together: cmf_verify_tree, cmf_model_set_window, cmf_score.

A plain f64 forward with any visibility (dequantized weights) is the reference
of hidden rows, keys and values, within relative L2 1e-4 as the other model
tests (the operators' own tolerances are in their tests); acceptance, paths and
commits are compared with what the same logits give in numpy, and the state
after a tree with that of plain forwards of the accepted stream (the oracle)."""
import numpy as np
import pytest

from conftest import rel_l2
from oracle import oracle as orc

pytestmark = pytest.mark.gpu

CFG = dict(n_layers=2, hidden=256, n_heads=4, n_kv=2, head_dim=128, inter=512, vocab=4096, max_seq=320, rope_theta=1e6,
           eps=1e-6)
TOL = 1e-4


def _rms(x, w, eps):
    return x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps) * w


def forward64(sm, toks, pos, see):
    """f64 forward: row i is token toks[i] at position pos[i] and sees the rows
    see[i]; returns the final hidden rows and each layer's (k, v)."""
    from cmf_amd import synth
    dq = lambda t: synth.dequant(t).astype(np.float64)  # noqa: E731
    c = sm["cfg"]
    n, nh, nkv, hd, eps = len(toks), c["n_heads"], c["n_kv"], c["head_dim"], c["eps"]
    hs = dq(sm["lm_head"])[toks]
    ang = np.asarray(pos)[:, None] * c["rope_theta"] ** (-np.arange(0, hd, 2) / hd)
    cos, sin = np.cos(ang)[:, None], np.sin(ang)[:, None]

    def rope(x):
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        return np.concatenate([a * cos - b * sin, a * sin + b * cos], -1)
    kvs = []
    for l in sm["layers"]:
        x = _rms(hs, l["input_norm"], eps)
        q = rope(_rms((x @ dq(l["wq"]).T).reshape(n, nh, hd), l["q_norm"], eps))
        k = rope(_rms((x @ dq(l["wk"]).T).reshape(n, nkv, hd), l["k_norm"], eps))
        v = (x @ dq(l["wv"]).T).reshape(n, nkv, hd)
        kvs.append((k.transpose(1, 0, 2), v.transpose(1, 0, 2)))
        att = np.zeros((n, nh, hd))
        for h in range(nh):
            g = h // (nh // nkv)
            s = np.where(see, q[:, h] @ k[:, g].T / np.sqrt(hd), -np.inf)
            w = np.exp(s - s.max(1, keepdims=True))
            att[:, h] = (w / w.sum(1, keepdims=True)) @ v[:, g]
        hs = hs + att.reshape(n, nh * hd) @ dq(l["wo"]).T
        x = _rms(hs, l["post_norm"], eps)
        g = x @ dq(l["gate"]).T
        hs = hs + (g / (1 + np.exp(-g)) * (x @ dq(l["up"]).T)) @ dq(l["down"]).T
    return hs, kvs


def causal(n, window=0, sinks=0):
    i, j = np.arange(n)[:, None], np.arange(n)[None]
    return (j <= i) & ((j > i - window) | (j < sinks) if window else True)


def logits64(sm, hs):
    from cmf_amd import synth
    return _rms(hs, sm["final_norm"], sm["cfg"]["eps"]) @ synth.dequant(sm["lm_head"]).astype(np.float64).T


def log_softmax(x):
    d = x - x.max(-1, keepdims=True)
    return d - np.log(np.exp(d).sum(-1, keepdims=True))


@pytest.fixture(scope="module")
def plain(gpu):
    from cmf_amd import synth
    from cmf_amd.model import Model
    sm = synth.synth_model(CFG, seed=41, norm_noise=0.1, sigma=0.05)
    g = Model(sm)
    yield sm, g
    g.free()


@pytest.fixture(scope="module")
def accepting(gpu):
    from cmf_amd import synth
    from cmf_amd.model import Model
    sm = synth.accept_model(CFG)
    g = Model(sm)
    yield sm, g
    g.free()


def random_tree(b, seed, back=6):
    r = np.random.RandomState(seed)
    return [-1] + [int(r.randint(max(0, i - back), i)) for i in range(1, b)]


def walk(parents, ok, lp):
    """The accepted path: the best accepted child from the root on."""
    path = [0]
    while True:
        kids = [i for i in range(1, len(parents)) if parents[i] == path[-1] and ok[i]]
        if not kids:
            return path
        path.append(max(kids, key=lambda i: (lp[i], -i)))


def check_results(toks, parents, eps, delta, r):
    """lp, entropy, argmax and the path are those of the returned logits."""
    lg = r["logits"].astype(np.float64)
    ls = log_softmax(lg)
    b = len(toks)
    lp = np.array([np.nan] + [ls[parents[i], toks[i]] for i in range(1, b)])
    ent = -(np.exp(ls) * ls).sum(1)
    am = np.array([np.flatnonzero(x == x.max())[-1] for x in r["logits"]])
    assert np.isnan(r["logprobs"][0]) and np.allclose(r["logprobs"][1:], lp[1:], rtol=1e-5, atol=2e-5)
    assert np.allclose(r["entropy"], ent, rtol=1e-5, atol=2e-5)
    assert r["argmax"].tolist() == am.tolist()
    if eps == 0:
        ok = [False] + [toks[i] == am[parents[i]] for i in range(1, b)]
    else:
        ok = [False] + [np.exp(lp[i]) >= min(eps, delta * np.exp(-ent[parents[i]])) for i in range(1, b)]
    assert r["path"].tolist() == walk(parents, ok, lp)
    assert r["next_token"] == am[r["path"][-1]]


@pytest.mark.parametrize("b,n", [(1, 5), (7, 40), (16, 33), (17, 64), (33, 100), (64, 40)])
def test_rows_of_a_tree(plain, b, n):
    """Every row's logits are those of its own path behind the prompt."""
    from cmf_amd import synth
    sm, g = plain
    prompt = synth.ids(51 + b, n, CFG["vocab"])
    toks = synth.ids(52 + b, b, CFG["vocab"])
    parents = random_tree(b, b)
    g.prefill(prompt)
    r = g.verify_tree(toks, parents, n, want_logits=True)
    depth = [0] * b
    see = np.zeros((n + b, n + b), bool)
    see[:n, :n] = causal(n)
    for i in range(b):
        see[n + i, :n] = True
        j = i
        while j >= 0:
            see[n + i, n + j] = True
            j = parents[j]
        depth[i] = int(see[n + i, n:].sum()) - 1
    hs, kvs = forward64(sm, np.concatenate([prompt, toks]), list(range(n)) + [n + d for d in depth], see)
    want = logits64(sm, hs[n:])
    for i in range(b):
        assert rel_l2(r["logits"][i], want[i]) < TOL, i
    check_results(toks, parents, 0, 0, r)
    a = len(r["path"]) - 1
    pos, tip = g.state()
    assert pos == n + a + 1
    rows = list(range(n)) + [n + p for p in r["path"]]
    assert rel_l2(tip, hs[rows[-1]]) < TOL
    for li, (k, v) in enumerate(kvs):
        gk, gv = g.kv_export(li, pos)
        assert rel_l2(gk, k[:, rows]) < TOL and rel_l2(gv, v[:, rows]) < TOL


def run_tree(g, prompt, t_next, seed, b=24):
    """A tree behind the prompt whose rows follow the model's own choices here
    and there: children repeat a token of the run, or are random."""
    r = np.random.RandomState(seed)
    parents = random_tree(b, seed, back=4)
    toks = [int(t_next)] + [int(t_next) if r.rand() < 0.6 else int(r.randint(CFG["vocab"])) for _ in range(1, b)]
    return np.array(toks, np.int32), parents


def check_state(sm, g, seq, mtp_rows):
    ref = orc.OracleModel(sm)
    ref.prefill(np.asarray(seq))
    for li in list(range(CFG["n_layers"])) + [-1]:
        n = len(seq) if li >= 0 else mtp_rows
        k, v = g.kv_export(li, n)
        rk, rv = ref.kv(li)
        assert rel_l2(k, rk[:, :n]) < TOL and rel_l2(v, rv[:, :n]) < TOL, li


@pytest.mark.parametrize("eps,delta", [(0.0, 0.0), (0.09, 0.3), (1e-6, 1e-6)])
@pytest.mark.parametrize("b", [9, 24, 64])
def test_accepted_paths_are_committed(accepting, b, eps, delta):
    """Two trees one after the other, then the decode goes on: caches, tip and
    MTP pairs are those of plain forwards of the accepted stream."""
    from cmf_amd import synth
    sm, g = accepting
    seq = list(synth.ids(23, 20, CFG["vocab"]))
    g.prefill(seq)
    nxt = int(np.argmax(g.forward_batch(seq[-1:], len(seq) - 1)[1][0]))
    for turn in range(2):
        toks, parents = run_tree(g, seq, nxt, 7 + turn, b)
        r = g.verify_tree(toks, parents, len(seq), eps, delta, want_logits=True)
        check_results(toks, parents, eps, delta, r)
        seq += [int(toks[i]) for i in r["path"]]
        nxt = r["next_token"]
        assert g.state()[0] == len(seq)
    # the pair of the last position waits for the next token
    check_state(sm, g, seq, len(seq) - 1)
    gt, _ = g.decode(8, spec=True, k=4)
    o = orc.OracleModel(sm)
    ot, _ = o.decode(o.prefill(np.asarray(seq)), len(seq), np.asarray(seq), 8, spec=True, k=4)
    assert gt.tolist() == ot.tolist()


@pytest.mark.parametrize("deep,wide", [(3, 1), (7, 2), (15, 4), (20, 3)])
def test_the_models_own_continuation_is_accepted(plain, deep, wide):
    """The oracle's greedy tokens, each among `wide - 1` other drafts whose rows
    come first or last: the path takes them all."""
    from cmf_amd import synth
    sm, g = plain
    prompt = synth.ids(91, 30, CFG["vocab"])
    want, _ = orc.OracleModel(sm).generate(prompt, deep + 2, spec=False)
    want = want.tolist()
    toks, parents, rows = [want[0]], [-1], [0]
    for d in range(1, deep + 1):
        at = rows[-1]
        for w in range(wide):
            if w == d % wide:
                rows.append(len(toks))
                toks.append(want[d])
            else:
                toks.append((want[d] + 17 * (w + 1)) % CFG["vocab"])
            parents.append(at)
    g.prefill(prompt)
    r = g.verify_tree(toks, parents, 30)
    assert r["path"].tolist() == rows and r["next_token"] == want[deep + 1]
    seq = list(prompt) + want[:deep + 1]
    check_state(sm, g, seq, len(seq) - 1)
    gt, _ = g.decode(4, spec=True, k=2)
    o = orc.OracleModel(sm)
    ot, _ = o.decode(o.prefill(np.asarray(seq)), len(seq), np.asarray(seq), 4, spec=True, k=2)
    assert gt.tolist() == ot.tolist()


@pytest.mark.parametrize("k", [1, 4, 8])
def test_a_chain_is_verify_step(accepting, k):
    from cmf_amd import synth
    from cmf_amd.model import Model
    sm, g = accepting
    twin = Model(sm)
    prompt = synth.ids(23, 20, CFG["vocab"])
    for m in (g, twin):
        m.prefill(prompt)
    nxt = int(np.argmax(g.forward_batch(prompt[-1:], 19)[1][0]))
    twin.forward_batch(prompt[-1:], 19)
    toks = np.array([nxt] * k + [5], np.int32)
    a, want, am, _ = twin.verify_step(toks, 20)
    r = g.verify_tree(toks, [i - 1 for i in range(k + 1)], 20)
    assert r["path"].tolist() == list(range(a + 1)) and r["next_token"] == want and r["argmax"].tolist() == am.tolist()
    assert g.state()[0] == twin.state()[0] and rel_l2(g.state()[1], twin.state()[1]) < TOL
    for li in (0, 1, -1):
        n = 20 + a + (li >= 0)
        for x, y in zip(g.kv_export(li, n), twin.kv_export(li, n)):
            assert rel_l2(x, y) < TOL
    twin.free()


def test_routed_experts(gpu):
    from cmf_amd import synth
    from cmf_amd.model import Model
    sm = synth.synth_model(CFG, seed=31, norm_noise=0.3, sigma=0.08, mtp=False,
                           moe=dict(n_experts=16, top_k=4, inter=128, layers=[0], router_dtype="f16"))
    g = Model(sm)
    prompt = synth.ids(61, 20, CFG["vocab"])
    for b in (6, 40):
        toks, parents = synth.ids(62, b, CFG["vocab"]), random_tree(b, 1)
        g.prefill(prompt)
        r = g.verify_tree(toks, parents, 20, want_logits=True)
        check_results(toks, parents, 0, 0, r)
        for leaf in (b - 1, b // 2):  # the same rows as chains
            chain, j = [], leaf
            while j >= 0:
                chain.insert(0, j)
                j = parents[j]
            g.prefill(prompt)
            lg = g.forward_batch(toks[chain], 20)[1]
            for c, row in zip(chain, lg):
                assert rel_l2(r["logits"][c], row) < TOL
    g.free()


def test_verify_tree_refuses(plain):
    import cmf_amd
    from cmf_amd import synth
    sm, g = plain
    g.prefill(synth.ids(1, 10, CFG["vocab"]))
    t = [1, 2, 3]
    for toks, parents, pos, eps, word in (
            (t, [-1, 0, 0], 9, 0, "committed"), (t, [-1, -1, 0], 10, 0, "only root"), (t, [0, 0, 0], 10, 0, "earlier"),
            (t, [-1, 2, 0], 10, 0, "earlier"), ([1, 5000, 2], [-1, 0, 0], 10, 0, "range"), (t, [-1, 0, 0], 10, -1.0, "eps"),
            (t, [-1, 0, 0], 10, float("nan"), "eps"), ([1] * 65, [-1] + [0] * 64, 10, 0, "64")):
        with pytest.raises(cmf_amd.CmfError, match=word):
            g.verify_tree(toks, parents, pos, eps)
        assert g.state()[0] == 10
    g.prefill(synth.ids(1, 310, CFG["vocab"]))
    with pytest.raises(cmf_amd.CmfError, match="max_seq"):
        g.verify_tree([1] * 10, [i - 1 for i in range(10)], 310)
    g.verify_tree([1] * 9, [i - 1 for i in range(9)], 310)  # the last one that fits
    assert g.state()[0] <= 319


# ---- the window -----------------------------------------------------------
@pytest.mark.parametrize("window,sinks,n", [(64, 4, 300), (17, 0, 130), (1, 0, 50), (33, 20, 200)])
def test_window(plain, window, sinks, n):
    """Prefill, a batch of rows, a tree and plain tokens through a window."""
    from cmf_amd import synth
    sm, g = plain
    ids = synth.ids(71, n, CFG["vocab"])
    m = n - 12
    g.set_window(window, sinks)
    try:
        g.prefill(ids[:m])
        hid, lg = g.forward_batch(ids[m:], m)
        hs, kvs = forward64(sm, ids, list(range(n)), causal(n, window, sinks))
        assert rel_l2(hid, hs[m:]) < TOL
        assert rel_l2(lg, logits64(sm, hs[m:])) < TOL
        for li, (k, v) in enumerate(kvs):
            gk, gv = g.kv_export(li, n)
            assert rel_l2(gk, k) < TOL and rel_l2(gv, v) < TOL
        # a chain as a tree: the same rows again
        g.prefill(ids[:m])
        r = g.verify_tree(ids[m:], [i - 1 for i in range(12)], m, want_logits=True)
        for i in range(12):
            assert rel_l2(r["logits"][i], lg[i]) < TOL
        # plain tokens, eager and captured rounds
        g.prefill(ids[:m])
        toks, _ = g.decode(8, spec=False)
        seq = list(ids[:m])
        for t in toks:
            hs, _ = forward64(sm, np.array(seq), list(range(len(seq))), causal(len(seq), window, sinks))
            top = logits64(sm, hs[-1:])[0]
            assert top[t] > top.max() - 1e-4 * np.abs(top).max()
            seq.append(int(t))
    finally:
        g.set_window(0)


def test_speculation_under_a_window(accepting):
    """Greedy speculative rounds emit the plain tokens, with accepted drafts."""
    from cmf_amd import synth
    sm, g = accepting
    prompt = synth.ids(23, 60, CFG["vocab"])
    g.set_window(24, 2)
    try:
        g.prefill(prompt)
        want, _ = g.decode(40, spec=False)
        g.prefill(prompt)
        got, st = g.decode(40, spec=True, k=4)
        assert got.tolist() == want.tolist() and st.accepted > 0
    finally:
        g.set_window(0)
    g.prefill(prompt)
    ot, _ = orc.OracleModel(sm).generate(prompt, 12, spec=True, k=4)
    assert g.decode(12, spec=True, k=4)[0].tolist() == ot.tolist()


def test_a_window_that_sees_everything_changes_nothing(plain):
    from cmf_amd import synth
    sm, g = plain
    ids = synth.ids(72, 100, CFG["vocab"])
    g.prefill(ids)
    want = g.forward_batch(ids[:5], 100)
    kv = g.kv_export(1, 105)
    g.set_window(90, 15)
    try:
        g.prefill(ids)
        got = g.forward_batch(ids[:5], 100)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        assert all(np.array_equal(x, y) for x, y in zip(kv, g.kv_export(1, 105)))
    finally:
        g.set_window(0)


def test_window_refuses(plain):
    import cmf_amd
    for w, s in ((-1, 0), (5, -1)):
        with pytest.raises(cmf_amd.CmfError):
            plain[1].set_window(w, s)


# ---- scores ---------------------------------------------------------------
@pytest.mark.parametrize("n,k,window", [(1, 3, 0), (2, 0, 0), (300, 8, 0), (257, 64, 0), (200, 2, 50)])
def test_score(plain, n, k, window):
    from cmf_amd import synth
    sm, g = plain
    ids = synth.ids(81, n, CFG["vocab"])
    g.set_window(window, 3)
    try:
        lp, ent, ti, tl = g.score(ids, top_k=k)
        hs, _ = forward64(sm, ids, list(range(n)), causal(n, window, 3))
    finally:
        g.set_window(0)
    lg = logits64(sm, hs)
    ls = log_softmax(lg)
    tol = 3 * TOL * np.abs(lg).max()  # a logit is off by TOL of the largest at most, a log probability by twice that
    assert np.isnan(lp[-1]) and lp.shape == (n,)
    assert np.abs(lp[:-1] - ls[np.arange(n - 1), ids[1:]]).max(initial=0) < tol
    assert np.abs(ent + (np.exp(ls) * ls).sum(1)).max() < 3 * tol
    if k:
        want = -np.sort(-ls, axis=1)[:, :k]
        assert np.abs(tl - want).max() < tol
        assert np.abs(np.take_along_axis(ls, ti.astype(np.int64), 1) - want).max() < 2 * tol
    # the state is the prefill's
    pos, tip = g.state()
    assert pos == n and rel_l2(tip, hs[-1]) < TOL
    if not window:
        got = g.decode(6, spec=True, k=4)[0]
        g.prefill(ids)
        assert got.tolist() == g.decode(6, spec=True, k=4)[0].tolist()


def test_score_refuses(plain):
    import cmf_amd
    from cmf_amd import synth
    g = plain[1]
    with pytest.raises(cmf_amd.CmfError, match="top_k"):
        g.score([1, 2], top_k=65)
    with pytest.raises(cmf_amd.CmfError, match="range"):
        g.score([1, 5000])
    with pytest.raises(cmf_amd.CmfError, match="max_seq"):
        g.score(synth.ids(1, 320, CFG["vocab"]))
