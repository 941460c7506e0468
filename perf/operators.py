"""The operators around the verification of drafted tokens, each against a plain
form in elementary torch operations:

  rope      the norm of every query and key head with the position rotation, the
            key and value rows stored in the cache's type (cmf_amd.ops.qk_rope)
  tree      attention of a tree of drafted tokens over a cache (ops.attention)
  window    attention with a sliding window and a few first positions that stay
            visible (ops.attention), one token to whole prompt chunks
  copy      rows of many caches copied by index: the commit of an accepted path,
            a forked prefix (ops.kv_copy)
  logprobs  log probabilities of given tokens, the entropy of their
            distributions and the top alternatives (ops.logprobs)

Activations are f32, caches and logits f32, f16 or bf16.  Head layouts are those
of the decoder shapes of this repository's benchmark (16 query heads on 8 KV
heads of 128) and generic ones.
"""
import math
import random

import torch

own = False

HD = 128
EPS = 1e-6
THETA = 1e6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
WS_BYTES = 64 << 20  # the scratch a program keeps for the attention


def listed():
    return [
        # one decoded token of the headline model: latency
        dict(name="rope_b1", kind="rope", b=1, nh=16, nkv=8, pos0=2047, dtype="f32", tree=False),
        # a ragged prompt chunk of a wider model into a 16-bit cache
        dict(name="rope_b2001_bf16", kind="rope", b=2001, nh=32, nkv=8, pos0=300, dtype="bf16", tree=False),
        # a small tree of drafts at the headline context
        dict(name="tree_b9_ctx2048", kind="tree", b=9, ctx=2048, nh=16, nkv=8, dtype="f32"),
        # a wider tree over a long context, odd sizes
        dict(name="tree_b29_ctx12001", kind="tree", b=29, ctx=12001, nh=16, nkv=8, dtype="f32"),
        # the largest tree over a very long 16-bit cache
        dict(name="tree_b64_ctx65536_bf16", kind="tree", b=64, ctx=65536, nh=32, nkv=8, dtype="bf16"),
        # a decoded token far into a stream of text
        dict(name="window_b1_ctx12000", kind="window", b=1, ctx=12000, window=1024, sinks=4, nh=16, nkv=8, dtype="f32"),
        # a verify batch with a wide window over a 16-bit cache
        dict(name="window_b5_ctx100000_f16", kind="window", b=5, ctx=100000, window=16000, sinks=64, nh=32, nkv=8,
             dtype="f16"),
        # a prompt chunk behind another one
        dict(name="window_b4100_ctx4000", kind="window", b=4100, ctx=4000, window=1024, sinks=4, nh=16, nkv=8,
             dtype="f32"),
        # an accepted path of five drafts into the caches of 28 layers
        dict(name="copy_n5_28layers", kind="copy", bufs=56, nkv=8, slots=512, n=5, pos0=300, src_rows=64, dtype="f32"),
        # a prompt's prefix forked into another cache
        dict(name="copy_n4001_8layers", kind="copy", bufs=16, nkv=8, slots=4096, n=4001, pos0=0, src_rows=4001,
             dtype="f32"),
        # the rows of a verify batch over the headline vocabulary
        dict(name="logprobs_5x151936", kind="logprobs", rows=5, vocab=151936, k=8, dtype="f32"),
        # a chunk of a text to be scored
        dict(name="logprobs_400x151936", kind="logprobs", rows=400, vocab=151936, k=5, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "tree", "tree", "window", "window", "copy", "logprobs"])
    dt = rng.choice(["f32", "f32", "f16", "bf16"])
    nh, nkv = rng.choice([(16, 8), (16, 8), (32, 8), (16, 4), (8, 8), (12, 4), (8, 1), (4, 2)])
    if kind == "rope":
        tree = rng.random() < 0.5
        return dict(kind=kind, b=_log(rng, 1, 64 if tree else 2000), nh=nh, nkv=nkv, pos0=rng.randint(0, 8000), dtype=dt,
                    tree=tree)
    if kind == "tree":
        return dict(kind=kind, b=_log(rng, 1, 64), ctx=_log(rng, 1, 50000), nh=nh, nkv=nkv, dtype=dt)
    if kind == "window":
        b = _log(rng, 1, 2048)
        return dict(kind=kind, b=b, ctx=_log(rng, 16, 100000), window=_log(rng, 16, 16000 if b <= 16 else 1024),
                    sinks=rng.choice([0, 1, 4, 37, 128]), nh=nh, nkv=nkv, dtype=dt)
    if kind == "copy":
        n, room = _log(rng, 1, 2000), rng.randint(0, 400)
        return dict(kind=kind, bufs=2 * rng.randint(1, 36 if n <= 64 else 6), nkv=nkv, slots=n + room, n=n,
                    pos0=rng.randint(0, room), src_rows=n + rng.randint(0, 60), dtype=dt)
    rows = _log(rng, 1, 600)
    return dict(kind=kind, rows=rows, vocab=min(_log(rng, 1000, 200000), 30000000 // rows), k=rng.choice([0, 1, 5, 20, 64]),
                dtype=dt)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
class _Rng:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed((int(seed) * 2654435761 + 97) % (1 << 62))

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda") * std

    def ints(self, lo, hi, n):
        return torch.randint(lo, hi, (n,), generator=self.g, device="cuda")


def _rope_table(n):
    """(cos, sin) of every position and frequency, as a model keeps it."""
    inv = 1.0 / THETA ** (torch.arange(0, HD, 2, device="cuda", dtype=torch.float64) / HD)
    ang = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], 2).float().contiguous()


def _tree(b, seed):
    """A drafted tree in the order of its drafting: the visible rows of each row
    as bits, and the depths.  Row 0 is the root, a row's parent one of the few
    rows before it."""
    rng = random.Random(seed * 7919 + b)
    mask, depth = [1], [0]
    for i in range(1, b):
        p = rng.randint(max(0, i - 6), i - 1)
        mask.append(mask[p] | (1 << i))
        depth.append(depth[p] + 1)
    signed = [m - (1 << 64) if m >> 63 else m for m in mask]
    return (torch.tensor(signed, dtype=torch.int64, device="cuda"), torch.tensor(depth, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    c, r, k = case, _Rng(seed), case["kind"]
    s = dict(case=c, stream=torch.cuda.current_stream().cuda_stream)
    if k == "rope":
        b, nh, nkv = c["b"], c["nh"], c["nkv"]
        s.update(qkv=r.normal(b, nh + 2 * nkv, HD), qn=1 + r.normal(HD, std=0.1), kn=1 + r.normal(HD, std=0.1),
                 rope=_rope_table(c["pos0"] + b), q=torch.empty(b, nh, HD, device="cuda"), depth=None)
        if c["tree"]:
            s["depth"] = _tree(b, seed)[1]
        rows = b if c["tree"] else c["pos0"] + b  # a tree's rows in a buffer of their own, others in the cache
        s["k"], s["v"] = (r.normal(nkv, rows, HD).to(DTYPES[c["dtype"]]) for _ in range(2))
        return s
    if k in ("tree", "window"):
        b, nh, nkv, ctx, dt = c["b"], c["nh"], c["nkv"], c["ctx"], DTYPES[c["dtype"]]
        rows = ctx if k == "tree" else ctx + b
        s.update(q=r.normal(b, nh, HD, std=1.5), k=r.normal(nkv, rows, HD).to(dt), v=r.normal(nkv, rows, HD, std=0.5).to(dt),
                 out=torch.empty(b, nh, HD, device="cuda"), ws=torch.empty(WS_BYTES, dtype=torch.uint8, device="cuda"))
        if k == "tree":
            s["mask"], s["depth"] = _tree(b, seed)
            s.update(kn=r.normal(nkv, b, HD).to(dt), vn=r.normal(nkv, b, HD, std=0.5).to(dt))
        return s
    if k == "copy":
        dt, nb, n = DTYPES[c["dtype"]], c["bufs"], c["n"]
        s.update(src=r.normal(nb, c["nkv"], c["src_rows"], HD).to(dt), dst=r.normal(nb, c["nkv"], c["slots"], HD).to(dt))
        # a path's rows in ascending order, out of all rows
        s["idx"] = torch.sort(torch.randperm(c["src_rows"], generator=r.g, device="cuda")[:n])[0].to(torch.int32)
        per = lambda t: torch.tensor([x.data_ptr() for x in t], dtype=torch.int64, device="cuda")  # noqa: E731
        s.update(dst_ptrs=per(s["dst"]), src_ptrs=per(s["src"]))
        return s
    rows, V = c["rows"], c["vocab"]
    x = r.normal(rows, V, std=2.0)
    tgt = r.ints(0, V, rows)
    # a model's logits: some tokens stand out, the given one often among them
    x.scatter_add_(1, r.ints(0, V, rows * 8).view(rows, 8), r.normal(rows, 8, std=4.0).abs() + 6)
    x.scatter_add_(1, tgt[:, None], r.normal(rows, 1, std=4.0).abs())
    s.update(x=x.to(DTYPES[c["dtype"]]), tgt=tgt.to(torch.int32), lp=torch.empty(rows, device="cuda"),
             ent=torch.empty(rows, device="cuda"), ids=torch.empty(rows, c["k"], dtype=torch.int32, device="cuda"),
             top=torch.empty(rows, c["k"], device="cuda"))
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def _rope_plain(s):
    c, x = s["case"], s["qkv"]
    b, nh, nkv = c["b"], c["nh"], c["nkv"]
    at = c["pos0"] + (s["depth"].long() if c["tree"] else torch.arange(b, device=x.device))
    cos, sin = s["rope"][at][:, None, :, 0], s["rope"][at][:, None, :, 1]

    def turned(h, w):
        y = h * torch.rsqrt((h * h).mean(2, keepdim=True) + EPS) * w
        a, z = y[..., :64], y[..., 64:]
        return torch.cat([a * cos - z * sin, a * sin + z * cos], 2)
    s["q"].copy_(turned(x[:, :nh], s["qn"]))
    rows = slice(0, b) if c["tree"] else slice(c["pos0"], c["pos0"] + b)
    s["k"][:, rows] = turned(x[:, nh:nh + nkv], s["kn"]).transpose(0, 1).to(s["k"].dtype)
    s["v"][:, rows] = x[:, nh + nkv:].transpose(0, 1).to(s["v"].dtype)
    return dict(q=s["q"], k=s["k"], v=s["v"])


def _seen(c):
    """The positions that some row sees: [0, first) and [lo, ctx) of the cache."""
    if c["kind"] == "tree":
        return 0, 0
    lo = max(0, c["ctx"] - c["window"] + 1)
    return min(c["sinks"], lo), lo


def _visible(s, at):
    """[b, keys] truth: row i sees key at position at[x] (cache keys, then the
    new rows)."""
    c, b = s["case"], s["case"]["b"]
    if c["kind"] == "tree":
        old = torch.ones(b, c["ctx"], dtype=torch.bool, device=at.device)
        bits = (s["mask"][:, None] >> torch.arange(b, device=at.device)) & 1
        return torch.cat([old, bits.bool()], 1)
    p = c["ctx"] + torch.arange(b, device=at.device)[:, None]
    return (at <= p) & ((at > p - c["window"]) | (at < c["sinks"]))


def _attention_plain(s):
    c = s["case"]
    b, nh, nkv, ctx = c["b"], c["nh"], c["nkv"], c["ctx"]
    first, lo = _seen(c)
    if c["kind"] == "tree":
        k, v = torch.cat([s["k"], s["kn"]], 1).float(), torch.cat([s["v"], s["vn"]], 1).float()
        at = torch.arange(ctx + b, device=k.device)
    else:
        at = torch.cat([torch.arange(first, device=s["k"].device), torch.arange(lo, ctx + b, device=s["k"].device)])
        k, v = s["k"][:, at].float(), s["v"][:, at].float()
    q = s["q"].view(b, nkv, nh // nkv, HD).permute(1, 2, 0, 3).reshape(nkv, -1, HD)
    sc = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(HD ** -0.5).view(nkv, nh // nkv, b, -1)
    sc.masked_fill_(~_visible(s, at), -math.inf)
    e = sc.sub_(sc.amax(3, keepdim=True)).exp_()
    o = torch.bmm(e.view(nkv, -1, e.shape[3]), v).view(nkv, -1, b, HD) / e.sum(3, keepdim=True)
    return o.permute(2, 0, 1, 3).reshape(b, nh, HD)


def _copy_plain(s):
    c = s["case"]
    s["dst"][:, :, c["pos0"]:c["pos0"] + c["n"]] = s["src"][:, :, s["idx"].long()]
    return s["dst"]


def _logprobs_plain(s):
    x, k = s["x"].float(), s["case"]["k"]
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    z = e.sum(1, keepdim=True)
    lp = d - z.log()
    ent = z.log()[:, 0] - (e * d).sum(1) / z[:, 0]
    out = dict(lp=lp.gather(1, s["tgt"].long()[:, None])[:, 0], ent=ent)
    if k:  # equal values: the lowest id first
        ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
        out.update(ids=ids.to(torch.int32), top=lp.gather(1, ids))
    return out


def _run_own(s):
    from cmf_amd import ops
    c, k = s["case"], s["case"]["kind"]
    if k == "rope":
        ops.qk_rope(s["qkv"], s["q"], s["k"], s["v"], s["qn"], s["kn"], s["rope"], pos0=c["pos0"], depth=s["depth"],
                    at_pos=not c["tree"], eps=EPS, stream=s["stream"])
        return dict(q=s["q"], k=s["k"], v=s["v"])
    if k == "tree":
        ops.attention(s["q"], s["k"], s["v"], s["out"], s["ws"], pos0=c["ctx"], k_new=s["kn"], v_new=s["vn"],
                      mask=s["mask"], depth=s["depth"], stream=s["stream"])
        return s["out"]
    if k == "window":
        ops.attention(s["q"], s["k"], s["v"], s["out"], s["ws"], pos0=c["ctx"], window=c["window"], sinks=c["sinks"],
                      stream=s["stream"])
        return s["out"]
    if k == "copy":
        ops.kv_copy(s["dst_ptrs"], s["src_ptrs"], s["dst"][0], s["src"][0], n=c["n"], pos0=c["pos0"], idx=s["idx"],
                    stream=s["stream"])
        return s["dst"]
    if "ws" not in s:  # the scratch, made once and kept as the attention's
        s["ws"] = torch.empty(WS_BYTES, dtype=torch.uint8, device="cuda")
    ops.logprobs(s["x"], s["tgt"], s["lp"], s["ent"], s["ids"] if c["k"] else None, s["top"] if c["k"] else None, s["ws"],
                 stream=s["stream"])
    return dict(lp=s["lp"], ent=s["ent"], **(dict(ids=s["ids"], top=s["top"]) if c["k"] else {}))


def run(state):
    if own:
        return _run_own(state)
    k = state["case"]["kind"]
    if k == "rope":
        return _rope_plain(state)
    if k in ("tree", "window"):
        return _attention_plain(state)
    return _copy_plain(state) if k == "copy" else _logprobs_plain(state)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    c, k = case, case["kind"]
    es = 4 if c["dtype"] == "f32" else 2
    if k == "rope":
        b, nh, nkv = c["b"], c["nh"], c["nkv"]
        return {"bytes": b * ((nh + 2 * nkv) * HD * 4 + HD * 4 + nh * HD * 4 + 2 * nkv * HD * es),
                "flops": b * (nh + nkv) * HD * 7}
    if k == "copy":
        return {"bytes": 2 * c["bufs"] * c["nkv"] * c["n"] * HD * es, "flops": 0}
    if k == "logprobs":
        return {"bytes": c["rows"] * (c["vocab"] * es + 12 + 8 * c["k"]), "flops": c["rows"] * c["vocab"] * 6}
    b, nh, nkv, ctx = c["b"], c["nh"], c["nkv"], c["ctx"]
    first, lo = _seen(c)
    keys = first + ctx - lo + b
    if k == "tree":
        pairs = b * (ctx + 1)  # and a few ancestors a row
    else:
        pairs = 0
        for i in range(b):
            p = ctx + i
            near = min(c["window"], p + 1)
            pairs += near + min(c["sinks"], p + 1 - near)
    return {"bytes": 2 * b * nh * HD * 4 + 2 * nkv * keys * HD * es, "flops": pairs * nh * 4 * HD}


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    c, k, s = case, case["kind"], prepare(case, seed)
    if k == "copy":
        want = s["dst"].clone()
        for i in range(c["bufs"]):
            want[i].narrow(1, c["pos0"], c["n"]).copy_(torch.index_select(s["src"][i], 1, s["idx"]))
        return want.double()
    if k == "rope":
        b, nh, nkv = c["b"], c["nh"], c["nkv"]
        x = s["qkv"].double()
        at = [c["pos0"] + d for d in (s["depth"].tolist() if c["tree"] else range(b))]
        t = s["rope"].double()[torch.tensor(at, device="cuda")]
        z = torch.complex(t[..., 0], t[..., 1])[:, None]
        heads = []
        for part, w in ((x[:, :nh], s["qn"]), (x[:, nh:nh + nkv], s["kn"])):
            y = part / (part.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
            o = torch.complex(y[..., :64], y[..., 64:]) * z
            heads.append(torch.cat([o.real, o.imag], -1))
        kk, vv, r0 = s["k"].double(), s["v"].double(), 0 if c["tree"] else c["pos0"]
        kk[:, r0:r0 + b], vv[:, r0:r0 + b] = heads[1].permute(1, 0, 2), x[:, nh + nkv:].permute(1, 0, 2)
        return dict(q=heads[0], k=kk, v=vv)
    if k == "logprobs":
        x, kk = s["x"].double(), c["k"]
        ls = torch.log_softmax(x, 1)
        ent = torch.distributions.Categorical(logits=x).entropy()
        out = dict(lp=ls[torch.arange(c["rows"], device="cuda"), s["tgt"].long()], ent=ent)
        if kk:
            out.update(ids=None, top=torch.topk(ls, kk, dim=1)[0])
        return out
    b, nh, nkv, ctx = c["b"], c["nh"], c["nkv"], c["ctx"]
    out = torch.empty(b, nh, HD, dtype=torch.float64, device="cuda")
    tree = k == "tree"
    n0 = 0 if tree else min(c["sinks"], max(0, ctx - c["window"] + 1))
    n1 = 0 if tree else max(0, ctx - c["window"] + 1)
    pos = list(range(n0)) + list(range(n1, ctx + b))
    pt = torch.tensor(pos, device="cuda")
    bias = torch.zeros(b, len(pos), dtype=torch.float64, device="cuda")
    if tree:
        m = [x & ((1 << 64) - 1) for x in s["mask"].tolist()]
        sees = torch.tensor([[m[i] >> j & 1 for j in range(b)] for i in range(b)], device="cuda")
        bias[:, ctx:] = torch.where(sees == 1, 0.0, -math.inf)
    else:
        mine = ctx + torch.arange(b, device="cuda")
        bias.masked_fill_(pt[None] > mine[:, None], -math.inf)
        bias.masked_fill_((pt[None] <= mine[:, None] - c["window"]) & (pt[None] >= c["sinks"]), -math.inf)
    for h in range(nh):
        g = h // (nh // nkv)
        keys, vals = (torch.cat([s[a][g], s[a + "n"][g]]).double() if tree else s[a][g][pt].double() for a in ("k", "v"))
        out[:, h] = torch.softmax(s["q"][:, h].double() @ keys.t().contiguous() / math.sqrt(HD) + bias, 1) @ vals
    return out
