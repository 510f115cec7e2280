"""The cases that the encoder-layer operators are measured on: masked and biased
attention, projections with an adapter for each request, and the step of norms,
gate and residual between two blocks.

``run`` makes one pass through an operator.  With ``own`` false it is the plain
form: elementary torch operations in 32 bits, rounded once at the end.  With
``own`` true it is the framework's call (``snapjudge_b200.ops``).  ``exact``
gives the same outputs in 64 bits from the definitions.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- cases --------------------------------------------------------------------
def _attn(name, **kw):
    # segs segments; each has lo..hi rows and, with docs > 0, that many documents of
    # doc_lo..doc_hi rows behind them.  prefix: "" none, "first" the rows before the
    # documents, "part" a random part of the segment.  q_rows > 0: at most that many
    # rows of a segment ask (its first among them), else all do.
    c = {"name": name, "op": "attn", "segs": 1, "lo": 1, "hi": 1, "docs": 0, "doc_lo": 8,
         "doc_hi": 32, "prefix": "", "H": 12, "Hkv": 12, "Dh": 64, "causal": False, "window": 0,
         "cap": 0.0, "rel": 0, "slopes": False, "short_keys": False, "q_rows": 0, "packed": True}
    c.update(kw)
    return c


def _lora(name, **kw):
    # segs requests of lo..hi rows, each with one of `adapters` adapters or none
    c = {"name": name, "op": "lora", "segs": 1, "lo": 1, "hi": 1, "K": 768, "N": 768, "rank": 16,
         "adapters": 4, "bias": False, "act": 0}
    c.update(kw)
    return c


def _norm(name, **kw):
    # M rows of D; gate: "" none, "channel" [D], "segment" [segs, D], "row" sigmoid of [M, D]
    c = {"name": name, "op": "norm", "M": 1, "D": 768, "kind": "ln", "post": True, "bias": False,
         "gate": "channel", "segs": 1, "alpha": 1.0, "x": "float32", "r": "bfloat16",
         "y": "bfloat16"}
    c.update(kw)
    return c


def listed():
    return [
        # one request alone: a state and its four questions in one segment (latency)
        _attn("attn one request", lo=180, hi=180, docs=4, doc_lo=14, doc_hi=30, prefix="first",
              rel=128),
        # a serving batch at the base width: 256 states, six questions about each
        _attn("attn shared states", segs=256, lo=96, hi=400, docs=6, doc_lo=10, doc_hi=40,
              prefix="first", rel=128),
        # the long-sequence batch at the large width: capped scores and a linear distance bias
        _attn("attn long capped", segs=16, lo=2048, hi=2048, H=16, Hkv=16, cap=30.0, slopes=True),
        # wide heads that share keys, causal behind a prefix, padded key ends, separate tensors
        _attn("attn wide heads", segs=12, lo=701, hi=1499, H=8, Hkv=2, Dh=128, prefix="part",
              causal=True, cap=50.0, short_keys=True, packed=False),
        # a batch's last layer, where only the [CLS] and option rows ask
        _attn("attn marker rows", segs=512, lo=32, hi=512, q_rows=4, rel=64),
        # one short request through the QKV projection with its adapter (latency)
        _lora("lora one request", lo=37, hi=37, N=2304),
        # a batch's [CLS] rows, each with the adapter of its own request
        _lora("lora single rows", segs=600, N=768, rank=8, adapters=64, bias=True),
        # a pass of short requests through the QKV projection
        _lora("lora short requests", segs=1024, lo=16, hi=112, N=2304, adapters=48),
        # longer requests at the large width, a feed-forward projection with its activation
        _lora("lora wide rank", segs=150, lo=100, hi=300, K=1024, N=2816, rank=64, adapters=12,
              bias=True, act=1),
        # the step between two blocks for one short request (latency)
        _norm("norm one request", M=37),
        # the same for a pass at the base width
        _norm("norm base pass", M=131072),
        # an odd width, root-mean-square norms, a gate for each request, a 16-bit stream
        _norm("norm odd width", M=30011, D=1001, kind="rms", gate="segment", segs=211, alpha=0.7,
              x="bfloat16", r="float32", y="float32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _unnamed(c):
    del c["name"]
    return c


def draw(rng):
    op = rng.choice(["attn", "attn", "lora", "norm"])
    if op == "attn":
        few = rng.random() < 0.3
        hi = _log(rng, 24, 1900)
        docs = 0 if few or rng.random() < 0.4 else rng.randint(1, 7)
        doc_hi = rng.randint(6, 32)
        Hkv, group = rng.choice([2, 3, 4]), rng.choice([1, 2, 4])
        # the padded scores stay below those of the largest listed case
        most = int(8e8 / (Hkv * group * (hi + docs * doc_hi) ** 2))
        return _unnamed(_attn(
            "", segs=max(1, min(_log(rng, 1, 300), most)), lo=max(1, int(hi * rng.uniform(0.2, 1))),
            hi=hi, docs=docs, doc_lo=5, doc_hi=doc_hi,
            prefix=rng.choice(["first", "part"]) if docs else rng.choice(["", "part"]),
            H=Hkv * group, Hkv=Hkv, Dh=rng.choice([64, 64, 128]), causal=rng.random() < 0.3,
            window=rng.choice([0, 0, 64, 128]), cap=rng.choice([0.0, 30.0, 50.0]),
            rel=rng.choice([0, 32, 128]), slopes=rng.random() < 0.3,
            short_keys=rng.random() < 0.3, q_rows=rng.randint(1, 8) if few else 0,
            packed=rng.random() < 0.5))
    if op == "lora":
        hi = _log(rng, 1, 400)
        return _unnamed(_lora(
            "", segs=max(1, min(_log(rng, 1, 1500), 40000 // hi)),
            lo=max(1, int(hi * rng.uniform(0.2, 1))), hi=hi, K=8 * rng.randint(32, 128),
            N=8 * rng.randint(32, 288), rank=rng.choice([8, 16, 24, 32, 64]),
            adapters=rng.randint(1, 12), bias=rng.random() < 0.5, act=rng.choice([0, 1, 2])))
    gate = rng.choice(["", "channel", "segment", "row"])
    M = _log(rng, 1, 60000)
    return _unnamed(_norm(
        "", M=M, D=rng.randint(200, 1600), kind=rng.choice(["ln", "rms"]),
        post=rng.random() < 0.7, bias=rng.random() < 0.5, gate=gate,
        segs=rng.randint(1, max(1, M // 20)), alpha=rng.choice([1.0, 0.5, 1.2]),
        x=rng.choice(["float32", "float32", "bfloat16"]), r=rng.choice(["bfloat16", "float32"]),
        y=rng.choice(["bfloat16", "float32"])))


# ---- shapes: the same for every seed ------------------------------------------------
def _cum(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


def _shape(c):
    """Lengths and masks of a case as host arrays."""
    r = np.random.default_rng(sum(ord(ch) * (k + 1) for k, ch in enumerate(
        repr(sorted((k, v) for k, v in c.items() if k != "name")))))
    if c["op"] == "norm":
        cuts = np.sort(r.integers(0, c["M"] + 1, c["segs"] - 1))
        return {"cu": np.concatenate([[0], cuts, [c["M"]]]).astype(np.int32)}
    state = r.integers(c["lo"], c["hi"] + 1, c["segs"])
    if c["op"] == "lora":
        return {"cu": _cum(state), "ids": r.integers(-1, c["adapters"], c["segs"]).astype(np.int32)
                if c["segs"] > 1 else np.zeros(1, np.int32)}
    parts = np.concatenate([state[:, None], r.integers(c["doc_lo"], c["doc_hi"] + 1,
                                                       (c["segs"], c["docs"]))], 1)
    n = parts.sum(1)
    cu = _cum(n)
    s = {"cu": cu, "docs": _cum(parts.reshape(-1)) if c["docs"] else None, "prefix": None,
         "kv_lens": None, "q_rows": None}
    if c["prefix"]:
        s["prefix"] = (state if c["prefix"] == "first" else
                       (n * r.random(c["segs"])).astype(int)).astype(np.int32)
    if c["short_keys"]:
        s["kv_lens"] = (n - (n * 0.3 * r.random(c["segs"])).astype(int)).astype(np.int32)
    if c["q_rows"]:
        more = cu[:-1, None] + (r.random((c["segs"], c["q_rows"] - 1)) * n[:, None]).astype(np.int32)
        s["q_rows"] = np.unique(np.concatenate([cu[:-1, None], more], 1)).astype(np.int32)
    return s


def _seg_of(cu, rows):
    return np.searchsorted(cu[1:], rows, side="right")


def _visible_pairs(c, s):
    """Pairs (query row, key row) that the masks leave."""
    T = int(s["cu"][-1])
    i = s["q_rows"].astype(np.int64) if s["q_rows"] is not None else np.arange(T)
    b = _seg_of(s["cu"], i)
    s0, e0 = s["cu"][b], s["cu"][b + 1]
    end = s0 + s["kv_lens"][b] if s["kv_lens"] is not None else e0
    lo, hi = s0, e0
    if s["docs"] is not None:
        d = _seg_of(s["docs"], i)
        lo, hi = s["docs"][d], s["docs"][d + 1]
    if c["causal"]:
        hi = np.minimum(hi, i + 1)
    if c["window"]:
        lo, hi = np.maximum(lo, i - c["window"]), np.minimum(hi, i + c["window"] + 1)
    hi = np.minimum(hi, end)
    pe = np.minimum(s0 + s["prefix"][b], end) if s["prefix"] is not None else s0
    both = np.maximum(0, np.minimum(hi, pe) - np.maximum(lo, s0))
    return int((np.maximum(0, hi - lo) + (pe - s0) - both).sum())


def work(case):
    s = _shape(case)
    if case["op"] == "attn":
        T = int(s["cu"][-1])
        Tq = T if s["q_rows"] is None else len(s["q_rows"])
        return {"bytes": 2 * case["Dh"] * (2 * Tq * case["H"] + 2 * T * case["Hkv"]),
                "flops": 4 * case["Dh"] * case["H"] * _visible_pairs(case, s)}
    if case["op"] == "lora":
        T, K, N, R = int(s["cu"][-1]), case["K"], case["N"], case["rank"]
        rows = int(np.diff(s["cu"])[s["ids"] >= 0].sum())
        used = len(set(s["ids"][s["ids"] >= 0].tolist()))
        return {"bytes": 2 * (T * K + N * K + T * N + used * R * (K + N)),
                "flops": 2 * T * K * N + 2 * rows * R * (K + N)}
    sz = {"bfloat16": 2, "float32": 4}
    per = 2 * sz[case["x"]] + sz[case["r"]] + sz[case["y"]] + (2 if case["gate"] == "row" else 0)
    extra = 4 * case["D"] * (4 + (case["segs"] if case["gate"] == "segment" else 0))
    return {"bytes": case["M"] * case["D"] * per + extra, "flops": 20 * case["M"] * case["D"]}


# ---- inputs -----------------------------------------------------------------------
def _tensors(c, s, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    f32 = torch.float32
    if c["op"] == "attn":
        T, H, Hkv, Dh = int(s["cu"][-1]), c["H"], c["Hkv"], c["Dh"]
        qs = 6.0 if c["cap"] else 1.0  # capped models have scores that reach their cap
        t = {}
        if c["packed"] and s["q_rows"] is None:
            qkv = rnd(T, H + 2 * Hkv, Dh)
            qkv[:, :H] *= qs
            t["q"], t["k"], t["v"] = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        else:
            t["q"] = rnd(T if s["q_rows"] is None else len(s["q_rows"]), H, Dh, scale=qs)
            kv = rnd(T, 2 * Hkv, Dh)
            t["k"], t["v"] = kv[:, :Hkv], kv[:, Hkv:]
        t["rel"] = rnd(H, 2 * c["rel"] + 1, dtype=f32) if c["rel"] else None
        t["slopes"] = (2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H)) \
            if c["slopes"] else None
        return t
    if c["op"] == "lora":
        T, K, N, R, n = int(s["cu"][-1]), c["K"], c["N"], c["rank"], c["adapters"]
        return {"x": rnd(T, K), "w": rnd(N, K, scale=K ** -0.5), "a": rnd(n, R, K, scale=K ** -0.5),
                "b": rnd(n, N, R, scale=0.3 * R ** -0.5),
                "scale": 0.5 + torch.rand(n, generator=g, device="cuda"),
                "bias": rnd(N, scale=0.1, dtype=f32) if c["bias"] else None}
    M, D = c["M"], c["D"]
    shape = {"channel": (D,), "segment": (c["segs"], D), "row": (M, D)}.get(c["gate"])
    t = {"x": rnd(M, D, scale=3.0, dtype=_TYPES[c["x"]]), "r": rnd(M, D, dtype=_TYPES[c["r"]]),
         "gate": None if shape is None else rnd(*shape, dtype=torch.bfloat16 if c["gate"] == "row"
                                                else f32)}
    for k, there in (("post_w", c["post"]), ("post_b", c["post"] and c["bias"]), ("pre_w", True),
                     ("pre_b", c["bias"])):
        t[k] = rnd(D, scale=0.2, dtype=f32) + (1.0 if k.endswith("w") else 0.0) if there else None
    return t


def prepare(case, seed):
    s = _shape(case)
    state = {"case": case, "shape": s, "t": _tensors(case, s, seed)}
    dev = {k: torch.from_numpy(v).cuda() for k, v in s.items() if v is not None}
    state["dev"] = dev  # lengths, documents and adapter numbers, as a program holds them
    if own:
        # the batch's plan, which a program makes once and uses in every layer
        from snapjudge_b200 import ops
        if case["op"] == "attn":
            state["plan"] = ops.AttnPlan(s["cu"], docs=s["docs"], prefix=s["prefix"],
                                         kv_lens=s["kv_lens"], q_rows=s["q_rows"],
                                         causal=case["causal"], window=case["window"])
        elif case["op"] == "lora":
            state["plan"] = ops.LoraPlan(s["cu"], s["ids"], rank=case["rank"],
                                         n_adapters=case["adapters"])
    return state


# ---- one pass -----------------------------------------------------------------------
def run(state):
    c, t = state["case"], state["t"]
    if not own:
        return {"attn": _plain_attn, "lora": _plain_lora, "norm": _plain_norm}[c["op"]](state)
    from snapjudge_b200 import ops
    if c["op"] == "attn":
        return ops.attn_masked(t["q"], t["k"], t["v"], state["plan"], softcap=c["cap"],
                               rel_bias=t["rel"], slopes=t["slopes"])
    if c["op"] == "lora":
        return ops.gemm_lora(t["x"], t["w"], t["a"], t["b"], state["plan"], scale=t["scale"],
                             bias=t["bias"], act=c["act"])
    return ops.norm_block(t["x"], t["r"], t["pre_w"], t["pre_b"], post_w=t["post_w"],
                          post_b=t["post_b"], kind=c["kind"], gate=t["gate"],
                          cu=state["dev"]["cu"] if c["gate"] == "segment" else None,
                          alpha=c["alpha"], out_dtype=_TYPES[c["y"]])


def _plain_attn(state):
    c, s, t, d = state["case"], state["shape"], state["t"], state["dev"]
    H, Hkv, Dh = c["H"], c["Hkv"], c["Dh"]
    cu = d["cu"].long()
    n = cu[1:] - cu[:-1]
    Lk = int(np.diff(s["cu"]).max())  # host arrays give the padded sizes
    jr = torch.arange(Lk, device="cuda")
    kidx = (cu[:-1, None] + jr).clamp(max=int(s["cu"][-1]) - 1)  # [B, Lk]
    if s["q_rows"] is None:
        pos, qidx, has_q = jr.expand(len(n), Lk), kidx, jr < n[:, None]
    else:
        rows = d["q_rows"].long()
        seg = torch.searchsorted(cu[1:].contiguous(), rows, right=True)
        first = torch.searchsorted(seg, torch.arange(len(n) + 1, device="cuda"))
        qidx = first[:-1, None] + torch.arange(c["q_rows"], device="cuda")
        has_q = qidx < first[1:, None]
        qidx = qidx.clamp(max=len(rows) - 1)
        pos = rows[qidx] - cu[:-1, None]
    q = t["q"].float()[qidx].transpose(1, 2)
    k = t["k"].float()[kidx].transpose(1, 2).repeat_interleave(H // Hkv, 1)
    v = t["v"].float()[kidx].transpose(1, 2).repeat_interleave(H // Hkv, 1)
    x = torch.matmul(q, k.transpose(2, 3))
    x *= Dh ** -0.5
    if c["cap"]:
        x.div_(c["cap"]).tanh_().mul_(c["cap"])
    dist = jr - pos[..., None]  # [B, Lq, Lk]
    if c["rel"]:
        x += t["rel"][:, dist.clamp(-c["rel"], c["rel"]) + c["rel"]].transpose(0, 1)
    if c["slopes"]:
        x -= t["slopes"][:, None, None] * dist.abs()[:, None]
    end = d["kv_lens"].long() if s["kv_lens"] is not None else n
    sees = torch.ones_like(dist, dtype=torch.bool)
    if s["docs"] is not None:
        doc = torch.searchsorted(d["docs"].long()[1:].contiguous(), kidx, right=True)
        sees &= doc[:, None, :] == doc.gather(1, pos.clamp(max=Lk - 1))[..., None]
    if c["causal"]:
        sees &= dist <= 0
    if c["window"]:
        sees &= dist.abs() <= c["window"]
    if s["prefix"] is not None:
        sees |= jr < d["prefix"].long()[:, None, None]
    sees &= jr < end[:, None, None]
    x.masked_fill_(~sees[:, None], -math.inf)
    m = x.amax(3, keepdim=True)
    x -= torch.where(m == -math.inf, 0.0, m)
    x.exp_()
    z = x.sum(3, keepdim=True)
    o = torch.matmul(x, v) / torch.where(z > 0, z, 1.0)
    return o.transpose(1, 2)[has_q].reshape(-1, H * Dh).to(torch.bfloat16)


def _plain_lora(state):
    c, t, d = state["case"], state["t"], state["dev"]
    x, n, R = t["x"].float(), c["adapters"], c["rank"]
    y = torch.matmul(x, t["w"].float().t())
    u = torch.matmul(x, t["a"].float().reshape(n * R, c["K"]).t()).reshape(-1, n, R)
    cu = d["cu"].long()
    mine = d["ids"].long()[torch.searchsorted(cu[1:].contiguous(),
                                              torch.arange(len(x), device="cuda"), right=True)]
    u *= ((mine[:, None] == torch.arange(n, device="cuda")) * t["scale"])[..., None]
    y += torch.matmul(u.reshape(-1, n * R), t["b"].float().transpose(1, 2).reshape(n * R, c["N"]))
    if t["bias"] is not None:
        y += t["bias"]
    if c["act"] == 1:
        y = 0.5 * y * (1 + torch.erf(y * 0.7071067811865476))
    elif c["act"] == 2:
        y = torch.where(y > 0, y, 0.0)
    return y.to(torch.bfloat16)


def _plain_one_norm(x, w, b, kind):
    if kind == "ln":
        x = x - x.mean(1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-5) * w
    return y if b is None else y + b


def _plain_norm(state):
    c, t, d = state["case"], state["t"], state["dev"]
    z = t["r"].float()
    if c["post"]:
        z = _plain_one_norm(z, t["post_w"], t["post_b"], c["kind"])
    if c["gate"] == "channel":
        z = z * t["gate"]
    elif c["gate"] == "segment":
        seg = torch.searchsorted(d["cu"].long()[1:].contiguous(),
                                 torch.arange(c["M"], device="cuda"), right=True)
        z = z * t["gate"][seg]
    elif c["gate"] == "row":
        z = z / (1 + torch.exp(-t["gate"].float()))
    x = t["x"].float() * c["alpha"] + z
    y = _plain_one_norm(x, t["pre_w"], t["pre_b"], c["kind"])
    return x.to(_TYPES[c["x"]]), y.to(_TYPES[c["y"]])


# ---- the definitions in 64 bits ---------------------------------------------------------
def exact(case, seed):
    s = _shape(case)
    t = {k: None if v is None else v.double() for k, v in _tensors(case, s, seed).items()}
    return {"attn": _exact_attn, "lora": _exact_lora, "norm": _exact_norm}[case["op"]](case, s, t)


def _exact_attn(c, s, t):
    H, g, Dh, cu = c["H"], c["H"] // c["Hkv"], c["Dh"], s["cu"]
    rows = s["q_rows"] if s["q_rows"] is not None else np.arange(cu[-1])
    out = torch.zeros(len(rows), H, Dh, dtype=torch.float64, device="cuda")
    for b in range(c["segs"]):
        a, e = np.searchsorted(rows, cu[b]), np.searchsorted(rows, cu[b + 1])
        keys = slice(int(cu[b]), int(cu[b + 1]))
        i = torch.from_numpy(rows[a:e].astype(np.int64)).cuda()[:, None]
        j = torch.arange(keys.start, keys.stop, device="cuda")[None]
        ok = torch.ones(e - a, keys.stop - keys.start, dtype=torch.bool, device="cuda")
        if s["docs"] is not None:
            at = torch.from_numpy(s["docs"]).cuda().long()[1:-1].contiguous()
            ok &= torch.bucketize(i, at, right=True) == torch.bucketize(j, at, right=True)
        if c["causal"]:
            ok &= i >= j
        if c["window"]:
            ok &= ((i - j) <= c["window"]) & ((j - i) <= c["window"])
        if s["prefix"] is not None:
            ok |= j < int(cu[b]) + int(s["prefix"][b])
        if s["kv_lens"] is not None:
            ok &= j < int(cu[b]) + int(s["kv_lens"][b])
        x = torch.einsum("ihd,jhd->hij", t["q"][a:e],
                         t["k"][keys].repeat_interleave(g, 1)) / math.sqrt(Dh)
        if c["cap"]:
            x = c["cap"] * torch.tanh(x / c["cap"])
        if c["rel"]:
            x = x + t["rel"][:, torch.clamp(j - i, -c["rel"], c["rel"]) + c["rel"]]
        if c["slopes"]:
            x = x - t["slopes"][:, None, None] * (i - j).abs()
        w = torch.softmax(torch.where(ok, x, -math.inf), 2)
        w = torch.where(ok.any(1)[None, :, None], w, 0.0)
        out[a:e] = torch.einsum("hij,jhd->ihd", w, t["v"][keys].repeat_interleave(g, 1))
    return out.reshape(len(rows), H * Dh)


def _exact_lora(c, s, t):
    out = t["x"] @ t["w"].t()
    if t["bias"] is not None:
        out += t["bias"]
    row_ids = np.repeat(s["ids"], np.diff(s["cu"]))
    for n in range(c["adapters"]):
        rows = torch.from_numpy(np.nonzero(row_ids == n)[0]).cuda()
        out[rows] += t["scale"][n] * ((t["x"][rows] @ t["a"][n].t()) @ t["b"][n].t())
    if c["act"] == 1:
        return torch.special.ndtr(out) * out
    return torch.relu(out) if c["act"] == 2 else out


def _exact_norm(c, s, t):
    def norm(v, w, b):
        if c["kind"] == "ln":
            v = (v - v.mean(1, keepdim=True)) / (v.var(1, correction=0, keepdim=True) + 1e-5).sqrt()
        else:
            v = v / (v.square().mean(1, keepdim=True) + 1e-5).sqrt()
        return v * w + (0.0 if b is None else b)

    z = norm(t["r"], t["post_w"], t["post_b"]) if c["post"] else t["r"]
    if c["gate"] == "channel":
        z = z * t["gate"]
    elif c["gate"] == "segment":
        z = z * t["gate"].repeat_interleave(torch.from_numpy(np.diff(s["cu"])).cuda(), 0)
    elif c["gate"] == "row":
        z = z * torch.sigmoid(t["gate"])
    x = c["alpha"] * t["x"] + z
    # the second norm reads the new stream before it is rounded
    return x, norm(x, t["pre_w"], t["pre_b"])
