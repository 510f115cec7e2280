"""The operators of an encoder layer against their definitions in 64 bits.

Tolerances, elementwise:
* attention: the output's rounding to bf16 (2^-8 |O|), and 2^-8 sum(p |v|) for
  the rounding of the probabilities to bf16 and of the sums; with a cap, a
  score x may be off by |x| 2^-10.9 (the tanh unit's bound), which changes a
  probability by that factor and the row's sum by as much again.
* projection: 2^-8 |y| for the output, 2^-8 sum_r |u_r b_r| for the rounding of
  the adapter's inner vector, 2^-16 sum_k |x_k w_k| for fp32 sums; times the
  activation's slope (at most 1.13).
* norms: 4e-6 of the terms for fp32 streams (fp32 statistics over up to some
  thousands of values), 1e-5 of value and weight for the norm that follows,
  plus 2^-8 of a value that is returned in bf16.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from snapjudge_b200 import ops  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rnd(shape, g, scale=1.0, dtype=BF):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def cum(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


# ---- attention ------------------------------------------------------------------
def sees(m):
    """bool [query rows, keys] from the definition."""
    cu = np.asarray(m["cu"])
    T = int(cu[-1])
    seg = np.repeat(np.arange(len(cu) - 1), np.diff(cu))
    doc = seg if m.get("docs") is None else np.repeat(np.arange(len(m["docs"]) - 1),
                                                      np.diff(m["docs"]))
    i = np.arange(T) if m.get("q_rows") is None else np.asarray(m["q_rows"], int)
    j = np.arange(T)
    jr = j - cu[seg]
    ok = doc[i][:, None] == doc[j][None]
    if m.get("causal"):
        ok &= j[None] <= i[:, None]
    if m.get("window"):
        ok &= np.abs(j[None] - i[:, None]) <= m["window"]
    if m.get("prefix") is not None:
        ok |= jr[None] < np.asarray(m["prefix"])[seg[i]][:, None]
    ok &= seg[i][:, None] == seg[j][None]
    if m.get("kv_lens") is not None:
        ok &= jr[None] < np.asarray(m["kv_lens"])[seg[i]][:, None]
    return torch.from_numpy(ok).to(DEV), torch.from_numpy(i).to(DEV)


def ref_attn(q, k, v, m, scale=None, softcap=0.0, rel_bias=None, slopes=None):
    """The definition in 64 bits -> (O, tolerance), both [rows, H * Dh]."""
    ok, i = sees(m)
    n, H, Dh = q.shape
    G = H // k.shape[1]
    scale = Dh ** -0.5 if scale is None else scale
    out = torch.zeros(n, H, Dh, dtype=F64, device=DEV)
    tol = torch.zeros_like(out)
    dist = torch.arange(k.shape[0], device=DEV)[None] - i[:, None]
    for h in range(H):
        kk, vv = k[:, h // G].double(), v[:, h // G].double()
        kk, vv = (torch.where(ok.any(0)[:, None], t, 0.0) for t in (kk, vv))
        x = (q[:, h].double() @ kk.t()) * scale
        e = 2.0 ** -8
        if softcap:
            x = softcap * torch.tanh(x / softcap)
            e += 2 * (float(x[ok].abs().max()) if ok.any() else 0.0) * 2.0 ** -10.9
        if rel_bias is not None:
            R = rel_bias.shape[1] // 2
            x = x + rel_bias[h].double()[dist.clamp(-R, R) + R]
        if slopes is not None:
            x = x - slopes[h].double() * dist.abs()
        x = torch.where(ok, x, -math.inf)
        mx = x.amax(1, keepdim=True) if x.shape[1] else x.new_full((n, 1), -math.inf)
        p = torch.exp(x - torch.where(mx == -math.inf, 0.0, mx))
        z = p.sum(1, keepdim=True)
        p = p / torch.where(z == 0, 1.0, z)
        out[:, h] = p @ vv
        tol[:, h] = 2.0 ** -8 * out[:, h].abs() + e * (p @ vv.abs()) + 1e-6
    return out.reshape(n, H * Dh), tol.reshape(n, H * Dh)


def close(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, at worst "
                           f"{float(((got.double() - want).abs() / tol).max()):.3g} tolerances")


def plan_of(m, form="auto"):
    return ops.AttnPlan(m["cu"], form=form, **{k: v for k, v in m.items() if k != "cu"})


both_forms = pytest.mark.parametrize("form", ["tiles", "few"])


def check_attn(m, H, Hkv, Dh, form, seed=1, qscale=1.0, **kw):
    plan = plan_of(m, form)
    g = gen(seed)
    q = rnd((plan.n_rows, H, Dh), g, qscale)
    k, v = rnd((plan.n_keys, Hkv, Dh), g), rnd((plan.n_keys, Hkv, Dh), g)
    if "rel" in kw:
        kw["rel_bias"] = rnd((H, 2 * kw.pop("rel") + 1), g, dtype=F32)
    if kw.pop("slope", False):
        kw["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=DEV) / H)
    got = ops.attn_masked(q, k, v, plan, **kw)
    assert got.dtype == BF and got.shape == (plan.n_rows, H * Dh)
    close(got, *ref_attn(q, k, v, m, **kw))
    return got


MASKS = {
    "one row": dict(cu=[0, 1]),
    "short and empty segments": dict(cu=cum([1, 0, 7, 33, 0, 127, 128, 129, 2, 64])),
    "long": dict(cu=cum([700, 65, 1000])),
    "window": dict(cu=cum([300, 200, 1]), window=64),
    "window of one": dict(cu=cum([130, 5]), window=1),
    "causal": dict(cu=cum([300, 1, 129]), causal=True),
    "causal behind a prefix": dict(cu=cum([300, 150]), causal=True, prefix=[100, 0]),
    "short keys": dict(cu=cum([200, 100, 90, 40]), kv_lens=[200, 37, 0, 1]),
    "documents": dict(cu=cum([260, 330, 3]), docs=[0, 100, 101, 190, 260, 500, 590, 593]),
    "state and questions": dict(cu=cum([260, 330]), docs=[0, 180, 200, 230, 260, 500, 530, 590],
                                prefix=[180, 240]),
    "everything": dict(cu=cum([260, 0, 330]), docs=[0, 180, 200, 230, 260, 260, 500, 530, 590],
                       prefix=[50, 0, 200], kv_lens=[240, 0, 329], causal=True, window=9),
    "few rows ask": dict(cu=cum([400, 300, 1, 200]), q_rows=[0, 17, 399, 400, 700, 701, 900],
                         prefix=[3, 0, 0, 200]),
    "one row of a long segment asks": dict(cu=[0, 3000], q_rows=[1234]),
    "nobody asks": dict(cu=[0, 40], q_rows=[]),
    "no rows": dict(cu=[0, 0]),
}


@pytest.mark.parametrize("name", MASKS)
@pytest.mark.parametrize("H,Hkv,Dh", [(3, 3, 64), (4, 2, 128), (2, 1, 16)])
@both_forms
def test_attn_masks(name, H, Hkv, Dh, form):
    check_attn(MASKS[name], H, Hkv, Dh, form)


MODS = [dict(softcap=30.0, qscale=6.0), dict(softcap=2.0, qscale=9.0), dict(rel=32), dict(rel=0),
        dict(rel=700), dict(slope=True), dict(scale=0.7), dict(scale=0.0), dict(scale=-0.3),
        dict(softcap=50.0, qscale=6.0, rel=128, slope=True)]


@pytest.mark.parametrize("mods", MODS, ids=str)
@pytest.mark.parametrize("name", ["long", "state and questions", "everything", "few rows ask"])
@pytest.mark.parametrize("H,Hkv,Dh", [(3, 3, 64), (4, 1, 128), (2, 2, 32)])
@both_forms
def test_attn_scores(name, mods, H, Hkv, Dh, form):
    check_attn(MASKS[name], H, Hkv, Dh, form, seed=2, **mods)


@pytest.mark.parametrize("Dh", [1, 7, 8, 40, 80, 96, 100])
def test_attn_other_head_dims(Dh):
    check_attn(MASKS["state and questions"], 2, 2, Dh, "auto", seed=3, rel=16)


@pytest.mark.parametrize("H,Hkv", [(16, 1), (12, 3), (5, 5)])
@pytest.mark.parametrize("name", ["long", "few rows ask"])
@both_forms
def test_attn_shared_heads(name, H, Hkv, form):
    check_attn(MASKS[name], H, Hkv, 64, form, seed=4, slope=True)


@pytest.mark.parametrize("Dh", [64, 128, 16])
@pytest.mark.parametrize("name", ["short and empty segments", "short keys", "state and questions",
                                  "everything", "few rows ask", "window"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@both_forms
def test_attn_masked_places_never_reach_the_output(name, value, Dh, form):
    """A key that some rows do not see: what it holds changes only the rows that
    see it."""
    m = MASKS[name]
    plan = plan_of(m, form)
    ok, _ = sees(m)
    g = gen(5)
    H = 2
    q = rnd((plan.n_rows, H, Dh), g)
    k, v = rnd((plan.n_keys, H, Dh), g), rnd((plan.n_keys, H, Dh), g)
    want, tol = ref_attn(q, k, v, m)
    # five of the twenty keys that the fewest rows see
    spoilt = torch.argsort(ok.sum(0), stable=True)[:20:4]
    k[spoilt[:3]] = value
    v[spoilt[2:]] = value
    free = ~ok[:, spoilt].any(1)
    assert free.any()
    got = ops.attn_masked(q, k, v, plan)
    close(got[free], want[free], tol[free])


@pytest.mark.parametrize("Dh", [64, 128, 16])
@both_forms
def test_attn_rows_of_lowest_scores(Dh, form):
    """A bias of the type's lowest value is a score like any other: a row whose
    every key has it weighs them alike; one whose every score is -inf gives 0."""
    m = dict(cu=cum([150, 90]))
    plan = plan_of(m, form)
    g = gen(6)
    q, k, v = (rnd((240, 1, Dh), g) for _ in range(3))
    low = torch.full((1, 1), torch.finfo(F32).min, device=DEV)
    got = ops.attn_masked(q, k, v, plan, rel_bias=low)
    want, tol = ref_attn(torch.zeros_like(q), k, v, m)
    close(got, want, tol)
    got = ops.attn_masked(q, k, v, plan, rel_bias=torch.full((1, 1), -math.inf, device=DEV))
    assert (got == 0).all()
    # half of the distances: keys behind the query only
    rel = torch.zeros(1, 2 * 150 + 1, device=DEV)
    rel[:, :150] = torch.finfo(F32).min
    got = ops.attn_masked(q, k, v, plan, rel_bias=rel)
    close(got, *ref_attn(q, k, v, m, rel_bias=rel))


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("pad", [0, 8, 1])
@pytest.mark.parametrize("name", ["state and questions", "few rows ask"])
@both_forms
def test_attn_strides_and_alignment(name, pad, Dh, form):
    """Slices of a packed tensor, row pitches that are no multiple of 16 bytes,
    and tensors that start anywhere give what contiguous ones give."""
    m = MASKS[name]
    plan = plan_of(m, form)
    H, Hkv, T = 4, 2, plan.n_keys
    g = gen(7)
    flat = rnd((T, (H + 2 * Hkv) * Dh + pad), g)
    parts = [flat[:, pad + a * Dh:pad + b * Dh].unflatten(1, (b - a, Dh))
             for a, b in ((0, H), (H, H + Hkv), (H + Hkv, H + 2 * Hkv))]
    q, k, v = parts
    if m.get("q_rows") is not None:
        big = torch.zeros(plan.n_rows, 2, H * Dh + pad, dtype=BF, device=DEV)
        big[:, 1, pad:] = q[torch.as_tensor(m["q_rows"], device=DEV)].flatten(1)
        q = big[:, 1, pad:].unflatten(1, (H, Dh))
    close(ops.attn_masked(q, k, v, plan), *ref_attn(q, k, v, m))


@both_forms
def test_attn_offsets_past_32_bits(form):
    """Key rows a million elements apart: offsets above 2^31 elements."""
    T, Dh = 2300, 64
    g = gen(8)
    big = torch.empty(T << 20, dtype=BF, device=DEV)
    kv = big.as_strided((T, 2, Dh), (1 << 20, Dh, 1))
    kv.copy_(rnd((T, 2, Dh), g))
    for m in (dict(cu=[0, 2000, T], q_rows=[3, 2299]), dict(cu=[0, 2000, T])):
        plan = plan_of(m, form)
        q = rnd((plan.n_rows, 1, Dh), g)
        close(ops.attn_masked(q, kv[:, :1], kv[:, 1:], plan),
              *ref_attn(q, kv[:, :1], kv[:, 1:], m))


@both_forms
def test_attn_many_short_segments_and_repeatable(form):
    lens = np.random.default_rng(9).integers(0, 90, 900)
    m = dict(cu=cum(lens))
    plan = plan_of(m, form)
    g = gen(9)
    q, k, v = (rnd((plan.n_keys, 2, 64), g) for _ in range(3))
    got = ops.attn_masked(q, k, v, plan)
    assert torch.equal(got, ops.attn_masked(q, k, v, plan))
    for a, b in ((0, 1500), (20000, 21500)):  # two stretches of whole segments
        s0, s1 = np.searchsorted(m["cu"], [a, b])
        rows = slice(int(m["cu"][s0]), int(m["cu"][s1]))
        sub = dict(cu=np.asarray(m["cu"][s0:s1 + 1]) - m["cu"][s0])
        close(got[rows], *ref_attn(q[rows], k[rows], v[rows], sub))


@both_forms
def test_attn_long_rows_keep_their_sum(form):
    """One row over 60,000 keys of equal score: the mean of the values."""
    T = 60000
    plan = ops.AttnPlan([0, T], q_rows=[T - 1], form=form)
    v = rnd((T, 1, 64), gen(10))
    got = ops.attn_masked(torch.zeros(1, 1, 64, dtype=BF, device=DEV), rnd((T, 1, 64), gen(11)), v,
                          plan)
    want = v.double().mean(0)
    close(got, want, 2.0 ** -8 * want.abs() + 2.0 ** -8 * v.double().abs().mean(0) / 100)


@both_forms
def test_attn_on_another_stream(form):
    m = MASKS["state and questions"]
    plan = plan_of(m, form)
    g = gen(12)
    q, k, v = (rnd((plan.n_keys, 3, 64), g) for _ in range(3))
    want = ops.attn_masked(q, k, v, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.attn_masked(q, k, v, plan)
    side.synchronize()
    assert torch.equal(got, want)


def test_attn_python_refusals():
    plan = ops.AttnPlan([0, 10])
    q = torch.zeros(10, 2, 64, dtype=BF, device=DEV)
    for bad in (lambda: ops.attn_masked(q.float(), q, q, plan),
                lambda: ops.attn_masked(q[:9], q, q, plan),
                lambda: ops.attn_masked(q, q[:9], q[:9], plan),
                lambda: ops.attn_masked(q, q, q[:, :1], plan),
                lambda: ops.attn_masked(q.transpose(0, 1).contiguous().transpose(0, 1), q, q, plan),
                lambda: ops.attn_masked(q, q, q, plan, rel_bias=torch.zeros(2, 4, device=DEV)),
                lambda: ops.attn_masked(q, q, q, plan, slopes=torch.zeros(3, device=DEV)),
                lambda: ops.attn_masked(q, q, q, plan, softcap=-1.0),
                lambda: ops.attn_masked(q.cpu(), q, q, plan),
                lambda: ops.AttnPlan([0, 10], prefix=[1, 2]),
                lambda: ops.AttnPlan([0, 10.5]),
                lambda: ops.AttnPlan([0, 10], form="both"),
                lambda: ops.AttnPlan([0, 2 ** 31])):
        with pytest.raises((ValueError, RuntimeError)):
            bad()


@pytest.mark.parametrize("H,Hkv,Dh", [(3, 3, 64), (6, 2, 64), (4, 1, 128), (3, 3, 128)])
@pytest.mark.parametrize("keys,parts", [(130, 2), (150, 3), (250, 4), (370, 6), (500, 8), (700, 11)])
def test_attn_masked_few_joins(H, Hkv, Dh, keys, parts):
    """Parts of a group joined in a block (up to 8) or by the second kernel; masked values
    hold NaN."""
    m = dict(cu=cum([keys, keys]), q_rows=[3, 11, keys - 1, keys, keys + 40],
             kv_lens=[keys - 3, keys - 6])
    plan = plan_of(m, "few")
    assert plan.info.n_parts == 2 * parts and plan.info.join == (parts if parts <= 8 else 0)
    g = gen(5)
    q = rnd((5, H, Dh), g)
    k, v = rnd((2 * keys, Hkv, Dh), g), rnd((2 * keys, Hkv, Dh), g)
    ok, _ = sees(m)
    slopes = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=DEV) / H)
    want, tol = ref_attn(q, k, v, m, slopes=slopes)
    clean = ops.attn_masked(q, k, v, plan, slopes=slopes)
    close(clean, want, tol)
    v[~ok.any(0)] = math.nan
    close(ops.attn_masked(q, k, v, plan, slopes=slopes), want, tol)


# ---- projection with adapters -------------------------------------------------------
def ref_lora(x, w, a, b, rows, scale=None, bias=None, act=0):
    x, w, a, b = (t.double() for t in (x, w, a, b))
    y = x @ w.t()
    tol = 2.0 ** -16 * (x.abs() @ w.abs().t())
    if bias is not None:
        y = y + bias.double()
    for n in range(a.shape[0]):
        mine = (rows == n).nonzero().flatten()
        u = x[mine] @ a[n].t() * (1.0 if scale is None else scale[n].double())
        y[mine] += u @ b[n].t()
        tol[mine] += 2.0 ** -8 * (u.abs() @ b[n].abs().t())
    if act == 1:
        y = y * torch.special.ndtr(y)
    elif act == 2:
        y = torch.relu(y)
    return y, 1.13 * tol + 2.0 ** -8 * y.abs() + 1e-6


def lora_inputs(cu, ids, N, K, R, n, seed, scaled=True, biased=False):
    g = gen(seed)
    M = int(cu[-1])
    t = dict(x=rnd((M, K), g), w=rnd((N, K), g, K ** -0.5), a=rnd((n, R, K), g, K ** -0.5),
             b=rnd((n, N, R), g, 0.5 * R ** -0.5))
    kw = dict(scale=rnd((n,), g, dtype=F32) if scaled else None,
              bias=rnd((N,), g, dtype=F32) if biased else None)
    rows = torch.from_numpy(np.repeat(np.asarray(ids), np.diff(cu))).to(DEV)
    return t, kw, rows, ops.LoraPlan(cu, ids, rank=R, n_adapters=n)


LORA = [
    # (lengths, adapters of the segments, n, N, K, R)
    ([1], [0], 1, 64, 64, 8),
    ([1], [-1], 2, 64, 64, 16),
    ([37], [2], 4, 2304, 768, 16),
    ([5, 0, 1, 130, 7], [1, 0, 1, -1, 0], 2, 96, 48, 16),
    ([100, 200, 300, 13], [3, 1, 3, 0], 4, 768, 768, 32),
    ([1] * 300, list(range(-1, 59)) * 5, 60, 768, 768, 8),  # a row each
    ([1] * 260, list(range(130)) * 2, 130, 128, 128, 64),   # more adapters than one pass holds
    ([90, 40, 128, 128, 3], [0, 1, 2, 1, 0], 3, 2816, 1024, 64),
    ([255, 1, 256, 2], [0, 1, 0, 1], 2, 136, 72, 24),       # widths that no tile divides
    ([700, 800, 900, 41], [2, 0, 1, 2], 3, 2304, 768, 16),  # tiles of two CTAs
    ([64, 32] * 40, [0, 1, -1, 2] * 20, 3, 1000, 520, 8),
    ([300], [0], 1, 100, 60, 12),                           # rows that are no whole 16 bytes
    ([33], [0], 1, 33, 31, 5),
    ([50], [0], 1, 256, 256, 130),
]


@pytest.mark.parametrize("lens,ids,n,N,K,R", LORA)
@pytest.mark.parametrize("act,biased,scaled", [(0, False, True), (1, True, True), (2, True, False)])
def test_lora(lens, ids, n, N, K, R, act, biased, scaled):
    cu = cum(lens)
    t, kw, rows, plan = lora_inputs(cu, ids, N, K, R, n, 21, scaled, biased)
    got = ops.gemm_lora(t["x"], t["w"], t["a"], t["b"], plan, act=act, **kw)
    assert got.dtype == BF and got.shape == (int(cu[-1]), N)
    close(got, *ref_lora(t["x"], t["w"], t["a"], t["b"], rows, act=act, **kw))


@pytest.mark.parametrize("lens,ids,n,N,K,R", [
    ([1] * 21, [0, 2, -1, 1, 3, 0, 0] * 3, 4, 72, 264, 8),  # adapters that change with every row
    ([17, 15, 1], [0, -1, 1], 2, 768, 8, 16),               # K below one step of a warp
    ([3, 30], [1, 0], 2, 40, 1000, 24),                     # two slabs an adapter, N within a tile
    ([16], [0], 1, 2304, 768, 64),                          # two rounds of slabs
    ([64], [0], 1, 2304, 768, 16),                          # the most rows in one launch there
    ([65], [0], 1, 2304, 768, 16),                          # ... and one more
    ([12, 12], [1, 0], 2, 64, 64, 40),                      # more slabs than one launch takes
])
def test_lora_few_rows(lens, ids, n, N, K, R):
    cu = cum(lens)
    t, kw, rows, plan = lora_inputs(cu, ids, N, K, R, n, 27, biased=True)
    want, tol = ref_lora(t["x"], t["w"], t["a"], t["b"], rows, act=1, **kw)
    close(ops.gemm_lora(t["x"], t["w"], t["a"], t["b"], plan, act=1, **kw), want, tol)
    for name in ("a", "b"):  # a spoilt adapter stays with its rows
        s = dict(t)
        s[name] = t[name].clone()
        s[name][0] = math.nan
        got = ops.gemm_lora(s["x"], s["w"], s["a"], s["b"], plan, act=1, **kw)
        close(got[rows != 0], want[rows != 0], tol[rows != 0])
        assert not torch.isfinite(got[rows == 0]).any()


@pytest.mark.parametrize("lens", [[40, 200, 60], [900, 900, 900]])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_lora_a_spoilt_adapter_stays_with_its_rows(lens, value):
    cu, ids = cum(lens), [0, 1, -1]
    t, kw, rows, plan = lora_inputs(cu, ids, 768, 768, 16, 2, 22)
    want, tol = ref_lora(t["x"], t["w"], t["a"], t["b"], rows, **kw)
    for name in ("a", "b"):
        s = dict(t)
        s[name] = t[name].clone()
        s[name][1, ::3, ::5] = value
        got = ops.gemm_lora(s["x"], s["w"], s["a"], s["b"], plan, **kw)
        others = rows != 1
        close(got[others], want[others], tol[others])
        assert not torch.isfinite(got[~others]).all()
    x = t["x"].clone()  # a spoilt row stays one row
    x[45] = value
    got = ops.gemm_lora(x, t["w"], t["a"], t["b"], plan, **kw)
    others = torch.arange(len(rows), device=DEV) != 45
    close(got[others], want[others], tol[others])
    assert not torch.isfinite(got[45]).any()


@pytest.mark.parametrize("pad", [8, 1])
def test_lora_row_pitch(pad):
    cu, ids = cum([130, 300]), [1, 0]
    t, kw, rows, plan = lora_inputs(cu, ids, 256, 192, 16, 2, 23)
    big = torch.full((430, 192 + pad), math.nan, dtype=BF, device=DEV)
    big[:, pad:] = t["x"]
    got = ops.gemm_lora(big[:, pad:], t["w"], t["a"], t["b"], plan, **kw)
    close(got, *ref_lora(t["x"], t["w"], t["a"], t["b"], rows, **kw))


def test_lora_repeatable_and_on_another_stream():
    cu, ids = cum([1000, 1200, 300]), [1, 0, 1]
    t, kw, rows, plan = lora_inputs(cu, ids, 768, 768, 16, 2, 24)
    call = lambda: ops.gemm_lora(t["x"], t["w"], t["a"], t["b"], plan, **kw)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert torch.equal(got, want)


def test_lora_without_rows_and_refusals():
    t, kw, _, plan = lora_inputs(cum([0]), [0], 64, 64, 8, 1, 25)
    assert ops.gemm_lora(t["x"], t["w"], t["a"], t["b"], plan).shape == (0, 64)
    t, kw, _, plan = lora_inputs(cum([4]), [0], 64, 64, 8, 1, 25)
    x, w, a, b = t["x"], t["w"], t["a"], t["b"]
    for bad in (lambda: ops.gemm_lora(x.float(), w, a, b, plan),
                lambda: ops.gemm_lora(x[:3], w, a, b, plan),
                lambda: ops.gemm_lora(x, w[:, :32], a, b, plan),
                lambda: ops.gemm_lora(x, w, a[:, :4], b, plan),
                lambda: ops.gemm_lora(x, w, a, b[:, :32], plan),
                lambda: ops.gemm_lora(x, w, a, b, plan, act=3),
                lambda: ops.gemm_lora(x, w, a, b, plan, bias=torch.zeros(63, device=DEV)),
                lambda: ops.LoraPlan([0, 4], [1], rank=8, n_adapters=1),
                lambda: ops.LoraPlan([0, 4], [0, 0], rank=8, n_adapters=1)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()


# ---- norms, gate and residual -----------------------------------------------------------
def ref_norm_block(x, r, pre_w, pre_b, post_w, post_b, kind, gate, mode, rows, alpha, beta, eps):
    d = lambda t: None if t is None else t.double()  # noqa: E731

    def norm(v, w, b):
        if kind == "ln":
            v = v - v.mean(1, keepdim=True)
        v = v / (v.square().mean(1, keepdim=True) + eps).sqrt() * d(w)
        return v if b is None else v + d(b)

    z = d(r) if post_w is None else norm(d(r), post_w, post_b)
    size = z.abs() if post_w is None else z.abs() + post_w.double().abs()
    if mode:
        g = d(gate)
        g = {"channel": lambda: g, "segment": lambda: g[rows], "row": lambda: torch.sigmoid(g)}[mode]()
        z, size = z * g, size * g.abs()
    xo = alpha * d(x) + beta * z
    xtol = 4e-6 * ((alpha * d(x)).abs() + abs(beta) * size) + 1e-12
    y = None if pre_w is None else norm(xo, pre_w, pre_b)
    return xo, xtol, y


def check_norm(M, D, kind="ln", post=True, bias=False, mode=None, xt=F32, rt=BF, yt=BF, gt=BF,
               alpha=1.0, beta=1.0, pre=True, inplace=False, seed=31, pad=0, lens=None):
    g = gen(seed)

    def mat(dtype, scale=1.0):
        return rnd((M, D + pad), g, scale, dtype)[:, pad:]

    x, r = mat(xt, 3.0), mat(rt)
    vec = lambda on, one: rnd((D,), g, 0.2, F32) + one if on else None  # noqa: E731
    post_w, post_b = vec(post, 1.0), vec(post and bias, 0.0)
    pre_w, pre_b = vec(pre, 1.0), vec(pre and bias, 0.0)
    gate = rows = cu = None
    if mode == "channel":
        gate = rnd((D,), g, dtype=F32)
    elif mode == "segment":
        lens = lens or [0, M // 3, 0, M - M // 3, 0]
        gate, cu = rnd((len(lens), D), g, dtype=F32), torch.from_numpy(cum(lens)).to(DEV)
        rows = torch.from_numpy(np.repeat(np.arange(len(lens)), lens)).to(DEV)
    elif mode == "row":
        gate = mat(gt, 2.0)
    x0 = x.clone()
    xo, y = ops.norm_block(x, r, pre_w, pre_b, post_w=post_w, post_b=post_b, kind=kind, eps=1e-5,
                           gate=gate, cu=cu, alpha=alpha, beta=beta, out_dtype=yt, inplace=inplace)
    assert (xo.data_ptr() == x.data_ptr()) == inplace or M == 0
    assert inplace or torch.equal(x, x0)
    want, xtol, wy = ref_norm_block(x0, r, pre_w, pre_b, post_w, post_b, kind, gate, mode, rows,
                                    alpha, beta, 1e-5)
    close(xo, want, xtol + (2.0 ** -8 * want.abs() if xt == BF else 0))
    if pre:
        assert y.dtype == yt
        close(y, wy, 1e-5 * (wy.abs() + pre_w.double().abs()) + (2.0 ** -8 * wy.abs() if yt == BF
                                                                 else 0))
    else:
        assert y is None


@pytest.mark.parametrize("M,D", [(1, 768), (37, 768), (300, 1024), (65, 64), (9, 100), (7, 1),
                                 (12, 3), (30, 7), (30, 9), (31, 130), (50, 257), (50, 385),
                                 (33, 510), (33, 641), (33, 774), (33, 899), (33, 1001), (40, 1021),
                                 (40, 1023), (20, 1536), (20, 2043), (9, 2048), (9, 2047),
                                 (5, 4093), (5, 4095), (6, 5599), (6, 5601),
                                 (3, 8192), (3, 16384), (2, 9001), (2, 20000)])
@pytest.mark.parametrize("kind,bias", [("ln", True), ("rms", False)])
def test_norm_block_widths(M, D, kind, bias):
    if D == 1 and kind == "ln":
        return  # a row of one value has no variance
    check_norm(M, D, kind, True, bias, "channel")


@pytest.mark.parametrize("mode", [None, "channel", "segment", "row"])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("D", [768, 515, 12000])
def test_norm_block_gates(mode, post, D):
    check_norm(130, D, "ln", post, True, mode, alpha=0.7, beta=1.3)


@pytest.mark.parametrize("xt", [F32, BF])
@pytest.mark.parametrize("rt", [F32, BF])
@pytest.mark.parametrize("yt", [F32, BF])
@pytest.mark.parametrize("D", [768, 1001, 8200, 9001])
def test_norm_block_types(xt, rt, yt, D):
    check_norm(41, D, "rms", True, False, "row", xt, rt, yt, gt=F32 if xt == BF else BF)


@pytest.mark.parametrize("D", [768, 1001, 2000, 20001])
def test_norm_block_in_place_and_without_a_following_norm(D):
    check_norm(19, D, inplace=True, mode="channel")
    check_norm(19, D, xt=BF, inplace=True, pre=False)


@pytest.mark.parametrize("pad", [1, 2, 4])
@pytest.mark.parametrize("D", [768, 1536])
def test_norm_block_row_pitch(pad, D):
    check_norm(33, D, mode="row", pad=pad)


def test_norm_block_many_segments():
    lens = np.random.default_rng(32).integers(0, 4, 3000).tolist()
    check_norm(sum(lens), 96, mode="segment", lens=lens)


def test_norm_block_no_rows_and_refusals():
    check_norm(0, 64, mode="channel")
    x = torch.zeros(4, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    for bad in (lambda: ops.norm_block(x.half(), x, w), lambda: ops.norm_block(x, x[:3], w),
                lambda: ops.norm_block(x, x, w[:63]), lambda: ops.norm_block(x, x, w, kind="l2"),
                lambda: ops.norm_block(x, x, w, gate=torch.ones(63, device=DEV)),
                lambda: ops.norm_block(x, x, w, gate=x[:3]),
                lambda: ops.norm_block(x, x, w, eps=-1.0),
                lambda: ops.norm_block(x, x, w, post_b=w),
                lambda: ops.norm_block(x.t().contiguous().t(), x, w)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
