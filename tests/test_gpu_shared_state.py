"""The shared-state example: its layers (adapters, masked attention, fused norms)
against the same layers in plain 64-bit torch, and its independence of how the
questions are packed."""
import importlib.util
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("shared_state",
                                                  os.path.join(ROOT, "examples", "shared_state.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain(m, ids, lens, kind):
    """encode() in 64 bits, one state at a time."""
    H, Dh = m["H"], m["D"] // m["H"]
    d = lambda t: t.double()  # noqa: E731

    def ln(v, w):
        v = v - v.mean(1, keepdim=True)
        return v / (v.square().mean(1, keepdim=True) + 1e-5).sqrt() * d(w)

    def project(x, w, a, b, kinds):
        y = x @ d(w).t()
        for n in range(m["types"]):
            mine = kinds == n
            y[mine] += 2.0 * (x[mine] @ d(a[n]).t()) @ d(b[n]).t()
        return y

    out, at = [], 0
    for row, kn in zip(lens, kind):
        n = int(row.sum())
        doc = torch.from_numpy(np.repeat(np.arange(len(row)), row)).cuda()
        kinds = torch.from_numpy(np.repeat(kn, row)).cuda()
        sees = (doc[:, None] == doc[None]) | (doc[None] == 0)
        dist = torch.arange(n, device="cuda")[None] - torch.arange(n, device="cuda")[:, None]
        x = d(m["emb"])[ids[at:at + n]]
        at += n
        x = x + 0
        for w in m["layers"]:
            q, k, v = project(ln(x, w["pre1"]), w["wqkv"], w["aqkv"], w["bqkv"],
                              kinds).view(n, 3, H, Dh).unbind(1)
            R = w["rel"].shape[1] // 2
            s = torch.einsum("ihd,jhd->hij", q, k) * Dh ** -0.5
            s = s + d(w["rel"])[:, dist.clamp(-R, R) + R]
            o = torch.softmax(s.masked_fill(~sees, -torch.inf), 2)
            o = torch.einsum("hij,jhd->ihd", o, v).reshape(n, -1)
            x = x + d(w["gate1"]) * ln(project(o, w["wo"], w["ao"], w["bo"], kinds), w["post1"])
            g, u = (ln(x, w["pre2"]) @ d(w["wi"]).t()).chunk(2, 1)
            f = (g * torch.special.ndtr(g) * u) @ d(w["wo2"]).t()
            x = x + d(w["gate2"]) * ln(f, w["post2"])
        first = np.cumsum(row)[:-1]
        out.append(ln(x, m["final"])[torch.from_numpy(first).cuda()] @ d(m["head"]))
    return torch.cat(out)


def test_example_against_plain_layers(ex):
    """Scores are sums of D = 128 products of normed values (unit size) with weights
    of size 1 / sqrt(D); three layers of bf16 activations leave each normed value
    within a few 2^-8, so a score within 8 x 2^-8."""
    m = ex.make_model(D=128, H=2, F=256, layers=3, rank=8, types=3, reach=16, vocab=50)
    ids, lens, kind = ex.make_batch(7, 4, 3, vocab=50, lo=3, hi=150, qlo=1, qhi=20)
    got = ex.encode(m, ids, ex.plans(m, lens, kind)).double()
    want = plain(m, ids, lens, kind)
    assert got.shape == want.shape == (28,)
    assert float((got - want).abs().max()) <= 8 * 2.0 ** -8


def test_questions_do_not_see_each_other(ex):
    """Other tokens in one question leave every other question's score as it was."""
    m = ex.make_model(D=128, H=2, F=256, layers=2, rank=8, types=3, reach=16, vocab=50)
    ids, lens, kind = ex.make_batch(3, 5, 3, vocab=50, lo=30, hi=150, qlo=5, qhi=20)
    plan = ex.plans(m, lens, kind)
    before = ex.encode(m, ids, plan)
    docs = np.concatenate([[0], np.cumsum(lens.reshape(-1))])
    other = ids.clone()
    a, b = docs[2], docs[3]  # the first state's second question
    other[a:b] = (other[a:b] + 1) % 50
    after = ex.encode(m, other, plan)
    assert after[1] != before[1]
    keep = torch.arange(15) != 1
    assert torch.equal(after[keep], before[keep])
