"""Many typed questions about one state, the state encoded once.

Asked one by one, every (state, question) pair is a sequence of its own and the
state is encoded again for each question.  Here a state and all of its questions
are one packed segment, [state | question 1 | question 2 | ...]: every question
sees the state (a prefix) and itself (a document), the state sees itself, and
question i uses the low-rank adapters of its type beside the shared projections.
A layer is

    qkv = X Wqkv^T + adapter;   a = attention(qkv) Wo^T + adapter
    x  += scale_1 * post_1(a);  y = pre_2(x)          (one norm_block)
    f   = GEGLU(y) Wo2^T
    x  += scale_2 * post_2(f);  y = pre_1 of the next layer (x)

with a distance bias instead of rotary positions (a distance counts packed rows,
so it also counts the questions between a question and the state; the table's
last entries stand for everything further away).  In the last layer only the
first row of each question asks.

    python examples/shared_state.py            # base width, 64 states of 8 questions
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from snapjudge_b200 import ops  # noqa: E402

BF = torch.bfloat16


def make_model(D=768, H=12, F=2048, layers=6, rank=16, types=4, reach=64, vocab=1000, seed=0):
    """Random weights: per layer the projections, their adapters (one pair for each
    question type) and norm, layer-scale and bias vectors."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, scale=0.05, dtype=BF):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def near(v):
        return rnd(D, scale=0.1, dtype=torch.float32) + v

    m = {"D": D, "H": H, "rank": rank, "types": types, "emb": rnd(vocab, D, scale=1.0,
                                                                  dtype=torch.float32),
         "final": near(1.0), "scale": torch.full((types,), 2.0, device="cuda"),
         "head": rnd(D, scale=D ** -0.5, dtype=torch.float32), "layers": []}
    for _ in range(layers):
        m["layers"].append({
            "pre1": near(1.0), "post1": near(1.0), "gate1": near(0.3), "pre2": near(1.0),
            "post2": near(1.0), "gate2": near(0.3),
            "wqkv": rnd(3 * D, D), "aqkv": rnd(types, rank, D), "bqkv": rnd(types, 3 * D, rank),
            "wo": rnd(D, D), "ao": rnd(types, rank, D), "bo": rnd(types, D, rank),
            "wi": rnd(2 * F, D), "wo2": rnd(D, F),
            "rel": rnd(H, 2 * reach + 1, scale=0.5, dtype=torch.float32)})
    return m


def make_batch(states, questions, types, vocab=1000, lo=96, hi=400, qlo=10, qhi=40, seed=1):
    """Token ids and lengths: row s holds the state's length and its questions'."""
    r = np.random.default_rng(seed)
    lens = np.concatenate([r.integers(lo, hi + 1, (states, 1)),
                           r.integers(qlo, qhi + 1, (states, questions))], 1)
    kind = np.concatenate([np.full((states, 1), -1), r.integers(0, types, (states, questions))], 1)
    ids = torch.from_numpy(r.integers(0, vocab, int(lens.sum()))).cuda()
    return ids, lens, kind


def plans(m, lens, kind):
    """What a batch's lengths fix for every layer."""
    cu = np.concatenate([[0], np.cumsum(lens.sum(1))]).astype(np.int32)
    docs = np.concatenate([[0], np.cumsum(lens.reshape(-1))]).astype(np.int32)
    ask = docs[:-1].reshape(lens.shape)[:, 1:].reshape(-1)  # first row of each question
    masks = dict(docs=docs, prefix=lens[:, 0])
    adapters = kind.reshape(-1)
    return {"all": ops.AttnPlan(cu, **masks), "ask": ops.AttnPlan(cu, q_rows=ask, **masks),
            "lora": ops.LoraPlan(docs, adapters, rank=m["rank"], n_adapters=m["types"]),
            "lora_ask": ops.LoraPlan(np.arange(len(ask) + 1), kind[:, 1:].reshape(-1),
                                     rank=m["rank"], n_adapters=m["types"]),
            "rows": torch.from_numpy(ask).cuda().long()}


def encode(m, ids, plan):
    """A score for each question, [questions]."""
    H, Dh = m["H"], m["D"] // m["H"]
    x = m["emb"][ids]
    y = ops.add_ln(x, None, m["layers"][0]["pre1"])
    for n, w in enumerate(m["layers"]):
        last = n == len(m["layers"]) - 1
        qkv = ops.gemm_lora(y, w["wqkv"], w["aqkv"], w["bqkv"], plan["lora"], scale=m["scale"])
        q, k, v = qkv.view(-1, 3, H, Dh).unbind(1)
        if last:
            q, x = q[plan["rows"]], x[plan["rows"]]
        o = ops.attn_masked(q, k, v, plan["ask" if last else "all"], rel_bias=w["rel"])
        a = ops.gemm_lora(o, w["wo"], w["ao"], w["bo"], plan["lora_ask" if last else "lora"],
                          scale=m["scale"])
        x, y = ops.norm_block(x, a, w["pre2"], post_w=w["post1"], gate=w["gate1"], inplace=True)
        f = ops.gemm(ops.gemm_geglu(y, w["wi"]), w["wo2"])
        after = m["final"] if last else m["layers"][n + 1]["pre1"]
        x, y = ops.norm_block(x, f, after, post_w=w["post2"], gate=w["gate2"], inplace=True,
                              out_dtype=torch.float32 if last else BF)
    return y @ m["head"]


def main():
    m = make_model()
    ids, lens, kind = make_batch(64, 8, m["types"])
    plan = plans(m, lens, kind)
    for _ in range(3):
        scores = encode(m, ids, plan)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(10):
        scores = encode(m, ids, plan)
    end.record()
    torch.cuda.synchronize()
    alone = int((lens[:, :1] + lens[:, 1:]).sum())
    print(f"{scores.numel()} questions about {len(lens)} states in {start.elapsed_time(end) / 10:.3f} "
          f"ms: {len(ids)} rows instead of {alone} with a sequence for each question")


if __name__ == "__main__":
    main()
