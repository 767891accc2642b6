"""Single operators through their public entry points: what a step of many answers to one prompt needs beside the layers' products.

``sample_tokens`` picks a token per row of logits from a given uniform number, with temperature, top-k, top-p and min-p.
``attention_shared_prefix`` is the attention of one new token per sequence where all sequences share their first cache rows
and each goes on in rows of its own.

Where ``own`` is false, ``run`` computes the operators' plain forms from elementary torch operations, in 32 bits (64 for the masses and cumulative
sums of sampling, whose borders decide on whole numbers).
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

VOCAB = 151936


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the vocabulary of the small test models, one row: a call's own latency
        dict(name="sample_1x4096", op="sample", rows=1, vocab=4096, type="fp32", filters="all"),
        # one sequence of the full vocabulary: token by token, interactive
        dict(name="sample_1x151936", op="sample", rows=1, vocab=VOCAB, type="fp32", filters="all"),
        # an odd vocabulary in fp16, rows behind one another without padding (no row but the first is aligned)
        dict(name="sample_7x32003_fp16", op="sample", rows=7, vocab=32003, type="fp16", filters="top_p"),
        # a step of 32 sequences with top-k and top-p
        dict(name="sample_32x151936", op="sample", rows=32, vocab=VOCAB, type="fp32", filters="all"),
        # a full step: 128 sequences, every row with its own options
        dict(name="sample_128x151936", op="sample", rows=128, vocab=VOCAB, type="fp32", filters="mixed"),
        # plain temperature sampling, nothing filtered, bf16 logits
        dict(name="sample_64x151936_bf16", op="sample", rows=64, vocab=VOCAB, type="bf16", filters="none"),
        # two answers behind a short prompt: latency
        dict(name="attend_2_128", op="attend", seqs=2, q_heads=16, kv_heads=8, dim=128, prefix=128, own=16, type="fp16"),
        # sixteen answers to a 2048-token prompt
        dict(name="attend_16_2048", op="attend", seqs=16, q_heads=16, kv_heads=8, dim=128, prefix=2048, own=256, type="fp16"),
        # other head layout, 64-wide bf16 heads, odd lengths, sequences without rows of their own
        dict(name="attend_33_1000_bf16", op="attend", seqs=33, q_heads=32, kv_heads=4, dim=64, prefix=1000, own=333, type="bf16"),
        # a few answers to a very long document
        dict(name="attend_8_32768", op="attend", seqs=8, q_heads=16, kv_heads=8, dim=128, prefix=32768, own=64, type="fp16"),
        # sixty-four requests behind a 4096-token system prompt
        dict(name="attend_64_4096", op="attend", seqs=64, q_heads=16, kv_heads=8, dim=128, prefix=4096, own=512, type="fp16"),
        # a full batch behind a long document
        dict(name="attend_128_16384", op="attend", seqs=128, q_heads=16, kv_heads=8, dim=128, prefix=16384, own=128, type="fp16"),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over the logarithm."""
    return int(round(low * (high / low) ** rng.random()))


def draw(rng: random.Random):
    if rng.random() < 0.5:
        vocab = rng.choice((4096, VOCAB, VOCAB, _between(rng, 1000, 200000)))
        return dict(op="sample", rows=_between(rng, 1, min(256, 128 * VOCAB // vocab)), vocab=vocab, type=rng.choice(("fp32", "fp32", "fp16", "bf16")),
                    filters=rng.choice(("all", "mixed", "top_p", "top_k", "none")))
    dim = rng.choice((64, 128, 128))
    kv_heads = rng.choice((1, 2, 4, 8, 8, 8))
    q_heads = kv_heads * rng.choice((1, 2, 2, 3, 4, 8))
    seqs = _between(rng, 1, 128)
    prefix = _between(rng, 1, 32768)
    while 4 * q_heads * dim * seqs * prefix > 4 * 16 * 128 * 128 * 16384:      # no more than the largest listed one
        prefix //= 2
    return dict(op="attend", seqs=seqs, q_heads=q_heads, kv_heads=kv_heads, dim=dim, prefix=prefix,
                own=_between(rng, 1, 512), type=rng.choice(("fp16", "fp16", "bf16")))


TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}


def _own_lengths(case):
    """Rows of their own that the sequences have, in no particular order: evenly spread over 0 .. own."""
    n = case["seqs"]
    return [case["own"] * (i + 1) // n if i or n < 3 else 0 for i in range(n)]


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZES[case["type"]] + case["rows"] * (5 * 4 + 2 * 4), "flops": 3 * n}
    heads, dim, e = case["q_heads"], case["dim"], SIZES[case["type"]]
    lens = sum(_own_lengths(case))
    return {"bytes": 2 * e * case["kv_heads"] * dim * (case["prefix"] + lens) + case["seqs"] * (heads * (2 * dim * e + 4) + 4),
            "flops": 4 * heads * dim * (case["seqs"] * case["prefix"] + lens)}


# ---------------------------------------------------------------------------------------------------------- inputs
def _options(case, rng):
    """Per row: temperature, top_k, top_p, min_p."""
    rows, kind = case["rows"], case["filters"]
    temperature = [rng.uniform(0.5, 1.3) for _ in range(rows)]
    top_k, top_p, min_p = [0] * rows, [1.0] * rows, [0.0] * rows
    for i in range(rows):
        use = rng.sample(("top_k", "top_p", "min_p"), rng.randrange(4)) if kind == "mixed" else ("top_k", "top_p") if kind == "all" else (kind,)
        if "top_k" in use:
            top_k[i] = rng.choice((1, 20, 50, 50, 200, 1000))
        if "top_p" in use:
            top_p[i] = rng.choice((0.5, 0.8, 0.9, 0.95, 0.99))
        if "min_p" in use:
            min_p[i] = rng.choice((0.01, 0.05, 0.1))
        if kind == "mixed" and rng.random() < 0.1:
            temperature[i] = 0.0
    return temperature, top_k, top_p, min_p


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    dt = TYPES[case["type"]]
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a language model's logits: a broad bulk, a few hundred plausible tokens, a handful of likely ones
        logits = torch.randn(rows, vocab, device="cuda", generator=gen).mul_(2.0)
        for count, low, high in ((max(1, vocab // 400), 2.0, 6.0), (8, 7.0, 12.0)):
            at = torch.randint(0, vocab, (rows, count), device="cuda", generator=gen)
            logits.scatter_add_(1, at, torch.empty(rows, count, device="cuda").uniform_(low, high, generator=gen))
        temperature, top_k, top_p, min_p = _options(case, rng)
        return dict(case=case, logits=logits.to(dt), uniforms=torch.rand(rows, device="cuda", generator=gen),
                    temperature=torch.tensor(temperature, dtype=torch.float32).cuda(), top_k=torch.tensor(top_k, dtype=torch.int32).cuda(),
                    top_p=torch.tensor(top_p, dtype=torch.float32).cuda(), min_p=torch.tensor(min_p, dtype=torch.float32).cuda())
    seqs, heads, dim = case["seqs"], case["kv_heads"], case["dim"]

    def rows_of(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=gen).mul_(scale).to(dt)

    lens = _own_lengths(case)
    rng.shuffle(lens)
    # normalised and rotated heads: entries around one, some larger
    gain = torch.empty(dim, device="cuda").uniform_(0.5, 2.0, generator=gen)
    return dict(case=case, q=(torch.randn(seqs, case["q_heads"], dim, device="cuda", generator=gen) * gain).to(dt),
                k_prefix=rows_of(heads, case["prefix"], dim), v_prefix=rows_of(heads, case["prefix"], dim),
                k_own=rows_of(seqs, heads, case["own"], dim), v_own=rows_of(seqs, heads, case["own"], dim),
                own_lens=torch.tensor(lens, dtype=torch.int32).cuda())


# ---------------------------------------------------------------------------------------------------------- the operators
def _ops():
    package = os.path.join(os.getcwd(), "qwen3-0.6b-megakernel-rtx-5090_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import qwen_megakernel_C
    return qwen_megakernel_C


def run(state):
    if state["case"]["op"] == "sample":
        args = [state[k] for k in ("logits", "uniforms", "temperature", "top_k", "top_p", "min_p")]
        tokens, logprobs = _ops().sample_tokens(*args) if own else _plain_sample(*args)
        return {"tokens": tokens, "logprobs": logprobs}
    args = [state[k] for k in ("q", "k_prefix", "v_prefix", "k_own", "v_own", "own_lens")]
    out, lse = _ops().attention_shared_prefix(*args) if own else _plain_attention(*args)
    return {"out": out, "lse": lse}


def _plain_sample(logits, uniforms, temperature, top_k, top_p, min_p):
    vocab = logits.shape[1]
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(1, keepdim=True)
    greedy = (~(temperature > 0))[:, None]
    t = torch.where(greedy, 1.0, temperature.double()[:, None])
    w = torch.where(x == top, 1.0, torch.where(x == -math.inf, 0.0, torch.exp((x - top) / t)))
    # the kept tokens are the first of the order: descending values, ties by ascending index
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    rank = torch.arange(vocab, device=x.device)[None]
    limit = torch.where((top_k <= 0) | (top_k > vocab), vocab, top_k)[:, None]
    ordered = torch.where(rank < limit, w.gather(1, order), 0.0)
    mass = ordered.cumsum(1)
    before = torch.cat((torch.zeros_like(mass[:, :1]), mass[:, :-1]), 1)
    p = top_p.double()[:, None]
    keep = (rank < limit) & ((before < p * mass[:, -1:]) | (p >= 1)) & (ordered >= min_p.double()[:, None]) & ~greedy
    keep[:, 0] = True
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    # lowest index whose cumulative mass exceeds u times the total
    w = torch.where(kept, w, 0.0)
    total = w.sum(1, keepdim=True)
    target = (uniforms.double()[:, None] * total).clamp_min(0.0)
    last = torch.where(kept, rank, -1).amax(1, keepdim=True)
    pick = torch.minimum(torch.searchsorted(w.cumsum(1), target, right=True), last)
    logprob = torch.log(w.gather(1, pick) / total)
    empty = top == -math.inf
    return torch.where(empty, 2 ** 31 - 1, pick)[:, 0].int(), torch.where(empty, math.nan, logprob)[:, 0].float()


def _plain_attention(q, k_prefix, v_prefix, k_own, v_own, own_lens):
    seqs, q_heads, dim = q.shape
    kv_heads = k_prefix.shape[0]
    group = q_heads // kv_heads
    qf = q.float().view(seqs, kv_heads, group, dim) / math.sqrt(dim)
    sp = torch.matmul(qf.permute(1, 0, 2, 3).reshape(kv_heads, seqs * group, dim), k_prefix.float().transpose(1, 2))
    sp = sp.view(kv_heads, seqs, group, -1).transpose(0, 1)
    visible = (torch.arange(k_own.shape[2], device=q.device) < own_lens[:, None])[:, None, None, :]
    so = torch.where(visible, torch.matmul(qf, k_own.float().transpose(2, 3)), -math.inf)
    s = torch.cat((sp, so), 3)
    top = s.amax(3, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(3, keepdim=True)
    ep, eo = e[..., :sp.shape[3]], e[..., sp.shape[3]:]
    o = torch.matmul(ep.transpose(0, 1).reshape(kv_heads, seqs * group, -1), v_prefix.float())
    o = o.view(kv_heads, seqs, group, dim).transpose(0, 1)
    o = o + torch.matmul(eo, torch.where(visible[:, :, 0, :, None], v_own.float(), 0.0))
    o = torch.where(total > 0, o / total, 0.0)
    return o.reshape(seqs, q_heads, dim).to(q.dtype), (top + torch.log(total)).view(seqs, q_heads)


# ---------------------------------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        tokens, logprobs = [], []
        x_all = s["logits"].double().cpu().numpy()
        opts = [s[k].double().cpu().numpy() for k in ("uniforms", "temperature", "top_k", "top_p", "min_p")]
        for x, u, t, k, p, mp in zip(x_all, *opts):
            by_value = np.argsort(-x, kind="stable")
            if t > 0:
                w = np.exp((x - x[by_value[0]]) / t).astype(np.longdouble)
                if 1 <= k < len(x):
                    by_value = by_value[:int(k)]
                if p < 1:
                    running = np.cumsum(w[by_value])
                    by_value = by_value[:1 + int(np.sum(running[:-1] < np.longdouble(p) * running[-1]))]
                by_value = by_value[:max(1, int(np.sum(w[by_value] >= mp)))]
            else:
                w, by_value = np.ones(len(x), np.longdouble), by_value[:1]
            ids = np.sort(by_value)
            running = np.cumsum(w[ids])
            at = min(int(np.sum(running <= np.longdouble(u) * running[-1])), len(ids) - 1)
            tokens.append(int(ids[at]))
            logprobs.append(float(np.log(w[ids[at]] / running[-1])))
        return {"tokens": torch.tensor(tokens, dtype=torch.int32), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}
    group = case["q_heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for h in range(case["q_heads"]):
        kp, vp = s["k_prefix"][h // group].double(), s["v_prefix"][h // group].double()
        scores = s["q"][:, h].double() @ kp.T * case["dim"] ** -0.5
        for b, n in enumerate(s["own_lens"].tolist()):
            k, v = s["k_own"][b, h // group, :n].double(), s["v_own"][b, h // group, :n].double()
            row = torch.cat((scores[b], k @ s["q"][b, h].double() * case["dim"] ** -0.5))
            lse[b, h] = torch.logsumexp(row, 0)
            weights = torch.exp(row - lse[b, h])
            out[b, h] = weights[:case["prefix"]] @ vp + weights[case["prefix"]:] @ v
    return {"out": out, "lse": lse}
