"""Caches kept in 4 or 8 bits, through their public entry points: rows quantised as they are written and read back, a cache read back
whole, and the attention of a decode step over such a cache.

A packed row (the keys or values that a head has at a position) is ``dim * bits / 8`` bytes of codes and a 16-byte trailer: per quarter of the
dimensions a scale s (fp16, four of them) and a centre z (fp16, four).  A value is z + s (n - 2^(bits - 1)) with n its code; s is a
(2^bits - 1)-th of the quarter's range, z its lowest value + 2^(bits - 1) s, n the nearest code.  Dimension ``dim/4 b + dim/32 g + j`` has the code at
index ``dim/8 g + dim/32 b + j`` of the row (4 bits: the low half of a byte first).

Where ``own`` is false, ``run`` computes the operators' plain forms from elementary torch operations, in 32 bits (64 where a value's
code is chosen: values next to a border).
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------- cases
def _update(name, seqs, rows, kv_heads=8, dim=128, bits=4, type="fp16", cache=2048, ragged=False):
    return dict(name=name, op="update", seqs=seqs, rows=rows, kv_heads=kv_heads, dim=dim, bits=bits, type=type, cache=cache, ragged=ragged)


def _read(name, seqs, rows, kv_heads=8, dim=128, bits=4, type="fp16", ragged=False):
    return dict(name=name, op="read", seqs=seqs, rows=rows, kv_heads=kv_heads, dim=dim, bits=bits, type=type, cache=rows, ragged=ragged)


def _attend(name, seqs, rows, q_heads=16, kv_heads=8, dim=128, bits=4, type="fp16", ragged=True):
    return dict(name=name, op="attend", seqs=seqs, rows=rows, q_heads=q_heads, kv_heads=kv_heads, dim=dim, bits=bits, type=type, cache=rows, ragged=ragged)


def listed():
    return [
        # a decode step of one sequence: its new row, a call's own latency
        _update("update_1x1", 1, 1),
        # a decode step of a full batch, every sequence at its own position
        _update("update_128x1", 128, 1, cache=4096),
        # prompts of different lengths in bf16, an odd head layout, 8 bits
        _update("update_7x333_bf16_b8", 7, 333, kv_heads=3, dim=64, bits=8, type="bf16", cache=1001, ragged=True),
        # a long prompt of a layer, as its prefill leaves it
        _update("update_4x4096", 4, 4096, cache=4096),
        # a short cache of odd lengths read back in bf16
        _read("read_5x777_bf16_b8", 5, 777, kv_heads=4, dim=64, bits=8, type="bf16", ragged=True),
        # a sequence that was set aside comes back: the rows of all 28 layers
        _read("read_28x4096", 28, 4096),
        # one sequence behind a short prompt: latency
        _attend("attend_1x128", 1, 128, ragged=False),
        # one sequence behind a very long document
        _attend("attend_1x32768", 1, 32768, ragged=False),
        # other head layout, 64-wide bf16 heads, 8 bits, odd lengths, a sequence that has no rows yet
        _attend("attend_33x1000_bf16_b8", 33, 1000, q_heads=32, kv_heads=4, dim=64, bits=8, type="bf16"),
        # a small batch at the usual context
        _attend("attend_16x2048", 16, 2048),
        # a batch of long contexts, 8 bits
        _attend("attend_64x4096_b8", 64, 4096, bits=8),
        # a full batch of long contexts
        _attend("attend_128x8192", 128, 8192),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over the logarithm."""
    return int(round(low * (high / low) ** rng.random()))


def draw(rng: random.Random):
    op = rng.choice(("update", "read", "attend", "attend"))
    kv_heads, dim = rng.choice((1, 2, 3, 4, 8, 8, 8)), rng.choice((64, 128, 128))
    case = dict(op=op, kv_heads=kv_heads, dim=dim, bits=rng.choice((4, 4, 8)), type=rng.choice(("fp16", "fp16", "bf16")), ragged=rng.random() < 0.6)
    seqs = _between(rng, 1, 128)
    if op == "attend":
        q_heads, rows = kv_heads * rng.choice((1, 2, 2, 3, 4, 8, 16)), _between(rng, 1, 32768)
        while seqs * rows * (4 * q_heads * dim + 8 * kv_heads * _row_bytes(case)) > 128 * 8192 * (4 * 16 * 128 + 8 * 8 * 80):      # no more than the largest listed one
            rows //= 2
        return dict(case, seqs=seqs, q_heads=q_heads, rows=max(rows, 1), cache=max(rows, 1))
    rows = 1 if op == "update" and rng.random() < 0.3 else _between(rng, 1, 4096)
    while seqs * rows * kv_heads * dim > (4 if op == "update" else 28) * 4096 * 8 * 128:
        rows //= 2
    rows = max(rows, 1)
    return dict(case, seqs=seqs, rows=rows, cache=max(rows, _between(rng, rows, 4096)) if op == "update" else rows)


def _row_bytes(case):
    return case["dim"] * case["bits"] // 8 + 16


def _lengths(case):
    """Rows that the sequences have, in no particular order: all of them, or evenly spread over 0 .. rows."""
    n, rows = case["seqs"], case["rows"]
    if not case["ragged"]:
        return [rows] * n
    return [rows * (i + 1) // n if i or n < 3 else 0 for i in range(n)]


def work(case):
    pairs = 2 * case["kv_heads"] * sum(_lengths(case))              # packed rows: keys and values
    dim, packed = case["dim"], _row_bytes(case)
    out = 2 * case["kv_heads"] * case["seqs"] * case["rows"]        # rows of the outputs, those that are zeros among them
    if case["op"] == "update":
        return {"bytes": pairs * (2 * dim + 2 * packed) + out * 2 * dim, "flops": 8 * pairs * dim}
    if case["op"] == "read":
        return {"bytes": pairs * packed + out * 2 * dim, "flops": 2 * pairs * dim}
    return {"bytes": pairs * packed + case["seqs"] * (case["q_heads"] * (4 * dim + 4) + 4), "flops": 4 * case["q_heads"] * dim * sum(_lengths(case))}


# ---------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    dt = TYPES[case["type"]]
    seqs, heads, rows, dim = case["seqs"], case["kv_heads"], case["rows"], case["dim"]
    # normalised and rotated keys: entries around one, some channels with an offset; values smaller, centred
    gain = torch.empty(dim, device="cuda").uniform_(0.5, 2.0, generator=gen)
    offset = torch.randn(heads, 1, dim, device="cuda", generator=gen) * (torch.rand(dim, device="cuda", generator=gen) < 0.1)

    def rows_of(n, keys):
        x = torch.randn(n, heads, rows, dim, device="cuda", generator=gen)
        return (x * gain + 4 * offset if keys else x * 0.5).to(dt)

    lens = _lengths(case)
    rng.shuffle(lens)
    state = dict(case=case, lens=torch.tensor(lens, dtype=torch.int32).cuda())
    if case["op"] == "update":
        # rows as a layer's projections make them: [sequence, row, head, dim], handed over as views with the heads in front
        k, v = (rows_of(seqs, keys).transpose(1, 2).contiguous().transpose(1, 2) for keys in (True, False))
        starts = [rng.randint(0, case["cache"] - rows) for _ in range(seqs)]
        caches = [torch.zeros(seqs, heads, case["cache"], _row_bytes(case), dtype=torch.uint8, device="cuda") for _ in range(2)]
        return dict(state, k=k, v=v, starts=torch.tensor(starts, dtype=torch.int32).cuda(), k_cache=caches[0], v_cache=caches[1])
    caches = []
    for keys in (True, False):
        cache = torch.empty(seqs, heads, rows, _row_bytes(case), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 26) // (heads * rows * dim))
        for at in range(0, seqs, step):
            n = min(step, seqs - at)
            cache[at:at + n] = _pack(rows_of(n, keys), case["bits"])
        caches.append(cache)
    state.update(k_cache=caches[0], v_cache=caches[1])
    if case["op"] == "attend":
        state["q"] = (torch.randn(seqs, case["q_heads"], dim, device="cuda", generator=gen) * gain).to(dt)
    return state


# ---------------------------------------------------------------------------------------------------------- the operators
def _ops():
    package = os.path.join(os.getcwd(), "qwen3-0.6b-megakernel-rtx-5090_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import qwen_megakernel_C
    return qwen_megakernel_C


def run(state):
    case = state["case"]
    if case["op"] == "attend":
        args = [state[k] for k in ("q", "k_cache", "v_cache", "lens")]
        out, lse = _ops().attention_packed_cache(*args) if own else _plain_attention(*args)
        return {"out": out, "lse": lse}
    caches, rows, dim, dt, lens = (state["k_cache"], state["v_cache"]), case["rows"], case["dim"], TYPES[case["type"]], state["lens"]
    starts = None
    if case["op"] == "update":
        starts = state["starts"]
        if own:
            _ops().write_cache_packed(state["k"], state["v"], *caches, starts, lens)
        else:
            _plain_write(state["k"], caches[0], starts, lens)
            _plain_write(state["v"], caches[1], starts, lens)
    if own:
        k, v = _ops().read_cache_packed(*caches, rows, dim, dt, starts=starts, lens=lens)
    else:
        k, v = _plain_read(caches[0], rows, dim, dt, starts, lens), _plain_read(caches[1], rows, dim, dt, starts, lens)
    return {"k": k, "v": v}


def _pack(x, bits):
    """Packed rows ``[..., dim * bits / 8 + 16]`` of values ``[..., dim]``."""
    dim, middle = x.shape[-1], 1 << (bits - 1)
    x = x.double().unflatten(-1, (4, dim // 4))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((high - low) / (2 ** bits - 1)).half()
    z = (low + middle * s.double()).half()
    n = torch.where(s > 0, torch.round((x - z.double()) / torch.where(s > 0, s, 1.0).double()), 0.0) + middle
    n = n.clamp(0, 2 ** bits - 1).to(torch.uint8)
    n = n.unflatten(-1, (8, dim // 32)).transpose(-2, -3).flatten(-3)
    if bits == 4:
        n = n[..., 0::2] | n[..., 1::2] << 4
    trailer = torch.cat((s, z), -2).squeeze(-1).contiguous().view(torch.uint8)
    return torch.cat((n, trailer), -1)


def _unpack(rows, dim):
    """The values, in 32 bits."""
    bits = (rows.shape[-1] - 16) * 8 // dim
    n, trailer = rows[..., :-16], rows[..., -16:].contiguous().view(torch.float16).float()
    if bits == 4:
        n = torch.stack((n & 15, n >> 4), -1).flatten(-2)
    n = n.float().unflatten(-1, (8, 4, dim // 32)).transpose(-2, -3).flatten(-2)
    return (trailer[..., 4:, None] + trailer[..., :4, None] * (n - (1 << (bits - 1)))).flatten(-2)


def _places(starts, lens, seqs, rows, device):
    """(row of the cache, whether it is there) of each sequence's rows."""
    t = torch.arange(rows, device=device)
    return (starts[:, None] if starts is not None else torch.zeros(seqs, 1, device=device, dtype=torch.int32)) + t, t < lens[:, None]


def _plain_write(x, cache, starts, lens):
    seqs, heads, rows, dim = x.shape
    at, there = _places(starts, lens, seqs, rows, x.device)
    packed = _pack(x, (cache.shape[-1] - 16) * 8 // dim).transpose(1, 2)
    b, t = torch.nonzero(there, as_tuple=True)
    cache.transpose(1, 2)[b, at[b, t]] = packed[b, t]


def _plain_read(cache, rows, dim, dt, starts, lens):
    at, there = _places(starts, lens, cache.shape[0], rows, cache.device)
    at = torch.where(there, at, 0).long()
    packed = cache.gather(2, at[:, None, :, None].expand(-1, cache.shape[1], -1, cache.shape[3])) if starts is not None else cache[:, :, :rows]
    return torch.where(there[:, None, :, None], _unpack(packed, dim), 0.0).to(dt)


def _plain_attention(q, k_cache, v_cache, lens):
    seqs, q_heads, dim = q.shape
    kv_heads, rows = k_cache.shape[1:3]
    visible = (torch.arange(rows, device=q.device) < lens[:, None])[:, None, None, :]
    qf = q.float().view(seqs, kv_heads, q_heads // kv_heads, dim) / math.sqrt(dim)
    s = torch.where(visible, torch.matmul(qf, _unpack(k_cache, dim).transpose(2, 3)), -math.inf)
    top = s.amax(3, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(3, keepdim=True)
    o = torch.matmul(e, torch.where(visible[:, :, 0, :, None], _unpack(v_cache, dim), 0.0))
    return torch.where(total > 0, o / total, 0.0).reshape(seqs, q_heads, dim).to(q.dtype), (top + torch.log(total)).view(seqs, q_heads)


# ---------------------------------------------------------------------------------------------------------- the definitions, in 64 bits
def _values(packed, dim):
    """Values of packed rows by the place of each dimension's code, in 64 bits."""
    bits = (packed.shape[-1] - 16) * 8 // dim
    d = np.arange(dim)
    quarter, g, j = d // (dim // 4), d % (dim // 4) // (dim // 32), d % (dim // 32)
    bit = bits * (dim // 8 * g + dim // 32 * quarter + j)
    at, shift, quarter = (torch.from_numpy(i).to(packed.device) for i in (bit // 8, bit % 8, quarter))
    n = (packed[..., at].long() >> shift & 2 ** bits - 1).double()
    pairs = packed[..., dim * bits // 8:].clone().view(torch.float16).double()
    return pairs[..., 4 + quarter] + pairs[..., quarter] * (n - 2 ** (bits - 1))


def _quantised(x, bits):
    """What the values of a row ``[..., dim]`` become, by their definition."""
    x = x.double().cpu().numpy()
    out = np.empty_like(x)
    for group in np.split(np.arange(x.shape[-1]), 4):
        part = x[..., group]
        low, high = part.min(-1, keepdims=True), part.max(-1, keepdims=True)
        s = ((high - low) / (2 ** bits - 1)).astype(np.float16).astype(np.float64)
        z = (low + 2 ** (bits - 1) * s).astype(np.float16).astype(np.float64)
        steps = np.rint(np.divide(part - z, s, out=np.zeros_like(part), where=s > 0))
        out[..., group] = z + s * np.clip(steps, -2 ** (bits - 1), 2 ** (bits - 1) - 1)
    return torch.from_numpy(out)


def exact(case, seed):
    s = prepare(case, seed)
    lens, dim = s["lens"].tolist(), case["dim"]
    if case["op"] == "update":
        both = {name: _quantised(s[name], case["bits"]) for name in ("k", "v")}
        for x in both.values():
            for b, n in enumerate(lens):
                x[b, :, n:] = 0.0
        return both
    if case["op"] == "read":
        both = {}
        for name in ("k", "v"):
            x = both[name] = torch.zeros(case["seqs"], case["kv_heads"], case["rows"], dim, dtype=torch.float64, device="cuda")
            for b, n in enumerate(lens):
                x[b, :, :n] = _values(s[name + "_cache"][b, :, :n], dim)
        return both
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if n:
            k, v = (_values(s[c][b, :, :n], dim).repeat_interleave(case["q_heads"] // case["kv_heads"], 0) for c in ("k_cache", "v_cache"))
            scores = torch.einsum("hd,hnd->hn", s["q"][b].double(), k) * dim ** -0.5
            lse[b] = torch.logsumexp(scores, 1)
            out[b] = torch.einsum("hn,hnd->hd", torch.exp(scores - lse[b][:, None]), v)
    return {"out": out, "lse": lse}
