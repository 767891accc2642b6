"""``write_cache_packed``, ``read_cache_packed`` and ``attention_packed_cache`` against their definitions in 64 bits.

Codes and scales are compared bit by bit.  A value that is read back is off by its own rounding, half a step of the type, and by the fp32 sum before
it (2^-24).  Tolerance of an output element of the attention, with w the weights, z and s the centre and scale of a row's quarter, n - M its code, A the sum of
w (|z| + |s (n - M)|), U the sum of w (|z| + s 2^bits): its own rounding, eps / 2 of it; weights and weights times scale rounded to fp16 before they
multiply, 2^-11 of A; the scores' fp32 sums over dim products, dim 2^-24 of the largest sum of |q| (|z| + s 2^bits) times scale as an absolute error of the
exponent, so the same relative error of a weight, twice (numerator and denominator), of U; the fp32 sums of the output, whose accumulator may truncate,
2^-23 for each of the n / 16 steps of U, and as much for the sum of weights.  exp2 in hardware adds 2^-21.  Weights below 2^-21 of the largest lose bits in fp16, at most 2^-32 of
the largest each, times codes of up to 2^bits of the largest scale.  The logarithm has the scores' error, 2^-22 of itself, and that of the sum."""

import ctypes
import math

import numpy as np
import pytest
import torch

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def C(built_library):
    import qwen_megakernel_C
    return qwen_megakernel_C


@pytest.fixture(scope="module")
def gpu(C):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return C


# ------------------------------------------------------------------------------------------------------------- the definition
def order(dim):
    """Index of each dimension's code."""
    d = np.arange(dim)
    return dim // 8 * (d % (dim // 4) // (dim // 32)) + dim // 32 * (d // (dim // 4)) + d % (dim // 32)


def packed(x, bits):
    """Packed rows (uint8) of values ``[..., dim]``, by the definition."""
    x = x.detach().cpu().double().numpy()
    dim, middle = x.shape[-1], 2 ** (bits - 1)
    quarters = x.reshape(*x.shape[:-1], 4, dim // 4)
    low, high = quarters.min(-1, keepdims=True), quarters.max(-1, keepdims=True)      # (NaN where one is)
    good = (low >= -65504) & (high <= 65504)
    low, high, quarters = (np.where(good, a, 0.0) for a in (low, high, quarters))
    s = np.where(good, (high - low) / (2 ** bits - 1), np.nan).astype(np.float16)
    z = (low + middle * s.astype(np.float64)).astype(np.float16)
    step = np.where(s > 0, s, 1).astype(np.float64)
    n = np.where(s > 0, np.rint((quarters - np.where(good, z, 0).astype(np.float64)) / step), 0) + middle
    n = np.clip(n, 0, 2 ** bits - 1).astype(np.uint8).reshape(x.shape)
    codes = np.empty_like(n)
    codes[..., order(dim)] = n
    if bits == 4:
        codes = codes[..., 0::2] | codes[..., 1::2] << 4
    trailer = np.concatenate((s[..., 0], z[..., 0]), -1)
    trailer[np.isnan(trailer)] = np.uint16(0x7fff).view(np.float16)
    return torch.from_numpy(np.concatenate((codes, np.ascontiguousarray(trailer).view(np.uint8)), -1))


def parts(rows, dim):
    """(z, s, n - M) of each dimension of packed rows, in 64 bits."""
    bits = (rows.shape[-1] - 16) * 8 // dim
    rows = rows.cpu().numpy()
    n = rows[..., :-16]
    if bits == 4:
        n = np.stack((n & 15, n >> 4), -1).reshape(*n.shape[:-1], dim)
    trailer = np.ascontiguousarray(rows[..., -16:]).view(np.float16).astype(np.float64)
    quarter = np.arange(dim) // (dim // 4)
    return tuple(torch.from_numpy(a) for a in (trailer[..., 4 + quarter], trailer[..., quarter], n[..., order(dim)].astype(np.float64) - 2 ** (bits - 1)))


def values(rows, dim):
    z, s, n = parts(rows, dim)
    return z + s * n


def made(*shape, dtype="fp16", seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * gain).to(DTYPES[dtype]).cuda()


def rounded_off(want, dtype):
    """How far a value of 64 bits may be from what is read back."""
    return want.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -23) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def check_attention(got, q, kc, vc, lens, scale=None):
    out, lse = got
    seqs, q_heads, dim = q.shape
    group = q_heads // kc[0].shape[0]
    bits = (kc[0].shape[-1] - 16) * 8 // dim
    scale = dim ** -0.5 if scale is None else scale
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous() and lse.dtype == torch.float32 and lse.shape == (seqs, q_heads)
    out, lse, eps = out.double().cpu(), lse.double().cpu(), torch.finfo(q.dtype).eps
    for b in range(seqs):
        n = min(max(int(lens[b]), 0), kc[b].shape[1])
        if n == 0:
            assert bool((out[b] == 0).all()) and bool((lse[b] == -math.inf).all())
            continue
        (kz, ks, kn), (vz, vs, vn) = (tuple(x.repeat_interleave(group, 0) for x in parts(c[b][:, :n], dim)) for c in (kc, vc))
        qb = q[b].double().cpu()
        s = torch.einsum("hd,hnd->hn", qb, kz + ks * kn) * scale
        w = torch.softmax(s, 1)
        want = torch.einsum("hn,hnd->hd", w, vz + vs * vn)
        a = torch.einsum("hn,hnd->hd", w, vz.abs() + (vs * vn).abs())
        u = torch.einsum("hn,hnd->hd", w, vz.abs() + vs * 2 ** bits)
        ds = dim * 2.0 ** -24 * torch.einsum("hd,hnd->hn", qb.abs(), kz.abs() + ks * 2 ** bits).amax(1, keepdim=True) * abs(scale) + s.abs().amax(1, keepdim=True) * 2.0 ** -23
        steps = (n / 16 + 2) * 2.0 ** -23
        tol = eps / 2 * want.abs() + 2.0 ** -11 * 1.001 * a + u * (2 * ds + 2 * steps + 2.0 ** -21) + n * 2.0 ** -32 * (vz.abs() + vs * 2 ** bits).amax()
        err = (out[b] - want).abs()
        assert bool((err <= tol).all()), (b, float((err / tol).max()))
        want_lse = torch.logsumexp(s, 1)
        err = (lse[b] - want_lse).abs()
        assert bool((err <= ds[:, 0] + 2.0 ** -22 * (1 + want_lse.abs()) + steps).all()), (b, float(err.max()))


def attention_inputs(seqs, q_heads, kv_heads, dim, bits, rows, dtype="fp16", seed=0, gain=1.0):
    k, v, q = made(seqs, kv_heads, rows, dim, seed=seed), made(seqs, kv_heads, rows, dim, seed=seed + 1, gain=0.5), made(seqs, q_heads, dim, dtype=dtype, seed=seed + 2, gain=gain)
    return q, packed(k, bits).cuda(), packed(v, bits).cuda()


def with_room(cache, rows):
    """The cache with room for ``rows`` rows, nothing sensible in those behind its own."""
    n, heads, have, size = cache.shape
    return torch.cat((cache, torch.full((n, heads, rows - have, size), 255, dtype=torch.uint8, device="cuda")), 2) if rows > have else cache


# ------------------------------------------------------------------------------------------------------------- refusals (no device)
def cache_args(C, **change):
    n = change.get("num_sequences", 2)
    one = (ctypes.c_void_p * max(n, 1))(*[4096] * max(n, 1))
    a = dict(bits=4, head_dim=128, num_sequences=2, kv_heads=8, rows=16, k=ctypes.addressof(one), v=ctypes.addressof(one), seq_stride=0, head_stride=1280, row_stride=80)
    a.update(change)
    cache = C._PackedCache(**a)
    cache.keep = one
    return cache


def row_args(C, **change):
    a = dict(type=0, rows=4, k=4096, v=4096, seq_stride=4096, head_stride=512, row_stride=128, start=0)
    a.update(change)
    return C._PackedRows(**a)


def attention_args(C, **change):
    a = dict(type=0, q_heads=16, q=4096, q_seq_stride=2048, q_head_stride=128, lens=4096, scale=1.0, out=4096, workspace=4096, workspace_bytes=1 << 30)
    a.update(change)
    return C._PackedAttention(**a)


def call(C, name, *args):
    return getattr(C._lib, name)(*[None if a is None else bytes(a) for a in args], None), C._lib.qmk_last_error()


CACHE_FAULTS = [(dict(bits=5), b"bits"), (dict(head_dim=96), b"head_dim"), (dict(num_sequences=0), b"num_sequences"), (dict(num_sequences=129), b"num_sequences"),
                (dict(kv_heads=0), b"kv_heads"), (dict(kv_heads=1025), b"kv_heads"), (dict(rows=-1), b"rows"), (dict(rows=(1 << 24) + 1), b"rows"),
                (dict(k=None), b"null"), (dict(v=None), b"null"), (dict(k=None, k_base=4096), b"null"), (dict(head_stride=1288), b"strides"), (dict(row_stride=84), b"strides"),
                (dict(row_stride=64), b"overlap"), (dict(row_stride=0), b"overlap"), (dict(k=None, k_base=4104, v_base=4096), b"multiple of 16"),
                (dict(k=None, k_base=4096, v_base=4096, seq_stride=8), b"strides")]


@pytest.mark.parametrize("change,text", CACHE_FAULTS)
def test_caches_are_refused_before_anything_runs(C, change, text):
    cache = cache_args(C, **change)
    for name, args in (("qmk_write_cache_packed", row_args(C)), ("qmk_read_cache_packed", row_args(C)), ("qmk_attention_packed_cache", attention_args(C))):
        rc, why = call(C, name, cache, args)
        assert rc == 2 and text in why and name.encode() in why, (name, why)


@pytest.mark.parametrize("change,text", [(dict(type=2), b"type"), (dict(rows=-1), b"rows"), (dict(rows=(1 << 24) + 1), b"rows"), (dict(k=None), b"null"), (dict(v=None), b"null"),
                                         (dict(k=4104), b"16"), (dict(seq_stride=4), b"strides"), (dict(head_stride=12), b"strides"), (dict(row_stride=130), b"strides")])
@pytest.mark.parametrize("name", ["qmk_write_cache_packed", "qmk_read_cache_packed"])
def test_rows_are_refused_before_anything_runs(C, name, change, text):
    rc, why = call(C, name, cache_args(C), row_args(C, **change))
    assert rc == 2 and text in why, why


def test_more_rows_than_an_index_holds_are_refused(C):
    rc, why = call(C, "qmk_write_cache_packed", cache_args(C, num_sequences=128), row_args(C, rows=1 << 21))
    assert rc == 2 and b"2^31" in why


@pytest.mark.parametrize("change,text", [(dict(type=2), b"type"), (dict(q_heads=12), b"q_heads"), (dict(q_heads=0), b"q_heads"), (dict(q_heads=136), b"q_heads"), (dict(q=None), b"null"),
                                         (dict(out=None), b"null"), (dict(lens=None), b"null"),
                                         (dict(scale=float("inf")), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(scale=3e38), b"scale"), (dict(q=4104), b"aligned"),
                                         (dict(out=4104), b"aligned"), (dict(workspace=4104), b"aligned"), (dict(q_seq_stride=2052), b"strides"), (dict(q_head_stride=4), b"strides")])
def test_attention_is_refused_before_anything_runs(C, change, text):
    rc, why = call(C, "qmk_attention_packed_cache", cache_args(C), attention_args(C, **change))
    assert rc == 2 and text in why, why


@pytest.mark.parametrize("change", [dict(workspace=None), dict(workspace_bytes=4), dict(workspace_bytes=-1)])
def test_a_workspace_that_is_needed_and_not_there_is_refused(C, change):
    rc, why = call(C, "qmk_attention_packed_cache", cache_args(C, rows=100000, head_stride=8000000), attention_args(C, **change))
    assert rc == 2 and b"workspace" in why


def test_null_arguments_are_refused(C):
    for name, args in (("qmk_write_cache_packed", row_args(C)), ("qmk_read_cache_packed", row_args(C)), ("qmk_attention_packed_cache", attention_args(C))):
        assert call(C, name, None, args)[0] == 2 and call(C, name, cache_args(C), None)[0] == 2
        holes = (ctypes.c_void_p * 2)(4096, None)
        rc, why = call(C, name, cache_args(C, v=ctypes.addressof(holes)), args)
        assert rc == 2 and b"null" in why


def test_no_workspace_for_sizes_that_are_refused(C):
    size = C._lib.qmk_attention_packed_cache_workspace
    assert size(1, 16, 8, 128, 4, 100) == 0 and size(1, 16, 8, 128, 4, 100000) > 0
    for bad in ((0, 16, 8, 128, 4, 100), (129, 16, 8, 128, 4, 100), (1, 12, 8, 128, 4, 100), (1, 136, 8, 128, 4, 100), (1, 16, 0, 128, 4, 100), (1, 16, 8, 96, 4, 100),
                (1, 16, 8, 128, 5, 100), (1, 16, 8, 128, 4, -1), (1, 16, 8, 128, 4, (1 << 24) + 1)):
        assert size(*bad) == -1


def test_packed_row_bytes(C):
    assert [C.packed_row_bytes(d, b) for d, b in ((128, 4), (128, 8), (64, 4), (64, 8))] == [80, 144, 48, 80]
    for bad in ((96, 4), (128, 5)):
        with pytest.raises(RuntimeError):
            C.packed_row_bytes(*bad)


@pytest.mark.gpu
def test_wrong_tensors_are_refused(gpu):
    q, kc, vc = attention_inputs(2, 4, 2, 64, 4, 8)
    k, v, lens = made(2, 2, 3, 64), made(2, 2, 3, 64), torch.tensor([1, 2], dtype=torch.int32).cuda()
    for bad in ((q.float(), kc, vc, lens), (q[0], kc, vc, lens), (q.cpu(), kc, vc, lens), (q, kc[:1], vc, lens), (q, kc.cpu(), vc.cpu(), lens), (q, kc.view(torch.int8), vc.view(torch.int8), lens),
                (q, kc[..., :40], vc[..., :40], lens), (q, kc, vc[:, :, :4], lens), (q, kc, vc, lens.long()), (q, kc, vc, lens[:1]), (q, kc, vc, lens.cpu()), (q, kc, vc, None),
                (q, list(kc)[:1], list(vc), lens), (q[:, :3], kc, vc, lens), (q, [kc[0], kc[1].transpose(0, 1)], list(vc), lens), (made(2, 4, 96), kc, vc, lens),
                (q, kc[:, :, :1].expand(-1, -1, 8, -1), vc[:, :, :1].expand(-1, -1, 8, -1), lens)):
        with pytest.raises(RuntimeError):
            gpu.attention_packed_cache(*bad)
    for bad in ((k.float(), v.float(), kc, vc), (k[0], v[0], kc, vc), (k.cpu(), v.cpu(), kc, vc), (k, v.bfloat16(), kc, vc), (k, v[:1], kc, vc), (k[:, :1], v[:, :1], kc, vc),
                (k, v.transpose(1, 2).contiguous().transpose(1, 2), kc, vc), (k[..., ::2], v[..., ::2], kc, vc), (k, v, kc.cpu(), vc.cpu()), (k, v, kc, vc, lens.long()),
                (k, v, kc, vc, 2 ** 31), (k, v, kc, vc, 0, lens.cpu()), (k, v, kc, vc, 1.5), (k[:1], v[:1], kc, vc)):
        with pytest.raises(RuntimeError):
            gpu.write_cache_packed(*bad)
    for bad, named in (((kc, vc, 3, 96), {}), ((kc, vc, -1, 64), {}), ((kc, vc, 3, 64, torch.float32), {}), ((kc, vc, 3, 128), {}), ((kc.cpu(), vc.cpu(), 3, 64), {}), (([], [], 3, 64), {}), ((list(kc), list(vc)[:1], 3, 64), {}),
                       ((kc, vc, 3, 64), dict(k_out=k)), ((kc, vc, 3, 64), dict(k_out=k, v_out=v.bfloat16())), ((kc, vc, 4, 64), dict(k_out=k, v_out=v)),
                       ((kc, vc, 3, 64), dict(k_out=k, v_out=v.transpose(1, 2).contiguous().transpose(1, 2)))):
        with pytest.raises(RuntimeError):
            gpu.read_cache_packed(*bad, **named)


# ------------------------------------------------------------------------------------------------------------- rows in and out
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
@pytest.mark.parametrize("seqs,heads,rows,cache", [(1, 1, 1, 1), (1, 8, 1, 40), (3, 2, 33, 50), (128, 8, 1, 5), (2, 5, 257, 300), (7, 3, 31, 31)])
def test_rows_become_their_codes_and_read_back(gpu, dtype, dim, bits, seqs, heads, rows, cache):
    """Rows of a projection's output (heads behind rows), at a start for each sequence, some sequences with fewer; everything else stays."""
    k, v = (made(seqs, rows, heads, dim, dtype=dtype, seed=seqs + i, gain=3.0).transpose(1, 2) for i in (0, 1))
    starts = torch.tensor([(5 * b) % (cache - rows + 1) for b in range(seqs)], dtype=torch.int32)
    lens = torch.tensor([rows if b % 3 != 1 else rows // 2 for b in range(seqs)], dtype=torch.int32)
    size = gpu.packed_row_bytes(dim, bits)
    kc, vc = (torch.randint(0, 256, (seqs, heads, cache, size), dtype=torch.uint8, generator=torch.Generator().manual_seed(9 + i)).cuda() for i in (0, 1))
    want = [c.cpu().clone() for c in (kc, vc)]
    for c, x in zip(want, (k, v)):
        new = packed(x, bits)
        for b in range(seqs):
            n, at = int(lens[b]), int(starts[b])
            c[b, :, at:at + n] = new[b, :, :n]
    gpu.write_cache_packed(k, v, kc, vc, starts.cuda(), lens.cuda())
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
    back = gpu.read_cache_packed(kc, vc, rows, dim, DTYPES[dtype], starts.cuda(), lens.cuda())
    for x, c in zip(back, want):
        assert x.dtype == DTYPES[dtype] and tuple(x.shape) == (seqs, heads, rows, dim)
        for b in range(seqs):
            n, at = int(lens[b]), int(starts[b])
            exact = values(c[b, :, at:at + n], dim)
            assert bool(((x[b, :, :n].double().cpu() - exact).abs() <= rounded_off(exact, DTYPES[dtype])).all())
            assert bool((x[b, :, n:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_values_that_quantise_badly(gpu, dtype, bits):
    """Constant quarters, values on the border of two codes, one far value, the smallest and largest ones, offsets, values that are no numbers."""
    x = torch.zeros(1, 1, 40, 128)
    x[0, 0, 1] = 7.25
    x[0, 0, 2] = torch.arange(128) % 32 * 0.5                                  # many quotients end in a half
    x[0, 0, 3, ::32] = 60000.0
    x[0, 0, 4] = torch.linspace(-65504, 65504, 128)
    x[0, 0, 5] = torch.arange(128) * 2.0 ** -24
    x[0, 0, 6] = 1000 + torch.arange(128) % 3
    x[0, 0, 7, 5], x[0, 0, 8, 40], x[0, 0, 9, 127] = math.nan, math.inf, -math.inf
    x[0, 0, 10] = 1e5                                                          # (infinite in fp16, too large for a scale in bf16)
    x[0, 0, 11] = -(2.0 ** -20) * (torch.arange(128) + 1)
    x[0, 0, 12:] = torch.randint(-8, 9, (28, 128), generator=torch.Generator().manual_seed(1)) / 8
    x[0, 0, 20:] += torch.randint(0, 2, (20, 128), generator=torch.Generator().manual_seed(2)) * 2.0 ** -12
    x[0, 0, 30:] *= 1024
    x = x.to(DTYPES[dtype]).cuda()
    kc, vc = (torch.zeros(1, 1, 40, gpu.packed_row_bytes(128, bits), dtype=torch.uint8, device="cuda") for _ in range(2))
    gpu.write_cache_packed(x, -x, kc, vc)
    for got, rows in ((kc, x), (vc, -x)):
        want, got = packed(rows, bits), got.cpu()
        bad = torch.isnan(values(want, 128))
        assert bool((got[..., -16:] == want[..., -16:]).all())
        # rows 7 to 9 a quarter each, row 10 all four; in bf16 the ends of row 4 are 65536 (65504 lies between 65280 and that): two quarters more
        assert bool(((values(got, 128) == values(want, 128)) | bad).all()) and int(bad.sum()) == 3 * 32 + 128 + (64 if dtype == "bf16" else 0)
    k, _ = gpu.read_cache_packed(kc, vc, 40, 128, DTYPES[dtype])
    assert torch.equal(torch.isnan(k.cpu()), torch.isnan(values(packed(x, bits), 128)))
    exact = values(packed(x, bits), 128)
    assert bool(((k.double().cpu() - exact).abs() <= rounded_off(exact, DTYPES[dtype])).nan_to_num(0).logical_or(torch.isnan(exact)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_rows_outside_the_caches(gpu, bits):
    """Starts in front of a cache and behind it, lengths below 0 and above the rows that are there."""
    heads, rows, cache = 2, 9, 12
    starts = torch.tensor([-4, 8, 100, -100, 2 ** 31 - 1, -2 ** 31, 0], dtype=torch.int32)
    lens = torch.tensor([9, 9, 9, 9, 9, 9, -3], dtype=torch.int32)
    k, v = made(7, heads, rows, 64, seed=1), made(7, heads, rows, 64, seed=2)
    kc, vc = (torch.full((7, heads, cache, gpu.packed_row_bytes(64, bits)), 170, dtype=torch.uint8, device="cuda") for _ in range(2))
    gpu.write_cache_packed(k, v, kc, vc, starts.cuda(), lens.cuda())
    want = torch.full(kc.shape, 170, dtype=torch.uint8)
    want[0, :, :5] = packed(k[0, :, 4:], bits)
    want[1, :, 8:] = packed(k[1, :, :4], bits)
    assert torch.equal(kc.cpu(), want)
    k2, v2 = gpu.read_cache_packed(kc, vc, rows, 64, starts=starts.cuda(), lens=lens.cuda())
    assert bool((k2[0, :, :4] == 0).all()) and bool((k2[1, :, 4:] == 0).all()) and bool((k2[2:] == 0).all()) and bool((v2[2:] == 0).all())
    assert bool((k2[0, :, 4:] != 0).any()) and bool((k2[1, :, :4] != 0).any())
    gpu.write_cache_packed(k, v, kc, vc, 3, torch.full((7,), 100, dtype=torch.int32).cuda())
    assert torch.equal(kc[:, :, 3:].cpu(), packed(k, bits)) and torch.equal(vc[:, :, 3:].cpu(), packed(v, bits)) and torch.equal(kc[:, :, :3].cpu(), want[:, :, :3])


@pytest.mark.gpu
def test_lists_of_caches_strides_and_no_rows(gpu):
    """Layers of caches that belong to different sequences, rows and outputs that are views; nothing to do is nothing done."""
    big = torch.zeros(3, 4, 2, 20, 2, 80, dtype=torch.uint8, device="cuda")               # [sequence, layer, head, row, k / v, bytes]
    kc, vc = [big[b, 1, :, :, 0] for b in (2, 0, 1)], [big[b, 1, :, :, 1] for b in (2, 0, 1)]
    k, v = made(3, 6, 4, 128, seed=3)[:, :5, 1:3].transpose(1, 2), made(3, 6, 4, 128, seed=4)[:, :5, 1:3].transpose(1, 2)
    gpu.write_cache_packed(k, v, kc, vc, 7)
    for i, b in enumerate((2, 0, 1)):
        assert torch.equal(big[b, 1, :, 7:12, 0].cpu(), packed(k[i], 4)) and torch.equal(big[b, 1, :, 7:12, 1].cpu(), packed(v[i], 4))
    assert int((big != 0).sum()) == int((big[:, 1, :, 7:12] != 0).sum())
    outs = [torch.full((2, 3, 9, 128), 5.0, dtype=torch.float16, device="cuda").transpose(0, 1) for _ in range(2)]
    got = gpu.read_cache_packed(kc, vc, 5, 128, starts=7, k_out=outs[0][:, :, 2:7], v_out=outs[1][:, :, 2:7])
    want = gpu.read_cache_packed(kc, vc, 5, 128, starts=7)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and bool((outs[0][:, :, :2] == 5).all()) and bool((outs[0][:, :, 7:] == 5).all())
    before = big.clone()
    gpu.write_cache_packed(k[:, :, :0], v[:, :, :0], kc, vc, 7)
    assert torch.equal(before, big) and gpu.read_cache_packed(kc, vc, 0, 128)[0].shape == (3, 2, 0, 128)


# ------------------------------------------------------------------------------------------------------------- attention
HEADS = [(16, 8), (4, 4), (6, 2), (8, 2), (10, 2), (8, 1), (16, 1), (9, 1), (32, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
@pytest.mark.parametrize("q_heads,kv_heads", HEADS)
@pytest.mark.parametrize("seqs,rows", [(1, 1), (1, 17), (2, 64), (3, 333), (19, 65)])
def test_attention_matches_the_definition(gpu, dtype, dim, bits, q_heads, kv_heads, seqs, rows):
    q, kc, vc = attention_inputs(seqs, q_heads, kv_heads, dim, bits, rows, dtype, seed=seqs + rows)
    lens = torch.tensor([rows * (i + 1) // seqs if i % 5 != 1 else 0 for i in range(seqs)], dtype=torch.int32)
    check_attention(gpu.attention_packed_cache(q, kc, vc, lens.cuda()), q, kc, vc, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("seqs,q_heads,kv_heads,rows", [(1, 16, 8, 20000), (128, 16, 8, 300), (40, 32, 2, 1500), (3, 8, 8, 5001)])
def test_long_caches_and_full_batches(gpu, bits, seqs, q_heads, kv_heads, rows):
    q, kc, vc = attention_inputs(seqs, q_heads, kv_heads, 128, bits, rows, seed=rows, gain=1.5)
    lens = torch.tensor([rows if seqs == 1 else (7919 * (i + 1)) % (rows + 1) for i in range(seqs)], dtype=torch.int32)
    check_attention(gpu.attention_packed_cache(q, kc, vc, lens.cuda()), q, kc, vc, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
@pytest.mark.parametrize("q_heads,kv_heads", HEADS)
@pytest.mark.parametrize("seqs,room,rows", [(1, 40000, 700), (5, 33000, 333), (37, 17000, 70)])
def test_caches_with_room_to_spare(gpu, dtype, dim, bits, q_heads, kv_heads, seqs, room, rows):
    """Caches made for more rows than the sequences have: the call is cut for long ones."""
    q, k, v = attention_inputs(seqs, q_heads, kv_heads, dim, bits, rows, dtype, seed=seqs + dim)
    kc, vc = (torch.full((seqs, kv_heads, room, x.shape[3]), 255, dtype=torch.uint8, device="cuda") for x in (k, v))
    lens = torch.tensor([rows * (i + 1) // seqs if i % 5 != 1 else 0 for i in range(seqs)], dtype=torch.int32)
    kc[:, :, :rows], vc[:, :, :rows] = k, v
    check_attention(gpu.attention_packed_cache(q, kc, vc, lens.cuda()), q, kc, vc, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("q_heads,kv_heads,dim,bits", [(16, 8, 64, 4), (32, 8, 64, 8), (64, 8, 64, 4), (16, 1, 128, 4)])
def test_full_batches_with_room_to_spare(gpu, q_heads, kv_heads, dim, bits):
    q, k, v = attention_inputs(128, q_heads, kv_heads, dim, bits, 90, seed=dim)
    kc, vc = (torch.full((128, kv_heads, 9000, x.shape[3]), 255, dtype=torch.uint8, device="cuda") for x in (k, v))
    kc[:, :, :90], vc[:, :, :90] = k, v
    for lens in ([(37 * i) % 91 for i in range(128)], [0] * 127 + [90], [1] * 128):
        lens = torch.tensor(lens, dtype=torch.int32)
        check_attention(gpu.attention_packed_cache(q, kc, vc, lens.cuda()), q, kc, vc, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("q_heads,kv_heads,dim,bits,dtype", [(2, 2, 128, 4, "fp16"), (4, 2, 128, 8, "bf16"), (16, 2, 64, 4, "fp16"), (16, 4, 128, 4, "bf16"), (5, 1, 128, 8, "fp16"), (16, 1, 64, 8, "fp16"), (4, 4, 64, 8, "fp16")])
def test_few_long_sequences(gpu, q_heads, kv_heads, dim, bits, dtype):
    """Clusters take parts of a sequence: lengths of no row, of fewer tiles than there are clusters, of one more than all tiles alike, of the whole cache."""
    q, kc, vc = attention_inputs(4, q_heads, kv_heads, dim, bits, 19000, dtype, seed=dim + q_heads)
    for lens in ([19000, 1, 0, 9001], [33, 32, 700, 0], [2369, 8 * 37 * 32 + 1, 18999, 64]):
        check_attention(gpu.attention_packed_cache(q, kc, vc, torch.tensor(lens, dtype=torch.int32).cuda()), q, kc, vc, lens)
    for b, n in ((0, 19000), (2, 18977)):
        check_attention(gpu.attention_packed_cache(q[b:b + 1], kc[b:b + 1], vc[b:b + 1], torch.tensor([n], dtype=torch.int32).cuda()), q[b:b + 1], kc[b:b + 1], vc[b:b + 1], [n])
    room = (with_room(kc, 40000), with_room(vc, 40000))
    lens = torch.zeros(4, dtype=torch.int32)
    check_attention(gpu.attention_packed_cache(q, *room, lens.cuda()), q, *room, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("q_heads,kv_heads,dim,bits", [(16, 8, 128, 4), (4, 2, 64, 8), (8, 2, 128, 8), (16, 2, 128, 4), (32, 2, 128, 8), (3, 1, 64, 4)])
def test_each_way_a_call_is_cut(gpu, q_heads, kv_heads, dim, bits):
    """The same rows in caches of their size, in long ones and in long ones of more sequences, then with a key and a value that are no numbers."""
    q, kc, vc = attention_inputs(4, q_heads, kv_heads, dim, bits, 700)
    lens = torch.tensor([0, 20, 700, 333], dtype=torch.int32)
    which = torch.tensor([0, 1, 2, 3, 2, 3, 1])

    def ways(kc, vc):
        at = which.cuda()
        long = with_room(kc, 20000), with_room(vc, 20000)
        lists = [long[0][i] for i in which], [long[1][i] for i in which]
        return [gpu.attention_packed_cache(q, kc, vc, lens.cuda()), gpu.attention_packed_cache(q, *long, lens.cuda()), gpu.attention_packed_cache(q[at], *lists, lens.cuda()[at])]

    want = ways(kc, vc)
    for got in want[:2]:
        check_attention(got, q, kc, vc, lens)
    check_attention(want[2], q[which.cuda()], [kc[i] for i in which], [vc[i] for i in which], lens[which])
    none = torch.full((1, kv_heads, 1, dim), math.nan, dtype=torch.float16, device="cuda")
    one = torch.ones_like(none)
    kn, vn = kc.clone(), vc.clone()
    gpu.write_cache_packed(none, one, kn[2:3], vn[2:3], 650)
    gpu.write_cache_packed(one, none, kn[3:], vn[3:], 332)
    gpu.write_cache_packed(none, none, kn[1:2], vn[1:2], 20)                   # (behind the last row)
    for i, (out, lse) in enumerate(ways(kn, vn)):
        seq = which if i == 2 else torch.arange(4)
        bad_key, bad = (seq == 2).cuda(), ((seq == 2) | (seq == 3)).cuda()
        assert torch.equal(lse.isnan(), bad_key[:, None].expand_as(lse)) and torch.equal(out.isnan(), bad[:, None, None].expand_as(out))
        assert torch.equal(out[~bad], want[i][0][~bad]) and torch.equal(lse[~bad], want[i][1][~bad])


@pytest.mark.gpu
def test_no_rows_and_lengths_outside_the_cache(gpu):
    q, kc, vc = attention_inputs(4, 4, 2, 64, 4, 30)
    for lens in ([0, 0, 0, 0], [-5, 1000, 2 ** 31 - 1, -2 ** 31]):
        check_attention(gpu.attention_packed_cache(q, kc, vc, torch.tensor(lens, dtype=torch.int32).cuda()), q, kc, vc, lens)
    out, lse = gpu.attention_packed_cache(q, kc[:, :, :0], vc[:, :, :0], torch.tensor([3, 0, 0, 1], dtype=torch.int32).cuda())
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_behind_the_last_are_not_looked_at(gpu, dim, bits):
    """Whatever bytes they hold, NaN in their trailers among them."""
    q, kc, vc = attention_inputs(3, 8, 2, dim, bits, 200)
    lens = torch.tensor([1, 77, 130], dtype=torch.int32)
    want = gpu.attention_packed_cache(q, kc, vc, lens.cuda())
    for c in (kc, vc):
        for b in range(3):
            c[b, :, int(lens[b]):] = 255
    got = gpu.attention_packed_cache(q, kc, vc, lens.cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("room", [100, 40000])
@pytest.mark.parametrize("q_heads", [8, 16, 32, 64])
def test_visible_rows_that_are_no_numbers(gpu, bits, room, q_heads):
    """A key without numbers leaves none in its head's outputs, a value in its quarter's; the other heads and sequences keep theirs."""
    group = q_heads // 4
    q, kc, vc = attention_inputs(2, q_heads, 4, 128, bits, 100)
    kc, vc = with_room(kc, room), with_room(vc, room)
    lens = torch.tensor([100, 90], dtype=torch.int32).cuda()
    want = gpu.attention_packed_cache(q, kc, vc, lens)
    k, v = gpu.read_cache_packed(kc, vc, 100, 128)
    k[0, 1, 50, 3] = math.nan
    v[1, 2, 7, 40] = math.inf
    v[1, 3, 95, 0] = math.nan                                                  # (behind the last row)
    kc2, vc2 = kc.clone(), vc.clone()
    gpu.write_cache_packed(k[:1, :, 50:51], v[:1, :, 50:51], kc2[:1], vc2[:1], 50)
    gpu.write_cache_packed(k[1:, :, 7:8], v[1:, :, 7:8], kc2[1:], vc2[1:], 7)
    gpu.write_cache_packed(k[1:, :, 95:96], v[1:, :, 95:96], kc2[1:], vc2[1:], 95)
    kc2[0, 0], kc2[0, 2:], vc2[0] = kc[0, 0], kc[0, 2:], vc[0]                # (read back and written again: not always the same codes)
    kc2[1], vc2[1, :2], vc2[1, 3, :95] = kc[1], vc[1, :2], vc[1, 3, :95]
    out, lse = gpu.attention_packed_cache(q, kc2, vc2, lens)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, group:2 * group] = True
    bad[1, 2 * group:3 * group, 32:64] = True
    assert torch.equal(torch.isnan(out), bad) and torch.equal(torch.isnan(lse), bad.all(2))
    other = ~bad
    other[1, 2 * group:3 * group] = False
    assert torch.equal(out[other], want[0][other]) and torch.equal(lse[~bad.all(2)], want[1][~bad.all(2)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("q_heads", [4, 8, 16, 32])
def test_sizes_of_values_and_scores(gpu, dtype, bits, q_heads):
    """Values from 2^-12 to 2^12 in quarters side by side and in rows behind one another, scores that rise and fall by hundreds, negative and zero scales."""
    seqs, rows = 3, 300
    k, q = made(seqs, 2, rows, 128, seed=5), made(seqs, q_heads, 128, dtype=dtype, seed=6, gain=8.0)
    v = made(seqs, 2, rows, 128, seed=7).float()
    v *= 2.0 ** torch.linspace(-12, 12, 4).repeat_interleave(32).cuda()
    v[1] *= 2.0 ** torch.linspace(0, -12, rows).cuda()[:, None]
    v[2] = v[2].flip(1) * 2.0 ** torch.linspace(-3, 0, rows).cuda()[:, None]
    kc, vc = packed(k, bits).cuda(), packed(v.half(), bits).cuda()
    lens = torch.tensor([300, 299, 170], dtype=torch.int32)
    for scale in (None, 3.0, -0.5, 0.0, 1e-30):
        check_attention(gpu.attention_packed_cache(q, kc, vc, lens.cuda(), scale=scale), q, kc, vc, lens, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads", [4, 8, 16, 32])
def test_queries_of_any_size(gpu, bits, heads):
    """Queries at both ends of their types, and tiny ones beside them."""
    _, kc, vc = attention_inputs(1, 4, 2, 128, bits, 50)
    lens = torch.tensor([50], dtype=torch.int32)
    for dtype, sizes in ((torch.float16, (6e4, 2.0 ** -14, 2.0 ** -24)), (torch.bfloat16, (1e30, 6e4, 1e-30, 2.0 ** -133))):
        for size in sizes:
            q = (made(1, heads, 128, seed=3).float().clamp(-1, 1) * size).to(dtype)
            q[0, 0, 0], q[0, 1, 5] = 0.0, size / 2 ** 12
            scale = 0.1 / max(size, 1e-30) if size > 1e-4 else 1e10
            check_attention(gpu.attention_packed_cache(q, kc, vc, lens.cuda(), scale=scale), q, kc, vc, lens, scale)
    zero = torch.zeros(1, heads, 128, dtype=torch.float16, device="cuda")
    check_attention(gpu.attention_packed_cache(zero, kc, vc, lens.cuda()), zero, kc, vc, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("room", [70, 30000])
@pytest.mark.parametrize("q_heads,bits", [(4, 4), (8, 8), (16, 4), (32, 8)])
def test_lists_views_and_strides(gpu, room, q_heads, bits):
    q, kc, vc = attention_inputs(5, q_heads, 2, 128, bits, 70)
    kc, vc = with_room(kc, room), with_room(vc, room)
    lens = torch.tensor([70, 1, 0, 33, 64], dtype=torch.int32)
    want = gpu.attention_packed_cache(q, kc, vc, lens.cuda())
    again = gpu.attention_packed_cache(q, list(kc), list(vc), lens.cuda())
    assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])
    both = torch.stack((kc, vc), 3).transpose(1, 2).contiguous().transpose(1, 2)           # [sequence, row, head, k / v, bytes] in memory
    qv = torch.cat((q, q), 2).view(5, q_heads, 256)[:, :, 128:]
    again = gpu.attention_packed_cache(qv, both[:, :, :, 0], both[:, :, :, 1], lens.cuda())
    assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])
    same = gpu.attention_packed_cache(q, kc[:1].expand(5, -1, -1, -1), vc[:1].expand(5, -1, -1, -1), lens.cuda())      # one cache for all
    check_attention(same, q, [kc[0]] * 5, [vc[0]] * 5, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("room", [700, 9000])
def test_results_do_not_depend_on_the_run(gpu, room):
    q, kc, vc = attention_inputs(33, 16, 8, 128, 4, 700)
    kc, vc = with_room(kc, room), with_room(vc, room)
    lens = torch.tensor([(131 * i) % 701 for i in range(33)], dtype=torch.int32).cuda()
    first = gpu.attention_packed_cache(q, kc, vc, lens)
    for _ in range(5):
        again = gpu.attention_packed_cache(q, kc, vc, lens)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ------------------------------------------------------------------------------------------------------------- together
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("cache", [64, 20000])
def test_prompt_then_steps_in_a_captured_graph(gpu, bits, cache):
    """A prompt's rows written, then decode steps - the new rows written, the attention over everything so far - replayed from one graph, on a stream of
    their own, with positions that move on the device."""
    seqs, q_heads, kv_heads, dim, room, prompt = 3, 16, 8, 128, 64, 30
    kc, vc = (torch.zeros(seqs, kv_heads, cache, gpu.packed_row_bytes(dim, bits), dtype=torch.uint8, device="cuda") for _ in range(2))
    k, v = made(seqs, kv_heads, room, dim, seed=1), made(seqs, kv_heads, room, dim, seed=2)
    lens = torch.tensor([30, 7, 0], dtype=torch.int32)
    gpu.write_cache_packed(k[:, :, :prompt], v[:, :, :prompt], kc, vc, 0, lens.cuda())
    at = lens.cuda()
    qs = made(10, seqs, q_heads, dim, seed=3)
    q, kn, vn = torch.empty_like(qs[0]), torch.empty(seqs, kv_heads, 1, dim, dtype=torch.float16, device="cuda"), torch.empty(seqs, kv_heads, 1, dim, dtype=torch.float16, device="cuda")
    gpu.attention_packed_cache(qs[0], kc, vc, at)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        gpu.write_cache_packed(kn, vn, kc, vc, at)
        after = at + 1
        out, lse = gpu.attention_packed_cache(q, kc, vc, after)
        at.copy_(after)
    for step in range(10):
        rows = [int(lens[b]) + step for b in range(seqs)]
        q.copy_(qs[step])
        for b in range(seqs):
            kn[b, :, 0].copy_(k[b, :, rows[b]])
            vn[b, :, 0].copy_(v[b, :, rows[b]])
        graph.replay()
        torch.cuda.synchronize()
        check_attention((out, lse), q, packed(k, bits), packed(v, bits), [r + 1 for r in rows])
    back, _ = gpu.read_cache_packed(kc, vc, room, dim)
    for b in range(seqs):
        n = int(lens[b]) + 10
        exact = values(packed(k[b, :, :n], bits), dim)
        assert bool(((back[b, :, :n].double().cpu() - exact).abs() <= rounded_off(exact, torch.float16)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("room", [500, 20000])
def test_two_streams_at_once(gpu, room):
    cases = [attention_inputs(9, 16, 8, 128, 4, 500, seed=s) for s in (1, 2)]
    cases = [(q, with_room(kc, room), with_room(vc, room)) for q, kc, vc in cases]
    lens = torch.tensor([500 - 50 * i for i in range(9)], dtype=torch.int32).cuda()
    want = [gpu.attention_packed_cache(*c, lens) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(gpu.attention_packed_cache(*cases[i], lens))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, want[i][0]) and torch.equal(e, want[i][1]) for o, e in got[i])


# ------------------------------------------------------------------------------------------------------------- sequences set aside
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_a_parked_sequence_comes_back(gpu, bits):
    """A slot's rows packed, the slot used for something else, the rows back in another slot: they are what the codes stand for, and decoding goes on exactly as from
    a cache that holds those values."""
    import synthetic as S
    from Model.Qwen06B_architecture import BatchDecoder
    w = S.make_weights(seed=31, num_layers=3, vocab_size=2048, norm_std=0.1, max_seq_len=16)
    eng = BatchDecoder(weights=S.weights_to(w, "cuda"), tokenizer=S.StubTokenizer(-1, 2048), num_sequences=3, max_seq_len=96, engine="gemm", prefill_mode="tensor")
    prompt = S.make_prompt(50, seed=3, vocab_size=2048)
    eng.prefill_slot(0, prompt[:-1])
    k, v = eng._k_caches[0][:, :, :49].clone(), eng._v_caches[0][:, :, :49].clone()
    parked = eng.park_slot(0, bits)
    assert parked.length == 49 and parked.bits == bits and parked.k.shape == (3, 8, 49, gpu.packed_row_bytes(128, bits))
    assert torch.equal(parked.k.cpu(), packed(k, bits)) and torch.equal(parked.v.cpu(), packed(v, bits)) and torch.equal(eng._k_caches[0][:, :, :49], k)
    eng.prefill_slot(0, S.make_prompt(20, seed=4, vocab_size=2048))
    eng.prefill_slot(2, S.make_prompt(30, seed=5, vocab_size=2048))
    behind = eng._k_caches[2][:, :, 49:].clone()
    eng.resume_slot(2, parked)
    assert eng.positions == [20, 0, 49]
    for cache, x in ((eng._k_caches[2], k), (eng._v_caches[2], v)):
        exact = values(packed(x, bits), 128)
        assert bool(((cache[:, :, :49].double().cpu() - exact).abs() <= rounded_off(exact, torch.float16)).all())
    assert torch.equal(eng._k_caches[2][:, :, 49:], behind)
    eng._k_caches[1][:, :, :49], eng._v_caches[1][:, :, :49] = eng._k_caches[2][:, :, :49], eng._v_caches[2][:, :, :49]
    torch.cuda.synchronize()
    eng.positions[1] = 49
    one, other = eng.decode_slots([1, 2], [prompt[-1]] * 2, 6)
    assert one == other and eng.positions == [20, 55, 55]
    for bad in (lambda: eng.park_slot(3), lambda: eng.resume_slot(-1, parked), lambda: eng.resume_slot(0, parked._replace(length=97)),
                lambda: eng.resume_slot(0, parked._replace(k=parked.k[:2]))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        eng.park_slot(0, 5)
    assert eng.positions == [20, 55, 55]
    eng.positions[0] = 0
    empty = eng.park_slot(0)
    eng.resume_slot(1, empty)
    assert empty.length == 0 and eng.positions[1] == 0


@pytest.mark.gpu
def test_a_graph_beside_another_and_other_sizes_in_between(gpu):
    """Two graphs of the two ways a call is cut, replayed in turn and with calls of their own between: each keeps its workspace."""
    cases = [attention_inputs(3, 16, 8, 128, 4, 300, seed=s) for s in (1, 2)]
    cases[1] = (cases[1][0], with_room(cases[1][1], 20000), with_room(cases[1][2], 20000))
    lens = torch.tensor([300, 0, 117], dtype=torch.int32).cuda()
    want = [gpu.attention_packed_cache(*c, lens) for c in cases]
    graphs, got = [], []
    for c in cases * 2:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(gpu.attention_packed_cache(*c, lens))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        again = gpu.attention_packed_cache(*cases[1], lens)
    torch.cuda.synchronize()
    for i, (out, lse) in enumerate(got):
        assert torch.equal(out, want[i % 2][0]) and torch.equal(lse, want[i % 2][1])
    assert torch.equal(again[0], want[1][0])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_caches_further_apart_than_32_bits(gpu, bits):
    """Sequences and heads more than 4 GiB apart."""
    size = gpu.packed_row_bytes(128, bits)
    apart = (1 << 32) + 4096
    memory = torch.empty(3 * apart + 20000 * size, dtype=torch.uint8, device="cuda")
    k, v, q = made(2, 2, 9, 128, seed=1), made(2, 2, 9, 128, seed=2), made(2, 4, 128, seed=3)
    kc, vc = (memory[first:].as_strided((2, 2, 10, size), (2 * apart, apart, size, 1)) for first in (0, 10 * size))
    gpu.write_cache_packed(k, v, kc, vc, 1)
    assert torch.equal(kc[:, :, 1:].cpu(), packed(k, bits)) and torch.equal(vc[:, :, 1:].cpu(), packed(v, bits))
    kc[:, :, 0], vc[:, :, 0] = kc[:, :, 1], vc[:, :, 1]
    back = gpu.read_cache_packed(kc, vc, 10, 128)
    exact = values(kc.cpu(), 128)
    assert bool(((back[0].double().cpu() - exact).abs() <= rounded_off(exact, torch.float16)).all())
    lens = torch.tensor([10, 7], dtype=torch.int32)
    check_attention(gpu.attention_packed_cache(q, kc, vc, lens.cuda()), q, kc, vc, lens)
    # the same with room for many rows: clusters of a sequence, the line of tiles
    long = memory.as_strided((1, 2, 20000, size), (0, apart, size, 1))
    long[:, :, :9] = packed(k[:1], bits).cuda()
    lens = torch.tensor([9], dtype=torch.int32)
    check_attention(gpu.attention_packed_cache(q[:1], long, long, lens.cuda()), q[:1], long, long, lens)
    long, lens = long.expand(40, -1, -1, -1), torch.tensor([9 - b % 4 for b in range(40)], dtype=torch.int32)
    check_attention(gpu.attention_packed_cache(q[:1].expand(40, -1, -1), long, long, lens.cuda()), q[:1].expand(40, -1, -1), long, long, lens)


# ------------------------------------------------------------------------------------------------------------- quarters that are no numbers beside others
def with_bad_quarters(dim, dtype, seed=0):
    """Rows of random values, each with a NaN or an infinity at one place of a quarter, at several, or in several quarters; rows without one between them."""
    x = torch.randn(1, 3, 4 * 3 * (dim // 4) + 9, dim, generator=torch.Generator().manual_seed(seed)).to(DTYPES[dtype])
    n = 0
    for quarter in range(4):
        for bad in (math.nan, math.inf, -math.inf):
            for d in range(dim // 4):
                x[0, n % 3, n, dim // 4 * quarter + d] = bad
                if n % 5 == 0:
                    x[0, n % 3, n, (dim // 4 * (quarter + 1) + d) % dim] = -bad
                if n % 7 == 0:
                    x[0, n % 3, n, dim // 4 * quarter:dim // 4 * (quarter + 1)] = bad
                n += 1
    x[0, 0, n] = math.nan
    x[0, 1, n + 1, 3], x[0, 1, n + 1, 4] = math.inf, -math.inf
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
def test_quarters_beside_one_without_numbers_keep_their_codes(gpu, dim, bits, dtype):
    """Every byte of such rows: the other quarters' codes, the middle code in the bad ones, the trailers."""
    x = with_bad_quarters(dim, dtype)
    want = packed(x, bits), packed(-x, bits)
    got = [torch.zeros(want[0].shape, dtype=torch.uint8, device="cuda") for _ in range(2)]
    gpu.write_cache_packed(x.cuda(), -x.cuda(), *got)
    for w, g in zip(want, got):
        assert torch.equal(g.cpu(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
@pytest.mark.parametrize("q_heads", [2, 4, 8, 16])
def test_outputs_beside_a_value_without_numbers(gpu, dim, bits, q_heads):
    """A value that is no number leaves the other three quarters of its head's outputs what the rows' values give, written by the operator itself."""
    rows = 40
    q, kc, vc = attention_inputs(4, q_heads, 1, dim, bits, rows)
    v = made(4, 1, rows, dim, seed=1, gain=0.5)
    for b in range(4):
        v[b, 0, 7 + b, dim // 4 * b + 1] = (math.nan, math.inf, -math.inf, math.nan)[b]
    gpu.write_cache_packed(made(4, 1, rows, dim, seed=0), v, kc, vc)
    lens = torch.full((4,), rows, dtype=torch.int32)
    out, lse = gpu.attention_packed_cache(q, kc, vc, lens.cuda())
    quarter = torch.arange(dim) // (dim // 4)
    bad = (quarter == torch.arange(4)[:, None])[:, None].expand(4, q_heads, dim).cuda()
    assert torch.equal(out.isnan(), bad)
    # a row's bad quarter made 0: what the others' outputs go by
    good = v.clone()
    for b in range(4):
        good[b, 0, 7 + b, dim // 4 * b:dim // 4 * (b + 1)] = 0.0
    check_attention((torch.where(bad, gpu.attention_packed_cache(q, kc, packed(good, bits).cuda(), lens.cuda())[0], out), lse), q, kc, packed(good, bits), lens)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_ranges_that_32_bits_do_not_hold(gpu, dtype, dim, bits):
    """Ranges beside a tie of the scale, where a difference rounded to 32 bits would lie on it: the scales and codes of exact arithmetic.  fp16: 316 pairs of lowest and
    highest value with 4 bits, 576 with 8; bf16: 12 with 8 and the smallest scales."""
    mantissa, levels, pairs = {"fp16": 10, "bf16": 7}[dtype], 2 ** bits - 1, [(15 * 2.0 ** -25, -2.0 ** -60), (45 * 2.0 ** -25, 2.0 ** -60)]
    high = np.arange(2 ** mantissa, 2 ** (mantissa + 1)) * 2.0 ** (14 - mantissa)
    for below in range(8, 24):
        low = -high * 2.0 ** -below
        exact = ((high[:, None] - low) / levels).astype(np.float16)
        rounded = ((high.astype(np.float32)[:, None] - low.astype(np.float32)) / np.float32(levels)).astype(np.float16)
        pairs += [(high[i], low[j]) for i, j in zip(*np.nonzero(exact != rounded))]
    pairs = np.array(pairs)
    assert len(pairs) == 2 + {("fp16", 4): 316, ("fp16", 8): 576, ("bf16", 4): 0, ("bf16", 8): 12}[dtype, bits]
    share = np.random.default_rng(1).random((1, 1, len(pairs), dim))
    share[..., ::dim // 4], share[..., 1::dim // 4] = 0.0, 1.0
    x = torch.from_numpy(pairs[:, 1:] + (pairs[:, :1] - pairs[:, 1:]) * share).to(DTYPES[dtype])
    got = [torch.zeros(1, 1, len(pairs), gpu.packed_row_bytes(dim, bits), dtype=torch.uint8, device="cuda") for _ in range(2)]
    gpu.write_cache_packed(x.cuda(), -x.cuda(), *got)
    assert torch.equal(got[0].cpu(), packed(x, bits)) and torch.equal(got[1].cpu(), packed(-x, bits))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
def test_values_beside_a_border_by_less_than_64_bits_hold(gpu, dim, bits):
    """Quarters from -L to L (L half the levels: scale 1, centre 1/2), so 0 lies between the codes M - 1 and M: bf16 values above it become M, those below it M - 1, 0 itself
    the even one, M."""
    levels, middle = 2 ** bits - 1, 2 ** (bits - 1)
    n = dim // 4 - 2
    sizes = 2.0 ** -torch.arange(20, 20 + 4 * n * 2, 2).double().clamp(max=133).view(4, 1, n).expand(4, 3, n)
    x = torch.zeros(4, 3, 4, n + 2, dtype=torch.float64)
    x[..., 0], x[..., 1] = -levels / 2, levels / 2
    x[..., 2:] = (sizes * torch.tensor([1.0, -1.0, 0.0]).double()[:, None])[:, :, None]
    x = x.view(1, 4, 3, dim).bfloat16()
    assert bool((x.double().view(4, 3, 4, n + 2)[:, :2, :, 2:].abs() == sizes[:, :2, None]).all())
    got = [torch.zeros(1, 4, 3, gpu.packed_row_bytes(dim, bits), dtype=torch.uint8, device="cuda") for _ in range(2)]
    gpu.write_cache_packed(x.cuda(), (-x).cuda(), *got)
    for sign, cache in zip((1.0, -1.0), got):
        z, s, n = parts(cache, dim)
        at = x.double() * sign
        want = torch.where(at.abs() == levels / 2, at - 0.5, torch.where(at < 0, -1.0, 0.0))
        assert bool((z == 0.5).all()) and bool((s == 1).all()) and torch.equal(n, want)


def check_hardest(got, q, kc, vc, lens, scale):
    """``check_attention`` where scores lie so far apart that the largest takes all: the output is its row, off by its rounding and by that of the scale to 11 bits; the
    logarithm is its score, which has the error of a fp32 sum.  Heads whose two largest scores are closer than that are left out of the first."""
    out, lse, sure_heads = *(x.double().cpu() for x in got), []
    dim, group, bits = q.shape[2], q.shape[1] // kc.shape[1], (kc.shape[3] - 16) * 8 // q.shape[2]
    for b in range(q.shape[0]):
        (kz, ks, kn), (vz, vs, vn) = (tuple(x.repeat_interleave(group, 0) for x in parts(c[b][:, :int(lens[b])], dim)) for c in (kc, vc))
        qb = q[b].double().cpu()
        s = torch.einsum("hd,hnd->hn", qb, kz + ks * kn) * scale
        error = (dim + 8) * 2.0 ** -24 * torch.einsum("hd,hnd->hn", qb.abs(), kz.abs() + ks * 2 ** bits).amax(1) * abs(scale)
        first, second = s.topk(2, 1).values.unbind(1)
        sure = first - second > 2 * error + 1e3
        sure_heads.append(sure)
        at = s.argmax(1)[:, None, None].expand(-1, 1, dim)
        z, move = vz.gather(1, at)[:, 0], (vs * vn).gather(1, at)[:, 0]
        tol = torch.finfo(q.dtype).eps / 2 * (z + move).abs() + 2.0 ** -11 * 1.001 * (z.abs() + move.abs()) + 2.0 ** -20 * (z.abs() + vs.gather(1, at)[:, 0] * 2 ** bits)
        assert bool(((out[b] - z - move).abs() <= tol)[sure].all()) and bool(out.isfinite().all()), (b, float(((out[b] - z - move).abs() / tol)[sure].max()))
        assert bool(((lse[b] - first).abs() <= error + 2.0 ** -22 * first.abs()).all()), (b, lse[b], first)
    assert float(torch.cat(sure_heads).double().mean()) >= 0.8                 # (of the inputs)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
@pytest.mark.parametrize("q_heads", [4, 8, 16, 32])
@pytest.mark.parametrize("room", [300, 20000])
def test_scores_far_apart(gpu, dim, bits, q_heads, room):
    """Scores of 1e9 to 1e37: large scales, bf16 queries of up to 2^118, and keys so small that the scale alone has no place in 32 bits."""
    seqs, rows = 3, 300
    lens = torch.tensor([300, 41, 230], dtype=torch.int32)
    for dtype, size, keys, scale in (("fp16", 1.0, 1.0, 1e9), ("fp16", 1.0, 1.0, -1e20), ("fp16", 2.0 ** -10, 1.0, 1e30), ("fp16", 1.0, 2.0 ** -8, 1e37), ("fp16", 1.0, 2.0 ** -12, -1.9e38),
                                     ("bf16", 1.0, 1.0, 1e36), ("bf16", 2.0 ** 107, 1.0, None), ("bf16", 2.0 ** 116, 1.0, None), ("bf16", 2.0 ** 118, 2.0 ** -9, -2.0),
                                     ("bf16", 2.0 ** 100, 2.0 ** -12, 2.0 ** 20), ("bf16", 2.0 ** -100, 1.0, 1e37)):
        q = (made(seqs, q_heads, dim, seed=6).float().clamp(-4, 4) * size).to(DTYPES[dtype])
        k, v = made(seqs, 2, rows, dim, seed=7, gain=keys), made(seqs, 2, rows, dim, seed=8)
        kc, vc = (with_room(packed(x, bits).cuda(), room) for x in (k, v))
        check_hardest(gpu.attention_packed_cache(q, kc, vc, lens.cuda(), scale=scale), q, kc, vc, lens, dim ** -0.5 if scale is None else scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
@pytest.mark.parametrize("q_heads", [4, 8, 16, 32])
@pytest.mark.parametrize("room", [300, 20000])
def test_fp16_outputs_are_as_near_as_their_rounding(gpu, dim, bits, q_heads, room):
    """Weights and their products with scales keep 22 bits or more: over all outputs the error is that of rounding the results in 64 bits to fp16, about 2^-12.2 of them.  A
    twentieth more leaves 2^-16.5 for the fp32 sums, whose steps of 2^-24 add up to some 2^-20."""
    rows = 300
    q, kc, vc = attention_inputs(4, q_heads, 2, dim, bits, rows, seed=q_heads)
    out, _ = gpu.attention_packed_cache(q, with_room(kc, room), with_room(vc, room), torch.full((4,), rows, dtype=torch.int32).cuda())
    k, v = (values(c, dim).repeat_interleave(q_heads // 2, 1) for c in (kc, vc))
    want = torch.einsum("bhn,bhnd->bhd", torch.softmax(torch.einsum("bhd,bhnd->bhn", q.double().cpu(), k) * dim ** -0.5, 2), v)
    assert float((out.double().cpu() - want).norm()) <= 1.05 * float((want.half().double() - want).norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
@pytest.mark.parametrize("q_heads", [4, 8, 16, 32])
@pytest.mark.parametrize("far", [2.0 ** 10, 2.0 ** 14])
def test_rows_beside_much_larger_ones(gpu, dim, bits, q_heads, far, dtype):
    """A row whose values are up to 2^16 times the others', and whose weight is next to nothing: the output is as near to that of 64 bits as its rounding.  A product of
    weight and scale is a number of 22 bits (11 for bf16), its last at 2^-25 of 2^7 times the largest scale: 2^-32 2^16 of a row's own values, and sums of 300 rows' errors are less than a row's."""
    rows = 300
    q, k = made(4, q_heads, dim, dtype=dtype, seed=1), made(4, 2, rows, dim, seed=2)
    v = made(4, 2, rows, dim, seed=3, gain=0.25)
    q[..., 0], k[:, :, ::97, 0] = 16.0, -40.0 * (dim / 64) ** 0.5
    v[:, :, ::97] = (made(4, 2, rows, dim, seed=4)[:, :, ::97].float().clamp(-3.5, 3.5) * far).half()
    kc, vc = packed(k, bits).cuda(), packed(v, bits).cuda()
    out, _ = gpu.attention_packed_cache(q, kc, vc, torch.full((4,), rows, dtype=torch.int32).cuda())
    kd, vd = (values(c, dim).repeat_interleave(q_heads // 2, 1) for c in (kc, vc))
    w = torch.softmax(torch.einsum("bhd,bhnd->bhn", q.double().cpu(), kd) * dim ** -0.5, 2)
    assert float(w[:, :, ::97].sum(2).max()) * far < 2.0 ** -40
    want = torch.einsum("bhn,bhnd->bhd", w, vd)
    assert float((out.double().cpu() - want).norm()) <= 1.05 * float((want.to(DTYPES[dtype]).double() - want).norm())


# ------------------------------------------------------------------------------------------------------------- the kernels of a call
def edges_of(graph):
    """Types of a captured graph's edges (cudaGraphEdgeData; 1: programmatic)."""
    class Edge(ctypes.Structure):
        _fields_ = [("from_port", ctypes.c_ubyte), ("to_port", ctypes.c_ubyte), ("type", ctypes.c_ubyte), ("reserved", ctypes.c_ubyte * 5)]
    nodes, edges, count = ((ctypes.c_void_p * 8)() for _ in range(2)), (Edge * 8)(), ctypes.c_size_t(8)
    assert ctypes.CDLL("libcudart.so.12").cudaGraphGetEdges_v2(ctypes.c_void_p(graph.raw_cuda_graph()), *nodes, edges, ctypes.byref(count)) == 0
    return [e.type for e in edges[:count.value]]


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,room,kernels", [(3, 100, 1), (2, 20000, 2), (40, 20000, 2)])
def test_kernels_of_a_call_one_after_the_other(gpu, seqs, room, kernels):
    """``no_overlap``: no edge between the call's kernels is a programmatic one, which it is without it; the same bits."""
    q, kc, vc = attention_inputs(seqs, 16, 8, 128, 4, 100)
    kc, vc = with_room(kc, room), with_room(vc, room)
    lens = torch.tensor([(37 * i) % 101 for i in range(seqs)], dtype=torch.int32).cuda()
    want = gpu.attention_packed_cache(q, kc, vc, lens)
    out, lse = torch.empty_like(q), torch.empty(seqs, 16, device="cuda")
    need = gpu._lib.qmk_attention_packed_cache_workspace(seqs, 16, 8, 128, 4, room)
    workspace = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    cache = cache_args(gpu, num_sequences=seqs, rows=room, k=None, v=None, k_base=kc.data_ptr(), v_base=vc.data_ptr(), seq_stride=8 * room * 80, head_stride=room * 80)
    for serial in (0, 1):
        a = attention_args(gpu, q=q.data_ptr(), lens=lens.data_ptr(), scale=128 ** -0.5, no_overlap=serial, out=out.data_ptr(), lse=lse.data_ptr(), workspace=workspace.data_ptr(), workspace_bytes=need)
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph):
            assert gpu._lib.qmk_attention_packed_cache(bytes(cache), bytes(a), torch.cuda.current_stream().cuda_stream) == 0
        assert edges_of(graph) == [0 if serial else 1] * (kernels - 1)
        graph.instantiate()
        out.zero_()
        graph.replay()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.gpu
def test_a_call_without_rows_waits_for_the_kernel_before_it(gpu):
    """More items than clusters take and caches of no rows: one kernel, which writes zeros, no programmatic dependent of what runs before the call."""
    q = made(128, 40, 64)
    kc = torch.empty(128, 20, 0, 48, dtype=torch.uint8, device="cuda")
    lens = torch.full((128,), 5, dtype=torch.int32, device="cuda")
    gpu.attention_packed_cache(q, kc, kc, lens)
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        lens.add_(1)
        out, lse = gpu.attention_packed_cache(q, kc, kc, lens)
    assert edges_of(graph) == [0]
    graph.instantiate()
    out.fill_(1.0)
    graph.replay()
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_no_address_of_a_cache_without_rows_is_looked_at(C):
    """Host arrays or bases that are not there: the calls go on to their next check, or have nothing to do."""
    for where in (dict(v=None), dict(k=None), dict(k=None, v=None), dict(k=None, v=None, k_base=None, v_base=None)):
        cache = cache_args(C, rows=0, **where)
        for name in ("qmk_write_cache_packed", "qmk_read_cache_packed"):
            assert call(C, name, cache, row_args(C, rows=0))[0] == 0
        rc, why = call(C, "qmk_attention_packed_cache", cache, attention_args(C, scale=math.inf))
        assert rc == 2 and b"scale" in why


@pytest.mark.parametrize("seqs,heads,tiles", [(42, 341, 149943), (1, 1, 1), (127, 129, 131081)])
def test_the_most_rows_of_all_heads(C, seqs, heads, tiles):
    """Caches shared by sequences and heads (strides of 0) may have this many rows: 2^31 - 2 tiles of 32 rows, which a warp's count would pass, are refused; fewer go on to the next check."""
    many = seqs * heads * tiles > 2 ** 31 - 16
    cache = cache_args(C, num_sequences=seqs, kv_heads=heads, rows=32 * tiles, head_stride=0)
    rc, why = call(C, "qmk_attention_packed_cache", cache, attention_args(C, q_heads=heads, scale=math.inf))
    assert rc == 2 and (b"2^36" if many else b"scale") in why
    assert (C._lib.qmk_attention_packed_cache_workspace(seqs, heads, heads, 128, 4, 32 * tiles) < 0) == many


def two_places(C, **change):
    return cache_args(C, **{**dict(k=None, v=None, k_base=1 << 20, v_base=1 << 21, seq_stride=1 << 16), **change})


@pytest.mark.parametrize("change", [dict(head_stride=0), dict(v_base=1 << 20)])
def test_caches_whose_rows_would_be_written_twice_are_refused(C, change):
    rc, why = call(C, "qmk_write_cache_packed", two_places(C, **change), row_args(C))
    assert rc == 2 and b"share" in why
    assert call(C, "qmk_write_cache_packed", two_places(C, **change), row_args(C, rows=0))[0] == 0
    one = (ctypes.c_void_p * 2)(1 << 20, 1 << 21), (ctypes.c_void_p * 2)(1 << 22, 1 << 21)
    rc, why = call(C, "qmk_write_cache_packed", cache_args(C, k=ctypes.addressof(one[0]), v=ctypes.addressof(one[1])), row_args(C))
    assert rc == 2 and b"share" in why


@pytest.mark.parametrize("change", [dict(v=4096), dict(seq_stride=0), dict(head_stride=0), dict(row_stride=0)])
def test_outputs_whose_rows_share_memory_are_refused(C, change):
    rc, why = call(C, "qmk_read_cache_packed", two_places(C), row_args(C, **{**dict(v=1 << 20), **change}))
    assert rc == 2 and b"share" in why


@pytest.mark.gpu
def test_rows_and_caches_that_may_be_shared(gpu):
    """One row for all heads, sequences and positions written, one cache read for all sequences and by keys and values alike, rows of sequences side by side in one cache."""
    size = gpu.packed_row_bytes(64, 4)
    row, kc, vc = made(1, 1, 1, 64), *(torch.zeros(3, 2, 12, size, dtype=torch.uint8, device="cuda") for _ in range(2))
    same = row.expand(3, 2, 4, 64)
    gpu.write_cache_packed(same, same, kc, vc, 5)
    assert torch.equal(kc[:, :, 5:9].cpu(), packed(row, 4).expand(3, 2, 4, size)) and torch.equal(kc, vc)
    k, v = gpu.read_cache_packed(kc[:1].expand(3, -1, -1, -1), kc[:1].expand(3, -1, -1, -1), 4, 64, starts=5)
    want = values(packed(row, 4), 64).expand(3, 2, 4, 64)
    assert torch.equal(k, v) and bool(((k.double().cpu() - want).abs() <= rounded_off(want, torch.float16)).all())
    rows = made(3, 2, 4, 64, seed=2)
    gpu.write_cache_packed(rows, rows, kc[:1].expand(3, -1, -1, -1), vc[:1].expand(3, -1, -1, -1), torch.tensor([8, 0, 4], dtype=torch.int32).cuda())
    for b, at in enumerate((8, 0, 4)):
        assert torch.equal(kc[0, :, at:at + 4].cpu(), packed(rows[b], 4)) and torch.equal(vc[0], kc[0])


@pytest.mark.gpu
def test_sizes_and_scales_that_no_structure_holds_are_refused(gpu):
    q, kc, vc = attention_inputs(2, 4, 2, 64, 4, 8)
    lens = torch.tensor([1, 2], dtype=torch.int32).cuda()
    many = kc[:1, :1, :1].expand(1, 1, 2 ** 31, -1), vc[:1, :1, :1].expand(1, 1, 2 ** 31, -1)
    for scale in (1e39, -1e300, math.inf, math.nan, 3e38):
        with pytest.raises(RuntimeError, match="scale"):
            gpu.attention_packed_cache(q, kc, vc, lens, scale=scale)
    none = torch.empty(2, 4, 0, dtype=torch.float16, device="cuda")
    for call in (lambda: gpu.attention_packed_cache(none, kc, vc, lens), lambda: gpu.write_cache_packed(none[:, :2, None], none[:, :2, None], kc, vc), lambda: gpu.read_cache_packed(kc, vc, 3, 0),
                 lambda: gpu.attention_packed_cache(q[:1, :1], *many, lens[:1]), lambda: gpu.read_cache_packed(*many, 3, 64), lambda: gpu.write_cache_packed(made(1, 1, 2, 64), made(1, 1, 2, 64), *many)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.gpu
def test_a_parked_sequence_is_resumed_up_to_its_rows(gpu):
    """Fewer rows than were parked come back if asked for; more than there are, which would read as zeros, are refused and change nothing."""
    import synthetic as S
    from Model.Qwen06B_architecture import BatchDecoder
    w = S.make_weights(seed=31, num_layers=2, vocab_size=2048, norm_std=0.1, max_seq_len=16)
    eng = BatchDecoder(weights=S.weights_to(w, "cuda"), tokenizer=S.StubTokenizer(-1, 2048), num_sequences=2, max_seq_len=96, engine="gemm", prefill_mode="tensor")
    eng.prefill_slot(0, S.make_prompt(30, seed=3, vocab_size=2048))
    parked = eng.park_slot(0)
    before = eng._k_caches[1].clone()
    for length in (31, 96, -1):
        with pytest.raises(ValueError):
            eng.resume_slot(1, parked._replace(length=length))
    assert eng.positions == [30, 0] and torch.equal(eng._k_caches[1], before)
    eng.resume_slot(1, parked._replace(length=20))
    assert eng.positions == [30, 20] and torch.equal(eng._k_caches[1][:, :, 20:], before[:, :, 20:]) and not torch.equal(eng._k_caches[1][:, :, :20], before[:, :, :20])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
@pytest.mark.parametrize("q_heads", [4, 8, 16, 32])
@pytest.mark.parametrize("room", [300, 20000])
def test_outputs_whose_terms_cancel(gpu, dim, bits, q_heads, room, dtype):
    """Element by element, behind nearly equal weights, whose scores have next to no error: an output that is small beside the sum A of its terms' sizes is as near.  Weights and
    products of weights and scales are two fp16 numbers: off by 2^-22 each of the largest weight's size, and of a scale 2^-4 times the largest 2^-18 of its product; the sums as above."""
    rows, scale = 300, 1e-4
    q, kc, vc = attention_inputs(3, q_heads, 2, dim, bits, rows, dtype, seed=q_heads + dim)
    out, _ = gpu.attention_packed_cache(q, with_room(kc, room), with_room(vc, room), torch.full((3,), rows, dtype=torch.int32).cuda(), scale=scale)
    (kz, ks, kn), (vz, vs, vn) = (tuple(x.repeat_interleave(q_heads // 2, 1) for x in parts(c, dim)) for c in (kc, vc))
    qd = q.double().cpu()
    w = torch.softmax(torch.einsum("bhd,bhnd->bhn", qd, kz + ks * kn) * scale, 2)
    want, a, u = (torch.einsum("bhn,bhnd->bhd", w, x) for x in (vz + vs * vn, vz.abs() + (vs * vn).abs(), vz.abs() + vs * 2 ** bits))
    ds = dim * 2.0 ** -24 * torch.einsum("bhd,bhnd->bhn", qd.abs(), kz.abs() + ks * 2 ** bits).amax(2, keepdim=True) * scale
    tol = torch.finfo(q.dtype).eps / 2 * want.abs() + 2.0 ** -18 * a + u * (2 * ds + 2 * (rows / 16 + 2) * 2.0 ** -23 + 2.0 ** -21)
    err = (out.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
@pytest.mark.parametrize("q_heads", [4, 8, 16, 32])
def test_scores_are_sums_of_32_bits(gpu, dim, bits, q_heads, dtype):
    """One row: the logarithm is its score.  S the sum of |q| (|z| + s 2^bits) times scale, of which the running sums are less than half: four groups of products and the sum over centres,
    each cut off at 2^-24 of its running sum or rounded, come to no more than the 2^-24 S that a rounding of S would."""
    q, kc, vc = attention_inputs(60, q_heads, 2, dim, bits, 1, dtype, seed=q_heads)
    _, lse = gpu.attention_packed_cache(q, kc, vc, torch.ones(60, dtype=torch.int32).cuda())
    z, s, n = (x.repeat_interleave(q_heads // 2, 1)[:, :, 0] for x in parts(kc, dim))
    qd = q.double().cpu()
    want, size = (torch.einsum("bhd,bhd->bh", a, b) * dim ** -0.5 for a, b in ((qd, z + s * n), (qd.abs(), z.abs() + s * 2 ** bits)))
    err = (lse.double().cpu() - want).abs() / size
    assert float(err.max()) <= 2.0 ** -24, math.log2(float(err.max()))
