"""``attention_shared_prefix`` against softmax(scale q k^T) v in 64 bits on the same rounded inputs.

Tolerance of an output element, with A = sum of weight * |v| for it: its own rounding, eps / 2 of it; the weights' rounding to the operand type before they
multiply v, eps / 2 of A; the scores' fp32 sums over dim products, dim 2^-24 of the largest sum of |q k| times scale as an absolute
error of the exponent, so the same relative error of a weight, twice (numerator and denominator); the fp32 sums of the output, whose accumulator may
truncate: 2^-23 for each of the n / 16 steps, and as much for the sum of weights.  exp2 in hardware adds 2^-22.  Weights below 2^-26 of the
largest lose bits in fp16: 2^-37 |v| each at most.  The logarithm has the scores' error, 2^-22 of itself, and that of the sum."""

import ctypes
import math

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


def inputs(seqs, q_heads, kv_heads, dim, prefix, own, lens, dtype, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    q, kp, vp, ko, vo = (torch.randn(*s, generator=g).mul_(gain if i == 0 else 1.0).to(DTYPES[dtype]).cuda() for i, s in enumerate(
        ((seqs, q_heads, dim), (kv_heads, prefix, dim), (kv_heads, prefix, dim), (seqs, kv_heads, own, dim), (seqs, kv_heads, own, dim))))
    return q, kp, vp, ko, vo, torch.tensor(lens, dtype=torch.int32).cuda()


def check(got, q, kp, vp, ko, vo, lens, scale=None):
    out, lse = got
    seqs, q_heads, dim = q.shape
    kv_heads, prefix = kp.shape[:2]
    group = q_heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous() and lse.dtype == torch.float32 and lse.shape == (seqs, q_heads)
    eps = torch.finfo(q.dtype).eps
    for b in range(seqs):
        n = min(max(int(lens[b]), 0), ko[b].shape[1])
        k = torch.cat((kp, ko[b][:, :n]), 1).double().repeat_interleave(group, 0)
        v = torch.cat((vp, vo[b][:, :n]), 1).double().repeat_interleave(group, 0)
        total = prefix + n
        if total == 0:
            assert bool((out[b] == 0).all()) and bool((lse[b] == -math.inf).all())
            continue
        s = torch.einsum("hd,hnd->hn", q[b].double(), k) * scale
        w = torch.softmax(s, 1)
        want, a = torch.einsum("hn,hnd->hd", w, v), torch.einsum("hn,hnd->hd", w, v.abs())
        ds = dim * 2.0 ** -24 * (torch.einsum("hd,hnd->hn", q[b].double().abs(), k.abs()).amax(1, keepdim=True) * abs(scale)) + s.abs().amax(1, keepdim=True) * 2.0 ** -23
        steps = (total / 16 + 2) * 2.0 ** -23
        tol = eps / 2 * (want.abs() + a * 1.001) + a * (2 * ds + 2 * steps + 2.0 ** -21) + total * 2.0 ** -37 * v.abs().amax()
        err = (out[b].double() - want).abs()
        assert bool((err <= tol).all()), (b, float((err / tol).max()))
        want_lse = torch.logsumexp(s, 1)
        err = (lse[b].double() - want_lse).abs()
        assert bool((err <= ds[:, 0] + 2.0 ** -22 * (1 + want_lse.abs()) + steps).all()), (b, float(err.max()))


# ------------------------------------------------------------------------------------------------------------- refusals (no device)
def args(C, **change):
    n = change.get("num_sequences", 2)
    own = (ctypes.c_void_p * max(n, 1))(*[4096] * max(n, 1))
    a = dict(type=0, num_sequences=2, q_heads=16, kv_heads=8, head_dim=128, q=4096, q_seq_stride=2048, q_head_stride=128, k_prefix=4096, v_prefix=4096,
             prefix_len=10, prefix_row_stride=128, prefix_head_stride=1280, k_own=ctypes.addressof(own), v_own=ctypes.addressof(own), own_rows=4,
             own_row_stride=128, own_head_stride=512, own_lens=4096, own_lens_add=0, scale=1.0, out=4096, lse=None, workspace=4096, workspace_bytes=1 << 30)
    a.update(change)
    made = C._SharedPrefixArgs(**a)
    made.keep = own
    return made


@pytest.mark.parametrize("change,text", [(dict(num_sequences=0), b"num_sequences"), (dict(num_sequences=129), b"num_sequences"), (dict(type=2), b"type"),
                                         (dict(head_dim=96), b"head_dim"), (dict(kv_heads=0), b"kv_heads"), (dict(q_heads=12), b"kv_heads"),
                                         (dict(q_heads=136), b"kv_heads"), (dict(prefix_len=-1), b"length"), (dict(own_rows=-1), b"length"), (dict(prefix_len=(1 << 24) + 1), b"length"), (dict(k_own=None, k_own_base=4096, v_own_base=4096, own_seq_stride=12), b"aligned"),
                                         (dict(q=None), b"null"), (dict(out=None), b"null"), (dict(k_prefix=None), b"null"), (dict(own_lens=None), b"null"),
                                         (dict(k_own=None), b"null"), (dict(v_own=None), b"null"), (dict(k_own=None, k_own_base=4096), b"null"), (dict(scale=float("inf")), b"scale"), (dict(scale=float("nan")), b"scale"),
                                         (dict(q=4098), b"aligned"), (dict(v_prefix=4104), b"aligned"), (dict(workspace=4112), b"aligned"), (dict(q_seq_stride=2049), b"strides"),
                                         (dict(prefix_row_stride=132), b"strides"), (dict(own_head_stride=4), b"strides"),
                                         (dict(workspace=None), b"workspace"), (dict(workspace_bytes=100), b"workspace")])
def test_refused_before_anything_runs(C, change, text):
    assert C._lib.qmk_attention_shared_prefix(ctypes.byref(args(C, **change)), None) == 2 and text in C._lib.qmk_last_error()


def test_null_arguments_and_null_caches_are_refused(C):
    assert C._lib.qmk_attention_shared_prefix(None, None) == 2
    holes = (ctypes.c_void_p * 2)(4096, None)
    assert C._lib.qmk_attention_shared_prefix(ctypes.byref(args(C, v_own=ctypes.addressof(holes))), None) == 2 and b"null" in C._lib.qmk_last_error()


@pytest.mark.gpu
def test_wrong_tensors_are_refused(gpu):
    good = inputs(2, 4, 2, 64, 8, 8, [1, 2], "fp16")
    q, kp, vp, ko, vo, lens = good
    bad = [(q.float(), *good[1:]), (q[0], *good[1:]), (q.cpu(), *good[1:]), (q, kp.bfloat16(), vp, ko, vo, lens), (q, kp[:1], vp[:1], ko, vo, lens),
           (q, kp, vp[:, :4], ko, vo, lens), (q, kp, vp, ko[:1], vo[:1], lens), (q, kp, vp, ko, vo[:, :, :4], lens), (q, kp, vp, ko, vo, lens.long()),
           (q, kp, vp, ko, vo, lens[:1]), (q, kp, vp, ko, vo, lens.cpu()), (q, kp, vp, list(ko)[:1], list(vo), lens), (q, kp, vp, ko.float(), vo.float(), lens),
           (q[:, :3], *good[1:]), (q, kp, vp, [ko[0], ko[1].transpose(0, 1)], list(vo), lens)]
    for case in bad:
        with pytest.raises(RuntimeError):
            gpu.attention_shared_prefix(*case)


# ------------------------------------------------------------------------------------------------------------- results
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("q_heads,kv_heads,dim", [(16, 8, 128), (4, 4, 64), (6, 2, 128), (8, 1, 64), (16, 1, 128), (32, 4, 64)])
@pytest.mark.parametrize("seqs,prefix,own", [(1, 1, 1), (1, 0, 5), (2, 63, 16), (3, 64, 64), (5, 65, 300), (17, 1000, 33), (40, 129, 65), (128, 200, 20), (37, 64, 1), (100, 448, 7)])
def test_matches_the_definition(gpu, dtype, q_heads, kv_heads, dim, seqs, prefix, own):
    lens = [(own * (i + 1) // seqs) if i % 5 else (0 if i else own) for i in range(seqs)]
    case = inputs(seqs, q_heads, kv_heads, dim, prefix, own, lens, dtype, seed=seqs + prefix)
    check(gpu.attention_shared_prefix(*case), *case)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,q_heads,kv_heads,prefix,own", [(8, 16, 8, 32768, 64), (64, 16, 8, 4097, 513), (128, 16, 8, 2049, 100), (33, 32, 4, 5000, 1), (100, 8, 8, 777, 1025)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_long_prefixes_and_full_batches(gpu, dtype, seqs, q_heads, kv_heads, prefix, own):
    case = inputs(seqs, q_heads, kv_heads, 128, prefix, own, [(7919 * i) % (own + 1) for i in range(seqs)], dtype, seed=prefix, gain=1.5)
    check(gpu.attention_shared_prefix(*case), *case)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,own,lens", [(1, 20000, [19999]), (3, 9001, [9001, 0, 300]), (40, 6000, [5999] + [0] * 20 + [64 * i for i in range(19)])])
@pytest.mark.parametrize("prefix", [0, 77])
def test_long_caches_of_their_own(gpu, seqs, own, lens, prefix):
    """Caches of more rows than sixteen short ranges, most of them behind the sequence's last."""
    case = inputs(seqs, 16, 8, 128, prefix, own, lens, "fp16", seed=own)
    check(gpu.attention_shared_prefix(*case), *case)


@pytest.mark.gpu
def test_no_rows_at_all_and_lengths_outside_the_cache(gpu):
    q, kp, vp, ko, vo, _ = inputs(6, 16, 8, 128, 0, 40, [0] * 6, "fp16")
    lens = torch.tensor([0, -3, 40, 41, 10 ** 6, 1], dtype=torch.int32).cuda()     # taken into [0, 40]
    check(gpu.attention_shared_prefix(q, kp, vp, ko, vo, lens), q, kp, vp, ko, vo, lens)
    none = ko[:, :, :0]
    out, lse = gpu.attention_shared_prefix(q, kp, vp, none, none, lens)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    q, kp, vp, ko, vo, _ = inputs(6, 16, 8, 128, 100, 0, [0] * 6, "fp16")
    check(gpu.attention_shared_prefix(q, kp, vp, ko, vo, lens), q, kp, vp, ko, vo, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [3, 20, 70])
@pytest.mark.parametrize("garbage", [float("nan"), float("inf"), -65504.0])
def test_rows_behind_the_last_are_not_looked_at(gpu, garbage, seqs):
    """Views of larger buffers: what lies behind the prefix, behind a sequence's last row and between heads is garbage."""
    q, kp, vp, ko, vo, lens = inputs(seqs, 16, 8, 128, 301, 77, [(13 * i) % 78 for i in range(seqs)], "fp16", seed=4)
    def bury(t, dim):
        shape = list(t.shape)
        shape[dim] += 51
        wide = torch.full(shape, garbage, dtype=t.dtype, device="cuda")
        wide.narrow(dim, 0, t.shape[dim]).copy_(t)
        return wide.narrow(dim, 0, t.shape[dim])
    kp, vp, ko, vo = bury(kp, 1), bury(vp, 1), bury(ko, 2), bury(vo, 2)
    for b, n in enumerate(lens.tolist()):
        ko[b, :, n:] = garbage
        vo[b, :, n:] = garbage
    got = gpu.attention_shared_prefix(q, kp, vp, ko, vo, lens)
    assert not bool(got[0].isnan().any())
    check(got, q, kp, vp, ko, vo, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [9, 70])
def test_other_strides_and_lists_of_caches(gpu, seqs):
    """Heads between rows ([rows, heads, dim] caches), queries in a wider buffer, caches of separate allocations: views of one layer of
    the engine's [layer][head][position] caches."""
    prefix, own = 150, 60
    lens = torch.tensor([(11 * i) % 61 for i in range(seqs)], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(8)
    caches = [[torch.randn(3, 8, prefix + own, 128, generator=g).half().cuda() for _ in range(seqs)] for _ in range(2)]
    q = torch.randn(seqs, 40, 128, generator=g).half().cuda()[:, 8:24]
    kp, vp = caches[0][0][1][:, :prefix], caches[1][0][1][:, :prefix]
    ko, vo = ([c[1][:, prefix:] for c in side] for side in caches)
    check(gpu.attention_shared_prefix(q, kp, vp, ko, vo, lens), q, kp, vp, ko, vo, lens)
    turned = [torch.randn(*s, generator=g).half().cuda() for s in ((prefix, 8, 128), (prefix, 8, 128), (seqs, own, 8, 128), (seqs, own, 8, 128))]
    case = (q, turned[0].transpose(0, 1), turned[1].transpose(0, 1), turned[2].transpose(1, 2), turned[3].transpose(1, 2), lens)
    check(gpu.attention_shared_prefix(*case), *case)
    same = q[:1].expand(seqs, 16, 128)               # one query for all: stride 0
    check(gpu.attention_shared_prefix(same, *case[1:]), same, *case[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0, 3.0])
@pytest.mark.parametrize("seqs", [20, 80])
def test_scales(gpu, scale, seqs):
    case = inputs(seqs, 16, 8, 128, 333, 50, [(17 * i) % 51 for i in range(seqs)], "fp16", seed=2, gain=0.5)
    check(gpu.attention_shared_prefix(*case, scale=scale), *case, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [4, 66])
def test_a_maximum_that_rises_late(gpu, seqs):
    """Scores that grow along the rows: the running maximum is raised again and again, by more than any threshold."""
    q, kp, vp, ko, vo, lens = inputs(seqs, 16, 8, 128, 2000, 40, [40] * seqs, "fp16", seed=6)
    q[:] = q[:1, :1]
    kp += (torch.linspace(-2, 2, 2000).cuda()[None, :, None] * q[0, 0]).half()
    case = (q, kp, vp, ko, vo, lens)
    check(gpu.attention_shared_prefix(*case), *case)


@pytest.mark.gpu
def test_same_bits_again_on_other_streams_and_in_graphs(gpu):
    case = inputs(30, 16, 8, 128, 999, 99, [(31 * i) % 100 for i in range(30)], "fp16", seed=5)
    want = gpu.attention_shared_prefix(*case)
    for _ in range(3):
        again = gpu.attention_shared_prefix(*case)
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    q2 = case[0].flip(0).contiguous()
    lens2 = case[5].flip(0).contiguous()
    want2 = gpu.attention_shared_prefix(q2, *case[1:5], lens2)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(8):                               # two at a time
        with torch.cuda.stream(streams[i % 2]):
            got.append(gpu.attention_shared_prefix(*(case if i % 2 == 0 else (q2, *case[1:5], lens2))))
    torch.cuda.synchronize()
    for i, (o, l) in enumerate(got):
        w = want if i % 2 == 0 else want2
        assert torch.equal(o, w[0]) and torch.equal(l, w[1])
    q, lens = case[0].clone(), case[5].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(streams[0]):
        gpu.attention_shared_prefix(q, *case[1:5], lens)
        with torch.cuda.graph(graph, stream=streams[0]):
            out, lse = gpu.attention_shared_prefix(q, *case[1:5], lens)
        for new_q, new_lens, w in ((case[0], case[5], want), (q2, lens2, want2), (case[0], case[5], want)):
            q.copy_(new_q)
            lens.copy_(new_lens)
            graph.replay()
            assert torch.equal(out, w[0]) and torch.equal(lse, w[1])


# ------------------------------------------------------------------- many queries against many rows (from 96 M products on)
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("q_heads,kv_heads,dim,seqs,prefix", [(16, 8, 128, 49, 1024), (16, 8, 128, 65, 1100), (16, 8, 128, 128, 513), (4, 4, 64, 128, 3333), (6, 2, 128, 128, 1153),
                                                              (8, 1, 64, 111, 2000), (16, 1, 128, 127, 449), (32, 4, 64, 97, 640), (32, 4, 64, 5, 10000), (16, 16, 128, 33, 1500)])
def test_many_queries_and_rows(gpu, dtype, q_heads, kv_heads, dim, seqs, prefix):
    assert seqs * q_heads * dim * prefix >= 96 << 20
    own = 90
    case = inputs(seqs, q_heads, kv_heads, dim, prefix, own, [(19 * i) % (own + 1) for i in range(seqs)], dtype, seed=prefix)
    check(gpu.attention_shared_prefix(*case), *case)


@pytest.mark.gpu
@pytest.mark.parametrize("garbage", [float("nan"), float("inf"), -65504.0])
def test_many_queries_do_not_look_behind_the_last_row(gpu, garbage):
    q, kp, vp, ko, vo, lens = inputs(70, 16, 8, 128, 1001, 77, [(13 * i) % 78 for i in range(70)], "fp16", seed=14)
    wide = [torch.full((8, 1301, 128), garbage, dtype=torch.float16, device="cuda") for _ in range(2)]
    for w, t in zip(wide, (kp, vp)):
        w[:, :1001] = t
    for b, n in enumerate(lens.tolist()):
        ko[b, :, n:] = garbage
        vo[b, :, n:] = garbage
    case = (q, wide[0][:, :1001], wide[1][:, :1001], ko, vo, lens)
    got = gpu.attention_shared_prefix(*case)
    assert not bool(got[0].isnan().any())
    check(got, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0, 3.0])
def test_many_queries_and_scales(gpu, scale):
    case = inputs(80, 16, 8, 128, 899, 50, [(17 * i) % 51 for i in range(80)], "fp16", seed=2, gain=0.5)
    check(gpu.attention_shared_prefix(*case, scale=scale), *case, scale=scale)


@pytest.mark.gpu
def test_many_queries_whose_maximum_rises_late(gpu):
    q, kp, vp, ko, vo, lens = inputs(66, 16, 8, 128, 4000, 40, [40] * 66, "fp16", seed=6)
    q[:] = q[:1, :1]
    kp += (torch.linspace(-2, 2, 4000).cuda()[None, :, None] * q[0, 0]).half()
    case = (q, kp, vp, ko, vo, lens)
    check(gpu.attention_shared_prefix(*case), *case)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [9, 100])
def test_broadcast_inputs_and_heads_between_rows(gpu, seqs):
    """A kv head expanded to all, one query expanded to all, one own cache for all sequences, [rows, heads, dim] caches."""
    q, kp, vp, ko, vo, lens = inputs(seqs, 16, 8, 128, 1001, 50, [(7 * i) % 51 for i in range(seqs)], "fp16", seed=31)
    one = (q, kp[:1].expand(8, 1001, 128), vp[:1].expand(8, 1001, 128), ko[:1].expand(seqs, 8, 50, 128), vo[:1].expand(seqs, 8, 50, 128), lens)
    check(gpu.attention_shared_prefix(*one), *one)
    check(gpu.attention_shared_prefix(*one[:3], [ko[0]] * seqs, [vo[0]] * seqs, lens), *one)
    same = (q[:1].expand(seqs, 16, 128), *one[1:])
    check(gpu.attention_shared_prefix(*same), *same)
    row = (q, kp[:, :1].expand(8, 1001, 128), vp[:, :1].expand(8, 1001, 128), ko, vo, lens)
    check(gpu.attention_shared_prefix(*row), *row)
    between = (q, kp.transpose(0, 1).contiguous().transpose(0, 1), vp.transpose(0, 1).contiguous().transpose(0, 1), ko, vo, lens)
    check(gpu.attention_shared_prefix(*between), *between)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [9, 100])
def test_offsets_of_more_than_32_bits(gpu, seqs):
    """Rows 2^22 and heads 2^31 elements apart; own caches 2^25 apart, so the last from 2^31 on."""
    q, kp, vp, ko, vo, lens = inputs(seqs, 4, 2, 128, 1100, 40, [(7 * i) % 41 for i in range(seqs)], "fp16", seed=41)
    buf = torch.empty(1100 * (1 << 22) + (1 << 12), dtype=torch.float16, device="cuda")
    rows = [buf.as_strided((2, 1100, 128), (256, 1 << 22, 1), at) for at in (0, 128)]
    heads = [buf.as_strided((2, 1100, 128), (1 << 31, 256, 1), at) for at in (1024, 1152)]
    own = [buf.as_strided((seqs, 2, 40, 128), (1 << 25, 128 * 128, 128, 1), at) for at in (1 << 20, (1 << 20) + 128 * 40)]
    for k, v in (rows, heads):
        k.copy_(kp)
        v.copy_(vp)
        check(gpu.attention_shared_prefix(q, k, v, ko, vo, lens), q, kp, vp, ko, vo, lens)
    own[0].copy_(ko)
    own[1].copy_(vo)
    check(gpu.attention_shared_prefix(q, kp, vp, *own, lens), q, kp, vp, ko, vo, lens)


@pytest.mark.gpu
def test_many_queries_two_calls_at_once_and_in_graphs(gpu):
    case = inputs(90, 16, 8, 128, 2000, 99, [(31 * i) % 100 for i in range(90)], "fp16", seed=5)
    other = (case[0].flip(0).contiguous(), *case[1:5], case[5].flip(0).contiguous())
    want = gpu.attention_shared_prefix(*case), gpu.attention_shared_prefix(*other)
    check(want[0], *case)
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, results = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for stream, graph, c in zip(streams, graphs, (case, other)):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=stream):
            results.append(gpu.attention_shared_prefix(*c))
    torch.cuda.synchronize()
    for _ in range(10):
        for out, lse in results:
            out.zero_()
            lse.zero_()
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        got = gpu.attention_shared_prefix(*case)
        torch.cuda.synchronize()
        for (o, l), w in zip((*results, got), (*want, want[0])):
            assert torch.equal(o, w[0]) and torch.equal(l, w[1])


# ------------------------------------------------------------------------------------------------------------- waits that run out
def test_a_negative_budget_of_the_waits_is_refused(C):
    assert C._lib.qmk_attention_shared_prefix(ctypes.byref(args(C, timeout_ms=-1)), None) == 2 and b"timeout_ms" in C._lib.qmk_last_error()
    for budget in (0, -5, 1000001):
        assert C._lib.qmk_selftest_shared_prefix_wait_timeout(budget) == 2 and b"budget_us" in C._lib.qmk_last_error()


@pytest.mark.gpu
def test_waits_run_out_and_leave_the_device_usable(gpu):
    """Score products that stop behind the second tile, with keys and values in flight: status 4 after the budget, NaN for the rows concerned,
    copies landed and TMEM freed (the calls behind it allocate all of it), their results as before."""
    case = inputs(90, 16, 8, 128, 2000, 99, [(31 * i) % 100 for i in range(90)], "fp16", seed=5)
    want = gpu.attention_shared_prefix(*case)
    check(want, *case)
    for _ in range(3):
        assert gpu.selftest_shared_prefix_wait_timeout(300) == 4
        got = gpu.attention_shared_prefix(*case)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,prefix", [(3, 200), (90, 2000)])
def test_the_callers_status_word(gpu, seqs, prefix):
    """A call whose waits end leaves the word as it is, on both ways through."""
    case = inputs(seqs, 16, 8, 128, prefix, 40, [(7 * i) % 41 for i in range(seqs)], "fp16", seed=9)
    q, kp, vp, ko, vo, lens = case
    want = gpu.attention_shared_prefix(*case)
    out, lse, word = torch.empty_like(q), torch.empty(seqs, 16, device="cuda"), torch.tensor([0, 7], dtype=torch.int32, device="cuda")
    need = gpu._lib.qmk_attention_shared_prefix_workspace(seqs, 16, 8, 128, prefix, 40)
    workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
    for i, budget in ((0, 0), (1, 500)):
        a = gpu._SharedPrefixArgs(type=0, num_sequences=seqs, q_heads=16, kv_heads=8, head_dim=128, q=q.data_ptr(), q_seq_stride=2048, q_head_stride=128,
                                  k_prefix=kp.data_ptr(), v_prefix=vp.data_ptr(), prefix_len=prefix, prefix_row_stride=128, prefix_head_stride=128 * prefix,
                                  k_own_base=ko.data_ptr(), v_own_base=vo.data_ptr(), own_seq_stride=8 * 40 * 128, own_rows=40, own_row_stride=128,
                                  own_head_stride=40 * 128, own_lens=lens.data_ptr(), scale=128 ** -0.5, out=out.data_ptr(), lse=lse.data_ptr(),
                                  workspace=workspace.data_ptr(), workspace_bytes=need, status=word.data_ptr() + 4 * i, timeout_ms=budget)
        assert gpu._lib.qmk_attention_shared_prefix(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and word.tolist() == [0, 7]


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,prefix,kernels", [(3, 200, 2), (90, 2000, 3)])
def test_kernels_of_a_call_one_after_the_other(gpu, seqs, prefix, kernels):
    """``no_overlap``: no edge between the call's kernels is a programmatic one, which all of them are without it; the same bits."""
    class Edge(ctypes.Structure):                                # cudaGraphEdgeData; type 1: programmatic
        _fields_ = [("from_port", ctypes.c_ubyte), ("to_port", ctypes.c_ubyte), ("type", ctypes.c_ubyte), ("reserved", ctypes.c_ubyte * 5)]
    runtime = ctypes.CDLL("libcudart.so.12")
    q, kp, vp, ko, vo, lens = case = inputs(seqs, 16, 8, 128, prefix, 40, [(7 * i) % 41 for i in range(seqs)], "fp16", seed=9)
    want = gpu.attention_shared_prefix(*case)
    out, lse = torch.empty_like(q), torch.empty(seqs, 16, device="cuda")
    need = gpu._lib.qmk_attention_shared_prefix_workspace(seqs, 16, 8, 128, prefix, 40)
    workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
    a = gpu._SharedPrefixArgs(type=0, num_sequences=seqs, q_heads=16, kv_heads=8, head_dim=128, q=q.data_ptr(), q_seq_stride=2048, q_head_stride=128,
                              k_prefix=kp.data_ptr(), v_prefix=vp.data_ptr(), prefix_len=prefix, prefix_row_stride=128, prefix_head_stride=128 * prefix,
                              k_own_base=ko.data_ptr(), v_own_base=vo.data_ptr(), own_seq_stride=8 * 40 * 128, own_rows=40, own_row_stride=128,
                              own_head_stride=40 * 128, own_lens=lens.data_ptr(), scale=128 ** -0.5, out=out.data_ptr(), lse=lse.data_ptr(),
                              workspace=workspace.data_ptr(), workspace_bytes=need)
    for serial in (0, 1):
        a.no_overlap = serial
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph):
            assert gpu._lib.qmk_attention_shared_prefix(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
        nodes, edges, count = ((ctypes.c_void_p * 8)() for _ in range(2)), (Edge * 8)(), ctypes.c_size_t(8)
        assert runtime.cudaGraphGetEdges_v2(ctypes.c_void_p(graph.raw_cuda_graph()), *nodes, edges, ctypes.byref(count)) == 0
        assert [e.type for e in edges[:count.value]] == [0 if serial else 1] * (kernels - 1)
        graph.instantiate()
        out.zero_()
        graph.replay()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


# ------------------------------------------------------------------------------------------------------------- visible rows whose scores are no numbers
def _hidden_by_scores(seqs, prefix, own, dtype, seed):
    """Inputs some of whose rows have scores of -inf with every query, and the same without these rows."""
    q, kp, vp, ko, vo, lens = inputs(seqs, 16, 8, 128, prefix, own, [(11 * i) % (own + 1) for i in range(seqs)], dtype, seed=seed)
    q[..., 5] = q[..., 5].abs() + 0.5
    g = torch.Generator().manual_seed(seed)
    out_prefix = torch.rand(prefix, generator=g) < 0.3
    out_prefix[:min(prefix, 300)] = True                         # whole tiles at the beginning
    out_own = torch.rand(seqs, own, generator=g) < 0.3
    out_own[0] = True
    out_own[1::3, :16] = True
    kp[:, out_prefix.cuda(), 5] = -math.inf
    ko.transpose(1, 2)[out_own.cuda()] = ko.transpose(1, 2)[out_own.cuda()].index_fill(2, torch.tensor([5], device="cuda"), -math.inf)
    keep = (~out_prefix).cuda()
    rows = [[j for j in range(int(lens[b])) if not out_own[b, j]] for b in range(seqs)]
    fewer = (q, kp[:, keep], vp[:, keep], [ko[b][:, r] for b, r in enumerate(rows)], [vo[b][:, r] for b, r in enumerate(rows)], [len(r) for r in rows])
    return (q, kp, vp, ko, vo, lens), fewer


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("seqs,prefix,own", [(3, 0, 40), (3, 130, 40), (5, 700, 300), (20, 700, 40), (100, 600, 40), (100, 300, 300), (100, 620, 20)])
def test_rows_whose_scores_are_minus_infinity_weigh_nothing(gpu, dtype, seqs, prefix, own):
    """As a mask inside the keys has it: single rows, whole tiles and ranges, all rows of a sequence (zeros and -inf, as without rows)."""
    case, fewer = _hidden_by_scores(seqs, prefix, own, dtype, seqs + prefix + own)
    got = gpu.attention_shared_prefix(*case)
    check(got, *fewer)
    if prefix <= 300:
        assert bool((got[0][0] == 0).all()) and bool((got[1][0] == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("seqs,prefix", [(3, 130), (20, 700), (100, 600)])
def test_a_score_that_is_no_number_makes_its_head_none(gpu, bad, seqs, prefix):
    """A NaN or +inf score of a visible row: NaN for the heads and sequences that see it, the bits of the others as without it."""
    q, kp, vp, ko, vo, lens = inputs(seqs, 16, 8, 128, prefix, 40, [40] * seqs, "fp16", seed=3)
    q[..., 5] = q[..., 5].abs() + 0.5
    want = gpu.attention_shared_prefix(q, kp, vp, ko, vo, lens)
    own = ko.clone()
    own[1, 3, 17, 5] = bad                                       # kv head 3 of sequence 1 alone: query heads 6 and 7
    out, lse = gpu.attention_shared_prefix(q, kp, vp, own, vo, lens)
    assert bool(out[1, 6:8].isnan().all()) and not bool(lse[1, 6:8].isfinite().any())
    rest = torch.ones(seqs, 16, dtype=torch.bool, device="cuda")
    rest[1, 6:8] = False
    assert torch.equal(out[rest], want[0][rest]) and torch.equal(lse[rest], want[1][rest])
    for rows in ([prefix // 2], list(range(prefix))):            # one shared row of kv head 2, and all of them
        k = kp.clone()
        k[2, rows, 5] = bad
        out, lse = gpu.attention_shared_prefix(q, k, vp, ko, vo, lens)
        assert bool(out[:, 4:6].isnan().all()) and not bool(lse[:, 4:6].isfinite().any())
        rest = torch.ones(16, dtype=torch.bool, device="cuda")
        rest[4:6] = False
        assert torch.equal(out[:, rest], want[0][:, rest]) and torch.equal(lse[:, rest], want[1][:, rest])


# ------------------------------------------------------------------------------------------------------------- more refusals
@pytest.mark.gpu
@pytest.mark.parametrize("which", range(1, 6))
@pytest.mark.parametrize("lists", [False, True])
def test_a_tensor_of_the_host_is_refused(gpu, which, lists):
    """Each of the caches and lengths in turn, own caches as one tensor or a list: no address of the host's memory reaches a kernel."""
    case = list(inputs(2, 4, 2, 64, 8, 8, [1, 2], "fp16"))
    case[which] = case[which].cpu()
    if lists:
        case[3], case[4] = list(case[3]), list(case[4])
    with pytest.raises(RuntimeError):
        gpu.attention_shared_prefix(*case)


@pytest.mark.parametrize("sizes", [(128, 1 << 30, 1 << 30, 128, 100, 10), (128, 2 ** 31 - 1, 1, 128, 100, 10), (1, 16, 8, 128, 2 ** 31 - 1, 10), (1, 16, 8, 128, 10, 2 ** 31 - 1),
                                   (1, 16, 8, 128, (1 << 24) + 1, 0), (1, 16, 8, 96, 10, 10), (1, 16, 8, 0, 10, 10), (0, 16, 8, 128, 10, 10), (129, 16, 8, 128, 10, 10),
                                   (1, 17, 1, 128, 10, 10), (1, 12, 8, 128, 10, 10), (1, 0, 0, 128, 10, 10), (1, 16, 8, 128, -1, 10)])
def test_no_workspace_for_sizes_that_are_refused(C, sizes):
    """... nor sums that leave 32 bits on the way to it."""
    assert C._lib.qmk_attention_shared_prefix_workspace(*sizes) == 0


def test_workspace_of_the_largest_sizes(C):
    """128 sequences of 1024 query heads of 128 dims, prefix and own caches of 2^24 rows: a state of 130 floats for each, in at most 17 parts a head."""
    need = C._lib.qmk_attention_shared_prefix_workspace(128, 1024, 64, 128, 1 << 24, 1 << 24)
    assert 17 * 128 * 1024 * 130 * 4 <= need <= 17 * 128 * 1024 * 130 * 4 + 16
