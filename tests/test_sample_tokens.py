"""``sample_tokens`` against its definition in 64 bits.

A pick is a whole number and has to be equal, except where the given number lies on a border: the kernel's masses are whole multiples of
2^-45 of the largest token's, each off by at most half of one, so a running sum of n of them is off by at most n 2^-46, and exp and the division
in 64 bits add less than 2^-48 of each mass (a few units in the last place of 2^-53).  A row whose target u * total or whose top-p target
lies closer than n 2^-45 + total 2^-46 to a border is not held to an equal pick; with inputs drawn once and for all those are counted and hardly
any.  The logarithm is rounded to fp32: half a step, 2^-24 of it, and 2^-46 n / total <= 2^-28 for the total."""

import math

import numpy as np
import pytest
import torch

NO_TOKEN = 2 ** 31 - 1
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def definition(x, u, t, k, p, mp):
    """(token, logprob, on a border) of one row: x in float64, NaN as -inf already; plain numpy."""
    n = len(x)
    if not np.any(x > -np.inf):
        return NO_TOKEN, np.nan, False
    order = np.argsort(-x, kind="stable")
    if not t > 0:
        return int(order[0]), 0.0, False
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.exp(np.where(np.isinf(top), -np.inf, (x - top) / t)))).astype(np.longdouble)
    near = False
    if 1 <= k < n:
        order = order[:k]
    slack = n * 2.0 ** -45 + float(w.sum()) * 2.0 ** -46
    if p < 1:
        run = np.cumsum(w[order])
        want = np.longdouble(np.float32(p)) * run[-1]
        near |= bool(np.min(np.abs(run - want)) < slack)
        order = order[:1 + int(np.sum(run[:-1] < want))]
    order = order[:max(1, int(np.sum(w[order] >= np.float32(mp))))]
    ids = np.sort(order)
    run = np.cumsum(w[ids])
    want = np.longdouble(np.float32(u)) * run[-1]
    near |= bool(np.min(np.abs(run - want)) < slack)
    at = min(int(np.sum(run <= want)), len(ids) - 1)
    return int(ids[at]), float(np.log(w[ids[at]] / run[-1])), near


def check(C, logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, skipped=0.02, exact=False):
    rows = logits.shape[0]

    def of(v, i):
        return v[i].item() if isinstance(v, torch.Tensor) else np.float32(v).item() if isinstance(v, float) else v

    def cuda(v):
        return v.cuda() if isinstance(v, torch.Tensor) else v
    got, logp = C.sample_tokens(logits.cuda() if not logits.is_cuda else logits, cuda(uniforms), cuda(temperature), cuda(top_k), cuda(top_p), cuda(min_p))
    assert got.dtype == torch.int32 and logp.dtype == torch.float32 and got.shape == logp.shape == (rows,)
    got, logp = got.cpu(), logp.cpu()
    x = logits.double().cpu().numpy()
    x = np.where(np.isnan(x), -np.inf, x)
    on_border = 0
    for i in range(rows):
        token, lp, near = definition(x[i], of(uniforms, i), of(temperature, i), of(top_k, i), of(top_p, i), of(min_p, i))
        near &= not exact                          # (sums that are whole numbers on both sides)
        on_border += near
        if near:
            continue
        assert int(got[i]) == token, (i, int(got[i]), token)
        if np.isnan(lp):
            assert math.isnan(float(logp[i]))
        else:
            assert abs(float(logp[i]) - lp) <= abs(lp) * 2.0 ** -24 + 2.0 ** -28 + 1e-45, (i, float(logp[i]), lp)
    assert on_border <= skipped * rows
    return got


def rows_of_logits(rows, vocab, seed, sigma=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * sigma
    at = torch.randint(0, vocab, (rows, 8), generator=g)
    return x.scatter_add_(1, at, torch.rand(rows, 8, generator=g) * 8), torch.rand(rows, generator=g), g


@pytest.fixture(scope="module")
def C(built_library):
    import qwen_megakernel_C
    return qwen_megakernel_C


@pytest.fixture(scope="module")
def gpu(C):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return C


# ------------------------------------------------------------------------------------------------------------- refusals (no device)
@pytest.mark.parametrize("change,text", [(dict(rows=-1), b"rows"), (dict(rows=65537), b"rows"), (dict(vocab=0), b"vocabulary"),
                                         (dict(vocab=262145), b"vocabulary"), (dict(kind=3), b"fp32"), (dict(logits=None), b"null"),
                                         (dict(uniforms=None), b"null"), (dict(tokens=None), b"null"), (dict(stride=99), b"overlap"),
                                         (dict(t=-0.5), b"temperature"), (dict(t=float("nan")), b"temperature"), (dict(p=0.0), b"top_p"),
                                         (dict(p=float("nan")), b"top_p"), (dict(mp=-0.1), b"min_p"), (dict(mp=1.5), b"min_p"), (dict(mp=float("nan")), b"min_p")])
def test_refused_before_anything_runs(C, change, text):
    a = dict(logits=4096, kind=0, stride=100, rows=2, vocab=100, uniforms=4096, t=1.0, k=0, p=1.0, mp=0.0, tokens=4096)
    a.update(change)
    rc = C._lib.qmk_sample_tokens(a["logits"], a["kind"], a["stride"], a["rows"], a["vocab"], a["uniforms"], None, a["t"], None, a["k"], None,
                                  a["p"], None, a["mp"], a["tokens"], None, None)
    assert rc == 2 and text in C._lib.qmk_last_error()


def test_no_rows_is_no_work(C):
    assert C._lib.qmk_sample_tokens(None, 0, 0, 0, 100, None, None, 1.0, None, 0, None, 1.0, None, 0.0, None, None, None) == 0


@pytest.mark.gpu
def test_wrong_tensors_are_refused(gpu):
    x, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    bad = [(x.cpu(), u, {}), (x.double(), u, {}), (x[0], u, {}), (x.t(), u, {}), (x, u.cpu(), {}), (x, u.double(), {}), (x, u[:1], {}),
           (x, u, dict(top_k=torch.zeros(2, device="cuda"))), (x, u, dict(top_p=torch.ones(3, device="cuda"))),
           (x, u, dict(temperature=torch.ones(2))), (x, u, dict(min_p=torch.ones(4, device="cuda")[::2])), (x, u, dict(temperature=-1.0))]
    for logits, uniforms, more in bad:
        with pytest.raises(RuntimeError):
            gpu.sample_tokens(logits, uniforms, **more)


# ------------------------------------------------------------------------------------------------------------- picks
@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 255, 257, 1000, 4096, 12288, 12289, 32003, 98305, 151936, 262144])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_every_combination_of_filters(gpu, vocab, dtype):
    kinds = [(k, p, m) for k in (0, 1, 7, 300) for p in (1.0, 0.9, 0.3) for m in (0.0, 0.02)]
    x, u, g = rows_of_logits(len(kinds), vocab, vocab)
    check(gpu, x.to(DTYPES[dtype]), u, temperature=torch.rand(len(kinds), generator=g) + 0.4, top_k=torch.tensor([k for k, _, _ in kinds], dtype=torch.int32),
          top_p=torch.tensor([p for _, p, _ in kinds]), min_p=torch.tensor([m for _, _, m in kinds]), skipped=0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("top_k", [0, 2, 40, 41, 5000, 39999, 40000])
@pytest.mark.parametrize("top_p", [1.0, 0.999, 0.5, 0.01])
def test_ties_go_to_the_lowest_index(gpu, top_k, top_p):
    """Values in steps of a half: a threshold has thousands of tokens on it, of which the first few by index stay."""
    x, u, _ = rows_of_logits(6, 40000, 3)
    # (two tokens: where they tie, both masses are 1 and every sum and border is exact on both sides)
    check(gpu, (x * 2).round() / 2, u, temperature=2.0, top_k=top_k, top_p=top_p, exact=top_k == 2)
    equal = torch.zeros(6, 40000)                  # all the same: u = i / 6 picks the token at that share of what stays
    check(gpu, equal, torch.arange(6) / 6 + 0.01, top_k=top_k, top_p=top_p, exact=True)


@pytest.mark.gpu
@pytest.mark.parametrize("sigma,temperature", [(0.05, 1.0), (1.0, 1.0), (8.0, 1.0), (30.0, 0.7), (2.0, 1e-3), (2.0, 1e-30), (2.0, 50.0), (1e4, 1.0), (1e37, 1.0)])
@pytest.mark.parametrize("top_p", [1.0, 0.95, 0.6])
def test_flat_and_peaked_rows(gpu, sigma, temperature, top_p):
    x, u, _ = rows_of_logits(8, 50000, 11, sigma)
    check(gpu, x, u, temperature=temperature, top_p=top_p)
    check(gpu, x, u, temperature=temperature, top_p=top_p, top_k=20000)


@pytest.mark.gpu
def test_infinite_values_and_numbers_that_are_none(gpu):
    inf, nan = float("inf"), float("nan")
    x = torch.randn(8, 5000, generator=torch.Generator().manual_seed(1))
    x[0] = -inf                                    # nothing there
    x[1] = nan
    x[2] = -inf; x[2, 4321] = -1e30                # one token left
    x[3, ::2] = -inf; x[3, 1::4] = nan
    x[4, 77] = inf; x[4, 4000] = inf               # these two share the mass
    x[5, :4999] = nan
    x[6] = -3.0e38; x[6, 9] = 3.0e38
    x[7, 100] = -0.0; x[7, 50] = 0.0; x[7, :50] = -9.0; x[7, 51:] = -9.0; x[7, 100] = -0.0   # zeros of both signs are equal
    for u in (0.0, 0.4, 0.6, 0.9999999):
        for kw in ({}, dict(top_k=3), dict(top_p=0.7), dict(min_p=0.5), dict(top_k=4000, top_p=0.99), dict(temperature=0.0)):
            # (u = 0 is on a border wherever the first token's mass is next to nothing)
            check(gpu, x, torch.full((8,), u), skipped=0.5 if u else 1.0, **kw)
    tokens, logp = gpu.sample_tokens(x[:2].cuda(), torch.zeros(2, device="cuda"))
    assert tokens.tolist() == [NO_TOKEN] * 2 and bool(logp.isnan().all())
    assert gpu.sample_tokens(x[7:].cuda(), torch.zeros(1, device="cuda"), temperature=0.0)[0].item() == 50


@pytest.mark.gpu
def test_numbers_outside_the_interval_are_drawn_into_it(gpu):
    x = torch.zeros(6, 10, device="cuda")
    x[:, 0] = x[:, 9] = -float("inf")
    u = torch.tensor([-1.0, float("nan"), 0.0, 1.0, 5.0, float("inf")], device="cuda")
    assert gpu.sample_tokens(x, u)[0].tolist() == [1, 1, 1, 8, 8, 8]


@pytest.mark.gpu
def test_every_share_of_the_interval_goes_to_its_token(gpu):
    """A thousand even numbers over one small row: the tokens come in the order of their indices, each as often as its probability says."""
    x = torch.tensor([0.3, -1.0, 2.0, 0.0, 1.2]).repeat(1000, 1)
    got, _ = gpu.sample_tokens(x.cuda(), ((torch.arange(1000) + 0.5) / 1000).cuda())
    counts = torch.bincount(got.cpu(), minlength=5)
    assert torch.equal(got.cpu(), got.cpu().sort().values)
    assert float((counts / 1000 - torch.softmax(x[0].double(), 0)).abs().max()) <= 1.01e-3


@pytest.mark.gpu
def test_rows_apart_and_rows_that_are_not_aligned(gpu):
    x, u, _ = rows_of_logits(5, 7003, 5)
    wide = torch.full((5, 7100), float("nan"))
    for at in (0, 1, 3, 97):
        wide[:, at:at + 7003] = x
        check(gpu, wide.cuda()[:, at:at + 7003], u, top_k=100, top_p=0.9)
        check(gpu, wide.half().cuda()[:, at:at + 7003], u, top_p=0.9)
        wide[:, at:at + 7003] = float("nan")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(15, 151936), (33, 100001), (70, 30000), (150, 9001), (400, 2500), (3000, 40)])
def test_every_number_of_ctas_a_row(gpu, rows, vocab):
    """Few rows have eight CTAs each, many one: every row with its own options, fp16 and fp32."""
    x, u, g = rows_of_logits(rows, vocab, rows)
    pick = lambda *v: [v[i % len(v)] for i in range(rows)]
    for dtype in ("fp32", "fp16"):
        check(gpu, x.to(DTYPES[dtype]), u, temperature=torch.tensor(pick(0.8, 1.3, 0.0, 0.5, 1.0)), top_k=torch.tensor(pick(0, 50, 1000, 3, 0, 0, 1), dtype=torch.int32),
              top_p=torch.tensor(pick(1.0, 0.9, 0.99)), min_p=torch.tensor(pick(0.0, 0.0, 0.03, 0.0)), skipped=0.03)


@pytest.mark.gpu
def test_a_pick_does_not_depend_on_its_batch(gpu):
    x, u, _ = rows_of_logits(64, 151936, 9)
    x, u = x.cuda(), u.cuda()
    for kw in (dict(top_k=50, top_p=0.9), dict(top_p=0.95), {}):
        all_tokens, all_logp = gpu.sample_tokens(x, u, **kw)
        for i in (0, 13, 63):
            token, logp = gpu.sample_tokens(x[i:i + 1], u[i:i + 1], **kw)
            assert token.item() == all_tokens[i].item() and logp.item() == all_logp[i].item()
        again = gpu.sample_tokens(x, u, **kw)
        assert torch.equal(again[0], all_tokens) and torch.equal(again[1], all_logp)


@pytest.mark.gpu
def test_on_other_streams_and_in_graphs(gpu):
    x, u, _ = rows_of_logits(4, 20000, 21)
    x, u = x.cuda(), u.cuda()
    want = [gpu.sample_tokens(x + 0.0, u, top_p=0.9)[0].tolist(), gpu.sample_tokens(-x, u, top_p=0.9)[0].tolist()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert gpu.sample_tokens(x, u, top_p=0.9)[0].tolist() == want[0]
        buf = x.clone()
        graph = torch.cuda.CUDAGraph()
        gpu.sample_tokens(buf, u, top_p=0.9)
        with torch.cuda.graph(graph, stream=stream):
            tokens, _ = gpu.sample_tokens(buf, u, top_p=0.9)
        for sign, w in ((1, want[0]), (-1, want[1]), (1, want[0])):
            buf.copy_(sign * x)
            graph.replay()
            assert tokens.tolist() == w


@pytest.mark.gpu
def test_many_draws_from_one_row(gpu):
    x, _, g = rows_of_logits(1, 32003, 3)
    u = torch.rand(200, generator=g)
    for kw in ({}, dict(top_k=50, top_p=0.9), dict(top_p=0.9)):
        got = gpu.sample_tokens(x.cuda().expand(200, 32003), u.cuda(), **kw)
        want = gpu.sample_tokens(x.expand(200, 32003).contiguous().cuda(), u.cuda(), **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_offsets_of_more_than_32_bits(gpu):
    """Rows 2^27 + 1 elements apart, the last from 2^32 on."""
    x, u, _ = rows_of_logits(36, 5000, 7)
    wide = torch.empty(36 * ((1 << 27) + 1), dtype=torch.float16, device="cuda").as_strided((36, 5000), ((1 << 27) + 1, 1))
    wide.copy_(x)
    for kw in ({}, dict(top_k=50), dict(top_p=0.9)):
        got, want = gpu.sample_tokens(wide, u.cuda(), **kw), gpu.sample_tokens(x.half().cuda(), u.cuda(), **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_numbers_of_tokens_of_more_than_32_bits_are_all(gpu):
    x, u, _ = rows_of_logits(4, 3000, 8)
    x, u = x.cuda(), u.cuda()
    want = gpu.sample_tokens(x, u)
    for k in (3000, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, -1, 1 - 2 ** 32):
        got = gpu.sample_tokens(x, u, top_k=k)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_two_calls_at_once(gpu):
    x, u, _ = rows_of_logits(20, 151936, 22)
    x, u = x.cuda(), u.cuda()
    want = [gpu.sample_tokens(x, u, top_p=0.9), gpu.sample_tokens(-x, u, top_k=40)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    minus = -x
    torch.cuda.synchronize()
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            got.append(gpu.sample_tokens(minus, u, top_k=40) if i % 2 else gpu.sample_tokens(x, u, top_p=0.9))
    torch.cuda.synchronize()
    for i, (tokens, logp) in enumerate(got):
        assert torch.equal(tokens, want[i % 2][0]) and torch.equal(logp, want[i % 2][1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("vocab", [3001, 40000, 151936])
def test_top_p_alone(gpu, dtype, vocab):
    """From a few tokens that stay to nearly all, sharp and flat, a temperature per row; values of bf16 are equal in hundreds."""
    ps, ts = (0.001, 0.3, 0.6, 0.9, 0.97, 0.999, 0.99999), (0.1, 0.17, 0.4, 0.8, 1.3, 2.5)
    rows = len(ps) * len(ts)
    x, u, _ = rows_of_logits(rows, vocab, 17)
    # (equal values on both sides of a border of 64-bit sums: skipped as elsewhere)
    check(gpu, x.to(DTYPES[dtype]), u, temperature=torch.tensor([t for t in ts for _ in ps]), top_p=torch.tensor(ps * len(ts)), skipped=0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [-3.4028234663852886e38, -65504.0, -1e4, -100.0, -60.0, -40.0, float("-inf"), float("nan")])
@pytest.mark.parametrize("stay", [1, 30, 5000])
def test_top_p_of_rows_with_masked_tokens(gpu, masked, stay):
    """Whole ranges of a row masked by low values, at its beginning, end or between; a few other outliers far below and above."""
    x, u, g = rows_of_logits(12, 30000, 23)
    for i in range(12):
        at = (0, 30000 - stay, 12345)[i % 3]
        keep = x[i, at:at + stay].clone()
        x[i] = masked
        x[i, at:at + stay] = keep
        if i % 4 == 3:
            x[i, at] = 90.0
            x[i, 29999] = -70.0
    for p in (0.5, 0.95):
        check(gpu, x, u, temperature=0.8, top_p=p, skipped=0.1)
    check(gpu, x, u, temperature=0.8, top_p=0.9, min_p=0.02, skipped=0.1)


def _garbage_outputs(rows):
    """What the next outputs of this size are made of: neither tokens nor logarithms."""
    for _ in range(4):
        torch.full((rows,), -77, dtype=torch.int32, device="cuda")
        torch.full((rows,), 77.0, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("vocab", [1, 300, 40000])
def test_a_min_p_above_one_keeps_the_first_token(gpu, vocab, dtype):
    """In an array, where it is not refused: no token's mass is above the largest one's, and one token always stays - the first of equal ones."""
    ways = [(0, 1.0), (0, 0.9), (0, 0.99999), (50, 1.0), (50, 0.9), (20000, 1.0), (20000, 0.9), (20000, 0.99999)]
    rows = len(ways)
    x, u, _ = rows_of_logits(rows, vocab, 41)
    x = (x - x.amax(1, keepdim=True)).to(DTYPES[dtype])          # (bounds around the largest value are closest to it at 0)
    ties = x.clone()
    at = [vocab // 3, vocab // 2, vocab - 1]
    ties[:, at] = 0.0
    flat = torch.zeros_like(x)
    for case in (x, x + 5.0, ties, flat, -40.0 + ties):
        for least in (1.0000001, 1.5, 1e30, float("inf")):
            options = dict(top_k=torch.tensor([k for k, _ in ways], dtype=torch.int32), top_p=torch.tensor([p for _, p in ways]),
                           min_p=torch.full((rows,), least))
            _garbage_outputs(rows)
            got = check(gpu, case, u, temperature=torch.tensor([0.05, 0.7, 1.0, 2.5] * (rows // 4)), skipped=1.0, **options)
            assert got.tolist() == case.float().argmax(1).tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [50, 20000])
def test_what_arrays_of_options_may_hold(gpu, vocab):
    """Values that a scalar may not have: a row's meaning is that of the valid value beside it, and the rows around it are as they were."""
    nan, inf = float("nan"), float("inf")
    means = [  # (temperature, top_k, top_p, min_p), and the same in valid values
        ((0.8, 0, 1.0, 0.0), None), ((-1.0, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0)), ((nan, 5, 1.0, 0.1), (0.0, 0, 1.0, 0.0)), ((-inf, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0)),
        ((-0.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0)), ((inf, 0, 1.0, 0.0), (2.0 ** 100, 0, 1.0, 0.0)), ((1e38, 7, 1.0, 0.0), (2.0 ** 100, 7, 1.0, 0.0)),
        ((0.8, -3, 1.0, 0.0), (0.8, 0, 1.0, 0.0)), ((0.8, -2 ** 31, 0.9, 0.0), (0.8, 0, 0.9, 0.0)), ((0.8, 2 ** 31 - 1, 0.9, 0.0), (0.8, 0, 0.9, 0.0)),
        ((0.8, 0, 0.0, 0.0), (0.8, 1, 1.0, 0.0)), ((0.8, 40, -0.5, 0.0), (0.8, 1, 1.0, 0.0)), ((0.8, 0, -inf, 0.3), (0.8, 1, 1.0, 0.0)), ((0.8, 0, 1e-45, 0.0), (0.8, 1, 1.0, 0.0)),
        ((0.8, 0, nan, 0.0), (0.8, 0, 1.0, 0.0)), ((0.8, 30, nan, 0.05), (0.8, 30, 1.0, 0.05)), ((0.8, 0, 2.0, 0.0), (0.8, 0, 1.0, 0.0)), ((0.8, 0, inf, 0.0), (0.8, 0, 1.0, 0.0)),
        ((0.8, 0, 1.0, nan), (0.8, 0, 1.0, 0.0)), ((0.8, 30, 0.9, nan), (0.8, 30, 0.9, 0.0)), ((0.8, 0, 1.0, -1.0), (0.8, 0, 1.0, 0.0)), ((0.8, 0, 0.95, -inf), (0.8, 0, 0.95, 0.0)),
        ((0.8, 0, 1.0, 1.0), None), ((0.8, 0, 0.9, 1.0), None), ((0.8, 0, 0.9, 0.2), None)]
    rows = len(means)
    x, u, _ = rows_of_logits(rows, vocab, 43)
    given = list(zip(*(g for g, _ in means)))
    got, logp = gpu.sample_tokens(x.cuda(), u.cuda(), torch.tensor(given[0]).cuda(), torch.tensor(given[1], dtype=torch.int32).cuda(),
                                  torch.tensor(given[2]).cuda(), torch.tensor(given[3]).cuda())
    got, logp, borders = got.cpu(), logp.cpu(), 0
    for i, (g, same) in enumerate(means):
        t, k, p, mp = same or g
        token, lp, near = definition(x[i].double().numpy(), float(u[i]), float(np.float32(t)), k, p, mp)
        borders += near
        if not near:
            assert int(got[i]) == token, (i, g)
            assert abs(float(logp[i]) - lp) <= abs(lp) * 2.0 ** -24 + 2.0 ** -28, (i, g)
    assert borders <= 1


@pytest.mark.parametrize("address,kind,refused", [(4097, 0, True), (4098, 0, True), (4099, 1, True), (4097, 2, True), (4098, 1, False), (4098, 2, False), (4100, 0, False)])
def test_logits_between_addresses_of_their_type_are_refused(C, address, kind, refused):
    """(A stride below the vocabulary is refused behind it, so that nothing runs.)"""
    rc = C._lib.qmk_sample_tokens(address, kind, 99, 2, 100, 4096, None, 1.0, None, 0, None, 1.0, None, 0.0, 4096, None, None)
    assert rc == 2 and (b"aligned" if refused else b"overlap") in C._lib.qmk_last_error()
