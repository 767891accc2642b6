"""``BatchDecoder.sample_ids`` / ``sample_batched``: sampled decode steps over a shared prefix, against the CPU oracle and the definition of a pick.

Logits are compared with the oracle's on the same tokens under the bar of the batched decode (GEMM operands and queries are fp16: 3e-2).  Picks are
compared for equality with the definition applied to the step's own logits, rows on a border excepted (see test_sample_tokens.py)."""

import ctypes

import pytest
import torch

import synthetic as S
from oracle.decoder_ref import Decoder as OracleDecoder
from test_sample_tokens import definition

LOGIT_TOL = 3e-2
VOCAB = 2048


@pytest.fixture(scope="module")
def C(built_library):
    import qwen_megakernel_C
    return qwen_megakernel_C


@pytest.fixture(scope="module")
def gpu(C):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return C


def _engine(w, n, max_seq_len, eos=-1, **kw):
    from Model.Qwen06B_architecture import BatchDecoder
    return BatchDecoder(weights=S.weights_to(w, "cuda"), tokenizer=S.StubTokenizer(eos, VOCAB), num_sequences=n, max_seq_len=max_seq_len, **kw)


def _oracle_logits(w, prompt, tokens, max_seq_len):
    """The oracle's logits of every step that picks one of ``tokens`` behind ``prompt``."""
    o = OracleDecoder(w, max_seq_len=max_seq_len)
    if len(prompt) > 1:
        o.prefill(prompt[:-1])
    rows = []
    for token in [prompt[-1], *tokens[:-1]]:
        o.step(token)
        rows.append(o.last_logits.clone())
    return torch.stack(rows)


def _run(gpu, eng, prompts, steps, **kw):
    dump = torch.zeros(len(prompts), steps, VOCAB, device="cuda")
    gpu.set_logits_dump(dump)
    try:
        return (*eng.sample_ids(prompts, steps, **kw), dump.cpu())
    finally:
        gpu.set_logits_dump(None)


def _check(w, eng, prompts, steps, tokens, logprobs, dump, uniforms, options, max_seq_len, which=None):
    borders = 0
    for b in which if which is not None else range(len(prompts)):
        assert len(tokens[b]) == steps == len(logprobs[b])
        assert float((dump[b] - _oracle_logits(w, prompts[b], tokens[b], max_seq_len)).abs().max()) < LOGIT_TOL, f"sequence {b}"
        for i in range(steps):
            t, k, p, m = (o[b] for o in options)
            want, lp, near = definition(dump[b, i].double().numpy(), float(uniforms[i, b]), t, k, p, m)
            borders += near
            if not near:
                assert tokens[b][i] == want, (b, i)
                assert abs(logprobs[b][i] - lp) <= abs(lp) * 2.0 ** -24 + 2.0 ** -28
    assert borders <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("n,prompt_len", [(1, 1), (2, 2), (5, 300), (20, 65), (70, 129)])
def test_many_answers_to_one_prompt(gpu, n, prompt_len):
    steps, L = 4, 384
    w = S.make_weights(seed=31, num_layers=3, vocab_size=VOCAB, norm_std=0.1, max_seq_len=16)
    prompts = [S.make_prompt(prompt_len, seed=3, vocab_size=VOCAB)] * n
    g = torch.Generator().manual_seed(n)
    uniforms = torch.rand(steps, n, generator=g)
    options = [[0.7 + 0.1 * (i % 5) for i in range(n)], [(0, 50, 7)[i % 3] for i in range(n)], [(1.0, 0.9)[i % 2] for i in range(n)],
               [(0.0, 0.0, 0.02)[i % 3] for i in range(n)]]
    eng = _engine(w, n, L, engine="gemm", prefill_mode="tensor")
    kw = dict(uniforms=uniforms.cuda(), temperature=options[0], top_k=options[1], top_p=options[2], min_p=options[3])
    tokens, logprobs, dump = _run(gpu, eng, prompts, steps, **kw)
    _check(w, eng, prompts, steps, tokens, logprobs, dump, uniforms, options, L, which=sorted({0, 1, n // 2, n - 1} & set(range(n))))
    assert n < 5 or len({tuple(t) for t in tokens}) > 1
    assert eng.positions[:n] == [prompt_len - 1 + steps] + [0] * (n - 1)
    for _ in range(2):                               # without the dump a captured step is replayed: the same picks
        again, again_lp = eng.sample_ids(prompts, steps, **kw)
        assert again == tokens and again_lp == logprobs


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["fp16", "fp8", "nvfp4"])
def test_prompts_with_a_common_beginning(gpu, fmt):
    """Prompts that share their first 90 tokens and go on differently, at different lengths; their slots go on greedily behind it."""
    n, steps, L = 6, 3, 256
    w = S.make_weights(seed=33, num_layers=2, vocab_size=VOCAB, norm_std=0.1, max_seq_len=16)
    import quantize as Q
    packed = {"fp16": lambda x: x, "fp8": lambda x: Q.quantize_weights_fp8(x)[0], "nvfp4": lambda x: Q.quantize_weights_nvfp4(x)[0]}[fmt](w)
    w = {"fp16": lambda x: x, "fp8": lambda x: Q.expand_weights_fp8(x)[1], "nvfp4": lambda x: Q.expand_weights_nvfp4(x)[1]}[fmt](w)
    system = S.make_prompt(90, seed=5, vocab_size=VOCAB)
    prompts = [system + S.make_prompt(1 + 13 * i, seed=50 + i, vocab_size=VOCAB) for i in range(n)]
    uniforms = torch.rand(steps, n, generator=torch.Generator().manual_seed(1))
    options = [[0.9] * n, [0] * n, [0.95] * n, [0.0] * n]
    eng = _engine(packed, n, L, engine="gemm", prefill_mode="tensor", weight_format=fmt)
    tokens, logprobs, dump = _run(gpu, eng, prompts, steps, uniforms=uniforms.cuda(), temperature=0.9, top_p=0.95)
    _check(w, eng, prompts, steps, tokens, logprobs, dump, uniforms, options, L)
    assert eng.positions == [len(p) - 1 + steps for p in prompts]
    more = eng.decode_slots(list(range(n)), [t[-1] for t in tokens], 2)
    gpu.set_weight_format("fp16")
    for b in range(n):
        o = OracleDecoder(w, max_seq_len=L)
        o.prefill(prompts[b] + tokens[b][:-1])
        assert more[b] == [o.step(tokens[b][-1]), o.step(more[b][0])]


@pytest.mark.gpu
def test_temperature_zero_is_the_greedy_decode(gpu):
    n, steps, L = 7, 6, 256
    w = S.make_weights(seed=35, num_layers=3, vocab_size=VOCAB, norm_std=0.1, max_seq_len=16)
    prompts = [S.make_prompt(5 + 20 * i, seed=70 + i, vocab_size=VOCAB) for i in range(n)]
    eng = _engine(w, n, L, engine="gemm", prefill_mode="tensor")
    greedy = eng.generate_ids(prompts, steps)
    tokens, logprobs = eng.sample_ids(prompts, steps, temperature=0.0)
    assert tokens == greedy and logprobs == [[0.0] * steps] * n
    assert eng.generate_ids(prompts, steps) == greedy            # (graphs of both kinds of steps side by side)


@pytest.mark.gpu
def test_seeds_ends_and_other_engines(gpu):
    steps, L = 12, 128
    w = S.make_weights(seed=37, num_layers=2, vocab_size=VOCAB, norm_std=0.1, max_seq_len=16)
    prompt = S.make_prompt(30, seed=8, vocab_size=VOCAB)

    def draw(eng, seed, **kw):
        return eng.sample_ids([prompt] * 3, steps, temperature=1.0, top_k=40, generator=torch.Generator("cuda").manual_seed(seed), **kw)[0]
    eng = _engine(w, 3, L)                           # the engine that decodes greedily in one persistent launch
    first = draw(eng, 1)
    assert draw(eng, 1) == first and draw(eng, 2) != first and all(0 <= t < VOCAB for ids in first for t in ids)
    eos = first[1][4]
    cut = draw(_engine(w, 3, L, eos=eos), 1)
    assert cut == [ids[:ids.index(eos)] if eos in ids else ids for ids in first]
    assert eng.sample_ids([prompt], 0) == ([[]], [[]])
    for bad in (dict(prompts=[]), dict(prompts=[prompt] * 4), dict(prompts=[[]]), dict(prompts=[prompt], max_tokens=200),
                dict(prompts=[prompt], top_k=[1, 2]), dict(prompts=[prompt], uniforms=torch.zeros(3, 1, device="cuda"))):
        with pytest.raises(ValueError):
            eng.sample_ids(**{"max_tokens": steps, **bad})
    for bad in (dict(temperature=-1.0), dict(top_p=0.0), dict(min_p=2.0)):
        with pytest.raises(RuntimeError):
            eng.sample_ids([prompt], steps, **bad)
    assert draw(eng, 1) == first


@pytest.mark.gpu
def test_refusals_leave_a_text(gpu):
    eng = _engine(S.make_weights(seed=37, num_layers=2, vocab_size=VOCAB, norm_std=0.1, max_seq_len=16), 2, 64)
    base = eng._base
    base.apply_options()
    logs = [torch.zeros(4, dtype=torch.int32, device="cuda") for _ in range(2)]
    scores = [torch.zeros(4, device="cuda") for _ in range(2)]
    def call(**change):
        a = dict(first=[1, 2], start=[8, 9], steps=4, prefix=(eng._k_caches[0], eng._v_caches[0], 8), k=eng._k_caches, v=eng._v_caches, t=[1.0, 1.0])
        a.update(change)
        gpu.sample_batched(a["first"], a["start"], a["steps"], base._embed_weight, base._layer_weights_packed, base._final_norm_weight, base._lm_head_weight,
                           base._cos_table, base._sin_table, *a["prefix"], a["k"], a["v"], torch.rand(a["steps"], 2, device="cuda"), a["t"], [0, 0], [1.0, 1.0],
                           [0.0, 0.0], logs, scores, base.num_layers, 64, base._attn_scale)
    call()
    for change, text in ((dict(start=[8, 7]), "inside the shared prefix"), (dict(prefix=(None, None, 8)), "prefix"), (dict(prefix=(eng._k_caches[0], eng._v_caches[0], -1)), "prefix"),
                         (dict(start=[8, 61]), "max_seq_len"), (dict(first=[1, VOCAB]), "vocab"), (dict(k=[eng._k_caches[0]] * 2), "share"), (dict(t=[1.0, -1.0]), "temperature")):
        with pytest.raises(RuntimeError, match=text):
            call(**change)
    call()


def test_null_pointers_are_refused(C):
    lib = C._lib
    if torch.cuda.is_available():
        assert lib.qmk_sample_batched(1, None, None, 1, *[None] * 8, 0, *[None] * 9, 1, 64, 1.0, None) != 0 and b"null" in lib.qmk_last_error()
    else:
        assert lib.qmk_sample_batched(1, None, None, 1, *[None] * 8, 0, *[None] * 9, 1, 64, 1.0, None) != 0 and lib.qmk_last_error() == b"no CUDA device"


def _past_the_borders(gpu, n, prefix, tails, L, steps, check):
    """``n`` prompts of ``prefix`` tokens in common and ``tails[i]`` of their own: picks, logarithms and logits of the sequences ``check`` against the oracle;
    captured steps, their replay and kernels one after the other give the same bits."""
    w = S.make_weights(seed=39, num_layers=2, vocab_size=VOCAB, norm_std=0.1, max_seq_len=16)
    system = S.make_prompt(prefix, seed=6, vocab_size=VOCAB)
    prompts = [system + S.make_prompt(tails[i], seed=200 + i, vocab_size=VOCAB) if tails[i] else list(system) for i in range(n)]
    uniforms = torch.rand(steps, n, generator=torch.Generator().manual_seed(prefix))
    options = [[0.8] * n, [(0, 40)[i % 2] for i in range(n)], [0.95] * n, [0.0] * n]
    eng = _engine(w, n, L, engine="gemm", prefill_mode="tensor")
    kw = dict(uniforms=uniforms.cuda(), temperature=options[0], top_k=options[1], top_p=options[2], min_p=options[3])
    tokens, logprobs, dump = _run(gpu, eng, prompts, steps, **kw)
    _check(w, eng, prompts, steps, tokens, logprobs, dump, uniforms, options, L, which=check)
    try:
        for overlap in (True, True, False, True):
            gpu.set_step_overlap(overlap)
            again, again_lp = eng.sample_ids(prompts, steps, **kw)
            assert again == tokens and again_lp == logprobs, overlap
            assert torch.equal(_run(gpu, eng, prompts, steps, **kw)[2], dump), overlap
    finally:
        gpu.set_step_overlap(True)


@pytest.mark.gpu
def test_a_full_batch_of_answers_whose_prefix_is_on_tcgen05(gpu):
    """256 query rows a kv head against 410 prefix rows: 107 M products, from 96 M on on tcgen05."""
    assert 128 * 16 * 128 * 410 >= 96 << 20
    _past_the_borders(gpu, 128, 411, [0] * 128, 512, 3, [0, 63, 64, 127])


@pytest.mark.gpu
def test_long_tails_behind_a_long_prefix(gpu):
    """48 query rows a kv head against 2100 prefix rows on tcgen05, and up to three ranges of 256 rows of their own."""
    assert 24 * 16 * 128 * 2100 >= 96 << 20
    _past_the_borders(gpu, 24, 2100, [1 + (173 * i) % 700 for i in range(24)], 2816, 3, [0, 4, 11, 23])


@pytest.mark.gpu
def test_long_tails_behind_a_short_prefix(gpu):
    """Prefix and several ranges of own rows in one grid (mma.sync): sequences start up to 600 rows behind the prefix."""
    _past_the_borders(gpu, 9, 50, [1 + (307 * i) % 600 for i in range(9)], 768, 3, [0, 1, 7])


@pytest.mark.gpu
def test_refused_options_leave_the_slots_as_they_were(gpu):
    """What ``sample_ids`` refuses it refuses before it fills a slot: positions and caches go on as if the call had not been made."""
    w = S.make_weights(seed=37, num_layers=2, vocab_size=VOCAB, norm_std=0.1, max_seq_len=16)
    prompts = [S.make_prompt(20 + 9 * i, seed=90 + i, vocab_size=VOCAB) for i in range(3)]
    eng = _engine(w, 3, 128, engine="gemm", prefill_mode="tensor")
    first = [ids[-1] for ids in eng.generate_ids(prompts, 4)]
    positions, rows = list(eng.positions), [(k.clone(), v.clone()) for k, v in zip(eng._k_caches, eng._v_caches)]
    other = [S.make_prompt(33, seed=99, vocab_size=VOCAB)]
    good = torch.rand(4, 2, device="cuda")
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_p=0.0), dict(top_p=1e-60), dict(top_p=[1.0, float("nan")]), dict(min_p=2.0),
                dict(min_p=-0.1), dict(uniforms=good.cpu()), dict(uniforms=good.double()), dict(uniforms=good.half()), dict(uniforms=good[:3]), dict(top_k=[1]),
                dict(temperature="warm"), dict(top_k=float("nan"))):
        for prompts_ in (other * 2, [other[0], other[0][:-3]]):
            with pytest.raises((RuntimeError, ValueError)):
                eng.sample_ids(prompts_, 4, **bad)
        assert eng.positions == positions
        assert all(torch.equal(k, a) and torch.equal(v, b) for k, v, (a, b) in zip(eng._k_caches, eng._v_caches, rows)), bad
    more = eng.decode_slots([0, 1, 2], first, 3)
    again = _engine(w, 3, 128, engine="gemm", prefill_mode="tensor")
    assert [ids[4:] for ids in again.generate_ids(prompts, 7)] == more


@pytest.mark.gpu
def test_two_sequences_with_one_log_of_logarithms_are_refused(gpu):
    eng = _engine(S.make_weights(seed=37, num_layers=2, vocab_size=VOCAB, norm_std=0.1, max_seq_len=16), 2, 64)
    base = eng._base
    base.apply_options()
    logs, scores = [torch.zeros(4, dtype=torch.int32, device="cuda") for _ in range(2)], [torch.zeros(4, device="cuda") for _ in range(2)]

    def call(scores):
        gpu.sample_batched([1, 2], [8, 9], 4, base._embed_weight, base._layer_weights_packed, base._final_norm_weight, base._lm_head_weight, base._cos_table,
                           base._sin_table, None, None, 0, eng._k_caches, eng._v_caches, torch.rand(4, 2, device="cuda"), [1.0, 1.0], [0, 0], [1.0, 1.0],
                           [0.0, 0.0], logs, scores, base.num_layers, 64, base._attn_scale)
    with pytest.raises(RuntimeError, match="share"):
        call([scores[0]] * 2)
    call(scores)


@pytest.mark.gpu
@pytest.mark.parametrize("engine,vocab,last", [("gemm", VOCAB, VOCAB), ("gemm", VOCAB, -1), ("persistent", VOCAB, VOCAB + 5), ("persistent", 1000, 3)])
def test_refused_tokens_and_vocabularies_leave_the_slots_as_they_were(gpu, engine, vocab, last):
    """A last token outside the vocabulary, and an engine whose vocabulary the sampled steps do not read."""
    from Model.Qwen06B_architecture import BatchDecoder
    w = S.make_weights(seed=37, num_layers=2, vocab_size=vocab, norm_std=0.1, max_seq_len=16)
    eng = BatchDecoder(weights=S.weights_to(w, "cuda"), tokenizer=S.StubTokenizer(-1, vocab), num_sequences=2, max_seq_len=128, engine=engine)
    prompts = [S.make_prompt(20 + 9 * i, seed=90 + i, vocab_size=vocab) for i in range(2)]
    eng.generate_ids(prompts, 4)
    positions, rows = list(eng.positions), [(k.clone(), v.clone()) for k, v in zip(eng._k_caches, eng._v_caches)]
    with pytest.raises(RuntimeError):
        eng.sample_ids([[5, 6, 7, 8], [5, 6, 7, last]], 4)
    assert eng.positions == positions
    assert all(torch.equal(k, a) and torch.equal(v, b) for k, v, (a, b) in zip(eng._k_caches, eng._v_caches, rows))
    assert eng.sample_ids([[5, 6, 7, 8]], 0, temperature=-1.0) == ([[]], [[]])


@pytest.mark.gpu
def test_caches_that_the_steps_could_not_read_are_refused(gpu):
    """Of the host's memory, of fewer rows than the call says, not contiguous, or none: the prefix's caches and the sequences' own."""
    eng = _engine(S.make_weights(seed=37, num_layers=2, vocab_size=VOCAB, norm_std=0.1, max_seq_len=16), 2, 64)
    base = eng._base
    base.apply_options()
    logs, scores = [torch.zeros(4, dtype=torch.int32, device="cuda") for _ in range(2)], [torch.zeros(4, device="cuda") for _ in range(2)]

    def call(k_prefix, v_prefix, k, v, max_seq_len=64):
        gpu.sample_batched([1, 2], [8, 9], 4, base._embed_weight, base._layer_weights_packed, base._final_norm_weight, base._lm_head_weight, base._cos_table,
                           base._sin_table, k_prefix, v_prefix, 8, k, v, torch.rand(4, 2, device="cuda"), [1.0, 1.0], [0, 0], [1.0, 1.0],
                           [0.0, 0.0], logs, scores, base.num_layers, max_seq_len, base._attn_scale)
    good = [eng._k_caches[0], eng._v_caches[0], eng._k_caches, eng._v_caches]
    for which in range(4):
        for bad in (lambda t: t.cpu(), lambda t: t[:, :, :60].contiguous(), lambda t: t[:1], lambda t: torch.cat((t, t), 3)[..., :128], lambda t: None):
            case = list(good)
            case[which] = bad(good[which]) if which < 2 else [good[which][0], bad(good[which][1])]
            with pytest.raises(RuntimeError, match="cache"):
                call(*case)
    with pytest.raises(RuntimeError, match="cache"):
        call(*good, max_seq_len=65)
    call(*good)
