"""Beam search of the engine (qd_generate_beams) against the CPU oracle: the same
search with a cache of its own for every beam, log probabilities in 64 bits."""
import numpy as np
import pytest

import qwen_decode as qd
import qwen_oracle as qo

LAYERS, VOCAB, CAPACITY, SEED = 2, 1003, 96, 3
# Scores reach 215 over 45 steps. Each step rounds one to FP32, by at most 2^-24 x 256 = 1.5e-5, and
# adds a log probability whose logits (below 4) are off by 1e-5 of them (sums of up to 4,864 FP32
# products, as in the batched step's tests): in the mean by a tenth of that. Added up with one sign
# 45 x (1.5e-5 + 4e-6) = 9e-4; two candidates further apart than NEAR are out of order only if the
# errors of 20 steps and more all have one sign.
NEAR, SCORE = 4e-4, 1e-3


def say(*a):
    print("[gpu-case]", *a, flush=True)


def log_softmax(x):
    x = x.astype(np.float64)
    return x - x.max() - np.log(np.exp(x - x.max()).sum())


def search(model, prompt, beams, steps, eos=None):
    """[(tokens, score)] of the best beams, and the smallest gap between two candidates that the
    search put in order."""
    def grown(cache, n):
        c = qo.Cache(model, CAPACITY)
        for layer in range(LAYERS):
            for value in (False, True):
                c.layer(layer, value)[:n] = cache.layer(layer, value)[:n]
        return c

    start = qo.Cache(model, CAPACITY)
    if len(prompt) > 1:
        start.prefill(prompt[:-1], want_logits=False)
    alive, gap = [([], 0.0, start, False)], np.inf
    for step in range(steps):
        at = len(prompt) - 1 + step
        candidates = []
        for b, (tokens, score, cache, done) in enumerate(alive):
            if done:
                candidates.append((score, b, eos))
                continue
            _, _, logits = cache.decode_step(int(tokens[-1] if tokens else prompt[-1]), at)
            logp = score + log_softmax(logits)
            candidates += [(float(logp[t]), b, int(t)) for t in np.argsort(-logp, kind="stable")[:beams + 1]]
        candidates.sort(key=lambda c: (-c[0], c[1], c[2]))
        gap = min([gap] + [a[0] - b[0] for a, b in zip(candidates[:beams], candidates[1:])])
        alive = [(alive[b][0] + [t], s, grown(alive[b][2], at + 1), alive[b][3] or t == eos) for s, b, t in candidates[:beams]]
    return [(tokens, score) for tokens, score, _, _ in alive], gap


@pytest.fixture(scope="module")
def model():
    m = qo.Model(qo.ModelShape(layers=LAYERS, vocab=VOCAB))
    m.fill_synthetic(SEED)
    yield m
    m.close()


@pytest.fixture(scope="module")
def engine():
    eng = qd.Engine(layers=LAYERS, vocab=VOCAB, capacity=CAPACITY, max_batch=2)
    eng.load_synthetic(SEED)
    yield eng
    eng.close()


def prompt_of(n, stream=0x720000):
    return qo.fill_tokens(n, SEED, stream + n, VOCAB)


# Prompts that end inside a page, at its end, after one token, in the third page; beams to the full batch.
CASES = [(1, 4, 20), (16, 3, 40), (17, 16, 18), (37, 5, 45), (48, 1, 12)]


def check(got, scores, want, length=lambda tokens: 1.0):
    assert [t.tolist() for t in got] == [t for t, _ in want]
    for s, (tokens, score) in zip(scores, want):
        assert abs(float(s) - score / length(tokens)) < SCORE


@pytest.mark.gpu
@pytest.mark.parametrize("n,beams,steps", CASES)
def test_beams_match_oracle(engine, model, n, beams, steps):
    say("beam search", n, beams, steps)
    prompt = prompt_of(n)
    want, gap = search(model, prompt, beams, steps)
    assert gap > NEAR, gap
    engine.kv_reset(1, 0)
    if n > 1:
        engine.prefill(1, prompt[:-1], want_logits=False)
    got, scores = engine.generate_beams(1, int(prompt[-1]), beams, steps)
    check(got, scores, want)


@pytest.mark.gpu
def test_slot_stays_and_greedy_is_one_beam(engine):
    say("the slot after a search; one beam")
    prompt = prompt_of(20)
    engine.kv_reset(0, 0)
    engine.prefill(0, prompt[:-1])
    before = [engine.read_kv(0, layer, 0, CAPACITY) for layer in range(LAYERS)]
    state, logits = engine.decode_state(0), engine.read_logits(0)
    first, scores = engine.generate_beams(0, int(prompt[-1]), 16, 60)
    after = engine.decode_state(0)
    assert [getattr(state, f) for f, _ in state._fields_] == [getattr(after, f) for f, _ in after._fields_]
    assert np.array_equal(engine.read_logits(0), logits)
    for layer in range(LAYERS):
        assert all(np.array_equal(a, b) for a, b in zip(engine.read_kv(0, layer, 0, CAPACITY), before[layer]))
    again, scores2 = engine.generate_beams(0, int(prompt[-1]), 16, 60)
    assert all(np.array_equal(a, b) for a, b in zip(first, again)) and np.array_equal(scores, scores2)
    one, _ = engine.generate_beams(0, int(prompt[-1]), 1, 30)
    greedy, _, _ = engine.generate(0, int(prompt[-1]), 30)
    assert np.array_equal(one[0], greedy)


def eos_of(model, prompt, beams, steps):
    """A token that the plain search produces midway on one of its beams."""
    want, _ = search(model, prompt, beams, steps)
    return want[beams // 2][0][steps // 2]


@pytest.mark.gpu
@pytest.mark.parametrize("penalty", [0.0, 1.0])
def test_beams_that_end(engine, model, penalty):
    say("beams that end", penalty)
    prompt, beams, steps = prompt_of(30), 4, 20
    eos = eos_of(model, prompt, beams, steps)
    want, gap = search(model, prompt, beams, steps, eos)
    assert gap > NEAR
    ended = [(t[: t.index(eos) + 1] if eos in t else t, s) for t, s in want]
    assert any(len(t) < steps for t, _ in ended)
    ended.sort(key=lambda x: -x[1] / len(x[0]) ** penalty)
    engine.kv_reset(0, 0)
    engine.prefill(0, prompt[:-1])
    got, scores = engine.generate_beams(0, int(prompt[-1]), beams, steps, eos=eos, length_penalty=penalty)
    check(got, scores, ended, lambda tokens: len(tokens) ** penalty)


@pytest.mark.gpu
def test_a_search_that_ends_early_equals_a_short_one(engine):
    """All beams at their end after a few steps: the search stops and says so."""
    say("every beam ends")
    eng = qd.Engine(layers=1, vocab=2, capacity=400, max_batch=1)
    eng.load_synthetic(1)
    got, scores = eng.generate_beams(0, 1, 2, 390, eos=0)
    assert all(t[-1] == 0 or len(t) == 390 for t in got)
    assert all(len(t) == 1 or 0 not in t[:-1].tolist() for t in got)
    assert scores[0] >= scores[1] and np.isfinite(scores).all()
    eng.close()


@pytest.mark.gpu
def test_from_an_empty_slot_to_the_last_position(engine, model):
    say("from position 0 to the capacity")
    engine.kv_reset(0, 0)
    got, _ = engine.generate_beams(0, 7, 2, CAPACITY)
    assert all(len(t) == CAPACITY for t in got)
    engine.kv_reset(0, CAPACITY - 1)
    got, _ = engine.generate_beams(0, 7, 2, 1)
    assert all(len(t) == 1 for t in got)


@pytest.mark.gpu
def test_refusals(engine):
    say("beam search refusals")
    engine.kv_reset(0, 10)
    for args, status in (((2, 1, 4, 8), qd.INVALID_ARGUMENT), ((0, VOCAB, 4, 8), qd.INVALID_ARGUMENT),
                         ((0, 1, 0, 8), qd.INVALID_ARGUMENT), ((0, 1, 17, 8), qd.INVALID_ARGUMENT),
                         ((0, 1, 4, 0), qd.INVALID_ARGUMENT), ((0, 1, 4, CAPACITY - 9), qd.INVALID_ARGUMENT),
                         ((0, 1, 4, 8, VOCAB), qd.INVALID_ARGUMENT), ((0, 1, 4, 8, 0, float("nan")), qd.INVALID_ARGUMENT)):
        with pytest.raises(qd.QdError) as e:
            engine.generate_beams(*args)
        assert e.value.status == status, args
    with qd.Engine(layers=1, vocab=64, capacity=8, decoder_dtype="bf16") as narrow:
        narrow.load_synthetic(1)
        with pytest.raises(qd.QdError) as e:
            narrow.generate_beams(0, 1, 2, 4)
        assert e.value.status == qd.NOT_SUPPORTED
    with qd.Engine(layers=1, vocab=64, capacity=8) as empty:
        with pytest.raises(qd.QdError) as e:
            empty.generate_beams(0, 1, 2, 4)
        assert e.value.status == qd.NOT_INITIALIZED


@pytest.mark.gpu
def test_a_search_without_room_for_its_memory(monkeypatch):
    """Its memory is the searches' once all of it is there: one that finds no room leaves nothing half made."""
    say("beam memory refused by QD_DEVICE_BYTES_LIMIT")
    config = dict(layers=LAYERS, vocab=VOCAB, capacity=4000, max_batch=1)
    with qd.Engine(**config) as ref:
        ref.load_synthetic(SEED)
        before = ref.device_bytes()
        want = ref.generate_beams(0, 7, 4, 20)
        small = ref.device_bytes()
        monkeypatch.setenv("QD_DEVICE_BYTES_LIMIT", str(small))
        with qd.Engine(**config) as eng:
            monkeypatch.delenv("QD_DEVICE_BYTES_LIMIT")
            eng.load_synthetic(SEED)
            for _ in range(2):
                with pytest.raises(qd.QdError) as err:
                    eng.generate_beams(0, 7, 16, 3000)
                assert err.value.status == qd.RUNTIME and before < eng.device_bytes() < small
                got = eng.generate_beams(0, 7, 4, 20)
                assert all(np.array_equal(a, b) for a, b in zip(got[0], want[0])) and np.array_equal(got[1], want[1])
                assert eng.device_bytes() == small


@pytest.mark.gpu
def test_24_layers_at_a_long_context():
    """The whole model deep in a context: each beam's score equals the sum of its log
    probabilities when its tokens are consumed one by one."""
    say("24 layers at 1,100")
    eng = qd.Engine(layers=24, vocab=qo.QWEN25_05B.vocab, capacity=1200, max_batch=1)
    eng.load_synthetic(SEED)
    prompt = qo.fill_tokens(1100, SEED, 0x710000, qo.QWEN25_05B.vocab)
    eng.prefill(0, prompt[:-1], want_logits=False)
    got, scores = eng.generate_beams(0, int(prompt[-1]), 6, 20)
    assert all(a >= b for a, b in zip(scores, scores[1:])) and len({tuple(t) for t in got}) == 6
    for tokens, score in zip(got, scores):
        eng.kv_reset(0, 1099)
        feed, total = int(prompt[-1]), 0.0
        for t in tokens.tolist():
            _, _, logits = eng.step(0, feed)
            total += log_softmax(logits)[t]
            feed = t
        # 20 steps, logits below 8 and 1e-5 of that off, in both terms: 3e-3 at most.
        assert abs(total - float(score)) < 3e-3
    eng.close()


def test_oracle_search_of_one_beam_is_greedy(model):
    prompt = prompt_of(5)
    (found,), _ = search(model, prompt, 1, 6)
    cache = qo.Cache(model, CAPACITY)
    token, _, _ = cache.prefill(prompt)
    want = [token]
    for i in range(5):
        token, _, _ = cache.decode_step(want[-1], len(prompt) + i)
        want.append(token)
    assert found[0] == want


@pytest.mark.gpu
def test_runner_prints_the_beams(engine):
    say("qd_run --beams")
    import os
    import re
    import subprocess

    runner = os.path.join(os.path.dirname(qd.LIB_PATH), "qd_run")
    prompt = [5, 17, 400]
    r = subprocess.run([runner, "1", "--synthetic-seed", str(SEED), "--layers", str(LAYERS), "--vocab", str(VOCAB),
                        "--prompt-token-ids", "5,17,400", "--max-new-tokens", "7", "--beams", "3", "--length-penalty", "1",
                        "--no-warmup", "--e2e-check"], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr
    engine.kv_reset(0, 0)
    engine.prefill(0, prompt[:-1])
    got, scores = engine.generate_beams(0, 400, 3, 7, length_penalty=1.0)
    lines = re.findall(r"^beam (\d) score=(\S+) generated_tokens=7 token_ids=\[([0-9,]+)\]$", r.stdout, re.M)
    assert [int(n) for n, _, _ in lines] == [1, 2, 3]
    assert [[int(t) for t in ids.split(",")] for _, _, ids in lines] == [t.tolist() for t in got]
    assert all(abs(float(s) - float(x)) < 1e-4 for (_, s, _), x in zip(lines, scores))
    assert "generated_token_ids=[" + lines[0][2] + "]" in r.stdout and "path=beams" in r.stdout


@pytest.mark.parametrize("flags,needle", [(("--beams", "0"), "--beams takes 1 to 16"), (("--beams", "4"), "requires --max-new-tokens"),
                                          (("--beams", "4", "--resident", "--max-new-tokens", "2"), "--beams excludes"),
                                          (("--length-penalty", "x"), "requires a number")])
def test_runner_refusals(flags, needle):
    import os
    import subprocess

    runner = os.path.join(os.path.dirname(qd.LIB_PATH), "qd_run")
    r = subprocess.run([runner, "--synthetic-seed", "1", "--prompt-token-ids", "1", *flags], capture_output=True, text=True, timeout=60)
    assert r.returncode == 2 and needle in r.stderr, r.stderr
