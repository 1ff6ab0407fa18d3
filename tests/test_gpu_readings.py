"""Several sampled readings of one window: sampled steps and the shared-window engine.

* A sampled step at temperature 0 is the greedy step, token for token, on every
  step path (one slot, several slots, tensor cores) and grammar.
* A sampled step at a temperature draws what the definition draws (float64,
  ``test_gpu_sample.draw64``) from the masked logits of a twin engine that is
  forced along the drawn tokens (engines are deterministic, so the twin's
  logits are the same bits).
* An engine with a shared window agrees with one that holds a copy per slot:
  logits within the parity tolerance of the other comparisons (the shared cross
  attention rounds unnormalised weights to bfloat16 where the decode kernel
  rounds scores and normalised weights), and a slot does not depend on the
  other slots, bit for bit.
* ``shard.decode_readings`` on it, end to end.
"""

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import scenarios as sc
from helpers import LOGIT_WITHIN_FRACTION, cuda_engine, loader, logit_error, logit_within, weights
from oracle.grammar import make_grammar_oracle
from sheetsage2_refined_b200 import _lib
from sheetsage2_refined_b200.shard import Song, decode_readings
from sheetsage2_refined_b200.vocab_table import OUT, SOS, VocabTable
from sheetsage2_refined_b200.weights import DecoderWeights, memory_array
from test_gpu_sample import draw64

pytestmark = pytest.mark.gpu
MODE_BIAS = [0.0, 1.5, -0.5, 2.0, 0.25, -1.0, 3.0, 0.5, -2.0]


@pytest.fixture(autouse=True)
def _needs_cuda():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")


def table_engine(batch, frames=sc.BATCH_FRAMES, **kw):
    return cuda_engine(sc.C1_SHORT, sc.BATCH_SEED, sc.batch_grammar(), batch, frames, **kw)


def real_engine(batch, prompts=sc.REAL_PROMPT_SETS[1], **kw):
    from sheetsage2_refined_b200 import BatchDecoder

    dec = DecoderWeights(sc.REAL_TINY, weights(sc.REAL_TINY, sc.REAL_SEED))
    return BatchDecoder(dec, VocabTable(), batch=batch, frames=sc.REAL_FRAMES, prompts=prompts, mode_bias=MODE_BIAS, **kw)


def start(eng, real, batch):
    load = loader(eng, eng.config.width, eng.frames)
    prefix = VocabTable().prompt_prefix(sc.REAL_PROMPT_SETS[1]) if real else [SOS, OUT]
    for slot in range(batch):
        load(slot, 20 + slot, prefix, None, eng.frames - 7 * (slot % 5), None if real else 60 + 9 * slot)


@pytest.mark.parametrize("batch", [1, 3, 16])
@pytest.mark.parametrize("real", [False, True], ids=["table", "class"])
def test_temperature_zero_is_the_greedy_step(batch, real):
    make = real_engine if real else table_engine
    greedy, sampled = make(batch), make(batch)
    for eng in (greedy, sampled):
        start(eng, real, batch)
    for n in (1, 20, 27):
        greedy.run(n)
        sampled.run_sampled(torch.rand(n, batch, device="cuda"), temperature=0.0, top_k=3, top_p=0.5)
    assert torch.equal(greedy.out, sampled.out)
    for name in greedy.state:
        assert torch.equal(greedy.state[name], sampled.state[name]), name


@pytest.mark.parametrize("batch,real,flags", [(1, False, 0), (3, True, 0), (16, True, 0), (2, False, _lib.S2R_FLAG_NO_GRAPH)])
def test_a_sampled_step_draws_from_the_masked_logits(batch, real, flags):
    make = real_engine if real else table_engine
    eng, twin = make(batch, flags=flags), make(batch)
    for e in (eng, twin):
        start(e, real, batch)
    grammar = make_grammar_oracle(eng.grammar)
    g = torch.Generator().manual_seed(batch)
    steps = 12
    u = torch.rand(steps, batch, generator=g)
    t = 0.5 + torch.rand(batch, generator=g)
    k = torch.randint(0, 40, (batch,), generator=g, dtype=torch.int32)
    lp = torch.zeros(steps, batch, device="cuda")
    args = dict(temperature=t.cuda(), top_k=k.cuda(), top_p=0.97, min_p=0.001)
    eng.run_sampled(u[:5].cuda(), logprobs=lp[:5], **args)
    eng.run_sampled(u[5:].cuda(), logprobs=lp[5:], **args)
    drawn = eng.out.cpu().numpy()
    total = np.zeros(batch)
    first = [len(VocabTable().prompt_prefix(sc.REAL_PROMPT_SETS[1])) if real else 2] * batch
    bias = eng._bias if real else None
    for i in range(steps):
        state = {n: v.cpu().numpy().copy() for n, v in twin.state.items()}
        live = state["finished"] == 0
        allowed = np.asarray(grammar.allowed(state))
        forced = np.array([drawn[s, first[s] + i] if live[s] else -1 for s in range(batch)], np.int64)
        logits, _ = twin.step_debug(forced)
        x = logits if bias is None else (logits + bias).astype(np.float32)
        for s in range(batch):
            if live[s]:
                token, logprob = draw64(x[s], allowed[s], float(u[i, s]), float(t[s]), int(k[s]),
                                        float(np.float32(0.97)), float(np.float32(0.001)))
                assert token == forced[s], (i, s, token, int(forced[s]))
                assert abs(float(lp[i, s]) - logprob) <= 1e-5 + 2.0**-22 * abs(logprob)
                total[s] += float(lp[i, s])
    # the sums are the same float32 values added in float64
    assert np.allclose(eng.logprob.cpu().numpy(), total, rtol=0, atol=1e-12)


def test_rescoring_reaches_the_draw():
    """With frame-head rescoring on, temperature 0 still gives the greedy tokens (eight terms, three slots)."""

    from sheetsage2_refined_b200 import BatchDecoder

    vocab = VocabTable()
    dec = DecoderWeights(sc.REAL_TINY, weights(sc.REAL_TINY, sc.REAL_SEED))
    engines = [BatchDecoder(dec, vocab, batch=3, frames=sc.REAL_FRAMES, prompts=sc.RESCORE_PROMPTS,
                            frame_weight={**sc.RESCORE_CASES["chords"], "meter": 2.0, "downbeat": 2.0}) for _ in range(2)]
    prefix = vocab.prompt_prefix(sc.RESCORE_PROMPTS)
    for eng in engines:
        for slot in range(3):
            eng.load(slot, memory_array(sc.REAL_FRAMES, sc.REAL_TINY.width, 60 + slot), prefix, None,
                     frame_logp=sc.rescore_tables(sc.REAL_FRAMES, 70 + slot))
    engines[0].run(50)
    engines[1].run_sampled(torch.rand(50, 3, device="cuda"), temperature=0.0)
    assert torch.equal(engines[0].out, engines[1].out)


# ---------------------------------------------------------------- the shared window

PREFIXES = ([SOS, OUT], [SOS, 5, OUT, 17, 200, 301], [SOS, OUT, 9, 11] + [(7 * i) % 500 + 4 for i in range(60)])


def shared_pair(batch, frames_engine=300, frames=277):
    own = table_engine(batch, frames_engine)
    shared = table_engine(batch, frames_engine, shared_window=True)
    memory = torch.from_numpy(memory_array(frames, sc.C1_SHORT.width, 31))
    for slot in range(batch):
        prefix = PREFIXES[slot % 3]
        own.load(slot, memory, prefix, None, frames, target=10_000)
        shared.load(slot, memory if slot == 0 else None, prefix, None, frames if slot == 0 else None, target=10_000)
    return own, shared


@pytest.mark.parametrize("batch", [1, 3, 16, 70])
def test_shared_window_agrees_with_a_copy_per_slot(batch):
    own, shared = shared_pair(batch)
    within = count = 0
    for _ in range(12):
        want, greedy = own.step_debug(None)
        got, _ = shared.step_debug(greedy)  # forced along the other engine's tokens
        assert logit_error(got, want) <= 1
        a, b = logit_within(got, want)
        within, count = within + a, count + b
    assert within >= LOGIT_WITHIN_FRACTION * count, (within, count)
    assert torch.equal(own.state["position"], shared.state["position"])


def test_a_shared_slot_does_not_depend_on_the_others():
    engines = [table_engine(5, 300, shared_window=True) for _ in range(2)]
    memory = memory_array(300, sc.C1_SHORT.width, 33)
    for n, eng in zip((1, 5), engines):
        for slot in range(n):
            eng.load(slot, memory if slot == 0 else None, PREFIXES[slot % 3], None, target=10_000)
        eng.run(40)
    assert torch.equal(engines[0].out[0], engines[1].out[0])


def test_shared_window_holds_one_copy_and_guards_it():
    eng = table_engine(4, 300, shared_window=True)
    memory = memory_array(300, sc.C1_SHORT.width, 34)
    with pytest.raises(_lib.EngineError, match="no window"):
        eng.load(0, None, [SOS, OUT], None)
    eng.load(0, memory, [SOS, OUT], None, 200, target=12)
    eng.load(2, None, [SOS, OUT], None, target=12)
    with pytest.raises(_lib.EngineError, match="slot 2 still decodes"):
        eng.load(0, memory, [SOS, OUT], None)
    eng.run(20)
    assert sorted(eng.finished()) == [0, 2]
    first, second = eng.take(0), eng.take(2)
    assert first == second  # the same reading, greedily
    eng.load(1, memory_array(300, sc.C1_SHORT.width, 35), [SOS, OUT], None, 300, target=12)  # the next window
    eng.run(20)
    single = table_engine(1, 300, shared_window=True)
    single.load(0, memory_array(300, sc.C1_SHORT.width, 35), [SOS, OUT], None, 300, target=12)
    single.run(20)
    assert eng.take(1) == single.take(0)
    own = table_engine(4, 300)
    with pytest.raises(ValueError, match="shared_window"):
        own.load(0, None, [SOS, OUT], None)


def test_prompt_sets_of_one_window_decode_side_by_side():
    """The real grammar: one slot per prompt set, against engines that decode each alone on a copy."""

    vocab = VocabTable()
    memory = memory_array(sc.REAL_FRAMES, sc.REAL_TINY.width, 41)
    both = real_engine(2, shared_window=True)
    both.load(0, memory, vocab.prompt_prefix(sc.REAL_PROMPT_SETS[1]), None)
    both.load(1, None, vocab.prompt_prefix(sc.REAL_PROMPT_SETS[0]), None)
    alone = real_engine(2)
    for slot, prompts in enumerate((sc.REAL_PROMPT_SETS[1], sc.REAL_PROMPT_SETS[0])):
        alone.load(slot, memory, vocab.prompt_prefix(prompts), None)
    for _ in range(10):
        want, greedy = alone.step_debug(None)
        got, _ = both.step_debug(greedy)
        assert logit_error(got, want) <= 1


# ---------------------------------------------------------------- readings, end to end

def test_decode_readings_ranks_reproducible_draws():
    memory = memory_array(300, sc.C1_SHORT.width, 51)
    song = Song(memory, [SOS, OUT], target=25)
    runs = []
    for _ in range(2):
        eng = table_engine(4, 300, shared_window=True)
        gen = torch.Generator(device="cuda").manual_seed(9)
        runs.append(decode_readings(eng, song, 7, generator=gen, temperature=1.2, top_p=0.98, poll_every=8))
        assert not any(eng.loaded) and eng.free_pages == 4 * 4
    assert runs[0] == runs[1]
    assert len(runs[0]) == 7 and len({tuple(r.tokens) for r in runs[0]}) > 1
    assert [r.logprob for r in runs[0]] == sorted((r.logprob for r in runs[0]), reverse=True)
    # a reading's log-probability is that of its tokens: teacher-force it through the engine
    eng = table_engine(4, 300, shared_window=True)
    best = runs[0][0]
    eng.load(0, memory, [SOS, OUT], None, target=25)
    grammar = make_grammar_oracle(eng.grammar)
    total = 0.0
    generated = best.tokens[2:27]
    for token in generated:
        state = {n: v.cpu().numpy().copy() for n, v in eng.state.items()}
        allowed = np.asarray(grammar.allowed(state))[0]
        assert allowed[token]
        logits, _ = eng.step_debug(np.array([token, -1, -1, -1]))
        x = logits[0].astype(np.float64)[allowed]
        total += float(logits[0][token]) - x.max() - np.log(np.exp(x - x.max()).sum())
    # each of the 25 draws within 1e-5 + 2^-22 of its float64 value (test_gpu_sample)
    assert abs(total - best.logprob) <= 25 * (1e-5 + 2.0**-22 * 10)


def test_greedy_readings_are_alike():
    eng = table_engine(3, 300, shared_window=True)
    song = Song(memory_array(300, sc.C1_SHORT.width, 52), [SOS, OUT], frames=250, target=20)
    readings = decode_readings(eng, song, 3, temperature=0.0)
    assert len({tuple(r.tokens) for r in readings}) == 1 and readings[0].ended == "eos"


CAPTURED_FIRST = """
import torch
from sheetsage2_refined_b200 import ops
g = torch.Generator(device="cuda").manual_seed(1)
def rand(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
q, k, v = rand(40, 8, 64), rand(300, 2, 64), rand(300, 2, 64)
pool = rand(40, 2, 64, 64)
own = dict(own_k=pool, own_v=pool, page_table=torch.arange(40, device="cuda", dtype=torch.int32).view(40, 1),
           own_len=torch.arange(40, device="cuda", dtype=torch.int32))
w, u = rand(512, 700, dtype=torch.float32), torch.rand(40, generator=g, device="cuda")
def step():
    out, lse = ops.shared_attention(q, k, v, **own)
    logits = out.float().reshape(40, 512)[:, :, None].mul(w).sum(1)
    return out, lse, *ops.sample(logits, u, top_k=20, top_p=0.9)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("equal")
"""


def test_the_first_calls_of_a_process_may_be_captured():
    """Attention, then a draw from what it gives, captured before either kernel has been set up."""

    run = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parents[1])
    assert run.returncode == 0 and "equal" in run.stdout, run.stderr[-2000:]
