"""Generation with keys and values held in 4 bits under load: a request's tokens are those that it gets alone, whatever other requests leave
of a step's tokens and of the pages: prompts cut anywhere (into portions of one token too), requests that give way and are fed again."""
import random

import pytest
import torch

import axon_amd
from axon_amd.engine import StepEntry, StepError
from axon_amd.parts import attention
from gpu_helpers import DTYPES
from helpers import TINY, prompts_for, run_trace

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
def test_requests_that_give_way_continue_with_the_same_tokens(model_dirs, dtype):
    d = model_dirs("D", "float32" if dtype == "float32" else "bfloat16")
    prompts = prompts_for("D", (20, 25, 18, 30, 1), seed=6)
    roomy = axon_amd.load(d, dtype=dtype, cache_bits=4, page_size=16, num_pages=64, max_seqs=5)
    want = roomy.generate(prompts, max_new_tokens=40)
    assert roomy.last_stats.preemptions == 0
    alone = [roomy.generate(p, max_new_tokens=40)[0] for p in prompts]
    assert alone == want
    tight = axon_amd.load(d, dtype=dtype, cache_bits=4, page_size=16, num_pages=9, max_seqs=4, max_batch_tokens=32)
    assert tight.generate(prompts, max_new_tokens=40) == want
    assert tight.last_stats.preemptions > 0
    tight.engine.cache.check()
    assert tight.engine.cache.free_pages() == 9
    kw = dict(max_new_tokens=30, temperature=0.9, seed=3)
    sampled = roomy.generate(prompts, **kw)
    assert tight.generate(prompts, **kw) == sampled and tight.last_stats.preemptions > 0
    stop = sampled[1][7]
    for full, part in zip(sampled, tight.generate(prompts, stop=[stop], **kw)):
        assert part == (full[:full.index(stop)] if stop in full else full)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("budget", [1, 5, 17, 33])
def test_prompts_cut_by_the_budget(model_dirs, dtype, budget):
    d = model_dirs("E", "float32" if dtype == "float32" else "bfloat16")
    prompts = prompts_for("E", (40, 18, 3, 67), seed=9)
    page = TINY["E"]["page_size"]
    whole = axon_amd.load(d, dtype=dtype, cache_bits=4, page_size=page, num_pages=64, max_seqs=4)
    cut = axon_amd.load(d, dtype=dtype, cache_bits=4, page_size=page, num_pages=64, max_seqs=4, max_batch_tokens=budget)
    for kw in (dict(max_new_tokens=10), dict(max_new_tokens=10, temperature=0.8, seed=5)):
        assert cut.generate(prompts, **kw) == whole.generate(prompts, **kw)


def logits_by(llm, ids, cuts, prompt):
    """Logits of every position, fed in portions of `cuts` tokens, the first `prompt` tokens as the prompt's."""
    e, out, at = llm.engine, [], 0
    for n in cuts:
        out.append(e.step([StepEntry("r", ids[at:at + n], list(range(n)), max(0, min(n, prompt - at)))], end=["r"] if at + n == len(ids) else []).clone())
        at += n
    assert at == len(ids)
    return torch.cat(out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("graphs", [False, True])
def test_steps_that_are_told_the_prompts_tokens(model_dirs, monkeypatch, dtype, graphs):
    """However a request's tokens are cut, and whether its own tokens come one by one or in a portion behind its prompt: the same logits."""
    d = model_dirs("D", "float32" if dtype == "float32" else "bfloat16")
    llm = axon_amd.load(d, dtype=dtype, cache_bits=4, page_size=16, num_pages=32, max_seqs=2, use_graphs=graphs)
    ids = prompts_for("D", (130,), seed=3)[0]
    prompt = 90
    want = logits_by(llm, ids, [90] + [1] * 40, prompt)
    for cuts in ([130], [89] + [1] * 41, [1] * 130, [16, 1, 17, 2, 54, 30, 10], [95, 35], [88, 1, 41]):
        assert torch.equal(logits_by(llm, ids, cuts, prompt), want), cuts
    for floats in (1, 6 * 66 * 7):                    # of partial results a call: a token, and seven, in the place of all
        monkeypatch.setattr(attention, "KV4_PARTIAL", floats)
        assert torch.equal(logits_by(llm, ids, [20, 110], prompt), want)
    for wrong in (-1, 4, 1.5, "2"):
        with pytest.raises(StepError):
            llm.engine.step([StepEntry("r", ids[:3], [0], wrong)])
    assert not llm.engine.live
    # what a step is not told: a portion of more tokens is a prompt's, a single one was generated
    assert torch.equal(llm.engine.step([StepEntry("r", ids[:90], list(range(90)))]), want[:90])
    for i in range(90, 93):
        assert torch.equal(llm.engine.step([StepEntry("r", [ids[i]], [0])], end=["r"] if i == 92 else []), want[i:i + 1])
    assert torch.equal(llm.logits(ids[:1]), llm.logits(ids[:1], all_positions=True)[0])
    assert torch.equal(llm.logits(ids[:1]), want[0])


def test_the_trace_program_is_told_them_too(model_dirs, tmp_path):
    d = model_dirs("D", "bfloat16")
    ids = prompts_for("D", (22,), seed=4)[0]
    llm = axon_amd.load(d, cache_bits=4, page_size=16, num_pages=16, max_seqs=2)
    want = llm.logits(ids, all_positions=True).cpu().numpy()
    steps = [{"step": 0, "entries": [{"id": "a", "tokens": ids[:20], "want": [19]}], "end": []},
             {"step": 1, "entries": [{"id": "a", "tokens": ids[20:21], "want": [0], "prompt": 1}], "end": []},
             {"step": 2, "entries": [{"id": "a", "tokens": ids[21:], "want": [0], "prompt": 1}], "end": ["a"]}]
    got = run_trace(d, "bfloat16", steps, str(tmp_path), 64, ["--cache-bits", "4"])
    assert all((got[i][0] == want[19 + i]).all() for i in range(3))


@pytest.mark.parametrize("seed", range(6))
def test_random_loads(model_dirs, seed):
    """Requests of random lengths under a random budget and too few pages: what each gets alone."""
    rng = random.Random(seed)
    name = rng.choice("DE")
    d = model_dirs(name, "bfloat16")
    prompts = prompts_for(name, [rng.choice([1, 2, 5, 16, 17, 40, 90, 130]) for _ in range(7)], seed=seed)
    page, kw = rng.choice([8, 16, 64]), dict(max_new_tokens=rng.choice([9, 30]))
    if rng.random() < 0.5:
        kw.update(temperature=0.8, seed=seed)
    roomy = axon_amd.load(d, cache_bits=4, page_size=page, num_pages=7 * (170 // page + 2), max_seqs=7)
    want = roomy.generate(prompts, **kw)
    assert roomy.last_stats.preemptions == 0
    tight = axon_amd.load(d, cache_bits=4, page_size=page, num_pages=170 // page + 2, max_seqs=5, max_batch_tokens=rng.choice([3, 18, 50, 200]),
                          use_graphs=rng.random() < 0.5)
    assert tight.generate(prompts, **kw) == want
