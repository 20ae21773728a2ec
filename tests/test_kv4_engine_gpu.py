"""The engine with its keys and values held in 4 bits: what a user is given, beside the plain implementation over keys and values that
went through the format, and beside itself (however steps are put together, replayed or resumed)."""
import json
import subprocess
import sys
import os

import numpy as np
import pytest
import torch

from axon_amd.config import ConfigError, EngineConfig, config_from_dict
from axon_amd.engine import Engine, Runtime
from axon_amd.engine.loading import load_model
from axon_amd.engine.step import StepError
from gpu_helpers import DTYPES
from helpers import ROOT, TINY, prompts_for
from plain import kv4_plain as F
from plain import qwen2_plain as P

pytestmark = pytest.mark.gpu


def engine(d, dtype, page, pages=96, max_seqs=4, **kw):
    rt = Runtime(dtype)
    model = load_model(d, rt, cache_bits=4)
    kw.setdefault("use_graphs", False)
    return Engine(model, rt, EngineConfig(dtype=dtype, page_size=page, num_pages=pages, max_seqs=max_seqs, **kw))


def feed(e, rid, ids, cuts, end=True):
    """Logits of every position, the prompt cut at `cuts`."""
    out, at = [], 0
    for n in cuts:
        out.append(e.step([(rid, ids[at:at + n], list(range(n)))], end=[rid] if end and at + n == len(ids) else []).clone())
        at += n
    assert at == len(ids)
    return torch.cat(out)


def plain_logits(d, ids, held):
    """The plain implementation; `held`: its keys (behind the rotation) and values through the 4-bit format."""
    pc, pw = P.load_plain(d)
    if not held:
        return P.forward_logits(pc, pw, ids)
    plain = P.causal_attention

    def through(x):
        n, words = F.quantise(x.float().numpy())
        return torch.from_numpy(F.values(n, words)).to(x.dtype)
    P.causal_attention = lambda q, k, v, window=0: plain(q, through(k), through(v), window)
    try:
        return P.forward_logits(pc, pw, ids)
    finally:
        P.causal_attention = plain


@pytest.mark.parametrize("name", ["D", "E"])
def test_logits_are_those_of_keys_and_values_in_the_format(model_dirs, name):
    """Against the plain implementation whose keys and values went through the format, in the float32 build: what is left is far less than
    what the format does.  (A number nearer to a border between two steps than 32 bits resolve may take the other step, one in some 2^18; all
    others take the same, so a tenth of the format's own effect is a wide bound.)"""
    d = model_dirs(name)
    ids = prompts_for(name, (120,), seed=2)[0]
    got = feed(engine(d, "float32", TINY[name]["page_size"]), "a", ids, [50, 1, 69]).double().cpu()
    held, free = (plain_logits(d, ids, h).double() for h in (True, False))
    effect = float((held - free).abs().max())
    assert effect > 1e-4 * float(free.abs().max())
    assert float((got - held).abs().max()) <= 0.1 * effect


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["D", "E"])
def test_any_batching_gives_the_same_bits(model_dirs, name, dtype):
    """Portions of more than 16 tokens cut anywhere, requests alone or side by side, single tokens in any batch."""
    d, page = model_dirs(name), TINY[name]["page_size"]
    a, b = prompts_for(name, (150, 97), seed=3)
    e = engine(d, dtype, page)
    alone = feed(e, "a", a, [150])
    assert torch.equal(alone, feed(e, "a", a, [40, 17, 93]))
    other = feed(e, "b", b, [97], end=False)
    both = e.step([("a", a[:60], list(range(60))), ("b", [5], [0])]).clone()
    assert torch.equal(both[:60], alone[:60])
    rest = e.step([("b", [7], [0]), ("a", a[60:], list(range(90)))]).clone()
    assert torch.equal(rest[1:], alone[60:])
    e.release_all()
    # single tokens, alone and in a batch
    feed(e, "b", b, [97], end=False)
    one = [e.step([("b", [t], [0])]).clone()[0] for t in (5, 7)]
    assert torch.equal(torch.stack(one), torch.stack([both[60], rest[0]]))
    # a single token and the same in a portion: within the outputs' rounding
    e.release_all()
    feed(e, "b", b[:60], [60], end=False)
    near = torch.cat([e.step([("b", [t], [0])]).clone() for t in b[60:]])
    span = float(other.max() - other.min())
    assert float((near - other[60:]).abs().max()) <= 2e-2 * span


@pytest.mark.parametrize("dtype", DTYPES)
def test_replayed_steps_are_the_launched_ones(model_dirs, dtype):
    """Decoding from graphs, several replays of each shape with eager work between: the same bits as launch by launch."""
    d, page = model_dirs("D"), 8
    prompts = prompts_for("D", (30, 61, 7), seed=5)
    rows = {}
    for graphs in (False, True):
        e = engine(d, dtype, page, use_graphs=graphs)
        for i, p in enumerate(prompts):
            e.step([(i, p, [])])
        got = []
        for step in range(12):
            ids = [0, 1, 2] if step % 4 else [0, 1]
            got.append(e.step([(i, [(step * 31 + i) % 300], [0]) for i in ids]).clone())
            torch.cuda.synchronize()
            if step % 3 == 0:
                feed(e, "other", prompts[1], [61])
        rows[graphs] = torch.cat(got)
    assert torch.equal(rows[False], rows[True])


def test_generation(model_dirs, tmp_path):
    """`load(..., cache_bits=4)` generates, with pages running out in between; the command line and the trace program take the option."""
    import axon_amd
    d = model_dirs("D", "bfloat16")
    prompts = prompts_for("D", (40, 90, 25), seed=8)
    llm = axon_amd.load(d, cache_bits=4, page_size=16, num_pages=64, max_seqs=3)
    out = llm.generate(prompts, max_new_tokens=12)
    assert [len(o) for o in out] == [12] * 3
    tight = axon_amd.load(d, cache_bits=4, page_size=16, num_pages=9, max_seqs=3)
    assert [len(o) for o in tight.generate(prompts, max_new_tokens=12)] == [12] * 3
    spec = llm.model.cache_plan.group_specs[0]
    assert spec.dtype == "uint8" and spec.head_dim == 36             # 64 numbers in 36 bytes
    line = subprocess.run([os.path.join(ROOT, "bin", "axon"), "gen", d, " ".join(map(str, prompts[0])), "-n", "12", "--cache-bits", "4",
                           "--page-size", "16"], capture_output=True, text=True, check=True, timeout=100).stdout
    assert [int(t) for t in line.split()] == out[0]
    steps = [{"step": 0, "entries": [{"id": 0, "tokens": prompts[0], "want": [39]}], "end": [0]}]
    run = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "trace_run"), "--model", d, "--dtype", "bfloat16", "--out", str(tmp_path),
                          "--max-tokens", "64", "--cache-bits", "4"], input="\n".join(map(json.dumps, steps)) + "\n", capture_output=True, text=True,
                         check=True, timeout=100)
    assert run.stdout.split() == ["done", "0"]
    logits = np.fromfile(tmp_path / "0.f32", dtype="<f4")
    assert int(logits.argmax()) == out[0][0]


def test_what_cannot_be_is_refused(model_dirs):
    for name in ("B", "C"):                                          # heads of 32 and 80
        with pytest.raises(ConfigError):
            load_model(model_dirs(name), Runtime("bfloat16"), cache_bits=4)
    with pytest.raises(ConfigError):
        load_model(model_dirs("D"), Runtime("bfloat16"), cache_bits=3)
    for page in (4, 24, 2048):
        with pytest.raises(StepError):
            engine(model_dirs("D"), "bfloat16", page)
