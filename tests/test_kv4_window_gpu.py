"""The 4-bit cache under layers that see a window of positions and give back the pages behind it, and under a layer that reads the keys and
values of another: the engine beside the plain implementation, and beside itself however steps are put together."""
from dataclasses import replace

import pytest
import torch

from axon_amd.config.base import PartSpec
from axon_amd.config.qwen2 import Qwen2Config
from gpu_helpers import DTYPES
from helpers import prompts_for
from plain import kv4_plain as F
from plain import qwen2_plain as P
from test_kv4_engine_gpu import engine, feed

pytestmark = pytest.mark.gpu
WINDOW = 40


def windowed(monkeypatch, shared=False):
    plain = Qwen2Config.model_spec

    def spec(self):
        s = plain(self)
        layers = [replace(layer, mixer=PartSpec(layer.mixer.kind, {**layer.mixer.params, "window": WINDOW})) for layer in s.layers]
        return replace(s, layers=layers, order=[replace(run, cache=0, writes_cache=i == 0) for i, run in enumerate(s.order)] if shared else s.order)
    monkeypatch.setattr(Qwen2Config, "model_spec", spec)


@pytest.mark.parametrize("name", ["D", "E"])
def test_logits_in_a_window(model_dirs, monkeypatch, name):
    """As without a window: what is left beside the plain implementation over keys and values that went through the format is a tenth of what
    the format does, at most; positions behind the window are not seen, nor are their pages kept."""
    d, page = model_dirs(name), 8
    ids = prompts_for(name, (150,), seed=2)[0]
    attention = P.causal_attention
    pc, pw = P.load_plain(d)

    def logits(held):
        def through(x):
            return torch.from_numpy(F.values(*F.quantise(x.float().numpy()))).to(x.dtype) if held else x
        monkeypatch.setattr(P, "causal_attention", lambda q, k, v, window=0: attention(q, through(k), through(v), WINDOW))
        return P.forward_logits(pc, pw, ids).double()
    held, free = logits(True), logits(False)
    windowed(monkeypatch)
    e = engine(d, "float32", page)
    got = feed(e, "a", ids, [70, 1, 30, 1, 48], end=False).double().cpu()
    effect = float((held - free).abs().max())
    assert effect > 1e-4 * float(free.abs().max())
    assert float((got - held).abs().max()) <= 0.1 * effect
    kept = e.cache.pages_of(0, e.live["a"].slot)
    assert kept <= -(-WINDOW // page) + 2 < -(-len(ids) // page)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shared", [False, True])
def test_any_batching_and_replays_give_the_same_bits(model_dirs, monkeypatch, dtype, shared):
    """Portions of more than 16 tokens cut anywhere, single tokens alone, in a batch and from graphs, with pages given back and used again."""
    d, page = model_dirs("D"), 8
    windowed(monkeypatch, shared)
    a, b = prompts_for("D", (160, 101), seed=4)
    rows = {}
    for graphs in (False, True):
        e = engine(d, dtype, page, pages=40, use_graphs=graphs)
        alone = feed(e, "a", a, [160])
        assert torch.equal(alone, feed(e, "a", a, [33, 17, 61, 49]))
        feed(e, "b", b, [101], end=False)
        both = e.step([("a", a[:90], list(range(90))), ("b", [5], [0])]).clone()
        assert torch.equal(both[:90], alone[:90])
        rest = e.step([("b", [7], [0]), ("a", a[90:], list(range(70)))]).clone()
        assert torch.equal(rest[1:], alone[90:])
        e.release_all()
        feed(e, "b", b, [101], end=False)
        feed(e, "a", a, [160], end=False)
        got = [e.step([("b", [5], [0])]).clone(), e.step([("b", [7], [0])]).clone()]
        assert torch.equal(torch.cat(got), torch.stack([both[90], rest[0]]))
        for step in range(30):
            got.append(e.step([(r, [(step * 31 + 3) % 300], [0]) for r in ("a", "b")]).clone())
            torch.cuda.synchronize()
        rows[graphs] = torch.cat(got)
    assert torch.equal(rows[False], rows[True])
