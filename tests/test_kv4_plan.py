"""How steps are planned for the 4-bit cache's prompt kernel: the workspace of tiles that are cut has a bound, which a cache pool sized from
the free memory leaves room for; which form of the kernel a step takes; and the models that cannot have such a cache."""
import importlib
from types import SimpleNamespace

import pytest
import torch

from axon_amd.config import ConfigError, EngineConfig, config_from_dict
from axon_amd.engine import Engine
from axon_amd.kernels import kernels
from axon_amd.models import build_model_description
from axon_amd.parts.attention import KV4_PARTIAL
from axon_amd.parts.base import CacheSpec
from helpers import TINY


@pytest.mark.parametrize("nh,nkv,dim", [(28, 4, 128), (1, 1, 64), (64, 8, 128), (14, 2, 64), (40, 8, 128)])
@pytest.mark.parametrize("longest", [1000, 1025, 9000, 131072, 1 << 20])
def test_the_workspace_of_a_step_has_a_bound(nh, nkv, dim, longest):
    k = kernels("bfloat16")
    one = k.kv4_prefill_workspace([(0, 1, -1, 0)], nh, dim)
    for tokens, requests in ((2048, 1), (2048, 7), (300, 3), (129, 1), (64, 1), (9000, 2), (16384, 64)):
        bound = k.kv4_prefill_most_workspace(tokens, requests, longest, nh, dim)
        # cut tiles 16,384 segments and heads, and those that are not cut one slot each
        assert bound <= ((1 << 14) // nh + -(-tokens // 128) + requests + 511 // nh) * one and (longest > 1024 or bound == 0)
        for window in (0, 5000):
            spans, n = [], -(-tokens // requests)
            for r in range(requests):
                mine = min(n, tokens - r * n)
                if mine > 0:
                    spans.append((r * n, mine, max(0, longest - mine - 37 * r)))
            if any(at + n > longest for _, n, at in spans):
                continue
            tiles = k.kv4_prefill_tiles(spans, window, nh, nkv)
            assert k.kv4_prefill_workspace(tiles, nh, dim) <= bound
            cut = [row for row in tiles if row[2] >= 0]
            assert len(cut) * nh <= 1 << 14
            assert sum(row[1] for row in tiles if row[2] < 0) + sum(row[1] for row in cut if row[4] > 0) == sum(m for _, m, _ in spans)
    # up to 131,072 positions everything is cut that is worth it: a tile, and what a step of four tiles holds
    if longest <= 131072 and nh <= 40:
        assert all(row[2] >= 0 for row in k.kv4_prefill_tiles([(0, 512, longest - 512)], 0, nh, nkv)) == (longest > 1024 + 512)


def test_mixers_say_what_steps_take():
    config = config_from_dict(TINY["D"]["config"])
    for bits in (0, 4):
        for block in build_model_description(config, bits).blocks:
            block.mixer._kernels = k = kernels("bfloat16")
            asked = block.mixer.step_scratch(2048, 4, 100000)
            assert asked is None if bits == 0 else asked[1] == k.kv4_prefill_most_workspace(2048, 4, 100000, 6, 64) + KV4_PARTIAL


def test_the_pool_leaves_room_for_them(monkeypatch):
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (1 << 30, 1 << 34))
    spec = CacheSpec(entries=2, heads=4, head_dim=72, dtype="uint8")
    engine = SimpleNamespace(cfg=EngineConfig(max_seqs=64, max_seq_len=1 << 20), rt=SimpleNamespace(device=None, elem_size=2), max_seq_len=1 << 20,
                             model=SimpleNamespace(cache_plan=SimpleNamespace(group_specs=[spec])), _scratch_sizes={"a": 1 << 20})
    per_page = 28 * 2 * 4 * 64 * 72
    free = int(((1 << 30) - 4 * (1 << 20)) * 0.85) // per_page
    assert Engine._pool_size(engine, spec, 28, 64) == free
    assert Engine._pool_size(engine, spec, 28, 64, of_steps=1 << 26) == int(((1 << 30) - 4 * (1 << 20) - 4 * (1 << 26)) * 0.85) // per_page < free


def test_which_steps_take_two_heads_a_workgroup():
    """The sizes of the tests that compare one and two heads a workgroup lie on both sides of the rule; the float32 build has one form."""
    k, f = kernels("bfloat16"), kernels("float32")
    for nh, nkv, portions in ((14, 2, 57), (28, 4, 29), (9, 3, 90), (5, 1, 160)):        # test_two_heads_a_workgroup
        assert k.kv4_prefill_heads(portions, nh, nkv) == k.kv4_prefill_heads(1 + 769 // nh + 1, nh, nkv) == 2
        assert k.kv4_prefill_heads(1, nh, nkv) == f.kv4_prefill_heads(portions, nh, nkv) == 1
    for nh, nkv, spans, window in ((7, 1, [(300, 5), (130, 0), (77, 1000)], 0), (4, 2, [(257, 700), (64, 64)], 130),
                                   (3, 1, [(128, 1990), (200, 4000)], 2500)):             # test_one_and_two_heads_a_workgroup_...
        firsts = [sum(n for n, _ in spans[:i]) for i in range(len(spans))]
        cut = len(k.kv4_prefill_tiles([(at, n, p) for at, (n, p) in zip(firsts, spans)], window, nh, nkv))
        whole, nothing = sum(-(-n // 128) for n, _ in spans), 769 // nh + 1
        assert [k.kv4_prefill_heads(n, nh, nkv) for n in (cut, cut + nothing, whole, whole + nothing)] == [1, 2, 1, 2]
    assert k.kv4_prefill_heads(65535, 8, 8) == 1                                          # a group of one has no second head


@pytest.mark.parametrize("design", ["pikesun", "figalorn", "napizen", "zugutar", "lilunex", "bafavik"])
def test_models_whose_mixers_cannot_hold_it_are_refused(design):
    """By the first mixer that keeps keys and values and has no form for 4 bits, paired ones among them; a model without such a mixer has nothing to
    hold."""
    for model in importlib.import_module(f"{design}_models").MODELS.values():
        config = config_from_dict(model["cfg"])
        kept = [b.mixer for b in build_model_description(config).blocks if b.mixer.cache_spec() is not None]
        expect = f"{type(kept[0]).__name__} does not hold its cache in 4 bits" if kept else "no mixer of this model keeps keys and values"
        with pytest.raises(ConfigError, match=expect):
            build_model_description(config, 4)
    for bits in (3, 8):
        for mixer in kept:
            with pytest.raises(ConfigError):
                mixer.hold_cache_in(bits)
