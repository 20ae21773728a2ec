"""The 4-bit cache without a device: how steps are split for its kernels, what the library's entry points refuse, which models take it,
and the reads of LDS that its prompt kernel writes as instructions."""
import random

import numpy as np
import pytest

from axon_amd.config import ConfigError, config_from_dict
from axon_amd.kernels import KernelError, kernels
from axon_amd.models import build_model_description
from gpu_helpers import DTYPES
from helpers import TINY
from plain import kv4_plain as P
from test_lds_reads import unwaited

TILE = 128


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("nh,nkv,window", [(28, 4, 0), (1, 1, 0), (64, 64, 0), (14, 2, 700), (8, 1, 1)])
def test_tiles_have_every_row_and_position_once(seed, nh, nkv, window):
    k, rng = kernels("bfloat16"), random.Random(seed)
    spans, first = [], 0
    for _ in range(rng.choice([1, 2, 9])):
        n, at = rng.choice([1, 17, 127, 128, 129, 700]), rng.choice([0, 1, 1900, 2047, 2048, 8191, 8192, 30000])
        spans.append((first, n, at))
        first += n + rng.choice([0, 3])
    tiles = k.kv4_prefill_tiles(spans, window, nh, nkv)
    start, segment = k.run.axk_kv4_prefill_segment_start, k.run.axk_kv4_prefill_segment
    at_of = {s + i: at + i for s, n, at in spans for i in range(n)}
    rows, slots, parts, work = [], set(), {}, []
    assert len({len(row) for row in tiles}) == 1 and (len(tiles[0]) == 5) == any(row[2] >= 0 for row in tiles)
    for first, count, which, slot, *n in tiles:
        assert 0 < count <= TILE
        p0, p1 = at_of[first], at_of[first + count - 1]
        assert p1 - p0 == count - 1                       # one portion's
        low = max(0, p0 + 1 - window) if window else 0
        s0, s1 = segment(low), segment(p1)
        if which >= 0:
            assert s0 <= which <= s1 and slot not in slots and n == [s1 - s0 + 1 if which == s0 else 0]
            slots.add(slot)
            parts.setdefault((first, count), {})[which] = slot
            work.append(min(p1, start(which + 1) - 1) - max(low, start(which)))
        else:
            assert which == -1 and n in ([], [0]) and (slot == -1) == (s0 == s1) and slot not in slots
            rows += range(first, first + count)
            slots |= {slot} - {-1}
            work.append(p1 - low)
    for (first, count), mine in parts.items():              # the slots of a tile's segments, in order
        p1 = at_of[first + count - 1]
        low = max(0, p1 - count + 2 - window) if window else 0
        assert [mine[s] for s in range(segment(low), segment(p1) + 1)] == list(range(mine[segment(low)], mine[segment(low)] + len(mine)))
        rows += range(first, first + count)
    assert sorted(rows) == sorted(at_of) and work == sorted(work, reverse=True)
    assert slots == set(range(len(slots)))
    one = k.kv4_prefill_workspace([(0, 1, -1, 0)], nh, 64)
    assert one > 0 and k.kv4_prefill_workspace(tiles, nh, 64) == len(slots) * one


def test_segments_follow_each_other():
    k = kernels("bfloat16")
    segment, start = k.run.axk_kv4_prefill_segment, k.run.axk_kv4_prefill_segment_start
    for s in range(300):
        assert start(s) < start(s + 1) and start(s) % 64 == 0
        assert segment(start(s)) == s == segment(start(s + 1) - 1)
    assert segment(2 ** 31 - 1) > 0 and start(segment(2 ** 31 - 1) + 1) == 2 ** 31 - 1


@pytest.mark.parametrize("window", [0, 1, 300, 9000])
def test_every_position_is_in_one_chunk(window):
    """What a token's work items cover, by the kernel's own chunk sizes, and the bounds that an engine plans by."""
    k = kernels("bfloat16")
    positions = [0, 1, 63, 255, 256, 2100, 8191, 8192, 16383, 16384, 40000, k.kv4_max_context - 1]
    factor, items, most = int(k.run.axk_kv4_decode_item_factor()), [], 0
    for slot, p in enumerate(positions):
        low = max(0, p + 1 - window) if window else 0
        size = int(k.run.axk_kv4_decode_chunk(p + 1 - low))
        assert size % 64 == 0
        n = p // size - low // size + 1
        items += [slot * factor + c for c in range(n)]
        most = max(most, n)
        assert n <= k.kv4_most_chunks(p + 1, window) <= factor
        assert k.kv4_decode_chunks([p], window) == n
    assert sorted(k.kv4_decode_work(positions, window)) == items and k.kv4_decode_chunks(positions, window) == most
    assert k.kv4_decode_work([], window) == [] and k.kv4_decode_chunks([], window) == 1
    if window == 0:
        with pytest.raises(KernelError):
            k.kv4_decode_work([k.kv4_max_context], 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_entry_points_refuse(dtype):
    """By the host's own checks, before anything is launched."""
    k = kernels(dtype)
    run, A = k.run, 4096                                  # an aligned address that nothing reads
    write = dict(qkv=A, qkv_stride=1024, q_out=A, q_stride=1024, table=A, pos=A, rows=A, block_table=A, table_stride=1, k=A, v=A, T=1, nh=4,
                 nkv=2, hd=64, rot=64, page=16, write_kv=1, stream=None)
    read = dict(k=A, v=A, block_table=A, table_stride=1, pos=A, rows=A, k_out=A, v_out=A, n=1, nkv=2, hd=64, page=16, stream=None)
    decode = dict(q=A, q_stride=256, k=A, v=A, block_table=A, table_stride=1, pos=A, rows=A, out=A, index=None, T=1, work=A, n_work=1,
                  partial=A, chunks=1, nh=4, nkv=2, hd=64, page=16, window=0, scale=0.1, stream=None)
    prompt = dict(q=A, q_stride=256, k=A, v=A, block_table=A, table_stride=1, pos=A, rows=A, out=A, tiles=A, n=1, columns=4, partial=A, floats=4, nh=4,
                  nkv=2, hd=64, page=16, window=0, scale=0.1, stream=None)
    cases = [(run.axk_rope_kv4_write, write, [dict(T=-1), dict(nh=0), dict(nkv=0), dict(hd=96), dict(hd=32), dict(page=4), dict(page=2048),
                                              dict(page=24), dict(rot=8), dict(rot=80), dict(rot=-16), dict(qkv=A + 8), dict(q_out=A + 4),
                                              dict(qkv_stride=1025), dict(q_stride=1025), dict(k=A + 8), dict(v=A + 8), dict(table=A + 4)]),
             (run.axk_kv4_read, read, [dict(n=-1), dict(nkv=0), dict(hd=256), dict(page=0), dict(k=A + 8), dict(v=A + 8), dict(k_out=A + 8),
                                       dict(v_out=A + 8)]),
             (run.axk_kv4_attention_decode, decode, [dict(hd=80), dict(page=12), dict(nh=0), dict(nkv=3), dict(nkv=0), dict(window=-1),
                                                     dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(T=-1), dict(chunks=0),
                                                     dict(chunks=1025), dict(n_work=-1), dict(work=None), dict(partial=None), dict(partial=A + 4),
                                                     dict(q=A + 8), dict(out=A + 8), dict(q_stride=257), dict(q_stride=-256)]),
             (run.axk_kv4_attention_prefill, prompt, [dict(hd=80), dict(page=12), dict(nh=5), dict(nh=65536), dict(window=-1), dict(scale=-1.0),
                                                      dict(n=-1), dict(n=65536), dict(tiles=None), dict(columns=3), dict(columns=6), dict(floats=-1), dict(partial=None),
                                                      dict(partial=A + 4), dict(k=A + 8), dict(q_stride=257)])]
    for entry, good, wrong in cases:
        for change in wrong:
            assert set(change) <= set(good)
            assert entry(*{**good, **change}.values()) < 0, change
            with pytest.raises(KernelError):
                k._check(entry(*{**good, **change}.values()))
    # nothing to do is done
    assert run.axk_rope_kv4_write(*{**write, "T": 0}.values()) == 0 and run.axk_kv4_read(*{**read, "n": 0}.values()) == 0
    assert run.axk_kv4_attention_decode(*{**decode, "T": 0, "partial": None}.values()) == 0
    assert run.axk_kv4_attention_prefill(*{**prompt, "n": 0, "tiles": None}.values()) == 0


def test_models_that_take_it():
    for name in ("D", "E"):
        config = config_from_dict(TINY[name]["config"])
        model = build_model_description(config, 4)
        specs = [b.mixer.cache_spec() for b in model.blocks]
        for spec, plain in zip(specs, (b.mixer.cache_spec() for b in build_model_description(config).blocks)):
            assert spec.dtype == "uint8" and (spec.heads, spec.window, spec.entries) == (plain.heads, plain.window, plain.entries)
            assert spec.head_dim == P.row_bytes(plain.head_dim)
        for bits in (1, 8, 16, None):
            with pytest.raises(ConfigError):
                build_model_description(config, bits)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_comes_between_a_read_and_its_wait(device_code, dtype):
    reads, faults = unwaited(device_code("kv4_attention.hip", dtype), "kv4_prefill_kernel")
    assert reads > 0 and not faults, faults[:5]


def test_quotients_by_a_scale_are_the_correctly_rounded_ones():
    """The kernels divide by a scale with its reciprocal and one correction: q = x r, q + (x - q s) r, each rounded once to 32 bits
    (the middle step exactly).  Over all scales and numbers of all sizes that is x / s to the last bit."""
    rng = np.random.default_rng(0)
    scales = P.scale_table()[0].astype(np.float32)
    scales = scales[scales > 0]
    x = (rng.standard_normal((200, 1)) * np.exp2(rng.integers(-30, 16, (200, 1)))).astype(np.float32)
    s = scales[None]
    r = np.float32(1) / s
    q = x * r
    rest = x.astype(np.float64) - q.astype(np.float64) * s                 # exact in 64 bits, as a fused step's input is
    fused = (rest.astype(np.float32).astype(np.float64) * r.astype(np.float64) + q.astype(np.float64)).astype(np.float32)
    assert np.array_equal(rest.astype(np.float32), rest)
    assert np.array_equal(fused, x / s)
