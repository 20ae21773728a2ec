"""What the 4-bit cache's calls check of their arguments before anything is launched, without a device: tensors of the host that say that they lie on
one, and entry points that note their calls."""
from types import SimpleNamespace

import copy

import pytest
import torch

from axon_amd.kernels import KernelError, kernels
from axon_amd.kernels import lib

NH, NKV, DIM, PAGE = 4, 2, 64, 8


class Placed(torch.Tensor):
    """A tensor that says it lies on device 0, or on the one named."""
    device_index = 0

    def get_device(self):
        return self.device_index

    @property
    def is_cuda(self):
        return True


def on(t, device=0):
    out = t.as_subclass(Placed)
    out.device_index = device
    return out


def i32(values, device=0):
    return on(torch.tensor(values, dtype=torch.int32), device)


@pytest.fixture
def calls(monkeypatch):
    """(kernels whose launches are noted instead, the list of them)."""
    monkeypatch.setattr(lib, "_device", lambda: 0)
    monkeypatch.setattr(lib, "_raw_stream", lambda device: 0)
    k, noted = copy.copy(kernels("bfloat16")), []
    real = k.run
    own = {name: getattr(real, name) for name in ("axk_kv4_ok", "axk_kv4_row_bytes", "axk_kv4_decode_workspace", "axk_kv4_prefill_workspace",
                                                  "axk_kv4_prefill_tile", "axk_kv4_prefill_segment", "axk_kv4_prefill_segment_start",
                                                  "axk_kv4_decode_chunk", "axk_kv4_decode_item_factor")}
    for name in ("axk_kv4_attention_decode", "axk_kv4_attention_prefill"):
        own[name] = lambda *a, name=name: noted.append(name) or 0
    k.run = SimpleNamespace(**own)
    return k, noted


def arguments(n):
    caches = [on(torch.zeros((3, NKV, PAGE, DIM // 2 + DIM // 16), dtype=torch.uint8)) for _ in range(2)]
    q = on(torch.zeros((n, NH * DIM), dtype=torch.bfloat16))
    return dict(q=q, q_stride=NH * DIM, k_cache=caches[0], v_cache=caches[1], block_table=i32([[0, 1]]), positions=i32([5] * n),
                seq_rows=i32([0] * n), out=on(torch.zeros_like(q)), n_heads=NH, n_kv_heads=NKV, head_dim=DIM, page_size=PAGE, window=0, scale=0.1)


def test_prompt_workspaces_that_are_too_small(calls):
    k, noted = calls
    tiles = k.kv4_prefill_tiles([(0, 200, 2000)], 0, NH, NKV)
    slots, floats = k.kv4_prefill_slots(tiles), k.kv4_prefill_workspace(tiles, NH, DIM)
    assert slots == 2 * 3 and floats == 6 * k.kv4_prefill_workspace([(0, 1, -1, 0)], NH, DIM)      # (two tiles, segments 0, 1 and 2 of each)
    good = dict(arguments(200), tiles=i32(tiles), partial=on(torch.zeros(floats)), slots=slots)
    k.kv4_attention_prefill(**good)
    for wrong in (dict(partial=on(torch.zeros(floats - 1))), dict(partial=on(torch.zeros(0))), dict(slots=slots + 1), dict(slots=-1)):
        with pytest.raises(KernelError, match="slots"):
            k.kv4_attention_prefill(**{**good, **wrong})
    assert noted == ["axk_kv4_attention_prefill"]
    one = k.kv4_prefill_tiles([(0, 100, 0)], 0, NH, NKV)
    assert k.kv4_prefill_slots(one) == k.kv4_prefill_slots([]) == 0
    k.kv4_attention_prefill(**dict(arguments(100), tiles=i32(one), partial=on(torch.zeros(0)), slots=0))


def test_named_tokens_on_another_device(calls):
    k, noted = calls
    good = dict(arguments(3), token_index=i32([2, 0]), partial=on(torch.zeros(k.kv4_decode_workspace(2, NH, DIM, 1))), max_chunks=1,
                work=i32(k.kv4_decode_work([5, 5], 0)))
    k.kv4_attention_decode(**good)
    with pytest.raises(KernelError):
        k.kv4_attention_decode(**{**good, "token_index": i32([2, 0], device=1)})
    assert noted == ["axk_kv4_attention_decode"]
