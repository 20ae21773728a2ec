"""Steps of which some tiles are cut into segments and others, beyond the room that there is for it, are not: the same bits, and right."""
import pytest
import torch

from axon_amd.kernels import kernels
from gpu_helpers import DTYPES, TORCH
from test_kv4_gpu import Held, check, i32, prefill_by

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,dim,spans,window", [(3, 1, 64, [(200, 2000), (140, 8100), (90, 0)], 0), (4, 2, 128, [(300, 4000), (129, 1000)], 2500)])
def test_tiles_that_there_is_no_room_for_are_not_cut(monkeypatch, dtype, nh, nkv, dim, spans, window):
    k, page = kernels(dtype), 32
    held = Held([n + at for n, at in spans], nkv, dim, page, seed=95)
    pos = [at + i for n, at in spans for i in range(n)]
    seq = [r for r, (n, _) in enumerate(spans) for _ in range(n)]
    first, listed = 0, []
    for n, at in spans:
        listed.append((first, n, at))
        first += n
    q = torch.randn((first, nh * dim), generator=torch.Generator().manual_seed(4)).to(TORCH[dtype]).cuda()
    counts, want = [], None
    for room in (k.KV4_CUT, 7 * nh, 3 * nh, 0):
        monkeypatch.setattr(k, "KV4_CUT", room)
        tiles = k.kv4_prefill_tiles(listed, window, nh, nkv)
        counts.append(sum(row[2] >= 0 for row in tiles))
        assert counts[-1] * nh <= room
        got = prefill_by(k, held, q, tiles, pos, seq, nh, nkv, dim, page, window, 0.1)
        want = got if want is None else want
        assert torch.equal(got, want)
    assert counts[0] > counts[1] > counts[2] > counts[3] == 0
    some = [0, 127, 128, 250, first - 1]
    check(dtype, want[some], q[some], held, [pos[i] for i in some], [seq[i] for i in some], window, 0.1, dim, nh)
