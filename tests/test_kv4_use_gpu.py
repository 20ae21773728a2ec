"""The 4-bit cache's kernels as a program uses them together: written in portions and then attended to, captured and replayed, on other
streams, with heads and lengths beyond one workgroup's.  (The kernels one by one, and the tolerance: test_kv4_gpu.py.)"""
import numpy as np
import pytest
import torch

from axon_amd.kernels import KernelError, kernels
from gpu_helpers import DTYPES, TORCH
from plain import kv4_plain as P
from test_kv4_gpu import Held, check, decode, i32, prefill, random_rows, step_of

pytestmark = pytest.mark.gpu


def empty_caches(n_pages, nkv, page, dim):
    return [torch.full((n_pages, nkv, page, P.row_bytes(dim)), 0xAB, dtype=torch.uint8, device="cuda") for _ in range(2)]


def plain_cache(x, table, pos, seq, n_pages, nkv, nh, page, dim):
    """What rows [T, nh + 2 nkv, dim] (already in the build's type, no rotation) leave in a cache of bytes 0xAB."""
    want = P.Cache(n_pages, nkv, page, dim, fill=0xAB)
    for t, (p, r) in enumerate(zip(pos, seq)):
        if p >= 0:
            want.store(table[r, p // page], p % page, x[t, nh:nh + nkv], x[t, nh + nkv:])
    return want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spans,nkv,nh,dim,page", [
    ([(1, 13)], 32, 32, 64, 16), ([(1, 0), (2, 6)], 12, 12, 128, 8),                # more keys and values of a token than threads
    ([(515, 3)], 2, 2, 64, 16), ([(300, 1), (1, 9), (230, 12)], 1, 3, 128, 32),     # eight tokens a block, octets across blocks
    ([(512, 4)], 1, 1, 64, 64), ([(513, 0)], 3, 3, 64, 8)])
def test_write_of_many_heads_and_of_portions_that_begin_anywhere(dtype, spans, nkv, nh, dim, page):
    k = kernels(dtype)
    pos, seq, table, n_pages = step_of(spans, page)
    for at in (len(pos) // 2, 0):                                                    # padding inside and before
        pos.insert(at, -1)
        seq.insert(at, 0)
    T = len(pos)
    x = random_rows(np.random.default_rng(6), T, nh + 2 * nkv, dim)
    qkv = torch.from_numpy(x.reshape(T, -1)).to(TORCH[dtype]).cuda()
    exact = qkv.float().cpu().numpy().reshape(T, -1, dim)
    want = plain_cache(exact, table, pos, seq, n_pages, nkv, nh, page, dim)
    caches = empty_caches(n_pages, nkv, page, dim)
    q = torch.empty((T, nh * dim), dtype=TORCH[dtype], device="cuda")
    k.rope_kv4_write(qkv, q, torch.zeros((T, 0, 2), device="cuda"), i32(pos), i32(seq), torch.from_numpy(table).cuda(), *caches, nh, nkv, dim, 0,
                     page)
    assert torch.equal(q, qkv[:, :nh * dim])
    assert np.array_equal(caches[0].cpu().numpy(), want.keys) and np.array_equal(caches[1].cpu().numpy(), want.values)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_request_from_its_prompt_to_its_last_token(dtype):
    """Written in portions that end inside octets, attended to by tiles, then token by token: what a layer does, step by step."""
    k, nh, nkv, dim, page, scale = kernels(dtype), 6, 2, 64, 16, 0.125
    total, cuts = 310, [200, 37, 61] + [1] * 12
    table = np.random.default_rng(1).permutation(24).astype(np.int32)[None, :20]
    x = random_rows(np.random.default_rng(2), total, nh + 2 * nkv, dim)
    qkv = torch.from_numpy(x.reshape(total, -1)).to(TORCH[dtype]).cuda()
    qkv[:, :nh * dim] = torch.randn((total, nh * dim), generator=torch.Generator().manual_seed(3)).to(TORCH[dtype]).cuda()
    exact = qkv.float().cpu().numpy().reshape(total, -1, dim)

    class Written:
        k, v = ([P.values(*P.quantise(exact[:, a:a + nkv]))] for a in (nh, nh + nkv))
        args = (*empty_caches(24, nkv, page, dim), torch.from_numpy(table).cuda())
    at = 0
    for n in cuts:
        part = qkv[at:at + n]
        q = torch.empty((n, nh * dim), dtype=qkv.dtype, device="cuda")
        k.rope_kv4_write(part, q, torch.zeros((n, 0, 2), device="cuda"), i32(list(range(at, at + n))), i32([0] * n), Written.args[2],
                         *Written.args[:2], nh, nkv, dim, 0, page)
        pos, seq = list(range(at, at + n)), [0] * n
        if n > 1:
            got = prefill(k, Written, q, [(n, at)], [0], nh, nkv, dim, page, 0, scale)[2]
        else:
            got = decode(k, Written, q, pos, seq, nh, nkv, dim, page, 0, scale)
        check(dtype, got, q, Written, pos, seq, 0, scale, dim, nh)
        at += n
    assert at == total


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_and_replayed(dtype):
    """A layer's calls in a graph, replayed over other contents of the same tensors, with eager work between: each replay gives what the
    calls give."""
    k, nh, nkv, dim, page, scale = kernels(dtype), 8, 2, 128, 16, 0.09
    lengths, n = [40, 700, 2300], 90
    held = Held(lengths, nkv, dim, page, seed=20)
    table = held.args[2]
    g = torch.Generator().manual_seed(8)
    T = len(lengths) + n
    pos_host = [[p - 1 - d for p in lengths] + list(range(2299 - n - d, 2299 - d)) for d in (5, 0, 17)]        # (no position twice)
    seq = i32([0, 1, 2] + [2] * n)
    pos, qkv = i32(pos_host[0]), torch.zeros((T, (nh + 2 * nkv) * dim), dtype=TORCH[dtype], device="cuda")
    rope = torch.zeros((T, 0, 2), device="cuda")
    caches = [c.clone() for c in held.args[:2]]
    chunks = max(k.kv4_decode_chunks(p[:3], 0) for p in pos_host)
    work, tiles = i32([0] * 64), None
    partial = torch.zeros(k.kv4_decode_workspace(3, nh, dim, chunks), device="cuda")
    lists = [k.kv4_prefill_tiles([(3, n, p[3])], 0, nh, nkv) for p in pos_host]
    rows = max(len(t) for t in lists)
    lists = [t + [(0, 0, -1, -1, 0)] * (rows - len(t)) for t in lists]
    tiles = i32(lists[0])
    state = torch.zeros(max(k.kv4_prefill_workspace(t, nh, dim) for t in lists), device="cuda")
    out = torch.zeros((T, nh * dim), dtype=qkv.dtype, device="cuda")
    back = [torch.zeros((T, nkv, dim), dtype=qkv.dtype, device="cuda") for _ in range(2)]

    def layer():
        q = qkv[:, :nh * dim]
        k.rope_kv4_write(qkv, q, rope, pos, seq, table, *caches, nh, nkv, dim, 0, page)
        k.kv4_attention_prefill(q, qkv.stride(0), *caches, table, pos, seq, out, tiles, state, nh, nkv, dim, page, 0, scale)
        k.kv4_attention_decode(q, qkv.stride(0), *caches, table, pos, seq, out, 3, partial, chunks, nh, nkv, dim, page, 0, scale, work=work)
        k.kv4_read(*caches, table, pos, seq, *back, nkv, dim, page)

    def contents(i):
        x = torch.randn(qkv.shape, generator=g).to(qkv.dtype)
        qkv.copy_(x)
        pos.copy_(i32(pos_host[i]))
        tiles.copy_(i32(lists[i]))
        items = k.kv4_decode_work(pos_host[i][:3], 0)
        work.copy_(i32(items + [-1] * (64 - len(items))))

    contents(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for i in (0, 1, 2, 1):
        contents(i)
        for c, h in zip(caches, held.args):
            c.copy_(h)
        layer()
        want = [t.clone() for t in (out, *back, *caches)]
        for c, h in zip(caches, held.args):
            c.copy_(h)
        out.fill_(3.0)
        partial.fill_(float("nan"))
        state.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip((out, *back, *caches), want):
            assert torch.equal(got, w)


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_streams_side_by_side(dtype):
    """Two calls of each kernel at once, on streams of their own with workspaces of their own: the bits of one after the other."""
    k, nh, nkv, dim, page = kernels(dtype), 4, 2, 64, 32
    held = [Held([3000, 90], nkv, dim, page, seed=s) for s in (30, 31)]
    q = torch.randn((60, nh * dim), generator=torch.Generator().manual_seed(1)).to(TORCH[dtype]).cuda()
    pos, seq = [2999, 89] * 30, [0, 1] * 30

    def both(h):
        single = decode(k, h, q, pos, seq, nh, nkv, dim, page, 0, 0.1)
        return single, prefill(k, h, q, [(40, 2960), (20, 70)], [0, 1], nh, nkv, dim, page, 0, 0.1)[2]
    want = [both(h) for h in held]
    streams, got = [torch.cuda.Stream() for _ in held], []
    torch.cuda.synchronize()
    for s, h in zip(streams, held):
        with torch.cuda.stream(s):
            got.append(both(h))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("last,nh,nkv,dim,window", [([8191, 8192, 8300], 4, 1, 64, 0), ([16383, 16384, 17000], 2, 1, 128, 0),
                                                    ([20000], 18, 1, 64, 9000), ([33000], 2, 2, 64, 0)])
def test_decode_of_long_contexts(dtype, last, nh, nkv, dim, window):
    """Where the chunks' size changes, and chunks that a window begins inside."""
    k, held = kernels(dtype), Held([p + 1 for p in last], nkv, dim, 64, seed=40)
    q = torch.randn((len(last), nh * dim), generator=torch.Generator().manual_seed(4)).to(TORCH[dtype]).cuda()
    seq = list(range(len(last)))
    got = decode(k, held, q, last, seq, nh, nkv, dim, 64, window, 0.1)
    check(dtype, got, q, held, last, seq, window, 0.1, dim, nh)


def test_more_work_items_than_a_grid_has_rows():
    """A list of more than 65,535 items, most of them padding or of tokens that see little."""
    k, nh, nkv, dim, page = kernels("bfloat16"), 1, 1, 64, 8
    held = Held([40], nkv, dim, page, seed=50)
    T = 66000
    q = torch.randn((T, dim), generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    pos = [i % 40 for i in range(T)]
    got = decode(k, held, q, pos, [0] * T, nh, nkv, dim, page, 0, 0.1)
    some = [0, 39, 65534, 65535, 65536, T - 1]
    check("bfloat16", got[some], q[some], held, [pos[i] for i in some], [0] * len(some), 0, 0.1, dim, nh)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_positions_do_not_reach_a_row(dtype):
    """Positions behind a token, before its window and in a page's unused slots hold NaN: nothing of them is seen."""
    k, nh, nkv, dim, page = kernels(dtype), 4, 2, 128, 64
    held = Held([400], nkv, dim, page, seed=60)
    q = torch.randn((50, nh * dim), generator=torch.Generator().manual_seed(4)).to(TORCH[dtype]).cuda()
    for window, at in ((0, 70), (33, 201)):
        pos, seq = list(range(at, at + 50)), [0] * 50
        want = [prefill(k, held, q, [(50, at)], [0], nh, nkv, dim, page, window, 0.1)[2], decode(k, held, q, pos, seq, nh, nkv, dim, page, window, 0.1)]
        nan = Held([400], nkv, dim, page, seed=60)
        for cache in nan.args[:2]:
            scales = cache.view(-1, nkv, page * P.row_bytes(dim))[..., page * dim // 2:].view(torch.int16)
            keys = cache is nan.args[0]
            for p in list(range(at + 50, 400)) + list(range(0, max(0, at + 1 - window) if window else 0)):
                row = scales[int(nan.table[0, p // page])]
                if keys:
                    row.view(nkv, page, dim // 32)[:, p % page] = 0x7FE0
                else:
                    row.view(nkv, page // 8, dim // 32, 8)[:, p % page // 8, :, p % 8] = 0x7FE0
        assert torch.equal(prefill(k, nan, q, [(50, at)], [0], nh, nkv, dim, page, window, 0.1)[2], want[0])
        # each token's own mask: the last ones of the portion are behind the first
        assert torch.equal(decode(k, nan, q, pos, seq, nh, nkv, dim, page, window, 0.1), want[1])
        assert all(w.isfinite().all() for w in want)


def test_refusals_of_write_and_read():
    k, nh, nkv, dim, page = kernels("bfloat16"), 4, 2, 64, 8
    keys, values = empty_caches(4, nkv, page, dim)
    qkv = torch.zeros((3, (nh + 2 * nkv) * dim), dtype=torch.bfloat16, device="cuda")
    step = dict(positions=i32([0, 1, -1]), seq_rows=i32([0, 0, 0]), block_table=i32([[1]]), k_cache=keys, v_cache=values, n_kv_heads=nkv,
                head_dim=dim, page_size=page)
    write = dict(qkv=qkv, q_out=qkv[:, :nh * dim], table=torch.zeros((3, 16, 2), device="cuda"), n_heads=nh, rotary_dim=32, **step)
    rows = [torch.zeros((3, nkv, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    read = dict(k_out=rows[0], v_out=rows[1], **step)
    k.rope_kv4_write(**write)
    k.kv4_read(**read)
    both = [dict(positions=i32([0, 1])), dict(seq_rows=i32([[0, 0, 0]])), dict(block_table=i32([1])), dict(k_cache=keys[:, :1]),
            dict(v_cache=values[:2]), dict(k_cache=keys.cpu()), dict(k_cache=keys.to(torch.int8)), dict(head_dim=128), dict(page_size=16),
            dict(n_kv_heads=1), dict(positions=torch.zeros(3, device="cuda")), dict(positions=i32([0, 1, -1]).cpu()),
            dict(seq_rows=torch.zeros(3, dtype=torch.int64, device="cuda")), dict(k_cache=keys.transpose(0, 1).contiguous().transpose(0, 1))]
    for wrong in both + [dict(qkv=qkv[:, :-8]), dict(qkv=qkv.float()), dict(q_out=qkv[:, :nh * dim - 8]), dict(rotary_dim=64), dict(rotary_dim=8),
                         dict(table=torch.zeros((3, 16, 2), dtype=torch.float16, device="cuda")), dict(qkv=qkv[:2]), dict(qkv=qkv.t().contiguous().t()),
                         dict(n_heads=nh + 1), dict(qkv=qkv.cpu())]:
        with pytest.raises(KernelError):
            k.rope_kv4_write(**{**write, **wrong})
    for wrong in both + [dict(k_out=rows[0][:2]), dict(v_out=rows[1].float()), dict(k_out=rows[0].cpu()), dict(v_out=rows[1].transpose(0, 1))]:
        with pytest.raises(KernelError):
            k.kv4_read(**{**read, **wrong})
    # nothing to do
    none = dict(positions=i32([]).reshape(0), seq_rows=i32([]).reshape(0))
    k.kv4_read(**{**read, **none, "k_out": rows[0][:0], "v_out": rows[1][:0]})
    k.rope_kv4_write(**{**write, **none, "qkv": qkv[:0], "q_out": qkv[:0, :nh * dim], "table": torch.zeros((0, 16, 2), device="cuda")})


@pytest.mark.parametrize("dim,nh,nkv,spans,window", [(128, 7, 1, [(300, 5), (130, 0), (77, 1000)], 0), (64, 4, 2, [(257, 700), (64, 64)], 130),
                                                     (128, 3, 1, [(128, 1990), (200, 4000)], 2500)])
def test_one_and_two_heads_a_workgroup_give_the_same_bits(dim, nh, nkv, spans, window):
    """With windows, segments and groups that are not numbers in the middle, at the edges of what is seen and beyond: rows of nothing make the
    step one of many tiles."""
    k, page = kernels("bfloat16"), 32
    held = Held([n + at for n, at in spans], nkv, dim, page, seed=80)
    rng = np.random.default_rng(4)
    for cache, keys in ((held.args[0], True), (held.args[1], False)):
        scales = cache.view(-1, nkv, page * P.row_bytes(dim))[..., page * dim // 2:].view(torch.int16)
        for r, (n, at) in enumerate(spans):
            for p in rng.integers(0, n + at, 3):
                row = scales[int(held.table[r, p // page])]
                if keys and p > at + n // 2:                            # (late keys: else every row is NaN throughout)
                    row.view(nkv, page, dim // 32)[0, p % page, 1] = 0x7FE0
                elif not keys:
                    row.view(nkv, page // 8, dim // 32, 8)[nkv - 1, p % page // 8, 0, p % 8] = 0x7FE0
    T = sum(n for n, _ in spans)
    pos = [at + i for n, at in spans for i in range(n)]
    seq = [r for r, (n, _) in enumerate(spans) for _ in range(n)]
    firsts = np.cumsum([0] + [n for n, _ in spans])[:-1]
    q = torch.randn((T, nh * dim), generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    cut = k.kv4_prefill_tiles([(int(f), n, at) for f, (n, at) in zip(firsts, spans)], window, nh, nkv)
    whole = [(int(f) + i, min(128, n - i), -1, -1) for f, (n, _) in zip(firsts, spans) for i in range(0, n, 128)]
    whole = [(a, b, c, i) for i, (a, b, c, _) in enumerate(whole)]
    few = len(cut) * nh, len(whole) * nh
    assert max(few) <= 768
    nothing = [(0, 0, -1, -1)] * (769 // nh + 1)
    want = None
    for tiles in (cut, cut + [row + (0,) * (len(cut[0]) - 4) for row in nothing], whole, nothing + whole):
        out = torch.full((T, nh * dim), 5.0, dtype=q.dtype, device="cuda")
        partial = torch.full((k.kv4_prefill_workspace(tiles, nh, dim),), float("nan"), device="cuda")
        k.kv4_attention_prefill(q, nh * dim, *held.args, i32(pos), i32(seq), out, i32(tiles), partial, nh, nkv, dim, page, window, 0.1)
        want = out if want is None else want
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))
    assert want.isnan().any() and want.isfinite().any() and not (want == 5.0).all(-1).any()
    single = decode(k, held, q, pos, seq, nh, nkv, dim, page, window, 0.1)
    assert torch.equal(single.isnan(), want.isnan())


def test_places_beyond_32_bits():
    """Pages that begin beyond 4 GiB of a cache: written, read back and attended to as the same positions in the first pages are."""
    k, nh, nkv, dim, page = kernels("bfloat16"), 8, 8, 128, 1024
    n_pages = (9 << 29) // (nkv * page * P.row_bytes(dim)) + 3
    assert (n_pages - 2) * nkv * page * P.row_bytes(dim) > 1 << 32
    caches = [torch.empty((n_pages, nkv, page, P.row_bytes(dim)), dtype=torch.uint8, device="cuda") for _ in range(2)]
    for c in caches:
        c[:2] = c[-2:] = 255                                         # (nothing else is looked at)
    n = 1100
    x = torch.from_numpy(random_rows(np.random.default_rng(1), n, nh + 2 * nkv, dim).reshape(n, -1)).bfloat16().cuda()
    angles = torch.randn((n, 32, 2), generator=torch.Generator().manual_seed(2)).cuda()
    pos, seq = list(range(n)), [0] * n
    got = []
    for table in (i32([[1, 0]]), i32([[n_pages - 1, n_pages - 2]])):
        q = torch.empty((n, nh * dim), dtype=x.dtype, device="cuda")
        k.rope_kv4_write(x, q, angles, i32(pos), i32(seq), table, *caches, nh, nkv, dim, 64, page)

        class Held:
            args = (*caches, table)
        back = [torch.empty((n, nkv, dim), dtype=x.dtype, device="cuda") for _ in range(2)]
        k.kv4_read(*caches, table, i32(pos), i32(seq), *back, nkv, dim, page)
        some = [1, 700, 1023, 1024, 1099]
        got.append([q, *back, prefill(k, Held, q, [(n, 0)], [0], nh, nkv, dim, page, 0, 0.05)[2],
                    decode(k, Held, q[some].contiguous(), some, [0] * 5, nh, nkv, dim, page, 0, 0.05)])
    for low, high in zip(*got):
        assert torch.equal(low.view(torch.int16), high.view(torch.int16)) and low.isfinite().all()
