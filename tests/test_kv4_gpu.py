"""The cache held in 4 bits against its plain implementation: what is written, what is read back, and the attention over it.

Attention's tolerance, an output o = sum p_j v_j against float64 over the same (exactly held) cache:
* the output's own rounding, eps/2 of |o|;
* the weights' rounding to the matrix cores' operands: bfloat16 build half precision, 2^-11 each, together 2^-11 sum p |v|;
  float32 build three such terms, whose rest is below 2^-24;
* scores in 32 bits: a sum of `dim` products, at most (dim + 8) 2^-24 of sum |q k| scale, which moves a weight by that much of itself,
  weights and their sum both: twice;
* half precision's smallest step is 2^-24.  Weights are 2^7 there at a reference that is no larger than a chunk's largest, so what is lost
  of one below that step is at most 2^-25-7 of the largest, which is at most their sum: 2^-32 sum |v| of an output.  A query's largest number is 2^14 at least there: what is
  lost of the others is at most 2^-39 max |q|, of a score 2^-39 max |q| sum |k| scale;
* the exponential and the multiply-add before it: 2^-20 of a weight;
* sums over positions in 32 bits: blocks of 64, then a fold a block: (64 + blocks) 2^-24 of sum p |v|, numerator and denominator."""
import numpy as np
import pytest
import torch

from axon_amd.kernels import KernelError, kernels
from gpu_helpers import DTYPES, TORCH
from plain import kv4_plain as P

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda").reshape(np.shape(v))


def random_rows(rng, *shape):
    """Rows whose channels differ in size, with groups of one sign, of zeros, tiny and large ones among them."""
    x = rng.standard_normal(shape).astype(np.float32) * np.exp(rng.standard_normal(shape[-1:])).astype(np.float32)
    flat = x.reshape(-1, 32)
    pick = rng.integers(0, 24, len(flat))
    flat[pick == 0] = 0
    flat[pick == 1] = np.abs(flat[pick == 1]) + 1
    flat[pick == 2] *= np.float32(2.0 ** -14)
    flat[pick == 3] *= 300
    flat[pick == 4] = -np.abs(flat[pick == 4])
    return x


class Held:
    """Requests of given lengths in a cache of shuffled pages, and what it holds in float64."""

    def __init__(self, lengths, nkv, dim, page, seed=0, fill=255):
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lengths]
        order = rng.permutation(sum(need) + 2)
        self.table, at = np.zeros((len(lengths), max(need) + 1), dtype=np.int32), 0
        self.keys = np.full((len(order), nkv, page, P.row_bytes(dim)), fill, dtype=np.uint8)
        self.vals = self.keys.copy()
        self.k, self.v = [], []
        for r, n in enumerate(lengths):
            pages = order[at:at + need[r]]
            at += need[r]
            self.table[r, :need[r]] = pages
            rows = [random_rows(rng, n, nkv, dim) for _ in range(2)]
            for held, cache, x, keys in ((self.k, self.keys, rows[0], True), (self.v, self.vals, rows[1], False)):
                padded = np.full((need[r] * page, nkv, dim), np.nan, dtype=np.float32)       # unwritten slots: scales that are NaN
                padded[:n] = x
                cache[pages] = P.pages_of(np.ascontiguousarray(padded.reshape(need[r], page, nkv, dim).swapaxes(1, 2)), page, dim, keys)
                numbers, words = P.quantise(x)
                held.append(P.values(numbers, words))
        self.args = (torch.from_numpy(self.keys).cuda(), torch.from_numpy(self.vals).cuda(), torch.from_numpy(self.table).cuda())


# ---------------------------------------------------------------------------- write, read

STEPS = [
    # (tokens, first position) a request; page; kv heads; heads; dim; rotated dims
    ([(1, 0)], 8, 1, 1, 64, 64),
    ([(1, 9), (1, 16), (1, 31)], 16, 2, 6, 128, 128),
    ([(37, 0), (1, 5), (13, 27), (8, 8)], 8, 3, 3, 64, 32),
    ([(130, 61)], 64, 2, 14, 128, 64),
    ([(19, 1021), (3, 7)], 1024, 1, 7, 128, 0),
]


def step_of(spans, page, seed=1):
    rng = np.random.default_rng(seed)
    need = [-(-(n + at) // page) for n, at in spans]
    order = rng.permutation(sum(need) + 2)
    table, first = np.zeros((len(spans), max(need)), dtype=np.int32), 0
    pos, rows = [], []
    for r, (n, at) in enumerate(spans):
        table[r, :need[r]] = order[first:first + need[r]]
        first += need[r]
        pos += range(at, at + n)
        rows += [r] * n
    return pos, rows, table, len(order)


def rotated(x, pos, rot, table):
    """Rotate-half in the kernel's 32-bit steps: x float32 [T, heads, dim]."""
    y, half = x.copy(), rot // 2
    s, c = table[:, None, :, 0], table[:, None, :, 1]
    y[..., :half] = x[..., :half] * c - x[..., half:rot] * s
    y[..., half:rot] = x[..., :half] * s + x[..., half:rot] * c
    return y


def write_case(dtype, spans, page, nkv, nh, dim, rot, seed=3, pad=0, rows=None):
    pos, seq, table, n_pages = step_of(spans, page)
    pos, seq = pos + [-1] * pad, seq + [0] * pad
    T, rng = len(pos), np.random.default_rng(seed)
    x = random_rows(rng, T, nh + 2 * nkv, dim) if rows is None else rows
    qkv = torch.from_numpy(x.reshape(T, -1)).to(TORCH[dtype]).cuda()
    angles = np.asarray(pos, dtype=np.float64)[:, None] * 10000.0 ** (-np.arange(rot // 2) * 2.0 / max(rot, 1))
    rope = np.stack([np.sin(angles), np.cos(angles)], axis=-1).astype(np.float32)
    keys = torch.full((n_pages, nkv, page, P.row_bytes(dim)), 0xAB, dtype=torch.uint8, device="cuda")
    vals = keys.clone()
    want = P.Cache(n_pages, nkv, page, dim, fill=0xAB)
    exact = qkv.float().cpu().numpy().reshape(T, nh + 2 * nkv, dim)
    turned = rotated(exact[:, :nh + nkv], pos, rot, rope)
    for t in range(T):
        if pos[t] >= 0:
            want.store(table[seq[t], pos[t] // page], pos[t] % page, turned[t, nh:], exact[t, nh + nkv:])
    step = (torch.from_numpy(rope.reshape(T, rot // 2, 2)).cuda(), i32(pos), i32(seq), torch.from_numpy(table).cuda(), keys, vals)
    return qkv, step, want, turned[:, :nh], exact


@pytest.mark.parametrize("spans,page,nkv,nh,dim,rot", STEPS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_write_is_the_format_byte_for_byte(dtype, spans, page, nkv, nh, dim, rot):
    k = kernels(dtype)
    qkv, step, want, q, _ = write_case(dtype, spans, page, nkv, nh, dim, rot, pad=2)
    out = torch.empty((qkv.shape[0], nh * dim), dtype=qkv.dtype, device="cuda")
    before = qkv.clone()
    k.rope_kv4_write(qkv, out, *step, nh, nkv, dim, rot, page)
    assert torch.equal(qkv, before)
    assert np.array_equal(step[4].cpu().numpy(), want.keys)
    assert np.array_equal(step[5].cpu().numpy(), want.values)
    expect = torch.from_numpy(q.reshape(q.shape[0], -1)).to(qkv.dtype)
    assert torch.equal(out.cpu(), expect)
    # in place, rows that lie apart, queries alone
    wide = torch.zeros((qkv.shape[0], qkv.shape[1] + 16), dtype=qkv.dtype, device="cuda")
    wide[:, :qkv.shape[1]] = before
    k.rope_kv4_write(wide, wide[:, :nh * dim], *step, nh, nkv, dim, rot, page, write_kv=False)
    assert torch.equal(wide[:, :nh * dim].cpu(), expect)
    assert torch.equal(wide[:, nh * dim:qkv.shape[1]], before[:, nh * dim:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_held_is_near_what_was_given(dtype):
    """|x - held| <= s / 2 (1 + 2^-20): the division's rounding moves a tie by no more."""
    k, dim, page, nkv, nh = kernels(dtype), 128, 16, 2, 2
    spans = [(50, 3), (1, 0)]
    qkv, step, _, _, exact = write_case(dtype, spans, page, nkv, nh, dim, 0)
    k.rope_kv4_write(qkv, qkv[:, :nh * dim], *step, nh, nkv, dim, 0, page)
    held = [torch.empty((51, nkv, dim), dtype=TORCH[dtype], device="cuda") for _ in range(2)]
    k.kv4_read(*step[4:], step[3], step[1], step[2], *held, nkv, dim, page)
    for got, x in zip(held, (exact[:, nh:nh + nkv], exact[:, nh + nkv:])):
        n, words = P.quantise(x)
        expect = torch.from_numpy(P.values(n, words)).to(TORCH[dtype])      # each number rounded once
        assert torch.equal(got.cpu(), expect)
        s = np.repeat((words & 0x7FE0).astype(np.uint16).view(np.float16).astype(np.float64), 32, axis=-1)
        assert (np.abs(P.values(n, words) - x) <= s / 2 * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_numbers_that_are_not_finite_and_too_large(dtype):
    """A group with one is NaN throughout, its neighbours are untouched; a range too wide saturates."""
    k, dim, page, nkv, nh = kernels(dtype), 64, 8, 1, 1
    x = random_rows(np.random.default_rng(0), 3, nh + 2 * nkv, dim)
    x[0, 1, 5], x[1, 2, 40], x[2, 1, 33] = np.nan, np.inf, -np.inf
    x[2, 2, :32] = np.linspace(-60000, 60000, 32)
    qkv, step, want, _, exact = write_case(dtype, [(3, 6)], page, nkv, nh, dim, 0, rows=x)
    k.rope_kv4_write(qkv, qkv[:, :dim], *step, nh, nkv, dim, 0, page)
    assert np.array_equal(step[4].cpu().numpy(), want.keys) and np.array_equal(step[5].cpu().numpy(), want.values)
    held = [torch.empty((3, 1, dim), dtype=TORCH[dtype], device="cuda") for _ in range(2)]
    k.kv4_read(*step[4:], step[3], step[1], step[2], *held, nkv, dim, page)
    keys, values = (h.float().cpu()[:, 0] for h in held)
    assert keys[0, :32].isnan().all() and keys[0, 32:].isfinite().all()
    assert values[1, 32:].isnan().all() and values[1, :32].isfinite().all()
    assert keys[2, 32:].isnan().all() and values[2].isfinite().all() and float(values[2, :32].abs().max()) >= 16000


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_of_one_octet_that_lie_apart_in_a_step(dtype):
    """Three requests' positions in turn: no token undoes what a neighbour of its octet stored."""
    k, dim, page, nkv, nh = kernels(dtype), 128, 16, 2, 2
    pos = [8, 3, 0, 9, 5, 1, 10, 4, 15, 11, 6, 2]
    seq = [0, 1, 2] * 4
    rng = np.random.default_rng(5)
    table = np.array([[3], [0], [4]], dtype=np.int32)
    x = random_rows(rng, 12, nh + 2 * nkv, dim)
    qkv = torch.from_numpy(x.reshape(12, -1)).to(TORCH[dtype]).cuda()
    want = P.Cache(5, nkv, page, dim, fill=0)
    exact = qkv.float().cpu().numpy().reshape(12, -1, dim)
    for t in range(12):
        want.store(table[seq[t], 0], pos[t], exact[t, nh:nh + nkv], exact[t, nh + nkv:])
    caches = [torch.zeros((5, nkv, page, P.row_bytes(dim)), dtype=torch.uint8, device="cuda") for _ in range(2)]
    rope = torch.zeros((12, 0, 2), device="cuda")
    k.rope_kv4_write(qkv, qkv[:, :nh * dim], rope, i32(pos), i32(seq), torch.from_numpy(table).cuda(), *caches, nh, nkv, dim, 0, page)
    assert np.array_equal(caches[0].cpu().numpy(), want.keys) and np.array_equal(caches[1].cpu().numpy(), want.values)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,page,nkv,dim", [([1], 8, 1, 64), ([130, 7, 64], 16, 3, 128), ([1025], 1024, 2, 64)])
def test_read_rows_in_any_order(dtype, lengths, page, nkv, dim):
    k, held = kernels(dtype), Held(lengths, nkv, dim, page, seed=2)
    rng = np.random.default_rng(3)
    rows = [(r, p) for r, n in enumerate(lengths) for p in range(n)]
    shuffled = [rows[i] for i in rng.integers(0, len(rows), 40)] + rows[-9:] + [(0, -1)]       # any order, some twice, padding
    for order in (rows, shuffled):
        pos, seq = i32([p for _, p in order]), i32([r for r, _ in order])
        got = [torch.full((len(order), nkv, dim), 7.0, dtype=TORCH[dtype], device="cuda") for _ in range(2)]
        k.kv4_read(*held.args, pos, seq, *got, nkv, dim, page)
        for g, of in zip(got, (held.k, held.v)):
            want = np.stack([of[r][p] if p >= 0 else np.zeros((nkv, dim)) for r, p in order])
            assert torch.equal(g.cpu(), torch.from_numpy(want).to(TORCH[dtype]))


# ---------------------------------------------------------------------------- attention

def tolerance(dtype, want, weight, score, size, spread, dim, positions):
    eps = 2.0 ** -24
    weights = 2.0 ** -11 if dtype == "bfloat16" else 2.0 ** -24
    rel = weights + 2 * ((dim + 8) * eps * score + 2.0 ** -39 * spread) + 2.0 ** -20 + 2 * (64 + positions / 64) * eps
    return torch.finfo(TORCH[dtype]).eps / 2 * np.abs(want) + rel * weight + 2.0 ** -32 * size + 1e-30


def check(dtype, got, q, held, pos, seq, window, scale, dim, nh):
    for t in range(len(pos)):
        want, *sizes = P.attention(q[t].double().cpu().numpy().reshape(nh, dim), held.k[seq[t]], held.v[seq[t]], pos[t], window, scale)
        off = np.abs(got[t].double().cpu().numpy().reshape(nh, dim) - want)
        bound = tolerance(dtype, want, *sizes, dim, pos[t] + 1)
        assert (off <= bound).all(), (t, pos[t], float((off / bound).max()))


def decode(k, held, q, pos, seq, nh, nkv, dim, page, window, scale, token_index=None, out=None, pad_work=0):
    T = len(pos)
    named = pos if token_index is None else [pos[i] for i in token_index]
    chunks = k.kv4_decode_chunks(named, window)
    work = k.kv4_decode_work(named, window) + [-1] * pad_work
    partial = torch.full((max(1, k.kv4_decode_workspace(len(named), nh, dim, chunks)),), float("nan"), device="cuda")
    out = torch.full((T, nh * dim), 5.0, dtype=q.dtype, device="cuda") if out is None else out
    index = T if token_index is None else i32(token_index)
    return k.kv4_attention_decode(q, q.stride(0), *held.args, i32(pos), i32(seq), out, index, partial, chunks, nh, nkv, dim, page, window,
                                  scale, work=i32(work))


DECODES = [
    # last positions of the requests; heads, kv heads, dim, page, window
    ([0], 1, 1, 64, 8, 0),
    ([0, 7, 8, 62, 63, 64], 4, 2, 64, 8, 0),
    ([127, 255, 256, 257, 300], 7, 1, 128, 16, 0),
    ([700, 1023, 1024, 31], 14, 2, 128, 64, 0),
    ([2113, 5], 28, 4, 128, 16, 0),
    ([600, 40, 299], 6, 3, 64, 32, 37),
    ([511, 1300], 8, 8, 128, 256, 256),
    ([900, 64], 16, 2, 64, 1024, 1),
    ([333], 40, 2, 128, 32, 0),
    ([100, 1500], 71, 1, 64, 64, 513),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("last,nh,nkv,dim,page,window", DECODES)
def test_decode(dtype, last, nh, nkv, dim, page, window):
    k, held = kernels(dtype), Held([p + 1 for p in last], nkv, dim, page, seed=len(last) + dim)
    g = torch.Generator().manual_seed(1)
    pos, seq = last + [-1], list(range(len(last))) + [0]
    q = torch.randn((len(pos), nh * dim + 32), generator=g).to(TORCH[dtype]).cuda()
    got = decode(k, held, q, pos, seq, nh, nkv, dim, page, window, dim ** -0.5, pad_work=3)
    check(dtype, got, q[:, :nh * dim], held, pos, seq, window, dim ** -0.5, dim, nh)
    assert not got[-1].any()
    # a token's bits do not depend on what else is in the step
    for t in range(len(last)):
        alone = decode(k, held, q[t:t + 1], [pos[t]], [seq[t]], nh, nkv, dim, page, window, dim ** -0.5)
        assert torch.equal(alone[0], got[t])


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_of_named_tokens(dtype):
    """Only the rows that are named are written, in any order."""
    nh, nkv, dim, page = 6, 2, 128, 16
    k, held = kernels(dtype), Held([400, 31, 66], nkv, dim, page, seed=4)
    q = torch.randn((5, nh * dim), generator=torch.Generator().manual_seed(2)).to(TORCH[dtype]).cuda()
    pos, seq = [399, 30, 3, 65, 200], [0, 1, 0, 2, 0]
    got = decode(k, held, q, pos, seq, nh, nkv, dim, page, 0, 0.1, token_index=[4, 1, 3])
    whole = decode(k, held, q, pos, seq, nh, nkv, dim, page, 0, 0.1)
    assert torch.equal(got[[4, 1, 3]], whole[[4, 1, 3]]) and (got[[0, 2]] == 5.0).all()


PROMPTS = [
    # (tokens, first position) a request; heads, kv heads, dim, page, window
    ([(2, 0)], 1, 1, 64, 8, 0),
    ([(63, 0), (64, 0), (65, 0), (3, 61)], 4, 2, 64, 8, 0),
    ([(129, 0), (1, 300), (31, 97)], 7, 1, 128, 16, 0),
    ([(200, 517), (128, 128)], 6, 2, 128, 64, 0),
    ([(300, 5), (40, 0)], 6, 3, 64, 32, 70),
    ([(150, 900)], 3, 3, 128, 1024, 64),
    ([(90, 200), (17, 0)], 9, 1, 64, 128, 1),
]


def prefill(k, held, q, spans, seq_of, nh, nkv, dim, page, window, scale, fill=5.0):
    pos = [at + i for n, at in spans for i in range(n)]
    seq = [seq_of[r] for r, (n, _) in enumerate(spans) for _ in range(n)]
    firsts = np.cumsum([0] + [n for n, _ in spans])[:-1]
    tiles = k.kv4_prefill_tiles([(int(f), n, at) for f, (n, at) in zip(firsts, spans)], window, nh, nkv)
    partial = torch.empty(k.kv4_prefill_workspace(tiles, nh, dim), device="cuda")
    out = torch.full((len(pos), nh * dim), fill, dtype=q.dtype, device="cuda")
    return pos, seq, k.kv4_attention_prefill(q, q.stride(0), *held.args, i32(pos), i32(seq), out, i32(tiles), partial, nh, nkv, dim, page,
                                             window, scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spans,nh,nkv,dim,page,window", PROMPTS)
def test_prefill(dtype, spans, nh, nkv, dim, page, window):
    k, held = kernels(dtype), Held([n + at for n, at in spans], nkv, dim, page, seed=7)
    T = sum(n for n, _ in spans)
    q = torch.randn((T, nh * dim + 16), generator=torch.Generator().manual_seed(1)).to(TORCH[dtype]).cuda()
    pos, seq, got = prefill(k, held, q, spans, range(len(spans)), nh, nkv, dim, page, window, dim ** -0.5)
    check(dtype, got, q[:, :nh * dim], held, pos, seq, window, dim ** -0.5, dim, nh)
    # a row's bits do not depend on the other portions of the step, nor on how its own was cut
    n, at = spans[0]
    cut = max(1, n // 3)
    if cut > 1:
        whole = got[:n]
        parts = [prefill(k, held, q[a:b], [(b - a, at + a)], [0], nh, nkv, dim, page, window, dim ** -0.5)[2] for a, b in ((0, cut), (cut, n))]
        assert torch.equal(torch.cat(parts), whole)


def prefill_by(k, held, q, tiles, pos, seq, nh, nkv, dim, page, window, scale):
    out = torch.full((len(pos), nh * dim), 5.0, dtype=q.dtype, device="cuda")
    partial = torch.full((k.kv4_prefill_workspace(tiles, nh, dim),), float("nan"), device="cuda")
    return k.kv4_attention_prefill(q, q.stride(0), *held.args, i32(pos), i32(seq), out, i32(tiles), partial, nh, nkv, dim, page, window, scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,at,nh,nkv,dim,window", [(70, 8150, 2, 1, 64, 0), (131, 1990, 3, 1, 128, 0), (40, 16390, 2, 2, 128, 9000),
                                                    (3, 2047, 4, 1, 64, 2048)])
def test_tiles_cut_at_segments(dtype, n, at, nh, nkv, dim, window):
    """Positions beyond a segment: the segments side by side and folded, or all by one workgroup: the same bits, and right."""
    k, page, held = kernels(dtype), 32, Held([n + at], nkv, dim, 32, seed=11)
    q = torch.randn((n, nh * dim), generator=torch.Generator().manual_seed(4)).to(TORCH[dtype]).cuda()
    pos, seq = list(range(at, at + n)), [0] * n
    cut = k.kv4_prefill_tiles([(0, n, at)], window, nh, nkv)
    assert sum(row[4] > 1 for row in cut) == -(-n // 128) and len(cut) == sum(row[4] for row in cut)
    got = prefill_by(k, held, q, cut, pos, seq, nh, nkv, dim, page, window, 0.1)
    whole = prefill_by(k, held, q, [(f, min(128, n - f), -1, i) for i, f in enumerate(range(0, n, 128))], pos, seq, nh, nkv, dim, page, window, 0.1)
    assert torch.equal(got, whole)
    some = [0, n // 2, n - 1]
    check(dtype, got[some], q[some], held, [pos[i] for i in some], [0] * 3, window, 0.1, dim, nh)
    # a slot that is not there: nothing is read or written behind the workspace, the tile's rows stay as they were
    empty = torch.empty(0, device="cuda")
    out = torch.full_like(q, 5.0)
    k.kv4_attention_prefill(q, q.stride(0), *held.args, i32(pos), i32(seq), out, i32(cut), empty, nh, nkv, dim, page, window, 0.1)
    assert (out == 5.0).all()


@pytest.mark.parametrize("nh,nkv,dim,portions", [(14, 2, 64, 57), (28, 4, 128, 29), (9, 3, 128, 90), (5, 1, 64, 160)])
def test_two_heads_a_workgroup(nh, nkv, dim, portions):
    """Steps of many tiles: a workgroup has two heads of a key head (an odd group leaves one out); the same bits as few tiles give."""
    k, page = kernels("bfloat16"), 16
    lengths = [(i * 37) % 90 + 2 for i in range(portions)]
    spans = [((i * 13) % n + 1, n - (i * 13) % n - 1) for i, n in enumerate(lengths)]
    held = Held(lengths, nkv, dim, page, seed=12)
    T = sum(n for n, _ in spans)
    q = torch.randn((T, nh * dim), generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    assert portions * nh > 768                       # the launch's rule
    pos, seq, got = prefill(k, held, q, spans, range(portions), nh, nkv, dim, page, 0, 0.1)
    first = 0
    for r, (n, at) in enumerate(spans):
        if r % 7 == 0:
            one = prefill(k, held, q[first:first + n], [(n, at)], [r], nh, nkv, dim, page, 0, 0.1)[2]
            assert torch.equal(one, got[first:first + n])
        first += n
    some = list(range(0, T, max(1, T // 12)))
    check("bfloat16", got[some], q[some], held, [pos[i] for i in some], [seq[i] for i in some], 0, 0.1, dim, nh)
    # longer than a segment
    held = Held([2300], nkv, dim, page, seed=13)
    tiles, n, at = [], 20, 2280
    q = torch.randn((n, nh * dim), generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    pos, seq = list(range(at, at + n)), [0] * n
    alone = prefill_by(k, held, q, [(0, n, -1, 0)], pos, seq, nh, nkv, dim, page, 0, 0.1)
    many = prefill_by(k, held, q, [(0, n, -1, 0)] + [(0, 0, -1, -1)] * (769 // nh + 1), pos, seq, nh, nkv, dim, page, 0, 0.1)
    assert torch.equal(alone, many)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_any_size_and_queries_of_zero(dtype):
    """Queries from 2^-60 to 2^60 times the ordinary, and a query of zeros: the softmax is as sharp as it should be."""
    nh, nkv, dim, page = 4, 2, 128, 16
    k, held = kernels(dtype), Held([200], nkv, dim, page, seed=9)
    q = torch.randn((6, nh * dim), generator=torch.Generator().manual_seed(6))
    q *= torch.tensor([2.0 ** -60, 2.0 ** -14, 1.0, 0.0, 2.0 ** 5, 2.0 ** -130])[:, None]
    q = q.to(TORCH[dtype]).cuda()
    pos, seq = [199, 150, 64, 63, 10, 70], [0] * 6
    got = decode(k, held, q, pos, seq, nh, nkv, dim, page, 0, 0.09)
    check(dtype, got, q, held, pos, seq, 0, 0.09, dim, nh)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_group_that_is_nan_reaches_whom_it_should(dtype):
    """A position whose keys hold a NaN makes the rows that see it NaN, and no others; a value's NaN its own 32 dims of them."""
    nh, nkv, dim, page = 2, 2, 64, 8
    k, held = kernels(dtype), Held([90], nkv, dim, page, seed=10)
    x = np.zeros((1, 64), dtype=np.float32)
    x[0, 40] = np.nan
    _, words = P.quantise(x)
    vals = held.vals[held.table[0, 3], 1].reshape(-1)          # position 29 (slot 5), head 1, group 1
    vals[page * dim // 2 + 2 * ((0 * 2 + 1) * 8 + 5):][:2] = [words[0, 1] & 255, words[0, 1] >> 8]
    keys = held.keys[held.table[0, 9], 0].reshape(-1)          # position 74 (slot 2), head 0, group 1
    keys[page * dim // 2 + 2 * (2 * 2 + 1):][:2] = [words[0, 1] & 255, words[0, 1] >> 8]
    held.args = (torch.from_numpy(held.keys).cuda(), torch.from_numpy(held.vals).cuda(), held.args[2])
    q = torch.randn((90, nh * dim), generator=torch.Generator().manual_seed(1)).to(TORCH[dtype]).cuda()
    pos, seq, rows = prefill(k, held, q, [(90, 0)], [0], nh, nkv, dim, page, 0, 0.125)
    single = decode(k, held, q, pos, seq, nh, nkv, dim, page, 0, 0.125)
    for got in (rows, single):
        nan = got.isnan().view(90, nh, dim).cpu()
        want = torch.zeros((90, nh, dim), dtype=torch.bool)
        want[29:, 1, 32:] = True
        want[74:, 0] = True
        assert torch.equal(nan, want)


# ---------------------------------------------------------------------------- refusals that want a device

def test_refusals():
    k = kernels("bfloat16")
    nh, nkv, dim, page = 4, 2, 64, 8
    held = Held([20], nkv, dim, page)
    q = torch.zeros((1, nh * dim), dtype=torch.bfloat16, device="cuda")
    good = dict(q=q, q_stride=nh * dim, k_cache=held.args[0], v_cache=held.args[1], block_table=held.args[2], positions=i32([3]),
                seq_rows=i32([0]), out=torch.zeros_like(q), token_index=1, partial=torch.zeros(4096, device="cuda"), max_chunks=1, n_heads=nh,
                n_kv_heads=nkv, head_dim=dim, page_size=page, window=0, scale=0.1, work=i32([0]))
    k.kv4_attention_decode(**good)
    for wrong in (dict(head_dim=128), dict(page_size=16), dict(n_kv_heads=3), dict(window=-1), dict(scale=float("nan")), dict(max_chunks=0),
                  dict(max_chunks=2000), dict(k_cache=held.args[0][:, :1]), dict(v_cache=held.args[1].float()), dict(q=q.float()),
                  dict(out=torch.zeros((1, nh * dim), device="cuda")), dict(out=torch.zeros((2, nh * dim), dtype=q.dtype, device="cuda")),
                  dict(positions=i32([3, 4])), dict(token_index=2), dict(work=i32([[0]])), dict(q_stride=nh * dim - 8),
                  dict(positions=torch.tensor([3], device="cuda")), dict(partial=torch.zeros(4, device="cuda")),
                  dict(block_table=held.args[2][0]), dict(q=q.cpu()), dict(v_cache=held.args[1].cpu())):
        with pytest.raises(KernelError):
            k.kv4_attention_decode(**{**good, **wrong})
    with pytest.raises(KernelError):
        k.kv4_decode_chunks([k.kv4_max_context], 0)
    for bad in ([(0, 0, 0)], [(-1, 3, 0)], [(0, 3, -1)]):
        with pytest.raises(KernelError):
            k.kv4_prefill_tiles(bad, 0, nh, nkv)
