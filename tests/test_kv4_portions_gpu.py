"""What the 4-bit cache's write stores of steps that its blocks take several tokens at a time: more than 1,024 (eight a block) and more than
4,096 (sixteen), byte for byte against the format, with portions that begin and end inside octets, runs across blocks, several runs of a block and
padding between them."""
import numpy as np
import pytest
import torch

from axon_amd.kernels import kernels
from gpu_helpers import DTYPES, TORCH
from plain import kv4_plain as P
from test_kv4_gpu import i32, random_rows, rotated, step_of

pytestmark = pytest.mark.gpu


def whole_pages(x, pos, seq, table, n_pages, page, fill):
    """The caches' bytes: keys and values [T, heads, dim] at the tokens' places.  Slots of no token keep `fill`, part words bit by bit."""
    caches = []
    for name, rows in zip("kv", x):
        heads, dim = rows.shape[1:]
        held = np.zeros((n_pages, heads, page, dim), dtype=np.float32)
        used = np.zeros((n_pages, page), dtype=bool)
        at = [(table[r, p // page], p % page) for p, r in zip(pos, seq) if p >= 0]
        there = [t for t, p in enumerate(pos) if p >= 0]
        pages, slots = (np.array(v) for v in zip(*at))
        held[pages, :, slots] = rows[there]
        used[pages, slots] = True
        want = P.pages_of(held, page, dim, name == "k")
        # which bits are a token's: those that numbers of fifteen, and scales of all ones, set
        bits = np.zeros((n_pages, heads, page * P.row_bytes(dim)), dtype=np.uint8)
        words = bits[..., :page * dim // 2].view("<u4")
        scales = bits[..., page * dim // 2:].view("<u2")
        if name == "k":
            words.reshape(n_pages, heads, page, dim // 8)[used[:, None].repeat(heads, 1)] = 0xFFFFFFFF
            scales.reshape(n_pages, heads, page, dim // 32)[used[:, None].repeat(heads, 1)] = 0xFFFF
        else:
            mask = np.zeros((n_pages, page // 8), dtype=np.uint32)
            for e in range(8):
                mask |= np.where(used.reshape(n_pages, -1, 8)[..., e], np.uint32(15 << P.place(e) & 0xFFFFFFFF | 15 >> (32 - P.place(e))), np.uint32(0))
            words.reshape(n_pages, heads, page // 8, dim)[:] = mask[:, None, :, None]
            scales.reshape(n_pages, heads, page // 8, dim // 32, 8)[:] = np.where(used.reshape(n_pages, 1, -1, 1, 8), 0xFFFF, 0)
        bits = bits.reshape(want.shape)
        caches.append((want & bits) | (np.uint8(fill) & ~bits))
    return caches


PORTIONS = [
    # (tokens, first position) a request; page, kv heads, heads, dim, rotated dims
    ([(1025, 0)], 16, 1, 2, 64, 64),                                                  # whole octets, one block behind them
    ([(700, 3), (1, 9), (5, 12), (2, 6), (333, 1021)], 32, 1, 3, 128, 64),            # octets across blocks, short runs in one
    ([(3, 5)] * 200 + [(611, 2)], 8, 2, 2, 64, 16),                                   # several runs a block
    ([(1900, 7), (14, 1)], 64, 2, 14, 64, 64),
    ([(4095, 0), (1, 77), (1, 4)], 128, 1, 1, 64, 32),
    ([(4097, 6)], 1024, 2, 2, 128, 0),
    ([(2100, 1), (1, 4000), (37, 9), (3, 30)] + [(2, 7)] * 900 + [(301, 13)], 16, 1, 2, 64, 64),
]


@pytest.mark.parametrize("spans,page,nkv,nh,dim,rot", PORTIONS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_write_of_many_tokens_is_the_format_byte_for_byte(dtype, spans, page, nkv, nh, dim, rot):
    k, fill = kernels(dtype), 0xAB
    pos, seq, table, n_pages = step_of(spans, page)
    for at in (len(pos) - 3, len(pos) * 2 // 3, 517, 9, 8, 0):                       # padding: before, inside and around blocks' ends
        pos.insert(at, -1)
        seq.insert(at, 0)
    T = len(pos)
    x = random_rows(np.random.default_rng(6), T, nh + 2 * nkv, dim)
    qkv = torch.from_numpy(x.reshape(T, -1)).to(TORCH[dtype]).cuda()
    exact = qkv.float().cpu().numpy().reshape(T, -1, dim)
    angles = np.asarray(pos, dtype=np.float64)[:, None] * 10000.0 ** (-np.arange(rot // 2) * 2.0 / max(rot, 1))
    rope = np.stack([np.sin(angles), np.cos(angles)], axis=-1).astype(np.float32)
    turned = rotated(exact[:, :nh + nkv], pos, rot, rope)
    want = whole_pages((turned[:, nh:], exact[:, nh + nkv:]), pos, seq, table, n_pages, page, fill)
    keys = torch.full((n_pages, nkv, page, P.row_bytes(dim)), fill, dtype=torch.uint8, device="cuda")
    vals = keys.clone()
    q = torch.empty((T, nh * dim), dtype=qkv.dtype, device="cuda")
    k.rope_kv4_write(qkv, q, torch.from_numpy(rope.reshape(T, rot // 2, 2)).cuda(), i32(pos), i32(seq), torch.from_numpy(table).cuda(), keys, vals, nh, nkv,
                     dim, rot, page)
    assert torch.equal(q.cpu(), torch.from_numpy(turned[:, :nh].reshape(T, -1)).to(qkv.dtype))
    assert np.array_equal(keys.cpu().numpy(), want[0])
    assert np.array_equal(vals.cpu().numpy(), want[1])


def test_whole_pages_are_what_slots_stored_one_by_one_give():
    """The oracle above, beside the one that stores a token at a time."""
    spans, page, nkv, dim = [(13, 3), (1, 9), (2, 6)], 16, 2, 64
    pos, seq, table, n_pages = step_of(spans, page)
    pos, seq = pos[:5] + [-1] + pos[5:], seq[:5] + [0] + seq[5:]
    x = random_rows(np.random.default_rng(1), len(pos), 2 * nkv, dim)
    one = P.Cache(n_pages, nkv, page, dim, fill=0xAB)
    for t, (p, r) in enumerate(zip(pos, seq)):
        if p >= 0:
            one.store(table[r, p // page], p % page, x[t, :nkv], x[t, nkv:])
    keys, vals = whole_pages((x[:, :nkv], x[:, nkv:]), pos, seq, table, n_pages, page, 0xAB)
    assert np.array_equal(keys, one.keys) and np.array_equal(vals, one.values)
