"""Attention over the 4-bit cache where scores are very large or nothing at all: both kernels, one chunk and several, one segment and
several.

Behind a gap of 64 or more (natural logarithms, beyond twice what 32 bits can lose of a score: test_kv4_gpu.py's (dim + 8) 2^-24 of
sum |q k| scale and 2^-39 of max |q| sum |k| scale) between the largest score and the next, all other weights together are below
n e^-64 < 2^-80, and the output is the largest's value: off by the output's rounding, the weight's own (2^-11 in half precision, 2^-24 as three
terms), the exponential's 2^-20 and the sums' 2 (64 + blocks) 2^-24.  Everywhere else test_kv4_gpu.py's bound holds."""
import numpy as np
import pytest
import torch

from axon_amd.kernels import kernels
from gpu_helpers import DTYPES, TORCH
from plain import kv4_plain as P
from test_kv4_gpu import Held, check, decode, prefill

pytestmark = pytest.mark.gpu


def check_sharp(dtype, got, q, held, pos, window, scale, dim, nh):
    """The rows of request 0 whose largest score is that far ahead; how many (row, head) there were."""
    weights, eps, sharp = 2.0 ** -11 if dtype == "bfloat16" else 2.0 ** -24, 2.0 ** -24, 0
    k, v = held.k[0], held.v[0]
    group = nh // k.shape[1]
    for t, p in enumerate(pos):
        lo = max(0, p + 1 - window) if window else 0
        for h in range(nh):
            row = q[t].double().cpu().numpy().reshape(nh, dim)[h]
            keys, values = k[lo:p + 1, h // group], v[lo:p + 1, h // group]
            s = keys @ row * scale
            lost = (dim + 8) * eps * (np.abs(keys) @ np.abs(row)).max() * scale + 2.0 ** -39 * np.abs(row).max() * np.abs(keys).sum(-1).max() * scale
            top = s.max()
            others = s[s < top]
            if others.size and top - others.max() < 64 + 2 * lost:
                continue
            sharp += 1
            want = values[s == top].mean(0)
            rel = weights + 2.0 ** -20 + 2 * (64 + p / 64) * eps
            bound = torch.finfo(TORCH[dtype]).eps / 2 * np.abs(want) + rel * np.abs(values[s == top]).mean(0) + 2.0 ** -80 * np.abs(values).max() + 1e-30
            off = np.abs(got[t].double().cpu().numpy().reshape(nh, dim)[h] - want)
            assert (off <= bound).all(), (t, p, h, float((off / bound).max()))
    return sharp


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,at,window,same", [(128, 30, 0, False), (128, 2250, 0, False), (64, 1000, 0, True), (64, 2200, 1500, False)])
def test_scores_of_any_size(dtype, dim, at, window, same):
    """Queries from 2^-60 to 2^60 times the ordinary ones, the largest score positive or negative (position 0 alone); `same`: every page is one page,
    so that each block has the largest score again."""
    nh, nkv, page, n = 4, 2, 16, 40
    k, held = kernels(dtype), Held([at + n], nkv, dim, page, seed=90)
    if same:
        first = int(held.table[0, 0])
        held.table[0] = first
        held.args = (*held.args[:2], torch.from_numpy(held.table).cuda())
        held.k, held.v = ([np.concatenate([x[0][:page]] * (-(-(at + n) // page)))[:at + n]] for x in (held.k, held.v))
    q = torch.randn((n, nh * dim), generator=torch.Generator().manual_seed(7))
    power = torch.tensor([-60, -14, 0, 3, 5, 8, 10, 12, 15, 20, 22, 25, 28, 30, 34, 40, 47, 50, 56, 60] * 2)
    q = (q * torch.exp2(power.float())[:, None]).to(TORCH[dtype]).cuda()
    pos, seq, rows = prefill(k, held, q, [(n, at)], [0], nh, nkv, dim, page, window, 0.09)
    check(dtype, rows, q, held, pos, seq, window, 0.09, dim, nh)
    assert check_sharp(dtype, rows, q, held, pos, window, 0.09, dim, nh) >= 40
    single = decode(k, held, q, pos, seq, nh, nkv, dim, page, window, 0.09)
    check(dtype, single, q, held, pos, seq, window, 0.09, dim, nh)
    assert check_sharp(dtype, single, q, held, pos, window, 0.09, dim, nh) >= 40
    # the first position alone, whose score is of either sign: its value
    early = decode(k, held, q, [0] * n, seq, nh, nkv, dim, page, window, 0.09)
    assert check_sharp(dtype, early, q, held, [0] * n, window, 0.09, dim, nh) == n * nh


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.09, 2.0 ** -100])
@pytest.mark.parametrize("dim,at,window", [(128, 70, 0), (64, 1100, 90)])
def test_queries_next_to_nothing(dtype, scale, dim, at, window):
    """Rows of the smallest numbers there are: every position seen has the same weight, and none that is not."""
    nh, nkv, page, n = 4, 2, 16, 12
    k, held = kernels(dtype), Held([at + n], nkv, dim, page, seed=91)
    smallest = torch.finfo(TORCH[dtype]).smallest_normal * torch.finfo(TORCH[dtype]).eps
    sign = torch.randn((n, nh * dim), generator=torch.Generator().manual_seed(8)).sign().double()
    q = (sign * smallest * torch.exp2(torch.arange(n).double() * 3)[:, None]).to(TORCH[dtype]).cuda()
    assert (q != 0).all()
    pos, seq, rows = prefill(k, held, q, [(n, at)], [0], nh, nkv, dim, page, window, scale)
    check(dtype, rows, q, held, pos, seq, window, scale, dim, nh)
    check(dtype, decode(k, held, q, pos, seq, nh, nkv, dim, page, window, scale), q, held, pos, seq, window, scale, dim, nh)
