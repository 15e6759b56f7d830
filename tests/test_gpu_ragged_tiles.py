"""Ragged decode attention over long requests, with inputs that give every tile of tokens a weight
of its own in the output (GPU): a tile that is lost or taken twice, or a part that is joined with
a wrong weight, moves some element by far more than the bound.

V is one-hot in a dim that goes round with the token, so that an element of the output is the
weight of the tokens of one dim, and all sums are of numbers that are not negative: rounding is
relative to the element itself.  With u = 2^-24 and h half a step of the output's type:

  flat logits: every weight is a power of two, every sum an integer times it (below 2^24, so
    exact), and what is left is the division, the output's rounding, and the logarithm:
      |out - exact| <= (h + 2^-20) exact,   |lse - exact| <= 2^-20 + 4 u |exact|;
  logits in steps of 1/2 up to 18 apart (exact in fp32): an exponent is at most 52 = 36 log2 e, off
    by two roundings, so a weight is off by e = 2 * 52 u + 2^-22 (the hardware's 2^x), and by h16^2
    where it enters the tensor cores as two 16-bit numbers.  Its part is rescaled by such powers at
    most 7 times (the base moves by 8 or more) and joined twice: 10 e in all.  A sum has at most the
    tokens of a warp's run, R = tokens of all segments / (148 * 4) + 64, then 8 warps and 148 CTAs,
    2 u each (tensor cores may truncate):
      |out - exact| <= (2 (10 e + h16^2 + 2 (R + 160) u) + h + 2^-20) exact,
      |lse - exact| <= 10 e + 2 (R + 160) u + 2^-20 + 4 u |exact|.
    fp16 adds absolute errors where numbers are subnormal.  The largest weight is at least 2^6 there,
    and the two halves of a weight lie on a grid of 2^-24, so that a token is off by 2^-25 of it, or
    2^-31 of the largest; and the output is off by 2^-25:
      + (tokens of the dim) 2^-31 (largest weight of the softmax) + 2^-25.
"""

import math

import pytest
import torch

import razorkv_b200 as R
from razorkv_b200.kernels import check_device_errors
from tests.test_gpu_ragged import HALF, U, _compare, _pool_case

pytestmark = pytest.mark.gpu

bf16, fp16, fp32 = torch.bfloat16, torch.float16, torch.float32
CASES = [
    (bf16, 28, 4, 128, 16, [131077], None), (bf16, 32, 8, 128, 16, [30011, 5, 0, 17000, 64, 9000], None),
    (fp16, 28, 4, 128, 16, [90001, 1, 33], [70, 0, 3]), (bf16, 16, 16, 64, 16, [20000, 20001, 7, 19999], None),
    (fp16, 32, 2, 128, 64, [60000, 300, 41000], [1, 290, 30007]), (bf16, 12, 4, 256, 5, [20000, 15, 20003], None),
    (fp16, 12, 1, 256, 16, [50001, 3], None), (fp32, 8, 4, 128, 16, [20000, 3, 30001], [0, 0, 29000]),
    (fp32, 8, 1, 64, 5, [40009], None), (fp32, 5, 1, 256, 16, [33333, 1], None), (bf16, 4, 2, 20, 7, [30011, 2, 9], None),
    (fp16, 64, 8, 128, 32, [4093, 0, 1, 17, 2200, 900, 3333, 64] * 8, None),
    (bf16, 32, 8, 128, 16, [250] * 64, None), (bf16, 32, 8, 128, 16, [500] * 64, None),
]


def _one_hot(case, step):
    """V one-hot in dim (t // step) % D of token t; K as levels (see _check)."""
    q, kp, vp, table, n, s = case
    P, D = kp.shape[2:]
    for b in range(len(n)):
        t = torch.arange(0 if s is None else min(int(s[b]), int(n[b])), int(n[b]), device="cuda")
        row = torch.zeros(len(t), 1, D, device="cuda", dtype=vp.dtype)
        row[torch.arange(len(t), device="cuda"), 0, (t // step) % D] = 1
        vp[table[b, t // P], :, t % P] = row.expand(-1, kp.shape[1], -1)
        k = torch.zeros_like(row)
        k[:, 0, 0] = _levels(len(n), b, t).to(kp.dtype)
        kp[table[b, t // P], :, t % P] = k.expand(-1, kp.shape[1], -1)


def _levels(batch, b, t):
    """A logit of token t of request b, in [-9, 9] by halves, the same for 64 tokens in a row."""
    g = torch.Generator(device="cuda").manual_seed(17 * batch + b)
    of_block = torch.randint(-18, 19, (int(t[-1]) // 64 + 1 if len(t) else 1,), generator=g, device="cuda") / 2
    return of_block[t // 64]


def _check(case, lse, got, step, flat):
    q, kp, vp, table, n, s = case
    B, Hq, _, D = q.shape
    Hkv = kp.shape[1]
    dtype, tokens = q.dtype, 0
    h16 = HALF[dtype] if dtype != fp32 else 0.0
    for b in range(B):
        tokens += (int(n[b]) - (0 if s is None else min(int(s[b]), int(n[b])))) * Hkv * -(-Hq // Hkv // 4)
    run = tokens / (148 * 4) + 64
    e = 2 * 52 * U + 2.0 ** -22
    rel = 2.0 ** -20 if flat else 2 * (10 * e + h16 * h16 + 2 * (run + 160) * U) + 2.0 ** -20
    off = 2.0 ** -20 if flat else 10 * e + 2 * (run + 160) * U + 2.0 ** -20
    assert rel < 1e-3 and off < 1e-3        # what a tile weighs is far beyond them
    for b in range(B):
        t = torch.arange(0 if s is None else min(int(s[b]), int(n[b])), int(n[b]), device="cuda")
        if not len(t):
            assert bool((got[b] == 0).all()) and bool((lse[b] == -math.inf).all())
            continue
        logit = torch.zeros_like(t, dtype=torch.float64) if flat else _levels(B, b, t).double()
        for sign in (1.0,) if flat else (1.0, -1.0):
            heads = torch.arange(Hq, device="cuda") if flat else torch.nonzero(q[b, :, 0, 0] == sign)[:, 0]
            if not len(heads):
                continue
            w = torch.softmax(sign * logit, 0)
            out = torch.zeros(D, device="cuda", dtype=torch.float64).index_add_(0, (t // step) % D, w)
            err = (got[b, heads, 0].double() - out).abs()
            tol = (rel + HALF[dtype]) * out
            if dtype == fp16:
                count = torch.zeros(D, device="cuda").index_add_(0, (t // step) % D, torch.ones(len(t), device="cuda"))
                tol += count * 2.0 ** -31 * w.max() + 2.0 ** -25
            assert bool((err <= tol).all()), (b, sign)
            want = torch.logsumexp(sign * logit, 0)
            assert bool(((lse[b, heads].double() - want).abs() <= off + 4 * U * want.abs()).all()), (b, sign)


@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("dtype,Hq,Hkv,D,P,lengths,starts", CASES)
def test_every_tile_counts_once(dtype, Hq, Hkv, D, P, lengths, starts, flat):
    case = _pool_case(lengths, Hq, Hkv, D, P, dtype, seed=D, starts=starts)
    step = 8 if flat else 64
    _one_hot(case, step)
    q, kp, vp, table, n, s = case
    q.zero_()
    if not flat:        # heads of both signs: what is heavy for one is light for the other
        q[:, ::2, :, 0] = 1
        q[:, 1::2, :, 0] = -1
    got, lse = R.ragged_decode_attention(q, kp, vp, table, n, scale=1.0, starts=s, return_lse=True)
    _check(case, lse, got, step, flat)
    check_device_errors()


@pytest.mark.parametrize("dtype", [bf16, fp16, fp32])
@pytest.mark.parametrize("Hq,Hkv", [(32, 8), (28, 4), (16, 1)])
@pytest.mark.parametrize("lengths", [[77], [250] * 8, [1, 500, 31], [256]])
def test_few_short_requests_in_a_wide_table(dtype, Hq, Hkv, lengths):
    """A table with room for 65,536 tokens, as a server's, beside one that just holds them."""
    for width in (4096, None):
        _compare(_pool_case(lengths, Hq, Hkv, 128, 16, dtype, seed=12, width=width))
