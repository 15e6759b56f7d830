"""Ragged decode attention on values at the ends of what its types hold (GPU): infinities and
NaN in tokens that are attended, and logits far beyond the exponents of their weights."""

import math

import pytest
import torch

import razorkv_b200 as R
from tests.test_gpu_ragged import HALF, U, _pool_case

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D,P", [(8, 2, 64, 16), (16, 1, 64, 8), (8, 2, 128, 16), (16, 1, 128, 5),
                                        (4, 2, 256, 16), (12, 1, 200, 32), (6, 2, 17, 16)])
@pytest.mark.parametrize("lengths", [[1, 7, 40], [3001, 2, 700]])
def test_infinite_values_that_are_attended(dtype, Hq, Hkv, D, P, lengths):
    """By the formula a column of V with an infinity of one sign gives it, of both signs NaN, and
    one with NaN NaN; every other element of the output is what it was."""
    q, kp, vp, table, n, s = _pool_case(lengths, Hq, Hkv, D, P, dtype, seed=D + P)
    clean, lse = R.ragged_decode_attention(q, kp, vp, table, n, return_lse=True)
    G = Hq // Hkv
    want = clean.clone()
    plant = [(0, 0, 3, math.inf), (0, lengths[0] - 1, 5, -math.inf), (2, 0, 0, -math.inf),
             (2, lengths[2] - 1, 0, -math.inf), (2, lengths[2] // 2, 1, math.inf), (2, 3, 1, -math.inf),
             (2, 5, 2, math.nan), (2, 6, 2, math.inf), (2, lengths[2] - 1, D - 1, math.inf)]
    for b, t, d, x in plant:
        h = b % Hkv
        vp[table[b, t // P], h, t % P, d] = x
        want[b, h * G: (h + 1) * G, 0, d] = x
    h = 2 % Hkv
    want[2, h * G: (h + 1) * G, 0, 1:3] = math.nan
    got, again = R.ragged_decode_attention(q, kp, vp, table, n, return_lse=True)
    assert torch.equal(again, lse)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(nan=7.0, posinf=math.inf, neginf=-math.inf),
                       want.nan_to_num(nan=7.0, posinf=math.inf, neginf=-math.inf))


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_value_in_a_part_of_little_weight(dtype):
    """The infinity's part of the request weighs e^-60 of the others."""
    q, kp, vp, table, n, s = _pool_case([4000], 4, 1, 128, 16, dtype, seed=2)
    q.zero_()
    q[..., 0] = 1
    kp[table[0], 0, :, 0] = 0
    kp[table[0, 100:150], 0, :, 0] = -60
    vp[table[0, 120], 0, 3, 9] = math.inf
    out = R.ragged_decode_attention(q, kp, vp, table, n, scale=1.0)
    assert bool((out[..., 9] == math.inf).all())
    out[..., 9] = 0
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D,lengths", [(8, 2, 64, [500, 1, 37]), (32, 8, 128, [400, 3]), (16, 1, 128, [300, 5]),
                                              (8, 2, 256, [200, 9]), (6, 2, 17, [333, 2]), (4, 1, 128, [20011])])
@pytest.mark.parametrize("scale,sign", [(1.0, 1), (0.037, 1), (1.37, -1)])
def test_logits_beyond_their_weights(dtype, Hq, Hkv, D, lengths, scale, sign):
    """Scaled logits of 2.7e7 to 1e9.  One product makes a logit, of two numbers of 7 bits, so that
    it is exact in fp32; every third token has the largest and the others lie 5e5 below and more, so
    exact weights are 1 and 0, and sums of ones below 2^24 are exact too.  What is left:
      lse = scale * top + log(count): one rounding of |lse|, one of the logarithm's factor, and the
        hardware's log2 (2^-22): 2 u |lse| + 2^-20;
      out = sum of V / count: N sums of 2 u A each, the division, and the output's rounding."""
    q, kp, vp, table, n, _ = _pool_case(lengths, Hq, Hkv, D, 16, dtype, seed=D)
    q.zero_()
    q[..., 0] = 99 * 256.0 * sign
    top, low = (113, 111) if sign > 0 else (111, 113)
    for b, m in enumerate(lengths):
        t = torch.arange(m, device="cuda")
        k = torch.where(t % 3 == (m - 1) % 3, top * 256.0, low * 256.0)
        kp[table[b, t // 16], :, t % 16] = 0
        kp[table[b, t // 16], :, t % 16, 0] = k[:, None].expand(-1, Hkv).to(dtype)
    got, lse = R.ragged_decode_attention(q, kp, vp, table, n, scale=scale, return_lse=True)
    s = float(torch.tensor(scale, dtype=torch.float32)) * sign * 99 * 256 * top * 256
    for b, m in enumerate(lengths):
        t = torch.arange((m - 1) % 3, m, 3, device="cuda")
        exact = s + math.log(len(t))
        assert bool(((lse[b].double() - exact).abs() <= 2 * U * abs(exact) + 2.0 ** -20).all())
        v = vp[table[b, t // 16], :, t % 16].double()
        out = v.mean(0).repeat_interleave(Hq // Hkv, 0)
        A = v.abs().mean(0).repeat_interleave(Hq // Hkv, 0)
        tol = (2 * len(t) * U + 2.0 ** -20) * A + HALF[dtype] * out.abs() + 2.0 ** -25
        assert bool(((got[b, :, 0].double() - out).abs() <= tol).all())
