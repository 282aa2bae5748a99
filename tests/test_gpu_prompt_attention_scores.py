"""qi_prompt_attention with scores far from zero, and with scales at the ends
of their range, against 64 bits.

q and k hold numbers whose products and sums FP32 holds exactly, so that the
scores q.k carry no error and what is left of the tolerance is (h the type's
half step, A = sum_j p_j |v_j|, n keys):
  - the output rounded once, h |o|, and the weights, h A;
  - a weight's exponent, sc (r_j - m): below 32 in size where the weight counts
    at all (2^-32 n is far below h), two products rounded, and where it is taken
    as sc r_j - sc m an sc m of at most 256 rounded once in each of two places:
    2^-16 in all, for weights and their sum alike: 2 A 2^-16;
  - FP32 sums: 2 (n + 16) 2^-23 A.
"""
import math

import pytest
import torch

import qib200 as Q

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def whole(shape, seed, dtype, most):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)


def normal(shape, seed, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def check(q, k, v, lq, lk, scale, causal=True):
    got = Q.prompt_attention(q, k, v, offsets(lq), offsets(lk), max(lk), causal=causal, scale=scale)
    torch.cuda.synchronize()
    Q.prompt_ops_check()
    h = torch.finfo(q.dtype).eps / 2
    G, q0, k0 = q.shape[1] // k.shape[1], 0, 0
    for nq, nk in zip(lq, lk):
        i, j = torch.arange(nq, device="cuda")[:, None], torch.arange(nk, device="cuda")[None]
        hidden = j > i + nk - nq if causal else torch.zeros(nq, nk, dtype=torch.bool, device="cuda")
        for head in range(q.shape[1]):
            qq, kk, vv = q[q0 : q0 + nq, head].double(), k[k0 : k0 + nk, head // G].double(), v[k0 : k0 + nk, head // G].double()
            r = qq @ kk.T
            far = r.masked_fill(hidden, -math.copysign(math.inf, scale)) * math.copysign(1, scale)
            s = (r - far.amax(1, keepdim=True) * math.copysign(1, scale)) * scale
            p = torch.softmax(s.masked_fill(hidden, -math.inf), 1)
            o, A = p @ vv, p @ vv.abs()
            tol = h * (o.abs() + A) + 2 * A * 2**-16 + 2 * (nk + 16) * 2**-23 * A
            d = (got[q0 : q0 + nq, head].double() - o).abs() - tol
            assert float(d.nan_to_num(math.inf).max()) <= 0, (nq, nk, head)
        q0, k0 = q0 + nq, k0 + nk


# sequences of queries and keys: packed prompts in one-tile and in two-tile CTAs, chunks and single tokens with split keys
CALLS = [([3, 150, 61], [3, 150, 61]), ([900, 1100], [900, 1100]), ([1, 1, 1], [2500, 1, 700]), ([40, 1], [3000, 129])]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("lq,lk", CALLS)
@pytest.mark.parametrize("scale", [1e3, -1e6, 1e10, 1e20, -1e30, 1e38, 1.9e38])
def test_one_key_takes_all(dtype, dim, lq, lk, scale):
    """Scores that are whole multiples of a huge scale: the keys with the largest
    share the row, however far the products are past what FP32 holds."""
    q, k, v = whole((sum(lq), 14, dim), 1, dtype, 4), whole((sum(lk), 2, dim), 2, dtype, 4), normal((sum(lk), 2, dim), 3, dtype)
    check(q, k, v, lq, lk, scale)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lq,lk", CALLS)
@pytest.mark.parametrize("base", [2.0**9, 2.0**13, -(2.0**13), 2.0**20, -(2.0**22)])
@pytest.mark.parametrize("causal", [True, False])
def test_far_scores_with_small_differences(dtype, lq, lk, base, causal):
    """All scores near `base` times the scale, and a few apart: the differences
    decide, and they are exact."""
    q, k, v = whole((sum(lq), 14, 128), 4, dtype, 3), whole((sum(lk), 2, 128), 5, dtype, 3), normal((sum(lk), 2, 128), 6, dtype)
    half = 2.0 ** (int(math.log2(abs(base))) // 2)
    q[:, :, 0], k[:, :, 0] = half, base / half
    check(q, k, v, lq, lk, 0.03, causal)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_maximum_that_comes_late(dtype):
    """Scores that rise from far below zero to far above along the keys, so that
    the maximum moves in every block."""
    lq, lk = [1, 30], [3000, 2000]
    q, k, v = whole((31, 14, 128), 7, dtype, 2), whole((5000, 2, 128), 8, dtype, 2), normal((5000, 2, 128), 9, dtype)
    q[:, :, 0] = 64
    ramp = torch.arange(5000, device="cuda") // 16 * 4.0 - 500
    k[:, :, 0] = (ramp.clamp(max=200)[:, None]).to(dtype)
    check(q, k, v, lq, lk, 0.05)


@pytest.mark.parametrize("dtype,big", [(BF, 2.0**62), (HF, 2.0**14)])
@pytest.mark.parametrize("lq,lk", CALLS)
@pytest.mark.parametrize("scale", [0.0, 2.0**-126, -(2.0**-127), 2.0**-128, 2.0**-140, 2.0**-149])
def test_smallest_scales(dtype, big, lq, lk, scale):
    """Scales down to the smallest subnormal number: with scores up to 3 x 2^124
    (BF16) they still decide, and scale 0 weighs all keys alike."""
    q, k, v = whole((sum(lq), 14, 64), 10, dtype, 3), whole((sum(lk), 2, 64), 11, dtype, 3), normal((sum(lk), 2, 64), 12, dtype)
    q[:, :, 1:], k[:, :, 1:] = 0, 0
    q[:, :, 0], k[:, :, 0] = big, k[:, :, 0] * big
    check(q, k, v, lq, lk, scale)
