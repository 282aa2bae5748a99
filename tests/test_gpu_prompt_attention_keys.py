"""qi_prompt_attention takes each key once: every key that a query sees, at the
borders of key blocks, of splits and of a cache's fill, and none twice.

The element bound of a long random sum hardly notices one key of thousands, so
these tests are built to: uniform weights that count keys, queries that pick one
key out, and a bound in norm that takes the roundings as independent.
"""
import pytest
import torch

import qib200 as Q

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def rand(shape, seed, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def slots(lens, gap):
    """Cache slots that hold `lens` keys, the rest of each `gap` wider slot unused."""
    cap = max(lens) + gap
    begin = torch.arange(len(lens), dtype=torch.int32, device="cuda") * cap
    return begin, begin + torch.tensor(lens, dtype=torch.int32, device="cuda"), cap


def call(q, k, v, lq, seq_k, max_k, causal=True):
    got = Q.prompt_attention(q, k, v, offsets(lq), seq_k, max_k, causal=causal)
    torch.cuda.synchronize()
    Q.prompt_ops_check()
    return got


# (queries, keys) per sequence: one token with several splits, chunks behind a prefix, packed prompts; lengths around
# whole key blocks and whole splits
CALLS = [
    ([1], [4096]), ([1], [4097]), ([1], [4000]), ([1], [16383]), ([1] * 5, [2500, 129, 1, 256, 3333]), ([1] * 16, [128 * i + i % 3 for i in range(1, 17)]),
    ([40, 100], [3000, 2049]), ([256], [4000]), ([3, 500, 127, 1], [3, 500, 127, 1]), ([1000], [1000]), ([2048, 129], [2048, 129]), ([50], [20]),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kv,dim", [(28, 4, 128), (16, 8, 64), (3, 3, 128)])
@pytest.mark.parametrize("lq,lk", CALLS)
@pytest.mark.parametrize("causal", [True, False])
def test_uniform_weights_count_the_keys(dtype, heads, kv, dim, lq, lk, causal):
    """q = 0: every key weighs 1, exactly, and out[d] is the share of keys whose
    v has a 1 at d: once the keys with number d in their stretch of `dim`, once
    those of the d-th stretch.  A key lost or taken twice moves a count c by 1 / c,
    1 / 128 or more (1 / 256 for 16383 keys and heads of 64, where BF16 may miss
    it and FP16 does not); the result is off by half a step h and a few FP32
    steps (2^-19)."""
    begin, end, cap = slots(lk, 37)
    rows = len(lk) * cap
    q = torch.zeros(sum(lq), heads, dim, dtype=dtype, device="cuda")
    k = torch.full((rows, kv, dim), float("nan"), dtype=dtype, device="cuda")
    for b, n in enumerate(lk):
        k[b * cap : b * cap + n] = rand((n, kv, dim), b, dtype)
    at = torch.arange(rows, device="cuda") % cap
    h = torch.finfo(dtype).eps / 2
    for number in (at % dim, at // dim):
        v = torch.zeros(rows, kv, dim, dtype=dtype, device="cuda")
        v[torch.arange(rows, device="cuda"), :, number % dim] = 1
        for b, n in enumerate(lk):
            v[b * cap + n : (b + 1) * cap] = float("nan")
        got = call(q, k, v, lq, (begin, end), max(lk), causal).double()
        i0 = 0
        for nq, nk in zip(lq, lk):
            hot = torch.nn.functional.one_hot(number[:nk] % dim, dim).double()
            seen = (torch.arange(nq, device="cuda") + nk - nq + 1).clamp(0, nk) if causal else torch.full((nq,), nk, device="cuda")
            count = torch.cat([torch.zeros(1, dim, dtype=torch.float64, device="cuda"), hot.cumsum(0)])[seen]
            want = (count / seen.clamp(min=1)[:, None])[:, None].expand(nq, heads, dim)
            assert bool(((got[i0 : i0 + nq] - want).abs() <= (h + 2**-19) * want).all()), (nq, nk)
            i0 += nq


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kv,dim", [(28, 4, 128), (16, 8, 64)])
@pytest.mark.parametrize("n", [1, 127, 128, 129, 1000, 4096, 4097, 8190])
@pytest.mark.parametrize("lq", [1, 3])
def test_every_border_key_can_be_picked(dtype, heads, kv, dim, n, lq):
    """Queries along one key each: first and last of every block of 128 and of the
    fill.  Its score is 8 sqrt(dim), the others' are 8 times a standard normal, so
    it is far above them (the gap is taken in 64 bits) and out is its v: rounded
    once, h |v|, with the others' weights, at most n e^-gap of the largest |v|."""
    g = torch.Generator(device="cuda").manual_seed(n)
    sign = lambda *s: (torch.randint(0, 2, s, generator=g, device="cuda") * 2 - 1).to(dtype)  # noqa: E731
    cap = n + 50
    k, v = torch.full((cap, kv, dim), float("nan"), dtype=dtype, device="cuda"), torch.full((cap, kv, dim), float("nan"), dtype=dtype, device="cuda")
    k[:n], v[:n] = sign(n, kv, dim), rand((n, kv, dim), 7, dtype)
    picks = sorted({j for b in range(0, n, 128) for j in (b, min(b + 127, n - 1))})
    B, G = len(picks), heads // kv
    # all sequences have the same keys; lq > 1: the pick is seen by all lq queries (not causal)
    q = (8 * k[picks]).repeat_interleave(G, 1).repeat_interleave(lq, 0)
    begin = torch.zeros(B, dtype=torch.int32, device="cuda")
    end = torch.full((B,), n, dtype=torch.int32, device="cuda")
    got = call(q, k, v, [lq] * B, (begin, end), n, causal=lq == 1).double()
    h = torch.finfo(dtype).eps / 2
    for head in range(heads):
        s = q[::lq, head].double() @ k[:n, head // G].double().T / dim**0.5
        mine = s[torch.arange(B), picks]
        s[torch.arange(B), picks] = -torch.inf
        gap = float((mine - s.amax(1)).min()) if n > 1 else 100.0
        assert gap > 10
        want = v[picks, head // G].double().repeat_interleave(lq, 0)
        tol = (h + 2**-19) * want.abs() + 2 * n * 2.718281828 ** -gap * float(v[:n].abs().max())
        assert bool(((got[:, head] - want).abs() <= tol).all()), head


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kv,dim", [(28, 4, 128), (16, 8, 64)])
@pytest.mark.parametrize("lq,lk", [c for c in CALLS if max(c[1]) >= 1000])
def test_random_values_in_norm(dtype, heads, kv, dim, lq, lk):
    """Per head, the roundings taken as independent: each weight's, h p_j |v_jd| at
    most, and the result's, h |o_d|.  A score's error (sums of dim products and two
    more, 2^-23 of sum |q k| at most each) reaches o as p_j e_j (v_j - o), with v
    independent of the scores; the FP32 sums, truncated every 16 keys, lose 2^-23
    of sums that are as random.  So the norm of the error is at most that of
    e = (h + (dim + 2) 2^-23 smax + 2^-20 + (n / 16 + 16) 2^-23) sqrt(sum_j p_j^2 v_jd^2) + h |o_d|."""
    begin, end, cap = slots(lk, 13)
    q, k, v = rand((sum(lq), heads, dim), 1, dtype), rand((len(lk) * cap, kv, dim), 2, dtype), rand((len(lk) * cap, kv, dim), 3, dtype)
    got = call(q, k, v, lq, (begin, end), max(lk)).double()
    h, G, i0 = torch.finfo(dtype).eps / 2, heads // kv, 0
    for b, (nq, nk) in enumerate(zip(lq, lk)):
        hidden = torch.arange(nk, device="cuda")[None] > torch.arange(nq, device="cuda")[:, None] + nk - nq
        for head in range(heads):
            qq, kk, vv = q[i0 : i0 + nq, head].double(), k[b * cap : b * cap + nk, head // G].double(), v[b * cap : b * cap + nk, head // G].double()
            p = torch.softmax((qq @ kk.T / dim**0.5).masked_fill(hidden, -torch.inf), 1)
            smax = float((qq.abs() @ kk.abs().T).max()) / dim**0.5
            o, spread = p @ vv, (p.square() @ vv.square()).sqrt()
            e = h + (dim + 2) * 2**-23 * smax + 2**-20 + (nk / 16 + 16) * 2**-23
            bound = (e * spread).square().sum() + (h * o).square().sum()
            assert float((got[i0 : i0 + nq, head] - o).square().sum()) <= float(bound), (nq, nk, head)
        i0 += nq
