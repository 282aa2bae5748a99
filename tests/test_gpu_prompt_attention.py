"""qi_prompt_attention against softmax attention in 64 bits, one sequence and
head at a time.

Tolerance per element, for the 16-bit type's half step h = finfo.eps / 2:
  - the result is rounded once: h |o|;
  - each weight 2^(s - m) is rounded to the 16-bit type before it meets v:
    h A, with A = sum_j p_j |v_j| (the attention of |v|, d by d);
  - a score is an FP32 sum of head_dim exact products: off by at most
    head_dim 2^-23 smax in units where smax is the row's largest
    scale * sum |q_d k_d|, the product with scale * log2(e) adds 2^-23 smax
    twice, and 2^x two more steps of 2^-22, in numerator and denominator alike:
    2 A ((head_dim + 2) 2^-23 smax + 2^-21);
  - the sums of the weights and of the products run in FP32, over n keys at
    most n + 16 additions each, every one off by 2^-23 of the partial sum:
    2 (n + 16) 2^-23 A.
"""
import math

import pytest
import torch

import qib200 as Q

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def rand(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def reference(q, k, v, ranges, causal, scale):
    """(out, tolerance) in 64 bits; ranges: (q0, q1, k0, k1) per sequence.
    Rows in no range are NaN."""
    G = q.shape[1] // k.shape[1]
    D = q.shape[2]
    h = torch.finfo(q.dtype).eps / 2
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for q0, q1, k0, k1 in ranges:
        lq, lk = q1 - q0, k1 - k0
        if lq == 0:
            continue
        i = torch.arange(lq, device=q.device)[:, None]
        j = torch.arange(lk, device=q.device)[None]
        seen = (j <= i + lk - lq) if causal else torch.ones(lq, lk, dtype=torch.bool, device=q.device)
        for head in range(q.shape[1]):
            qq, kk, vv = q[q0:q1, head].double(), k[k0:k1, head // G].double(), v[k0:k1, head // G].double()
            s = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
            smax = ((qq.abs() @ kk.abs().T) * abs(scale)).masked_fill(~seen, 0).amax(1, keepdim=True) if lk else 0
            p = torch.softmax(s, 1).masked_fill(~seen, 0)
            p = torch.nan_to_num(p) if lk else p  # rows that see nothing
            o, A = p @ vv, p @ vv.abs()
            out[q0:q1, head] = o
            steps = (D + 2) * 2**-23 * smax + 2**-21
            tol[q0:q1, head] = h * (o.abs() + A) + 2 * A * steps + 2 * (lk + 16) * 2**-23 * A
    return out, tol


def spans(seq_q, seq_k):
    qb, qe = seq_q if isinstance(seq_q, tuple) else (seq_q[:-1], seq_q[1:])
    kb, ke = seq_k if isinstance(seq_k, tuple) else (seq_k[:-1], seq_k[1:])
    return list(zip(qb.tolist(), qe.tolist(), kb.tolist(), ke.tolist()))


def check(q, k, v, seq_q, seq_k, max_k, causal=True, scale=None, out=None, ref=None):
    got = Q.prompt_attention(q, k, v, seq_q, seq_k, max_k, causal=causal, scale=scale, out=out)
    torch.cuda.synchronize()
    Q.prompt_ops_check()
    want, tol = ref or reference(q, k, v, spans(seq_q, seq_k), causal, q.shape[2] ** -0.5 if scale is None else scale)
    inside = ~want.isnan()
    assert bool(torch.isfinite(got[inside]).all())
    over = ((got.double() - want).abs() - tol)[inside]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{float(over.max())} over the tolerance"
    return got


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim", [(28, 4, 128), (3, 3, 64), (5, 1, 128), (8, 4, 80), (2, 1, 8), (6, 2, 96), (4, 2, 72),
                                          (130, 1, 64), (96, 1, 128)])
def test_packed_sequences(dtype, causal, heads, kv, dim):
    lens = [1, 130, 0, 17, 128, 64, 300, 2, 129]
    t = sum(lens)
    cu = offsets(lens)
    check(rand((t, heads, dim), 1, dtype), rand((t, kv, dim), 2, dtype), rand((t, kv, dim), 3, dtype), cu, cu, max(lens), causal)


@pytest.mark.parametrize("lens", [[1], [2], [18], [19], [127], [128], [129], [255], [256], [257], [1500], [1] * 70])
def test_lengths(lens):
    t, cu = sum(lens), offsets(lens)
    check(rand((t, 14, 128), 4, BF), rand((t, 2, 128), 5, BF), rand((t, 2, 128), 6, BF), cu, cu, max(lens))


@pytest.mark.parametrize("causal", [True, False])
def test_queries_and_keys_of_different_lengths(causal):
    """A chunk behind a prefix, one token, more queries than keys (the first
    ones see nothing when causal), no keys at all, no queries."""
    lq, lk = [5, 1, 300, 40, 0, 7, 1, 128], [700, 1000, 300, 9, 50, 0, 1, 127]
    cq, ck = offsets(lq), offsets(lk)
    q, k, v = rand((sum(lq), 14, 128), 7, BF), rand((sum(lk), 2, 128), 8, BF), rand((sum(lk), 2, 128), 9, BF)
    got = check(q, k, v, cq, ck, max(lk), causal)
    r = spans(cq, ck)
    assert not got[r[5][0] : r[5][1]].any()  # no keys: zeros
    if causal:
        assert not got[r[3][0] : r[3][0] + 31].any()  # 40 queries, 9 keys: 31 see nothing


@pytest.mark.parametrize("dtype,heads,kv,dim", [(BF, 28, 4, 128), (HF, 16, 8, 64), (BF, 4, 4, 128), (HF, 8, 1, 96)])
@pytest.mark.parametrize("batch,longest", [(1, 1), (1, 40), (1, 2500), (3, 5000), (16, 1000), (40, 300)])
def test_one_token_against_cache_slabs(dtype, heads, kv, dim, batch, longest):
    """Lq = 1; each sequence's keys fill part of its slot, the rest of the slot
    holds NaN; some sequences have few keys or none."""
    cap = longest + 13
    fill = [(longest * (7 * i + 1)) % (longest + 1) if i else longest for i in range(batch)]
    kb = torch.arange(batch, dtype=torch.int32, device="cuda") * cap
    ke = kb + torch.tensor(fill, dtype=torch.int32, device="cuda")
    q = rand((batch, heads, dim), 10, dtype)
    k, v = rand((batch * cap, kv, dim), 11, dtype), rand((batch * cap, kv, dim), 12, dtype)
    used = torch.zeros(batch * cap, dtype=torch.bool, device="cuda")
    for b, n in enumerate(fill):
        used[b * cap : b * cap + n] = True
    k[~used], v[~used] = float("nan"), float("nan")
    check(q, k, v, offsets([1] * batch), (kb, ke), longest)


@pytest.mark.parametrize("max_k", [0, 1, 100, 100000])
def test_max_k_is_only_a_hint(max_k):
    lk = [900, 3, 2600]
    q, k, v = rand((3, 14, 128), 13, BF), rand((sum(lk), 2, 128), 14, BF), rand((sum(lk), 2, 128), 15, BF)
    check(q, k, v, offsets([1, 1, 1]), offsets(lk), max_k)


@pytest.mark.parametrize("layout", ["qkv", "heads", "batch_heads"])
def test_strided_layouts_equal_the_contiguous_one(layout):
    lens, heads, kv, dim = [77, 200, 19, 128], 12, 4, 128
    t, cu = sum(lens), offsets(lens)
    if layout == "qkv":
        rows = rand((t, heads + 2 * kv, dim), 16, BF)
        q, k, v = rows[:, :heads], rows[:, heads : heads + kv], rows[:, heads + kv :]
        out = torch.empty(t, 3 * heads, dim, dtype=BF, device="cuda")[:, heads : 2 * heads]
    elif layout == "heads":
        q, k, v = (rand((n, t, dim), 17 + n, BF).transpose(0, 1) for n in (heads, kv, kv))
        out = torch.empty(heads, t, dim, dtype=BF, device="cuda").transpose(0, 1)
    else:  # head dimension inside a wider row
        q, k, v = (rand((t, n, dim + 24), 18 + n, BF)[:, :, 8 : 8 + dim] for n in (heads, kv, kv))
        out = torch.empty(t, heads, dim + 8, dtype=BF, device="cuda")[:, :, :dim]
    got = check(q, k, v, cu, cu, max(lens), out=out)
    assert got.data_ptr() == out.data_ptr()
    plain = Q.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, cu, max(lens))
    assert torch.equal(got, plain)


def test_rows_behind_the_last_sequence_are_left():
    lens = [50, 130]
    t, cu = sum(lens), offsets(lens)
    q, k, v = rand((t + 40, 4, 128), 19, BF), rand((t + 40, 2, 128), 20, BF), rand((t + 40, 2, 128), 21, BF)
    out = torch.full((t + 40, 4, 128), 7.0, dtype=BF, device="cuda")
    check(q, k, v, cu, cu, max(lens), out=out)
    assert bool((out[t:] == 7.0).all())


def test_ranges_are_clipped_to_the_tensors():
    """Offsets past the end or running backwards read and write nothing outside."""
    q, k, v = rand((40, 4, 128), 22, BF), rand((60, 2, 128), 23, BF), rand((60, 2, 128), 24, BF)
    out = torch.full((40, 4, 128), 7.0, dtype=BF, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    qb, qe = i32(-5, 20, 30, 40), i32(10, 15, 90, 2000000000)
    kb, ke = i32(-9, 0, 50, 0), i32(30, 10, 2000000000, 60)
    Q.prompt_attention(q, k, v, (qb, qe), (kb, ke), 60, out=out)
    want, tol = reference(q, k, v, [(0, 10, 0, 30), (30, 40, 50, 60)], True, 128**-0.5)
    inside = ~want.isnan()
    assert bool(((out.double() - want).abs() <= tol)[inside].all())
    assert bool((out[~inside] == 7.0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 128), (14, 2, 128), (4, 2, 64)])
def test_non_finite_values_stay_where_they_are_seen(bad, heads, kv, dim):
    """A non-finite key or value row reaches only the queries that see it: not
    other sequences, not earlier positions of its own."""
    lens = [100, 300, 60]
    t, cu = sum(lens), offsets(lens)
    q, k, v = rand((t, heads, dim), 25, BF), rand((t, kv, dim), 26, BF), rand((t, kv, dim), 27, BF)
    clean = Q.prompt_attention(q, k, v, cu, cu, max(lens))
    at = 100 + 170
    for which in ("v", "k", "q"):
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        {"v": v2, "k": k2, "q": q2}[which][at, :, 3] = bad
        got = Q.prompt_attention(q2, k2, v2, cu, cu, max(lens))
        same = torch.ones(t, dtype=torch.bool, device="cuda")
        same[at : (400 if which != "q" else at + 1)] = False
        assert torch.equal(got[same], clean[same]), which
        if which == "v":  # the row's own result in that dimension is not finite, the others are as they were
            d3 = got[at:400, :, 3].float()
            assert bool((d3.isnan() | d3.isinf()).all())
            if math.isinf(bad):  # queries with only this infinity: the infinity itself
                assert bool((got[at, :, 3].float() == bad).all())
            rest = [d for d in range(dim) if d != 3]
            assert torch.equal(got[:, :, rest], clean[:, :, rest])
        if which == "q" and math.isnan(bad):
            assert bool(got[at].isnan().all())


def test_large_scores_and_lowest_values():
    """Scores of the order of 1e4, and keys at the type's lowest value."""
    lens = [200]
    cu = offsets(lens)
    q, k, v = rand((200, 2, 128), 28, BF, 30.0), rand((200, 1, 128), 29, BF, 30.0), rand((200, 1, 128), 30, BF)
    check(q, k, v, cu, cu, 200)
    k[50] = torch.finfo(BF).min
    q[:, :, :64], q[:, :, 64:] = q[:, :, :64].abs() * 1e-3, q[:, :, 64:].abs() * 1e-3
    check(q, k, v, cu, cu, 200)


@pytest.mark.parametrize("scale", [0.0, 0.3, -0.2])
def test_scales(scale):
    cu = offsets([150, 33])
    q, k, v = rand((183, 4, 64), 31, HF), rand((183, 2, 64), 32, HF), rand((183, 2, 64), 33, HF)
    check(q, k, v, cu, cu, 150, scale=scale)


def test_offsets_past_32_bits():
    """Keys that start beyond 2^31 elements of the cache."""
    kv, dim, n = 8, 128, 2_200_000
    k = torch.empty(n, kv, dim, dtype=BF, device="cuda")
    v = torch.empty(n, kv, dim, dtype=BF, device="cuda")
    k[-700:], v[-700:] = rand((700, kv, dim), 34, BF), rand((700, kv, dim), 35, BF)
    q = rand((2, 16, dim), 36, BF)
    kb = torch.tensor([n - 700, n - 300], dtype=torch.int32, device="cuda")
    ke = torch.tensor([n - 300, n], dtype=torch.int32, device="cuda")
    ref = reference(q, k[-700:], v[-700:], [(0, 1, 0, 400), (1, 2, 400, 700)], True, dim**-0.5)
    check(q, k, v, offsets([1, 1]), (kb, ke), 400, ref=ref)


def test_same_result_every_time_and_on_two_streams_at_once():
    lens = [1, 1, 1, 200]
    lk = [4000, 900, 3000, 200]
    q, k, v = rand((203, 28, 128), 37, BF), rand((sum(lk), 4, 128), 38, BF), rand((sum(lk), 4, 128), 39, BF)
    cq, ck = offsets(lens), offsets(lk)
    first = Q.prompt_attention(q, k, v, cq, ck, 4000)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(Q.prompt_attention(q, k, v, cq, ck, 4000))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    Q.prompt_ops_check()


def test_captured_and_replayed_with_other_lengths():
    """The lengths are read on the device: a replay follows them."""
    heads, kv, dim, cap = 28, 4, 128, 3000
    q = rand((4, heads, dim), 40, BF)
    k, v = rand((4 * cap, kv, dim), 41, BF), rand((4 * cap, kv, dim), 42, BF)
    kb = torch.arange(4, dtype=torch.int32, device="cuda") * cap
    ke = kb + 1
    cq = offsets([1] * 4)
    out = torch.empty_like(q)
    Q.prompt_attention(q, k, v, cq, (kb, ke), cap, out=out)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        Q.prompt_attention(q, k, v, cq, (kb, ke), cap, out=out)
    out2 = torch.empty_like(q)
    with torch.cuda.graph(g2):
        Q.prompt_attention(q, k, v, cq, (kb, ke), cap, out=out2)
    for fill in ([3000, 1, 128, 2000], [5, 0, 2999, 700]):
        ke.copy_(kb + torch.tensor(fill, dtype=torch.int32, device="cuda"))
        want, tol = reference(q, k, v, spans(cq, (kb, ke)), True, dim**-0.5)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        for o in (out, out2):
            assert bool(((o.double() - want).abs() <= tol).all())
    Q.prompt_ops_check()


def test_empty_calls():
    cu = offsets([0, 0])
    e = lambda n, h: torch.empty(n, h, 64, dtype=BF, device="cuda")  # noqa: E731
    assert Q.prompt_attention(e(0, 4), e(0, 2), e(0, 2), cu, cu, 0).shape == (0, 4, 64)
    out = Q.prompt_attention(rand((3, 4, 64), 43, BF), e(0, 2), e(0, 2), offsets([1, 2]), cu, 0)
    assert not out.any()


def test_binding_refuses():
    q, k, v = rand((10, 4, 64), 44, BF), rand((10, 2, 64), 45, BF), rand((10, 2, 64), 46, BF)
    cu = offsets([4, 6])
    bad = [
        (q.half(), k, v, cu, cu), (q.float(), k.float(), v.float(), cu, cu), (q, k, v[:5], cu, cu),
        (q, k, v, cu.long(), cu), (q, k, v, cu, cu[:2]), (q, k, v, cu.cpu(), cu), (q[:, :, ::2], k[:, :, ::2], v[:, :, ::2], cu, cu),
        (q[:, :3], k, v, cu, cu), (q[:, :, :60], k[:, :, :60], v[:, :, :60], cu, cu),
        (q[:, :, 4:60], k[:, :, 4:60], v[:, :, 4:60], cu, cu), (q, k[:, :1].expand(10, 2, 64), v, cu, cu),
    ]
    for args in bad:
        with pytest.raises(Q.QIError):
            Q.prompt_attention(*args, 6)
    with pytest.raises(Q.QIError):
        Q.prompt_attention(q, k, v, cu, cu, 6, out=q[:1].expand(10, 4, 64))


@pytest.mark.parametrize("lq", ["same", "one"])
def test_many_sequences(lq):
    """More sequences than a CTA keeps in shared memory, short and long ones mixed."""
    lk = [(37 * i) % 90 for i in range(300)] + [700, 1, 0, 300]
    lq = lk if lq == "same" else [1] * len(lk)
    cq, ck = offsets(lq), offsets(lk)
    q, k, v = rand((sum(lq), 8, 128), 50, BF), rand((sum(lk), 2, 128), 51, BF), rand((sum(lk), 2, 128), 52, BF)
    check(q, k, v, cq, ck, max(lk))


@pytest.mark.parametrize("lens,lk", [([200, 31, 128], None), ([1, 1, 3], [2000, 700, 5])])
def test_output_over_the_queries(lens, lk):
    """out = q: the same results, also as views into one buffer of q, k and v rows."""
    lk = lk or lens
    cq, ck = offsets(lens), offsets(lk)
    q, k, v = rand((sum(lens), 8, 128), 53, BF), rand((sum(lk), 2, 128), 54, BF), rand((sum(lk), 2, 128), 55, BF)
    want = Q.prompt_attention(q, k, v, cq, ck, max(lk))
    mine = q.clone()
    assert Q.prompt_attention(mine, k, v, cq, ck, max(lk), out=mine).data_ptr() == mine.data_ptr()
    assert torch.equal(mine, want)
    if lk == lens:
        rows = torch.cat([q, k, v], 1)
        Q.prompt_attention(rows[:, :8], rows[:, 8:10], rows[:, 10:], cq, ck, max(lk), out=rows[:, :8])
        assert torch.equal(rows[:, :8], want) and torch.equal(rows[:, 8:10], k) and torch.equal(rows[:, 10:], v)


def test_output_over_keys_or_values_is_refused():
    rows = rand((40, 12, 64), 56, BF)
    q, k, v = rows[:, :4], rows[:, 4:8], rows[:, 8:]
    cu = offsets([40])
    for out in (k, v, rows[:, 2:6]):
        with pytest.raises(Q.QIError):
            Q.prompt_attention(q, k, v, cu, cu, 40, out=out)


def test_two_tiles_with_split_keys():
    """Enough queries for two-tile CTAs, few enough to split the keys."""
    lq, lk = [900, 700], [4000, 700]
    cq, ck = offsets(lq), offsets(lk)
    q, k, v = rand((1600, 14, 128), 57, BF), rand((4700, 1, 128), 58, BF), rand((4700, 1, 128), 59, BF)
    check(q, k, v, cq, ck, 4000)
    check(q, k, v, cq, ck, 4000, causal=False)


@pytest.mark.parametrize("heads,kv,dim", [(64, 8, 128), (20, 4, 64), (6, 6, 128)])
def test_tile_without_keys_next_to_one_with_keys(heads, kv, dim):
    """More queries than keys under a causal mask: where the first key is seen, a
    CTA has a tile of rows that see none (zeros) beside one of rows that do."""
    lq = [4, 297, 5, 7, 55, 571, 3, 116, 9, 3, 34, 85, 21, 6, 17, 2, 635, 1500]
    lk = [457, 667, 1338, 2193, 272, 42, 17, 114, 1123, 28, 1333, 24, 15, 48, 10, 20, 3, 700]
    q, k, v = rand((sum(lq), heads, dim), 1, BF), rand((sum(lk), kv, dim), 2, BF), rand((sum(lk), kv, dim), 3, BF)
    sq, sk = offsets(lq), offsets(lk)
    ref = reference(q, k, v, spans(sq, sk), True, dim**-0.5)
    for _ in range(5):
        check(q, k, v, sq, sk, max(lk), ref=ref)


def test_overlapping_query_ranges_read_nothing_outside_the_workspace():
    """Not allowed, and the rows' results mean nothing, but the lengths live on
    the device: a call whose ranges ask for more tiles than there are CTAs joins
    rows that no CTA has made, whatever the workspace held before."""
    heads, kv, dim, batch, tq, lk = 28, 4, 128, 64, 100, 4096
    q, k, v = rand((tq, heads, dim), 1, BF), rand((lk, kv, dim), 2, BF), rand((lk, kv, dim), 3, BF)
    begin = torch.tensor([0] * (batch - 1) + [90], dtype=torch.int32, device="cuda")
    end = torch.tensor([90] * (batch - 1) + [tq], dtype=torch.int32, device="cuda")
    ks, ke = torch.zeros(batch, dtype=torch.int32, device="cuda"), torch.full((batch,), lk, dtype=torch.int32, device="cuda")
    n = Q.lib().qi_prompt_attention_workspace(heads, kv, dim, batch, tq, lk, lk)
    assert n > 0
    ws = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(q)
    st = Q.lib().qi_prompt_attention(
        q.data_ptr(), heads * dim, dim, k.data_ptr(), kv * dim, dim, v.data_ptr(), kv * dim, dim, out.data_ptr(), heads * dim, dim,
        Q.DT_BF16, heads, kv, dim, begin.data_ptr(), end.data_ptr(), ks.data_ptr(), ke.data_ptr(), batch, tq, lk, lk,
        dim**-0.5, 0, ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
    assert st == 0
    torch.cuda.synchronize()
    Q.prompt_ops_check()
