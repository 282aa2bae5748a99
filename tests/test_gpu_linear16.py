"""qi_linear_16bit against the formula in 64 bits.

Tolerance per element, with h = finfo(out).eps / 2 and T = sum_k |x w| + |bias|:
  - the products are exact in FP32; the sum of K of them in the tensor core's
    order, one step of 2^-23 of the running sum each at most: K 2^-23 T (the
    bias adds one more);
  - silu and tanh-GELU have a slope of at most 1.13; their own arithmetic
    (2^x, one division, a few products) adds 2^-19 of the value;
  - SwiGLU: each factor's error times the other factor;
  - gate and residual: one more FP32 step each (2^-23);
  - the result is rounded once: h |y|.
"""
import math

import pytest
import torch

import qib200 as Q

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rand(shape, seed, dtype=F32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def reference(x, w, bias, act, gate, residual, out_dtype):
    K = x.shape[1]
    xd, wd = x.double(), w.double()
    a, t = xd @ wd.T, xd.abs() @ wd.abs().T
    if bias is not None:
        a, t = a + bias.double(), t + bias.double().abs()
    e = (K + 1) * 2**-23 * t
    if act == Q.ACT_GELU:
        y = a * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a**3))
        e = 1.13 * e + 2**-19 * y.abs()
    elif act == Q.ACT_SILU:
        y = a * torch.sigmoid(a)
        e = 1.13 * e + 2**-19 * y.abs()
    elif act == Q.ACT_SWIGLU:
        n = a.shape[1] // 2
        s = a[:, :n] * torch.sigmoid(a[:, :n])
        es = 1.13 * e[:, :n] + 2**-19 * s.abs()
        y = s * a[:, n:]
        e = es * a[:, n:].abs() + (s.abs() + es) * e[:, n:]
    else:
        y = a
    if gate is not None:
        y, e = y * gate.double(), e * gate.double().abs()
    e = e + 2**-23 * y.abs()
    if residual is not None:
        y = y + residual.double()
        e = e + 2**-23 * y.abs()
    return y, e + torch.finfo(out_dtype).eps / 2 * (y.abs() + e)


def check(x, w, out_dtype, bias=None, act=Q.ACT_NONE, gate=None, residual=None, out=None):
    want, tol = reference(x, w, bias, act, gate, residual.clone() if residual is not None else None, out_dtype)
    got = Q.linear_16bit(x, w, bias=bias, act=act, gate=gate, residual=residual, out_dtype=out_dtype, out=out)
    torch.cuda.synchronize()
    Q.prompt_ops_check()
    assert got.dtype == out_dtype and got.shape == want.shape
    assert bool(torch.isfinite(got).all())
    over = (got.double() - want).abs() - tol
    assert over.numel() == 0 or float(over.max()) <= 0, f"{float(over.max())} over the tolerance"
    return got


def operands(M, N, K, dtype, wide=1, seed=1):
    return rand((M, K), seed, dtype), rand((wide * N, K), seed + 1, dtype, K**-0.5)


@pytest.mark.parametrize("dtype,out_dtype", [(BF, BF), (HF, HF), (BF, F32), (HF, F32)])
@pytest.mark.parametrize("act", [Q.ACT_NONE, Q.ACT_GELU, Q.ACT_SILU, Q.ACT_SWIGLU])
@pytest.mark.parametrize("M,N,K", [(1, 64, 64), (7, 200, 136), (130, 264, 72), (300, 520, 1024), (1000, 776, 512)])
def test_every_epilogue(dtype, out_dtype, act, M, N, K):
    wide = 2 if act == Q.ACT_SWIGLU else 1
    x, w = operands(M, N, K, dtype, wide)
    check(x, w, out_dtype, act=act)
    check(x, w, out_dtype, act=act, bias=rand((wide * N,), 3, dtype), gate=rand((N,), 4), residual=rand((M, N), 5, out_dtype))


@pytest.mark.parametrize("M", [1, 2, 3, 8, 15, 16, 17, 31, 33, 64, 65, 96, 127, 128, 129, 255, 256, 257, 384, 511, 513, 700, 1025, 2100])
def test_rows(M):
    x, w = operands(M, 768, 1280, BF)
    check(x, w, BF, bias=rand((768,), 6, BF), residual=rand((M, 768), 7, BF))


@pytest.mark.parametrize("N", [1, 2, 8, 31, 32, 33, 63, 64, 65, 100, 127, 129, 250, 255, 257, 1001, 4111])
@pytest.mark.parametrize("M", [5, 300])
def test_odd_widths(M, N):
    x, w = operands(M, N, 320, BF)
    check(x, w, BF, bias=rand((N,), 8, BF), act=Q.ACT_GELU)
    x, w = operands(M, N, 320, HF, 2)
    check(x, w, F32, bias=rand((2 * N,), 9, HF), act=Q.ACT_SWIGLU)


@pytest.mark.parametrize("K", [1, 3, 8, 15, 16, 40, 63, 64, 65, 100, 127, 200, 1000, 4099, 14336])
@pytest.mark.parametrize("M", [1, 40, 600])
def test_odd_depths(M, K):
    """K may be odd as long as rows start on 16 bytes; what follows a row's K
    values in memory is not read into the product."""
    pad = -(-K // 8) * 8 + 8
    x = torch.full((M, pad), float("nan"), dtype=BF, device="cuda")
    w = torch.full((320, pad), float("nan"), dtype=BF, device="cuda")
    x[:, :K], w[:, :K] = operands(M, 320, K, BF)
    check(x[:, :K], w[:, :K], F32)
    check(x[:, :K], w[:, :K], BF)


@pytest.mark.parametrize("M", [3, 200, 1200])
def test_strided_rows_and_neighbours_left_alone(M):
    """Operands and output inside wider rows; what lies beside and behind the
    output stays as it was."""
    N, K = 328, 448
    x, w = rand((M, K + 64), 10, BF)[:, 32 : 32 + K], rand((N, K + 16), 11, BF, K**-0.5)[:, 8 : 8 + K]
    buf = torch.full((M + 5, N + 40), 7.0, dtype=BF, device="cuda")
    res = rand((M, N + 8), 12, BF)[:, :N]
    out = buf[:M, 16 : 16 + N]
    got = check(x, w, BF, residual=res, out=out)
    assert got.data_ptr() == out.data_ptr()
    buf[:M, 16 : 16 + N] = 7.0
    assert bool((buf == 7.0).all())


@pytest.mark.parametrize("M", [1, 64, 300, 900])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_residual_in_place(M, out_dtype):
    x, w = operands(M, 640, 512, BF)
    stream = rand((M, 640), 13, out_dtype)
    gate = rand((640,), 14)
    want = Q.linear_16bit(x, w, gate=gate, residual=stream.clone(), out_dtype=out_dtype)
    check(x, w, out_dtype, gate=gate, residual=stream, out=stream)
    assert torch.equal(stream, want)


@pytest.mark.parametrize("M,N,K", [(1, 3584, 3584), (4, 3584, 14336), (96, 4608, 3584), (700, 3584, 14336), (2048, 4608, 3584)])
def test_model_sizes(M, N, K):
    x, w = operands(M, N, K, BF)
    check(x, w, F32, bias=rand((N,), 15, BF), residual=rand((M, N), 16))


def test_large_and_lowest_values():
    """Infinities and saturating values where the formula has them: a silu or
    GELU of a large negative is 0, of a large positive the value itself."""
    x = torch.zeros(4, 64, dtype=BF, device="cuda")
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = 1e4, -1e4, 3e38, -3e38
    w = torch.zeros(64, 64, dtype=BF, device="cuda")
    w[:, 0] = 1.0
    for act in (Q.ACT_SILU, Q.ACT_GELU):
        y = Q.linear_16bit(x, w, act=act, out_dtype=F32)
        assert bool((y[0] == x[0, 0].float()).all()) and not y[1].any()
        assert bool((y[2] == x[2, 0].float()).all()) and not y[3].any()
    y = Q.linear_16bit(x, torch.cat([w, w]), act=Q.ACT_SWIGLU, out_dtype=F32)
    assert bool((y[0] == x[0, 0].float() ** 2).all()) and not y[1].any() and bool(y[2].isinf().all())
    x[0, 5] = float("nan")
    y = Q.linear_16bit(x, w, out_dtype=F32)
    assert bool(y[0].isnan().all()) and bool(torch.isfinite(y[1:]).all())


def test_same_result_every_time_and_on_two_streams_at_once():
    cases = [operands(M, 1280, 2048, BF, seed=20 + M) for M in (1, 48, 300, 1100)]
    first = [Q.linear_16bit(x, w) for x, w in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append([Q.linear_16bit(x, w) for x, w in cases])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, first))
    Q.prompt_ops_check()


def test_captured_and_replayed():
    x, w = operands(40, 512, 768, BF)
    x2, w2 = operands(700, 512, 768, BF, seed=30)
    out, out2 = torch.empty(40, 512, dtype=BF, device="cuda"), torch.empty(700, 512, dtype=BF, device="cuda")
    Q.linear_16bit(x, w, out=out)
    Q.linear_16bit(x2, w2, out=out2)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        Q.linear_16bit(x, w, out=out)
        Q.linear_16bit(x2, w2, out=out2)
    x.copy_(rand((40, 768), 31, BF))
    x2.copy_(rand((700, 768), 32, BF))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, Q.linear_16bit(x, w)) and torch.equal(out2, Q.linear_16bit(x2, w2))
    Q.prompt_ops_check()


def test_offsets_past_32_bits():
    """Output rows beyond 2^31 elements of their buffer."""
    M, N, K = 300, 64, 128
    ld = 7_400_000  # (M - 1) * ld > 2^31
    buf = torch.empty(M * ld, dtype=BF, device="cuda")
    out = buf.as_strided((M, N), (ld, 1))
    x, w = operands(M, N, K, BF)
    check(x, w, BF, out=out)


def test_empty_call():
    assert Q.linear_16bit(torch.empty(0, 64, dtype=BF, device="cuda"), rand((32, 64), 33, BF)).shape == (0, 32)


def test_binding_refuses():
    x, w = operands(8, 64, 64, BF)
    for kw in (dict(w=w.half()), dict(w=w[:, :32]), dict(bias=rand((63,), 34, BF)), dict(bias=rand((64,), 34)),
               dict(gate=rand((64,), 35, BF)), dict(residual=rand((8, 64), 36)), dict(out_dtype=HF), dict(out=x),
               dict(out=rand((8, 64), 37)[:, ::1].t().contiguous().t()), dict(w=w[:63], act=Q.ACT_SWIGLU),
               dict(bias=rand((72,), 38, BF)[1:65]), dict(x=rand((8, 68), 39, BF)[:, :64]), dict(w=w.cpu())):
        args = dict(x=x, w=w, out_dtype=BF)
        args.update(kw)
        with pytest.raises(Q.QIError):
            Q.linear_16bit(**args)
    buf = rand((8, 72), 40, BF)
    with pytest.raises(Q.QIError):  # residual shifted against out
        Q.linear_16bit(x, w, residual=buf[:, :64], out=buf[:, 8:])


@pytest.mark.parametrize("M", [3, 130, 600])
@pytest.mark.parametrize("act", [Q.ACT_NONE, Q.ACT_GELU, Q.ACT_SWIGLU])
def test_long_sums_in_fp32(M, act):
    """K past the length from which FP32 outputs add their accumulators up in
    parts of 2048: the error stays that of such a part.  Of n = 2048 / 16 = 128
    additions that round towards zero, on a sum that grows as the square root of
    their number, each loses 2^-24 of the sum on average: 2/3 n 2^-24 = 5.1e-6 of
    the part, so of the whole (1 / 7 of what K = 14336 in one sum loses).  GELU
    has a slope of at most 1.13, SwiGLU two such factors, one under a slope of 1.1."""
    bound = {Q.ACT_NONE: 5.1e-6, Q.ACT_GELU: 5.8e-6, Q.ACT_SWIGLU: 1.1e-5}[act]
    wide = 2 if act == Q.ACT_SWIGLU else 1
    for K in (4104, 14336):
        x, w = operands(M, 328, K, BF, wide, seed=60 + M)
        got = check(x, w, F32, act=act)
        want, _ = reference(x, w, None, act, None, None, F32)
        assert float((got.double() - want).norm() / want.norm()) <= bound
        # in place, with everything in the epilogue
        stream = rand((M, 328), 61)
        check(x, w, F32, act=act, bias=rand((wide * 328,), 62, BF), gate=rand((328,), 63), residual=stream, out=stream)


@pytest.mark.parametrize("M,N", [(130, 328), (2100, 4104)])
@pytest.mark.parametrize("K", [4160, 6200, 8192, 12288, 16384])
@pytest.mark.parametrize("act", [Q.ACT_NONE, Q.ACT_SWIGLU])
def test_long_sums_of_even_and_odd_parts(M, N, K, act):
    """2 to 8 parts of 2048, in the first tile of a CTA pair and in later ones:
    a tile's last part may be in either accumulator.  Bounds as above."""
    wide = 2 if act == Q.ACT_SWIGLU else 1
    x, w = operands(M, N, K, BF, wide, seed=70 + K)
    stream = rand((M, N), 71)
    got = check(x, w, F32, act=act, residual=stream)
    want, _ = reference(x, w, None, act, None, stream, F32)
    assert float((got.double() - want).norm() / want.norm()) <= (1.1e-5 if wide == 2 else 5.1e-6)
