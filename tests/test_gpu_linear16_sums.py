"""Accuracy of qi_linear_16bit's FP32 sums against 64 bits, for long K and in
norm: sharper than the element bounds of a K-long sum, which grow with K.

The tensor cores truncate: every product and every running sum of one of the
kernel's parts of 768 values of K at most loses at most one step of 2^-23 of that sum;
the parts' sums (K / 512 at most, and 8 warps') are rounded to nearest, again at
most 2^-23 each.
"""
import pytest
import torch

import qib200 as Q

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rand(shape, seed, dtype=F32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dtype,out_dtype", [(HF, HF), (BF, BF), (HF, F32), (BF, F32)])
@pytest.mark.parametrize("M", [1, 8, 16, 17, 300])
@pytest.mark.parametrize("act", [Q.ACT_NONE, Q.ACT_SWIGLU])
def test_long_sums_of_one_sign(dtype, out_dtype, M, act):
    """A million products of one sign: a single truncated sum would lose 7e-3 of
    them (measured), so would its 16-bit result.  Per element, with T the sum
    and h the half step of out: e = (768 + K / 512 + 16) 2^-23 T; silu of these
    sums (about 40) is the sum itself, plus 2^-19; SwiGLU multiplies two of them."""
    K, N = (1 << 20) + 8, 32
    wide = 2 if act == Q.ACT_SWIGLU else 1
    x, w = rand((M, K), 1, dtype, 2.0**-7).abs(), rand((wide * N, K), 2, dtype, 2.0**-7).abs()
    t = x.double() @ w.double().T
    assert 30 < float(t.min()) and float(t.max()) < 60
    e = (768 + K / 512 + 16) * 2**-23 * t
    want = t
    if act == Q.ACT_SWIGLU:
        s, u = t[:, :N] * torch.sigmoid(t[:, :N]), t[:, N:]
        es = e[:, :N] + 2**-19 * s
        want, e = s * u, es * u + (s + es) * e[:, N:] + 2**-23 * s * u
    tol = e + torch.finfo(out_dtype).eps / 2 * (want + e)
    got = Q.linear_16bit(x, w, act=act, out_dtype=out_dtype)
    torch.cuda.synchronize()
    Q.prompt_ops_check()
    assert float(((got.double() - want).abs() / tol).max()) <= 1


@pytest.mark.parametrize("out_dtype,K", [(HF, 16392), (HF, 20480), (BF, 131080), (BF, 135168)])
@pytest.mark.parametrize("M,N", [(130, 328), (2100, 1000)])
def test_first_lengths_in_parts(out_dtype, K, M, N):
    """The first K from which 16-bit outputs are made of parts, with everything in
    the epilogue, in a CTA pair's first tile and in later ones."""
    dtype = out_dtype
    x, w = rand((M, K), 3, dtype), rand((N, K), 4, dtype, K**-0.5)
    bias, gate, res = rand((N,), 5, dtype), rand((N,), 6), rand((M, N), 7, out_dtype)
    t = x.double().abs() @ w.double().abs().T + bias.double().abs()
    y = (x.double() @ w.double().T + bias.double()) * gate.double()
    e = (768 + K / 512 + 17) * 2**-23 * t * gate.double().abs() + 2**-23 * y.abs()
    want = y + res.double()
    e = e + 2**-23 * want.abs()
    tol = e + torch.finfo(out_dtype).eps / 2 * (want.abs() + e)
    stream = res.clone()
    got = Q.linear_16bit(x, w, bias=bias, gate=gate, residual=stream, out=stream)
    torch.cuda.synchronize()
    Q.prompt_ops_check()
    assert got.data_ptr() == stream.data_ptr()
    assert float(((got.double() - want).abs() / tol).max()) <= 1


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 16, 17, 130, 600])
@pytest.mark.parametrize("K", [64, 512, 520, 768, 776, 1000, 1032, 1544, 2048, 3584, 4096, 4104, 18944])
def test_fp32_results_in_norm(dtype, M, K):
    """FP32 outputs of every kernel and epilogue in norm, with random signs.  Of n
    additions to one sum, which grows as the square root of their number, each
    loses at most 2^-23 of it: 2/3 n 2^-23 of the result.  n = K / 16, at most 48
    (parts of 768, SwiGLU 24 of 384); with up to 16 rows eight warps share K.  A sum of few
    terms, of parts or of warps adds 2^-22.  The loss goes with the sums' size s,
    not with the result's: under a slope of 1.13 (silu, GELU) or times the other
    factor (SwiGLU) it is s times theirs; their own arithmetic adds 2^-18."""
    N = 328
    x, w, w2 = rand((M, K), 11, dtype), rand((N, K), 12, dtype, K**-0.5), rand((N, K), 13, dtype, K**-0.5)
    bias, gate, res = rand((N,), 14, dtype), rand((N,), 15), rand((M, N), 16)
    n = min(48, K / 128 if M <= 16 else K / 16)
    n_wide = min(24, K / 128 if M <= 8 else K / 16)
    b, b_wide = (2 / 3 * m * 2**-23 + 2**-22 for m in (n, n_wide))
    a, u = x.double() @ w.double().T, x.double() @ w2.double().T

    def close(got, want, bound):
        torch.cuda.synchronize()
        Q.prompt_ops_check()
        assert got.dtype == F32
        assert float((got.double() - want).norm()) <= bound

    close(Q.linear_16bit(x, w, out_dtype=F32), a, b * a.norm())
    y = (a + bias.double()) * gate.double()
    close(Q.linear_16bit(x, w, bias=bias, gate=gate, residual=res, out_dtype=F32), y + res.double(),
          b * (a * gate.double()).norm() + 2**-22 * (y.norm() + res.double().norm()))
    size = a.square().mean().sqrt() * a.numel() ** 0.5
    silu = a * torch.sigmoid(a)
    close(Q.linear_16bit(x, w, act=Q.ACT_SILU, out_dtype=F32), silu, 1.13 * b * size + 2**-18 * silu.norm())
    gelu = a * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (a + 0.044715 * a**3))
    close(Q.linear_16bit(x, w, act=Q.ACT_GELU, out_dtype=F32), gelu, 1.13 * b * size + 2**-18 * gelu.norm())
    s = a.square().mean().sqrt()
    close(Q.linear_16bit(x, torch.cat([w, w2]), act=Q.ACT_SWIGLU, out_dtype=F32), silu * u,
          b_wide * s * (1.13 * u.norm() + silu.norm()) + 2**-18 * (silu * u).norm())


def test_parts_are_added_up_the_same_every_time():
    """FP32 sums in parts: eager on two streams at once, and captured and replayed
    on other inputs."""
    cases = [(rand((M, K), 20 + M, BF), rand((648, K), 21 + M, BF, K**-0.5)) for M, K in ((5, 9000), (40, 3584), (300, 3584), (2600, 1544))]
    acts = (Q.ACT_NONE, Q.ACT_SWIGLU)
    run = lambda: [Q.linear_16bit(x, w, act=a, out_dtype=F32) for x, w in cases for a in acts]  # noqa: E731
    first = run()
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for x, _ in cases:
        x.copy_(x.flip(0) * 0.5)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, run()))
    Q.prompt_ops_check()
