"""The prompt operators together, as a causal text model uses them to make the
text states of qi_forward: two layers over packed prompts, then one token per
prompt against the caches the first pass filled, and the whole through a
captured graph.

Layer, on an FP32 residual stream r [T, 3584 / 4]:
  a = rms_norm(r); qkv = a Wqkv^T + b; q, k = rope(q), rope(k)
  r += attention(q, k, v) Wo^T;  m = rms_norm(r)
  r += (silu(m Wg^T) o (m Wu^T)) Wd^T

Tolerance: against 64 bits without any rounding.  Per layer a value passes at
most 8 roundings to BF16 (normed input, projection, RoPE, weights of the
softmax, attention output; normed input, gated product, and the weights'
effect on q.k counted once more), each off by at most 2^-8 of the value in
norm; random weights of norm one do not amplify them.  The residual stream
itself is FP32.  So after n layers the norm of the error is at most
8 n 2^-8 of the norm of what the layers added.
"""
import math

import pytest
import torch

import qib200 as Q

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
DIM, HEADS, KV, HD, MLP, LAYERS = 896, 7, 1, 128, 2048, 2
WIDE = HEADS + 2 * KV


def rand(shape, seed, dtype=F32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def weights():
    out = []
    for i in range(LAYERS):
        s = 100 * i
        out.append(dict(
            n1=rand((DIM,), s + 1, BF, 0.1) + 1, n2=rand((DIM,), s + 2, BF, 0.1) + 1, wqkv=rand((WIDE * HD, DIM), s + 3, BF, DIM**-0.5),
            b=rand((WIDE * HD,), s + 4, BF, 0.2), wo=rand((DIM, HEADS * HD), s + 5, BF, (HEADS * HD) ** -0.5),
            wgu=rand((2 * MLP, DIM), s + 6, BF, DIM**-0.5), wd=rand((DIM, MLP), s + 7, BF, MLP**-0.5)))
    return out


def rope(x, pos):
    """Rotates the halves of each head by pos / 10000^(2 i / HD)."""
    f = 10000.0 ** (-torch.arange(0, HD, 2, device=x.device, dtype=torch.float64) / HD)
    a = pos.double()[:, None, None] * f
    c, s = a.cos(), a.sin()
    x1, x2 = x[..., : HD // 2].double(), x[..., HD // 2 :].double()
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def layer(w, r, pos, cq, seq_k, max_k, kc, vc, slots):
    """One layer on r [T, DIM] in place; keys and values go to rows `slots` of the caches."""
    a = Q.rms_norm(r, w["n1"]).to(BF)
    qkv = Q.linear_16bit(a, w["wqkv"], bias=w["b"]).view(-1, WIDE, HD)
    q = rope(qkv[:, :HEADS], pos).to(BF)
    kc[slots] = rope(qkv[:, HEADS : HEADS + KV], pos).to(BF)
    vc[slots] = qkv[:, HEADS + KV :]
    o = Q.prompt_attention(q, kc, vc, cq, seq_k, max_k)
    Q.linear_16bit(o.view(-1, HEADS * HD), w["wo"], residual=r, out=r)
    m = Q.rms_norm(r, w["n2"]).to(BF)
    h = Q.linear_16bit(m, w["wgu"], act=Q.ACT_SWIGLU)
    Q.linear_16bit(h, w["wd"], residual=r, out=r)


def reference(ws, x, n):
    """The layers over one sequence of n positions, in 64 bits."""
    r = x.double()
    pos = torch.arange(n, device=x.device)
    norm = lambda t, g: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * g.double()  # noqa: E731
    for w in ws:
        qkv = (norm(r, w["n1"]) @ w["wqkv"].double().T + w["b"].double()).view(n, WIDE, HD)
        q, k, v = rope(qkv[:, :HEADS], pos), rope(qkv[:, HEADS : HEADS + KV], pos), qkv[:, HEADS + KV :]
        hide = torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1)
        o = torch.empty(n, HEADS, HD, dtype=torch.float64, device=x.device)
        for h in range(HEADS):
            s = (q[:, h] @ k[:, h * KV // HEADS].T / math.sqrt(HD)).masked_fill(hide, -math.inf)
            o[:, h] = torch.softmax(s, -1) @ v[:, h * KV // HEADS]
        r = r + o.reshape(n, -1) @ w["wo"].double().T
        g = norm(r, w["n2"]) @ w["wgu"].double().T
        r = r + (g[:, :MLP] * torch.sigmoid(g[:, :MLP]) * g[:, MLP:]) @ w["wd"].double().T
    return r


def test_prompts_then_one_token_each():
    lens = [77, 19, 301, 1]
    cap, B = 320, len(lens)
    ws = weights()
    full = [rand((n + 1, DIM), 900 + n) for n in lens]  # prompt rows and the token after it
    want = [reference(ws, x, x.shape[0]) for x in full]
    cq = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    kb = torch.arange(B, dtype=torch.int32, device="cuda") * cap
    caches = [(torch.full((B * cap, KV, HD), float("nan"), dtype=BF, device="cuda"),
               torch.full((B * cap, KV, HD), float("nan"), dtype=BF, device="cuda")) for _ in ws]
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    slots = torch.cat([torch.arange(n) + i * cap for i, n in enumerate(lens)]).cuda()
    n_t = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def close(got, x, ref):
        added = (ref - x.double()).norm()
        assert float((got.double() - ref).norm() / added) <= 8 * LAYERS * 2**-8

    r = torch.cat([x[:-1] for x in full])
    for w, (kc, vc) in zip(ws, caches):
        layer(w, r, pos, cq, (kb, kb + n_t), cap, kc, vc, slots)
    Q.prompt_ops_check()
    for i, n in enumerate(lens):
        close(r[cq[i] : cq[i] + n], full[i][:-1], want[i][:-1])

    # one token per prompt, through a captured graph
    one = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    x1 = torch.cat([x[-1:] for x in full])
    r1, slots1, pos1, ke1 = x1.clone(), (kb + n_t).long(), n_t.long(), kb + n_t + 1

    def step():
        for w, (kc, vc) in zip(ws, caches):
            layer(w, r1, pos1, one, (kb, ke1), cap, kc, vc, slots1)

    step()
    eager = r1.clone()
    for i in range(B):
        close(r1[i], full[i][-1], want[i][-1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r1.copy_(x1)
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    r1.copy_(x1)
    with torch.cuda.graph(g):
        step()
    for _ in range(2):
        r1.copy_(x1)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(r1, eager)
    Q.prompt_ops_check()
