"""Cases of the prompt operators: attention over packed prompts (prompt_attention) and the 16-bit linear layer with bias,
activation, gate and residual in its epilogue (linear_16bit).

run() computes a case in elementary torch operations, in 32 bits, rounded once at the end; with own = True it makes the
calls a user makes of the library.  exact() gives the same from the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _lib():
    at = os.path.join(os.getcwd(), "qwen-image.cu_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import qib200

    return qib200


# ---------------------------------------------------------------- cases
def _attn(name, q, k, heads, kv, dim, dtype, causal, layout):
    """q, k: lengths, as text.  layout: "qkv" (views into the rows of one QKV projection), "heads" ([head][token][dim]
    buffers), "slab" (queries packed, keys in a cache of a fixed capacity per sequence)."""
    c = {"op": "attention", "q": q, "k": k, "heads": heads, "kv": kv, "dim": dim, "dtype": dtype, "causal": causal, "layout": layout}
    return dict(c, name=name) if name else c


def _lin(name, m, n, k, dtype, out, act, bias, gate, residual):
    c = {"op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "out": out, "act": act, "bias": bias, "gate": gate, "residual": residual}
    return dict(c, name=name) if name else c


def listed():
    packed = "1,1024,17,333,64,512,129,40,77,255,901,2,640,31,448,100,7,768,203,58,128,385,11,290"
    token_k = "4096,1,777,2048,3000,129,1500,3583,64,2500,4000,910,333,1024,2777,1919"
    return [
        # one prompt and its negative prompt, as they are encoded before a denoising run: latency counts
        _attn("attn prompt pair", "77,19", "77,19", 28, 4, 128, "bf16", True, "qkv"),
        # a server's batch of prompts of all lengths, packed
        _attn("attn packed prompts", packed, packed, 28, 4, 128, "bf16", True, "qkv"),
        # one long prompt (a rewritten prompt with its examples, or a document)
        _attn("attn long prompt", "8192", "8192", 28, 4, 128, "bf16", True, "qkv"),
        # the joint text + image attention of two CFG halves, exact instead of quantized
        _attn("attn joint 4352", "4352,4352", "4352,4352", 24, 24, 128, "f16", False, "heads"),
        # a chunk of new tokens behind a cached prefix; heads of 64
        _attn("attn chunk", "256,100,511", "6000,2148,511", 16, 8, 64, "f16", True, "slab"),
        # one new token for each of 16 sequences
        _attn("attn one token x16", ",".join(["1"] * 16), token_k, 28, 4, 128, "bf16", True, "slab"),
        # one new token of one long sequence: the keys have to be split over the card
        _attn("attn one token 30000", "1", "30000", 28, 4, 128, "bf16", True, "slab"),
        # output projection of one token into the FP32 residual stream: latency and the weights' bytes
        _lin("linear 1 row", 1, 3584, 3584, "bf16", "f32", "none", False, False, True),
        # Q/K/V projection of a prompt pair
        _lin("linear prompt qkv", 96, 4608, 3584, "bf16", "bf16", "none", True, False, False),
        # gated MLP, first half, of packed prompts
        _lin("linear swiglu 1111", 1111, 14336, 3584, "bf16", "bf16", "swiglu", False, False, False),
        # MLP, second half, into a gated residual stream
        _lin("linear down 700", 700, 3584, 14336, "bf16", "f32", "none", True, True, True),
        # GELU MLP over the image tokens of a batch
        _lin("linear gelu 8192", 8192, 12288, 3584, "f16", "f16", "gelu", True, False, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.5:
        heads, kv = rng.choice([(28, 4), (16, 8), (24, 24), (8, 1), (32, 8), (12, 12), (20, 4)])
        dim = rng.choice([128, 128, 64, 96, 80])
        dtype = rng.choice(["bf16", "f16"])
        kind = rng.choice(["prompt", "token", "chunk", "joint"])
        if kind == "prompt":
            longest = _log(rng, 2, 6000)
            count = max(1, min(_log(rng, 1, 48), 30_000_000 // (longest * longest)))
            q = [_log(rng, 1, longest) for _ in range(count - 1)] + [longest]
            rng.shuffle(q)
            return _attn("", ",".join(map(str, q)), ",".join(map(str, q)), heads, kv, dim, dtype, True, rng.choice(["qkv", "heads"]))
        if kind == "joint":
            n, b = _log(rng, 16, 4200), rng.choice([1, 2])
            t = ",".join([str(n)] * b)
            return _attn("", t, t, heads, kv, dim, dtype, False, rng.choice(["qkv", "heads"]))
        longest = _log(rng, 8, 32000)
        count = max(1, min(_log(rng, 1, 64), 200_000 // longest))
        k = [_log(rng, 1, longest) for _ in range(count - 1)] + [longest]
        rng.shuffle(k)
        q = [1 if kind == "token" else min(x, _log(rng, 1, 512), max(1, 20_000_000 // (longest * count))) for x in k]
        return _attn("", ",".join(map(str, q)), ",".join(map(str, k)), heads, kv, dim, dtype, True, "slab")
    m = rng.choice([_log(rng, 1, 64), _log(rng, 1, 8192), _log(rng, 64, 8192)])
    k = 8 * _log(rng, 16, 1792)
    n = min(_log(rng, 64, 16384), max(64, int(3.0e11 / (m * k))))
    act = rng.choice(["none", "gelu", "silu", "swiglu"])
    n = max(16, n // 2 if act == "swiglu" else n)
    n = n // 8 * 8  # rows of the output start on 16 bytes
    dtype = rng.choice(["bf16", "f16"])
    out = rng.choice([dtype, dtype, "f32"])
    return _lin("", m, n, k, dtype, out, act, rng.random() < 0.5, rng.random() < 0.25, rng.random() < 0.5)


def _lens(text):
    return [int(x) for x in text.split(",")]


def _pairs(c):
    """Attended (query, key) pairs of one head."""
    total = 0
    for lq, lk in zip(_lens(c["q"]), _lens(c["k"])):
        if not c["causal"]:
            total += lq * lk
        else:  # query i sees keys 0 .. i + lk - lq
            n = min(lq, lk)
            total += n * lk - n * (n - 1) // 2
    return total


def work(c):
    if c["op"] == "attention":
        q, k = sum(_lens(c["q"])), sum(_lens(c["k"]))
        return {"bytes": 2 * c["dim"] * (2 * q * c["heads"] + 2 * k * c["kv"]), "flops": 4 * c["dim"] * c["heads"] * _pairs(c)}
    m, n, k, wide = c["m"], c["n"], c["k"], 2 if c["act"] == "swiglu" else 1
    o = 4 if c["out"] == "f32" else 2
    nbytes = 2 * m * k + 2 * wide * n * k + o * m * n * (2 if c["residual"] else 1)
    nbytes += 2 * wide * n * bool(c["bias"]) + 4 * n * bool(c["gate"])
    return {"bytes": nbytes, "flops": 2 * m * n * k * wide}


# ---------------------------------------------------------------- inputs
def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = _DT[c["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dt)

    if c["op"] == "attention":
        heads, kv, dim = c["heads"], c["kv"], c["dim"]
        lq, lk = _lens(c["q"]), _lens(c["k"])
        cq = torch.tensor([0] + lq, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
        if c["layout"] == "slab":
            cap = -(-max(lk) // 64) * 64
            kc, vc = normal(len(lk) * cap, kv, dim), normal(len(lk) * cap, kv, dim)
            q = normal(sum(lq), heads, dim)
            kb = torch.arange(len(lk), dtype=torch.int32, device="cuda") * cap
            ke = kb + torch.tensor(lk, dtype=torch.int32).cuda()
            seq_k = (kb, ke)
        else:
            t = sum(lq)
            if c["layout"] == "qkv":
                rows = normal(t, heads + 2 * kv, dim)
                q, kc, vc = rows[:, :heads], rows[:, heads : heads + kv], rows[:, heads + kv :]
            else:
                q, kc, vc = (normal(h, t, dim).transpose(0, 1) for h in (heads, kv, kv))
            seq_k = cq
        return {"case": c, "q": q, "k": kc, "v": vc, "seq_q": cq, "seq_k": seq_k, "max_q": max(lq), "max_k": max(lk)}
    m, n, k = c["m"], c["n"], c["k"]
    wide = 2 if c["act"] == "swiglu" else 1
    s = {"case": c, "x": normal(m, k), "w": normal(wide * n, k, scale=1.0 / math.sqrt(k))}
    s["bias"] = normal(wide * n, scale=0.5) if c["bias"] else None
    s["gate"] = torch.randn(n, device="cuda", generator=g) * 0.5 if c["gate"] else None
    s["residual"] = torch.randn(m, n, device="cuda", generator=g).to(_DT[c["out"]]) if c["residual"] else None
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if c["op"] == "attention":
        if own:
            return _lib().prompt_attention(s["q"], s["k"], s["v"], s["seq_q"], s["seq_k"], s["max_k"], causal=c["causal"])
        return _attention(s, c["causal"])
    if own:
        Q = _lib()
        act = {"none": Q.ACT_NONE, "gelu": Q.ACT_GELU, "silu": Q.ACT_SILU, "swiglu": Q.ACT_SWIGLU}[c["act"]]
        return Q.linear_16bit(s["x"], s["w"], bias=s["bias"], act=act, gate=s["gate"], residual=s["residual"], out_dtype=_DT[c["out"]])
    y = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if c["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    elif c["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif c["act"] == "swiglu":
        a, b = y[:, : c["n"]], y[:, c["n"] :]
        y = a / (1.0 + torch.exp(-a)) * b
    if s["gate"] is not None:
        y = y * s["gate"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(_DT[c["out"]])


def _attention(s, causal):
    """Padded to the longest of the batch, masked, and put back into packed rows."""
    q, k, v = s["q"], s["k"], s["v"]
    heads, kv, dim = q.shape[1], k.shape[1], q.shape[2]
    q0, q1 = s["seq_q"][:-1].long(), s["seq_q"][1:].long()
    k0, k1 = (t.long() for t in (s["seq_k"] if isinstance(s["seq_k"], tuple) else (s["seq_k"][:-1], s["seq_k"][1:])))
    lq, lk = q1 - q0, k1 - k0
    iq = torch.arange(s["max_q"], device=q.device)
    ik = torch.arange(s["max_k"], device=q.device)
    is_q = iq[None] < lq[:, None]
    at_q = torch.where(is_q, q0[:, None] + iq[None], 0)
    at_k = torch.where(ik[None] < lk[:, None], k0[:, None] + ik[None], 0)
    b = lq.numel()
    qp = q[at_q].float().view(b, s["max_q"], kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dim)
    kp = k[at_k].float().permute(0, 2, 3, 1)
    vp = v[at_k].float().permute(0, 2, 1, 3)
    sc = (qp @ kp).mul_(1.0 / math.sqrt(dim)).view(b, kv, heads // kv, s["max_q"], s["max_k"])
    last = torch.where(is_q, (iq[None] + (lk - lq)[:, None]) if causal else lk[:, None] - 1, -1)
    seen = (ik[None, None] <= last[:, :, None]) & (ik[None, None] < lk[:, None, None])
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, kv, -1, s["max_k"]) @ vp).view(b, kv, heads // kv, s["max_q"], dim)
    o = (o / torch.where(total == 0, 1.0, total)).permute(0, 3, 1, 2, 4).reshape(b, s["max_q"], heads, dim)
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    out[at_q[is_q]] = o[is_q].to(q.dtype)
    return out


# ---------------------------------------------------------------- 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "linear":
        acc = torch.matmul(s["x"].double(), s["w"].double().T)
        if s["bias"] is not None:
            acc += s["bias"].double()
        if c["act"] == "gelu":
            u = (2.0 / math.pi) ** 0.5 * (acc + 0.044715 * acc**3)
            acc = acc * torch.sigmoid(2.0 * u)  # (1 + tanh u) / 2
        elif c["act"] == "silu":
            acc = acc * torch.sigmoid(acc)
        elif c["act"] == "swiglu":
            left, right = acc.split(c["n"], dim=1)
            acc = left * torch.sigmoid(left) * right
        if s["gate"] is not None:
            acc = s["gate"].double()[None, :] * acc
        return acc if s["residual"] is None else s["residual"].double() + acc
    q, k, v = s["q"].double(), s["k"], s["v"]
    out = torch.zeros_like(q)
    group = c["heads"] // c["kv"]
    begin_q = s["seq_q"].tolist()
    begin_k = (s["seq_k"][0] if isinstance(s["seq_k"], tuple) else s["seq_k"]).tolist()
    for n, (lq, lk) in enumerate(zip(_lens(c["q"]), _lens(c["k"]))):
        rows = slice(begin_q[n], begin_q[n] + lq)
        keys = slice(begin_k[n], begin_k[n] + lk)
        for h in range(c["heads"]):
            score = q[rows, h] @ k[keys, h // group].double().T / c["dim"] ** 0.5
            if c["causal"]:
                hidden = torch.ones(lq, lk, dtype=torch.bool, device=score.device).triu_(lk - lq + 1)
                score[hidden] = -math.inf
            out[rows, h] = torch.softmax(score, dim=1) @ v[keys, h // group].double()
    return out
