"""Refusals of the prompt operators through the C ABI: every bad argument is
answered with a status before anything touches a device (pointers that are
never dereferenced stand in for buffers)."""
import ctypes

import pytest

import qib200 as Q

P = 4096  # 16-byte aligned stand-in
ARG, ALIGN, UNSUPPORTED = 1, 2, 5


def attention(**kw):
    a = dict(q=P, q_row=512, q_head=128, k=2 * P, k_row=256, k_head=128, v=3 * P, v_row=256, v_head=128, out=4 * P, o_row=512,
             o_head=128, dtype=0, heads=4, kv_heads=2, head_dim=128, qb=P, qe=P, kb=P, ke=P, batch=2, total_q=10, total_k=20,
             max_k=20, scale=0.1, causal=1, ws=0, nws=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return Q.lib().qi_prompt_attention(*a.values())


def linear(**kw):
    a = dict(x=P, ldx=64, M=4, K=64, w=1 << 20, ldw=64, N=32, dtype=0, bias=None, act=0, gate=None, residual=None, ldr=0,
             out=1 << 24, ldo=32, out_dtype=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return Q.lib().qi_linear_16bit(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(q=0), ARG), (dict(k=0), ARG), (dict(v=0), ARG), (dict(out=0), ARG), (dict(qb=0), ARG), (dict(qe=0), ARG),
    (dict(kb=0), ARG), (dict(ke=0), ARG), (dict(dtype=2), ARG), (dict(dtype=-1), ARG), (dict(heads=0), ARG),
    (dict(kv_heads=0), ARG), (dict(heads=5), ARG), (dict(head_dim=0), ARG), (dict(batch=-1), ARG), (dict(total_q=-1), ARG),
    (dict(total_k=-1), ARG), (dict(max_k=-1), ARG), (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG),
    (dict(head_dim=136), UNSUPPORTED), (dict(head_dim=100), UNSUPPORTED), (dict(heads=70000, kv_heads=70000), UNSUPPORTED),
    (dict(q=P + 8), ALIGN), (dict(k=P + 2), ALIGN), (dict(v=P + 4), ALIGN), (dict(out=P + 8), ALIGN),
    (dict(q_row=516), ALIGN), (dict(k_head=132), ALIGN), (dict(v_row=257), ALIGN), (dict(o_head=130), ALIGN),
    (dict(q_row=0), ARG), (dict(k_row=-256), ARG), (dict(k_head=0), ARG), (dict(v_row=1 << 40), ARG),
    (dict(o_row=256, o_head=128), ARG), (dict(o_row=128, o_head=1272), ARG), (dict(o_head=64), ARG), (dict(o_row=64), ARG),
    (dict(ws=P + 1, nws=1 << 30), ALIGN),
])
def test_attention_refuses(kw, status):
    assert attention(**kw) == status


def test_attention_without_work():
    assert attention(batch=0, q=0, k=0, v=0, out=0, qb=0, qe=0, kb=0, ke=0) == 0
    assert attention(total_q=0, q=0, out=0) == 0


def test_attention_workspace():
    ws = Q.lib().qi_prompt_attention_workspace
    assert ws(4, 2, 128, 2, 10, 20, 20) >= 0
    assert ws(4, 3, 128, 2, 10, 20, 20) == -ARG
    assert ws(4, 2, 130, 2, 10, 20, 20) == -UNSUPPORTED
    assert ws(4, 2, 128, 2, -1, 20, 20) == -ARG


@pytest.mark.parametrize("kw,status", [
    (dict(x=0), ARG), (dict(w=0), ARG), (dict(out=0), ARG), (dict(dtype=2), ARG), (dict(dtype=3), ARG), (dict(out_dtype=1), ARG),
    (dict(out_dtype=3), ARG), (dict(act=4), ARG), (dict(act=-1), ARG), (dict(M=-1), ARG), (dict(N=0), ARG), (dict(K=0), ARG),
    (dict(ldx=56), ARG), (dict(ldw=56), ARG), (dict(ldo=24), ARG), (dict(residual=1 << 28, ldr=24), ARG),
    (dict(ldx=68), ALIGN), (dict(ldw=66), ALIGN), (dict(ldo=36), ALIGN), (dict(out_dtype=2, ldo=34), ALIGN),
    (dict(residual=1 << 28, ldr=36), ALIGN), (dict(x=P + 8), ALIGN), (dict(w=P + 2), ALIGN), (dict(out=P + 4), ALIGN),
    (dict(bias=P + 2), ALIGN), (dict(gate=P + 4), ALIGN), (dict(residual=P + 8, ldr=32), ALIGN),
    (dict(ldx=1 << 40), ARG), (dict(N=1 << 30, act=3, ldo=1 << 30), UNSUPPORTED),
    (dict(out=P), ARG), (dict(out=P + 16), ARG), (dict(out=1 << 20), ARG), (dict(bias=1 << 24), ARG), (dict(gate=(1 << 24) + 64), ARG),
    (dict(residual=(1 << 24) + 16, ldr=32), ARG), (dict(residual=1 << 24, ldr=40), ARG),
])
def test_linear_refuses(kw, status):
    assert linear(**kw) == status


def test_linear_without_work():
    assert linear(M=0, x=0, out=0) == 0


def test_header_constants():
    assert (Q.DT_BF16, Q.DT_F16, Q.DT_F32) == (0, 1, 2)
    assert (Q.ACT_NONE, Q.ACT_GELU, Q.ACT_SILU, Q.ACT_SWIGLU) == (0, 1, 2, 3)
    src = open(Q.HEADER).read()
    assert "QI_DT_BF16 = 0, QI_DT_F16 = 1, QI_DT_F32 = 2" in src
    assert "QI_ACT_NONE = 0, QI_ACT_GELU = 1, QI_ACT_SILU = 2, QI_ACT_SWIGLU = 3" in src


def test_binding_refuses_cpu_tensors():
    import torch

    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(Q.QIError):
        Q.linear_16bit(x, x)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(Q.QIError):
        Q.prompt_attention(x.view(4, 1, 64), x.view(4, 1, 64), x.view(4, 1, 64), cu, cu, 4)
    assert ctypes.sizeof(ctypes.c_longlong) == 8


# stand-ins far apart, so that only what is changed can overlap
FAR = dict(q=1 << 20, k=1 << 24, v=1 << 25, out=1 << 26)


@pytest.mark.parametrize("kw,status", [
    (dict(q=0), ARG), (dict(k=0), ARG), (dict(v=0), ARG), (dict(out=0), ARG), (dict(qe=0), ARG), (dict(kb=0), ARG),
    (dict(out=1 << 24), ARG), (dict(out=1 << 25), ARG), (dict(out=(1 << 20) + 16), ARG),  # over k, v, part of q
    (dict(out=1 << 20, o_row=1024), ARG),  # q's memory, other strides
    (dict(q_row=1024, k_row=1024, v_row=1024, k=(1 << 20) + 1024, v=(1 << 20) + 1536, out=(1 << 20) + 512, o_row=1024), ARG),
    (dict(total_q=(1 << 30) + 1), UNSUPPORTED), (dict(total_k=(1 << 30) + 1), UNSUPPORTED),
])
def test_attention_refuses_overlaps_and_extents(kw, status):
    assert attention(**{**FAR, **kw}) == status


@pytest.mark.parametrize("kw", [dict(M=(1 << 30) + 1), dict(K=(1 << 30) + 8, ldx=(1 << 30) + 8, ldw=(1 << 30) + 8),
                                dict(N=(1 << 30) + 8, ldo=(1 << 30) + 8)])
def test_linear_refuses_extents(kw):
    assert linear(**kw) == UNSUPPORTED


@pytest.mark.parametrize("scale", [2.9e38, -2.9e38, 2.5e38])
def test_attention_refuses_scales_past_fp32_in_base_2(scale):
    """scale * log2(e) would be infinite, and times a score of 0 not a number."""
    assert attention(scale=scale) == ARG
    assert attention(scale=scale / 2, total_q=0) == 0
