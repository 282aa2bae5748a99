"""Refusals of the prompt operators through the C ABI, each one change away from
a call that is not refused: the stand-in buffers (never dereferenced) lie far
apart, so that nothing but the argument under test can be at fault, and the
unchanged calls are tested to pass every check.

Without a GPU an accepted call ends where it first asks the driver for
something (QI_ERR_CUDA).  With one it would start a kernel on the stand-ins, so
these tests run only where there is none.
"""
import pytest
import torch

import qib200 as Q

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="stand-in pointers: only where no kernel can start")

ARG, ALIGN, CUDA, UNSUPPORTED = 1, 2, 3, 5
M1 = 1 << 20
NAN, INF = float("nan"), float("inf")

ATTENTION = dict(q=16 * M1, q_row=512, q_head=128, k=32 * M1, k_row=256, k_head=128, v=48 * M1, v_row=256, v_head=128, out=64 * M1,
                 o_row=512, o_head=128, dtype=0, heads=4, kv_heads=2, head_dim=128, qb=80 * M1, qe=80 * M1, kb=80 * M1, ke=80 * M1,
                 batch=2, total_q=10, total_k=20, max_k=20, scale=0.1, causal=1, ws=0, nws=0, stream=None)
LINEAR = dict(x=16 * M1, ldx=64, M=4, K=64, w=32 * M1, ldw=64, N=32, dtype=0, bias=None, act=0, gate=None, residual=None, ldr=0,
              out=48 * M1, ldo=32, out_dtype=0, stream=None)


def attention(**kw):
    assert set(kw) <= set(ATTENTION)
    return Q.lib().qi_prompt_attention(*{**ATTENTION, **kw}.values())


def linear(**kw):
    assert set(kw) <= set(LINEAR)
    return Q.lib().qi_linear_16bit(*{**LINEAR, **kw}.values())


def qkv_rows(**kw):
    """q, k and v as views into rows of 8 heads of 128 (4 + 2 + 2)."""
    at = ATTENTION["q"]
    return {**dict(q_row=1024, k=at + 1024, k_row=1024, v=at + 1536, v_row=1024, total_k=10), **kw}


WS = 96 * M1
SPLIT = dict(total_k=100000, max_k=100000, k=1 << 31, v=1 << 32)  # one that splits its keys


@pytest.mark.parametrize("kw", [
    dict(), dict(dtype=1), dict(causal=0), dict(scale=0.0), dict(scale=-1.9e38), dict(scale=1.9e38), dict(head_dim=8), dict(head_dim=72),
    dict(heads=2), dict(kv_heads=4, k_row=512, v_row=512), dict(q_head=1280, q_row=128), dict(o_row=128, o_head=1280),
    dict(out=16 * M1), dict(out=16 * M1 + 10 * 1024), dict(out=32 * M1 - 10 * 1024), dict(total_k=0, k=0, v=0, max_k=0),
    dict(total_q=1, q_row=0, o_row=-8), dict(heads=1, kv_heads=1, q_head=3, k_head=0, v_head=-1, o_head=5), qkv_rows(),
    qkv_rows(out=16 * M1, o_row=1024), dict(k_row=1024, v=32 * M1 + 512, v_row=1024), dict(SPLIT, ws=WS, nws=1 << 30), dict(ws=WS),
    dict(max_k=1 << 30, ws=WS, nws=1 << 30), dict(total_q=1 << 30, out=1 << 42), dict(total_k=1 << 30, k=1 << 42, v=1 << 43),
])
def test_attention_accepts(kw):
    assert attention(**kw) == CUDA


@pytest.mark.parametrize("kw,status", [
    (dict(q=0), ARG), (dict(k=0), ARG), (dict(v=0), ARG), (dict(out=0), ARG), (dict(qb=0), ARG), (dict(qe=0), ARG), (dict(kb=0), ARG),
    (dict(ke=0), ARG), (dict(dtype=2), ARG), (dict(dtype=3), ARG), (dict(dtype=-1), ARG), (dict(heads=0), ARG), (dict(heads=-4), ARG),
    (dict(kv_heads=0), ARG), (dict(kv_heads=-2), ARG), (dict(heads=5), ARG), (dict(head_dim=0), ARG), (dict(head_dim=-8), ARG),
    (dict(batch=-1), ARG), (dict(total_q=-1), ARG), (dict(total_k=-1), ARG), (dict(max_k=-1), ARG),
    (dict(scale=NAN), ARG), (dict(scale=INF), ARG), (dict(scale=-INF), ARG), (dict(scale=2.1e38), ARG), (dict(scale=-2.5e38), ARG),
    (dict(head_dim=136), UNSUPPORTED), (dict(head_dim=100), UNSUPPORTED), (dict(heads=65536, kv_heads=65536), UNSUPPORTED),
    (dict(total_q=(1 << 30) + 1), UNSUPPORTED), (dict(total_k=(1 << 30) + 1), UNSUPPORTED),
    (dict(q=16 * M1 + 8), ALIGN), (dict(k=32 * M1 + 2), ALIGN), (dict(v=48 * M1 + 4), ALIGN), (dict(out=64 * M1 + 8), ALIGN),
    (dict(ws=WS + 1, nws=1 << 30), ALIGN),
    (dict(q_row=516), ALIGN), (dict(q_head=132), ALIGN), (dict(k_row=260), ALIGN), (dict(k_head=132), ALIGN), (dict(v_row=257), ALIGN),
    (dict(v_head=129), ALIGN), (dict(o_row=513), ALIGN), (dict(o_head=130), ALIGN),
    (dict(q_row=0), ARG), (dict(q_head=-128), ARG), (dict(k_row=-256), ARG), (dict(k_head=0), ARG), (dict(v_row=1 << 40), ARG),
    (dict(v_head=0), ARG), (dict(o_row=-512), ARG), (dict(o_head=1 << 38), ARG),
    (dict(o_row=256), ARG), (dict(o_row=128, o_head=1272), ARG), (dict(o_head=64), ARG), (dict(o_row=64, o_head=4096), ARG),
    (dict(out=16 * M1 + 16), ARG), (dict(out=16 * M1 + 10 * 1024 - 16), ARG), (dict(out=16 * M1, o_row=1024), ARG),
    (dict(out=16 * M1, o_row=128, o_head=1280), ARG), (dict(out=32 * M1), ARG), (dict(out=48 * M1), ARG),
    (dict(out=32 * M1 + 20 * 512 - 16), ARG), (dict(out=48 * M1 - 10 * 1024 + 16), ARG),
    (qkv_rows(out=16 * M1 + 256, o_row=1024), ARG), (qkv_rows(out=16 * M1 + 1024, o_row=1024), ARG),
    (qkv_rows(out=16 * M1 + 1536, o_row=1024), ARG), (qkv_rows(out=16 * M1 + 768, o_row=1024), ARG),
    (dict(heads=5, q_row=1024, o_row=1024), ARG), (dict(q_row=1024, out=16 * M1, o_row=1024, o_head=256), ARG),
    (dict(q_row=1024, out=16 * M1 + 1536, o_row=1024), ARG), (dict(q_row=1024, out=16 * M1 + 512, o_row=1024), ARG),  # the next row's q, the same row's
    (SPLIT, ARG), (dict(SPLIT, ws=WS), ARG), (dict(SPLIT, nws=1 << 30), ARG),
])
def test_attention_refuses(kw, status):
    assert attention(**kw) == status


def test_attention_workspace_to_the_byte():
    need = Q.lib().qi_prompt_attention_workspace(4, 2, 128, 2, 10, 100000, 100000)
    assert need > 0
    assert attention(**SPLIT, ws=WS, nws=need) == CUDA
    assert attention(**SPLIT, ws=WS, nws=need - 1) == ARG


@pytest.mark.parametrize("kw", [dict(batch=0), dict(total_q=0)])
def test_attention_without_work(kw):
    """Nothing to do: no pointer is asked for, sizes, type and scale still are."""
    none = dict(q=0, k=0, v=0, out=0, qb=0, qe=0, kb=0, ke=0)
    assert attention(**kw, **none) == 0
    assert attention(**kw, **none, scale=1e38) == 0
    for bad in (dict(scale=2.5e38), dict(scale=NAN), dict(dtype=2), dict(heads=0), dict(total_k=-1)):
        assert attention(**kw, **none, **bad) == ARG
    assert attention(**kw, **none, head_dim=12) == UNSUPPORTED


R = 64 * M1  # a residual


@pytest.mark.parametrize("kw", [
    dict(), dict(dtype=1, out_dtype=1), dict(out_dtype=2), dict(act=1), dict(act=2), dict(act=3), dict(bias=R), dict(gate=R),
    dict(residual=R, ldr=32), dict(residual=48 * M1, ldr=32), dict(residual=16 * M1, ldr=64, K=32), dict(K=1), dict(K=57), dict(N=1), dict(N=25),
    dict(M=1), dict(M=1 << 20, w=1 << 40, out=1 << 41), dict(out=16 * M1 + 512), dict(out=16 * M1 - 256), dict(bias=48 * M1 + 256),
    dict(M=17, K=1 << 30, ldx=1 << 30, ldw=1 << 30, x=1 << 40, w=1 << 41, out=1 << 42),
])
def test_linear_accepts(kw):
    assert linear(**kw) == CUDA


@pytest.mark.parametrize("kw,status", [
    (dict(x=0), ARG), (dict(w=0), ARG), (dict(out=0), ARG), (dict(dtype=2), ARG), (dict(dtype=-1), ARG), (dict(dtype=2, out_dtype=2), ARG),
    (dict(out_dtype=1), ARG), (dict(dtype=1), ARG), (dict(out_dtype=3), ARG), (dict(act=4), ARG), (dict(act=-1), ARG), (dict(M=-1), ARG),
    (dict(N=0), ARG), (dict(K=0), ARG), (dict(N=-1), ARG), (dict(K=-8), ARG),
    (dict(ldx=56), ARG), (dict(ldw=56), ARG), (dict(ldo=24), ARG), (dict(residual=R, ldr=24), ARG), (dict(residual=R), ARG),
    (dict(ldx=1 << 38, x=1 << 50), ARG), (dict(ldw=1 << 38, w=1 << 50), ARG), (dict(ldo=1 << 38), ARG), (dict(residual=R, ldr=1 << 38), ARG),
    (dict(ldx=68), ALIGN), (dict(ldw=66), ALIGN), (dict(ldo=36), ALIGN), (dict(out_dtype=2, ldo=34), ALIGN),
    (dict(residual=R, ldr=36), ALIGN), (dict(residual=R, ldr=34, out_dtype=2), ALIGN),
    (dict(x=16 * M1 + 8), ALIGN), (dict(w=32 * M1 + 2), ALIGN), (dict(out=48 * M1 + 4), ALIGN), (dict(bias=R + 2), ALIGN),
    (dict(gate=R + 4), ALIGN), (dict(residual=R + 8, ldr=32), ALIGN),
    (dict(M=(1 << 30) + 1), UNSUPPORTED), (dict(K=(1 << 30) + 8, ldx=(1 << 30) + 8, ldw=(1 << 30) + 8), UNSUPPORTED),
    (dict(N=(1 << 30) + 8, ldo=(1 << 30) + 8), UNSUPPORTED), (dict(N=(1 << 29) + 8, act=3, ldo=(1 << 29) + 8), UNSUPPORTED),
    (dict(out=16 * M1), ARG), (dict(out=16 * M1 + 496), ARG), (dict(out=16 * M1 - 240), ARG), (dict(out=32 * M1), ARG),
    (dict(out=32 * M1 + 32 * 128, act=3), ARG), (dict(bias=48 * M1), ARG), (dict(bias=48 * M1 - 64, act=3), ARG), (dict(gate=48 * M1 + 240), ARG),
    (dict(residual=48 * M1 + 16, ldr=32), ARG), (dict(residual=48 * M1, ldr=40), ARG), (dict(residual=48 * M1 - 240, ldr=32), ARG),
])
def test_linear_refuses(kw, status):
    assert linear(**kw) == status


def test_linear_without_work():
    assert linear(M=0, x=0, w=0, out=0) == 0
    for bad in (dict(dtype=2), dict(out_dtype=1), dict(act=4), dict(N=0), dict(K=0)):
        assert linear(M=0, **bad) == ARG
