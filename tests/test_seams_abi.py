"""Refusals of the C entry points of the embedding, the norms around a block and the head's log
probabilities: decided on the host, before any device call, so they need no GPU."""
import ctypes

import pytest
import torch

from if_i_could_turn_back_time_amd import (_capi as C, head_logprobs, residual_norm,
                                           token_embedding)

NULL, SHAPE, DTYPE, ALIGN, WORKSPACE, VALUE = -1, -2, -5, -7, -8, -10
BUF = (ctypes.c_uint8 * 1024)()
P = (ctypes.addressof(BUF) + 255) // 256 * 256
BIG = 1 << 50


def test_embedding():
    L = C.lib()

    def rc(w=P, stride=64, dt=0, V=10, K=64, t=P, rows=5, out=P):
        return L.fb_embed(w, stride, dt, V, K, t, rows, 1.0, out, None)

    def grad(g=P, stride=64, dt=0, V=10, K=64, t=P, rows=5, out=P, ws=P, nb=BIG):
        return L.fb_embed_grad(g, stride, dt, V, K, t, rows, 1.0, out, ws, nb, None)

    for f in (rc, grad):
        assert f(dt=3) == DTYPE and f(dt=-1) == DTYPE
        assert f(V=0) == SHAPE and f(K=0) == SHAPE and f(rows=-1) == SHAPE and f(stride=-1) == SHAPE
        assert f(K=(1 << 20) + 1) == SHAPE and f(rows=(1 << 30) + 1) == SHAPE
        assert f(t=None) == NULL and f(out=None) == NULL and f(t=P + 4) == ALIGN
    assert rc(w=None) == NULL and rc(w=P + 1) == ALIGN and rc(out=P + 2, dt=2) == ALIGN
    assert rc(rows=0, w=None) == 0
    assert grad(g=None) == NULL and grad(ws=None) == NULL
    assert grad(out=P + 8) == ALIGN and grad(ws=P + 16) == ALIGN and grad(g=P + 1) == ALIGN
    need = L.fb_embed_grad_workspace_bytes(5, 10, 64)
    assert need > 0 and grad(nb=need - 1) == WORKSPACE
    assert L.fb_embed_grad_workspace_bytes(0, 10, 64) == 0
    assert L.fb_embed_grad_workspace_bytes(5, 0, 64) == 0


def _norm(**kw):
    return C.FbNorm(**{**dict(x=P, branch=P, gate=P, weight=P, branch_weight=P, x_stride=64,
                              branch_stride=64, rows=5, gate_rows=5, width=64, dtype=0,
                              weight_dtype=2, branch_weight_dtype=0, gate_dtype=0, scale=1.0,
                              eps=1e-6), **kw})


BAD_NORMS = [(dict(x=None), NULL), (dict(weight=None), NULL), (dict(branch=None), NULL),
             (dict(branch=None, gate=None), NULL), (dict(rows=-1), SHAPE), (dict(rows=1 << 31), SHAPE),
             (dict(width=0), SHAPE), (dict(width=32769), SHAPE), (dict(x_stride=-1), SHAPE),
             (dict(gate_rows=0), SHAPE), (dict(dtype=3), DTYPE), (dict(weight_dtype=1), DTYPE),
             (dict(branch_weight_dtype=1), DTYPE), (dict(gate_dtype=3), DTYPE), (dict(x=P + 1), ALIGN),
             (dict(weight=P + 2), ALIGN), (dict(gate=P + 1), ALIGN), (dict(eps=-1.0), VALUE),
             (dict(eps=float("nan")), VALUE)]


@pytest.mark.parametrize("i", range(len(BAD_NORMS)))
def test_norms(i):
    kw, rc = BAD_NORMS[i]
    L, n = C.lib(), _norm(**kw)
    assert L.fb_residual_norm(ctypes.byref(n), P, P, P, None) == rc
    assert L.fb_residual_norm_grad(ctypes.byref(n), P, P, P, P, P, P, P, P, P, BIG, None) == rc
    assert L.fb_residual_norm_grad_workspace_bytes(ctypes.byref(n)) == 0


def test_norm_results():
    L, n = C.lib(), ctypes.byref(_norm())
    assert L.fb_residual_norm(None, P, P, P, None) == NULL
    assert L.fb_residual_norm(n, None, P, P, None) == NULL
    assert L.fb_residual_norm(n, P, None, P, None) == NULL
    assert L.fb_residual_norm(n, P + 1, P, P, None) == ALIGN
    assert L.fb_residual_norm(n, P, P, P + 2, None) == ALIGN
    need = L.fb_residual_norm_grad_workspace_bytes(n)

    def rc(n=n, stats=P, gh=P, dx=P, db=P, dw=P, dwb=P, dg=P, ws=P, nb=BIG):
        return L.fb_residual_norm_grad(n, stats, gh, P, dx, db, dw, dwb, dg, ws, nb, None)

    assert need > 0 and rc(nb=need - 1) == WORKSPACE and rc(ws=None) == NULL and rc(ws=P + 8) == ALIGN
    assert rc(stats=None) == NULL and rc(gh=P + 1) == ALIGN and rc(dw=P + 2) == ALIGN
    plain = ctypes.byref(_norm(branch=None, gate=None, branch_weight=None))
    assert rc(n=plain) == NULL and rc(n=plain, db=None, dwb=None) == NULL
    assert L.fb_residual_norm(ctypes.byref(_norm(rows=0, x=None)), None, None, None, None) == 0


def test_head():
    L = C.lib()

    def rc(x=P, xs=64, w=P, wst=64, dt=0, rows=5, K=64, V=10, t=P, lp=P, ent=P, st=P, ws=P, nb=BIG):
        return L.fb_head_logprobs(x, xs, w, wst, dt, rows, K, V, t, lp, ent, st, ws, nb, None)

    def grad(x=P, xs=64, w=P, wst=64, dt=0, rows=5, K=64, V=10, t=P, lp=P, ent=P, st=P, ws=P, nb=BIG,
             ge=P, gw=P):
        return L.fb_head_logprobs_grad(x, xs, w, wst, dt, rows, K, V, t, st, ent, lp, ge, P, gw, ws, nb,
                                       None)

    for f in (rc, grad):
        assert f(dt=2) == DTYPE and f(dt=-1) == DTYPE
        assert f(rows=-1) == SHAPE and f(rows=(1 << 23) + 1) == SHAPE and f(K=0) == SHAPE
        assert f(V=0) == SHAPE and f(V=(1 << 24) + 1) == SHAPE and f(xs=56) == SHAPE
        assert f(K=65, xs=72) == SHAPE and f(wst=1 << 21) == SHAPE
        assert f(xs=68) == ALIGN and f(x=P + 8) == ALIGN and f(w=P + 2) == ALIGN and f(t=P + 4) == ALIGN
        assert f(ws=P + 16) == ALIGN and f(ent=P + 2) == ALIGN and f(st=P + 1) == ALIGN
        assert f(x=None) == NULL and f(w=None) == NULL and f(t=None) == NULL and f(ws=None) == NULL
        assert f(nb=0) == WORKSPACE and f(rows=0, x=None) == 0
    assert rc(lp=None) == NULL and rc(ent=None) == NULL
    assert grad(st=None) == NULL and grad(ent=None) == NULL and grad(gw=P + 4) == ALIGN
    assert grad(rows=1 << 23, K=2048, xs=2048, wst=2048) == SHAPE
    need = L.fb_head_logprobs_workspace_bytes(5, 64, 10)
    assert need > 0 and rc(nb=need - 1) == WORKSPACE
    need = L.fb_head_logprobs_grad_workspace_bytes(5, 64, 10, 1, 1)
    assert need > 0 and grad(nb=need - 1) == WORKSPACE
    assert L.fb_head_logprobs_workspace_bytes(0, 64, 10) == 0


def test_pad_rows():
    L = C.lib()

    def rc(src=P + 2, stride=7, rows=5, K=7, dst=P, ld=8):
        return L.fb_pad_rows(src, stride, rows, K, dst, ld, None)

    assert rc(src=None) == NULL and rc(dst=None) == NULL
    assert rc(rows=0) == SHAPE and rc(rows=(1 << 24) + 1) == SHAPE and rc(K=0) == SHAPE
    assert rc(K=9) == SHAPE and rc(ld=12) == SHAPE and rc(stride=-1) == SHAPE
    assert rc(K=(1 << 20) + 1, ld=(1 << 20) + 8) == SHAPE
    assert rc(src=P + 1) == ALIGN and rc(dst=P + 8) == ALIGN


def test_packed_head():
    L = C.lib()

    def rc(wdev=P, x=P, t=P, st=P, ent=P, ge=P, gx=P, gdt=2, ws=P, nb=BIG, **kw):
        s = C.FbShape(**{**dict(N=32, K=128, B=5, group=32, fmt=1, fwht_block=0, x_dtype=1, y_dtype=2),
                         **kw})
        return L.fb_packed_head_grad(wdev, x, ctypes.byref(s), t, st, ent, P, ge, gx, gdt, ws, nb, None)

    assert rc(wdev=None) == NULL and rc(x=None) == NULL and rc(t=None) == NULL and rc(st=None) == NULL
    assert rc(ent=None) == NULL and rc(gx=None) == NULL and rc(ws=None) == NULL
    assert rc(K=100) == SHAPE and rc(group=64) == -3 and rc(fmt=7) == -4
    assert rc(fwht_block=128, x_dtype=0) == -6 and rc(fmt=0, group=128, x_dtype=1) == DTYPE
    assert rc(gdt=3) == DTYPE and rc(x_dtype=2) == DTYPE
    assert rc(wdev=P + 8) == ALIGN and rc(gx=P + 8) == ALIGN and rc(ws=P + 16) == ALIGN
    s = C.FbShape(N=32, K=128, B=5, group=32, fmt=1, fwht_block=0, x_dtype=1, y_dtype=2)
    need = L.fb_packed_head_grad_workspace_bytes(ctypes.byref(s))
    assert need > 0 and rc(nb=need - 1) == WORKSPACE
    assert L.fb_packed_head_grad_workspace_bytes(None) == 0


def test_tensors_on_the_cpu_are_refused():
    x, t = torch.randn(3, 16), torch.tensor([1, 2, 0])
    for call in (lambda: token_embedding(t, x), lambda: residual_norm(x, x[0], x),
                 lambda: head_logprobs(x.half(), x.half(), t)):
        with pytest.raises(ValueError, match="GPU"):
            call()
