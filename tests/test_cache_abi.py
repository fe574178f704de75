"""Refusals of the cache's and the log probabilities' C entry points: decided on the host, before
any device call, so they need no GPU."""
import ctypes

import pytest
import torch

from if_i_could_turn_back_time_amd import KVCache, _capi as C

NULL, SHAPE, DTYPE, ALIGN, WORKSPACE = -1, -2, -5, -7, -8
BUF = (ctypes.c_uint8 * 1024)()
P = (ctypes.addressof(BUF) + 255) // 256 * 256


def _cache(**kw):
    return C.FbCache(**{**dict(k=P, v=P, k_scale=P, v_scale=P, pages=4, heads=2, head_dim=64,
                               page=64), **kw})


def _seqs(**kw):
    return C.FbSeqs(**{**dict(table=P, table_stride=2, lens=P, cu=None, seqs=3, max_pages=2,
                              tokens=3, max_new=1, max_len=100), **kw})


BAD = [(_cache(k=None), _seqs(), NULL), (_cache(v_scale=None), _seqs(), NULL),
       (_cache(), _seqs(table=None), NULL), (_cache(), _seqs(lens=None), NULL),
       (_cache(pages=0), _seqs(), SHAPE), (_cache(pages=1 << 31), _seqs(), SHAPE),
       (_cache(heads=0), _seqs(), SHAPE), (_cache(heads=5000), _seqs(), SHAPE),
       (_cache(head_dim=72), _seqs(), SHAPE), (_cache(head_dim=272), _seqs(), SHAPE),
       (_cache(head_dim=0), _seqs(), SHAPE), (_cache(page=48), _seqs(), SHAPE),
       (_cache(page=0), _seqs(), SHAPE), (_cache(), _seqs(seqs=0), SHAPE),
       (_cache(), _seqs(seqs=70000, tokens=70000), SHAPE), (_cache(), _seqs(max_pages=0), SHAPE),
       (_cache(), _seqs(table_stride=1), SHAPE), (_cache(), _seqs(tokens=2), SHAPE),
       (_cache(), _seqs(max_new=-1), SHAPE), (_cache(), _seqs(max_len=-1), SHAPE),
       (_cache(k=P + 8), _seqs(), ALIGN), (_cache(v=P + 4), _seqs(), ALIGN),
       (_cache(), _seqs(table=P + 2), ALIGN), (_cache(), _seqs(cu=P + 1), ALIGN)]


@pytest.mark.parametrize("i", range(len(BAD)))
def test_cache_and_sequences(i):
    c, s, rc = BAD[i]
    L, r = C.lib(), ctypes.byref
    assert L.fb_cache_append(r(c), r(s), P, 128, 64, P, 128, 64, 0, None) == rc
    assert L.fb_cache_attention(r(c), r(s), P, 256, 64, 4, 0, 1.0, P, P, None, 0, 0, 0, P, 0,
                                None) == rc
    assert L.fb_cache_evict(r(c), r(s), P, 200, 100, 100, 8, 2, P, 1, 1, P, P, P, None) == rc
    assert L.fb_cache_attention_workspace_bytes(r(c), r(s), 4, 0) == 0


def test_append():
    L, r = C.lib(), ctypes.byref
    c, s = _cache(), _seqs()

    def rc(k=P, v=P, dt=0, s=s):
        return L.fb_cache_append(r(c), r(s), k, 128, 64, v, 128, 64, dt, None)

    assert rc(k=None) == NULL and rc(v=None) == NULL and rc(dt=3) == DTYPE and rc(dt=-1) == DTYPE
    assert rc(k=P + 1) == ALIGN and rc(v=P + 2, dt=2) == ALIGN
    assert rc(s=_seqs(cu=P, tokens=0), k=None) == 0  # nothing to do
    assert rc(s=_seqs(cu=P, tokens=1 << 30, max_new=1 << 30)) == SHAPE


def test_attention():
    L, r = C.lib(), ctypes.byref
    c = _cache()

    def rc(q=P, hq=4, dt=0, out=P, lse=P, w=None, wt=0, ws=P, nb=1 << 40, s=_seqs()):
        return L.fb_cache_attention(r(c), r(s), q, 256, 64, hq, dt, 1.0, out, lse, w, 200, 100, wt,
                                    ws, nb, None)

    assert rc(hq=3) == SHAPE and rc(hq=1) == SHAPE and rc(dt=2) == DTYPE
    assert rc(q=None) == NULL and rc(out=None) == NULL
    assert rc(w=P, lse=None, wt=100) == NULL and rc(w=P, wt=0) == SHAPE
    assert rc(q=P + 1) == ALIGN and rc(out=P + 8) == ALIGN and rc(lse=P + 2) == ALIGN
    assert rc(w=P + 1, wt=9) == ALIGN and rc(ws=P + 16) == ALIGN
    assert rc(s=_seqs(cu=P, tokens=0), q=None) == 0
    long = _seqs(max_pages=10000, table_stride=10000, max_len=500000)
    need = L.fb_cache_attention_workspace_bytes(r(c), r(long), 4, 0)
    assert need > 0
    assert rc(s=long, ws=None) == NULL and rc(s=long, nb=need - 1) == WORKSPACE


def test_evict():
    L, r = C.lib(), ctypes.byref
    c, s = _cache(), _seqs()

    def rc(w=P, wt=100, keep=8, recent=2, nt=P, ns=1, np_=1, kept=P, nw=P, nl=P):
        return L.fb_cache_evict(r(c), r(s), w, 200, 100, wt, keep, recent, nt, ns, np_, kept, nw,
                                nl, None)

    assert rc(w=None) == NULL and rc(nt=None) == NULL and rc(kept=None) == NULL
    assert rc(nl=None) == NULL and rc(wt=0) == SHAPE and rc(keep=0) == SHAPE
    assert rc(recent=9) == SHAPE and rc(recent=-1) == SHAPE and rc(keep=65) == SHAPE
    assert rc(np_=0) == SHAPE and rc(np_=2) == SHAPE
    assert rc(w=P + 2) == ALIGN and rc(kept=P + 2) == ALIGN and rc(nw=P + 1) == ALIGN


def test_logprobs():
    L = C.lib()

    def rc(x=P, dt=0, stride=50, rows=2, vocab=50, tok=P, top=3, lp=P, ent=P, tl=P, ti=P, st=P):
        return L.fb_token_logprobs(x, dt, stride, rows, vocab, tok, top, lp, ent, tl, ti, st, None)

    assert rc(dt=3) == DTYPE and rc(rows=-1) == SHAPE and rc(vocab=0) == SHAPE
    assert rc(vocab=(1 << 30) + 1) == SHAPE and rc(top=65) == SHAPE and rc(top=-1) == SHAPE
    assert rc(top=51) == SHAPE and rc(stride=-1) == SHAPE
    assert rc(x=None) == NULL and rc(tok=None) == NULL and rc(lp=None) == NULL
    assert rc(ent=None) == NULL and rc(tl=None) == NULL and rc(ti=None) == NULL
    assert rc(x=P + 1) == ALIGN and rc(x=P + 2, dt=2) == ALIGN and rc(tok=P + 4) == ALIGN
    assert rc(ti=P + 4) == ALIGN and rc(lp=P + 2) == ALIGN
    assert rc(rows=0, x=None, tok=None) == 0

    def gr(x=P, dt=0, rows=2, vocab=50, tok=P, top=3, ti=P, st=P, ent=P, gl=P, ge=P, gt=P, gx=P):
        return L.fb_token_logprobs_grad(x, dt, 50, rows, vocab, tok, top, ti, st, ent, gl, ge, gt,
                                        gx, None)

    assert gr(dt=7) == DTYPE and gr(top=70) == SHAPE
    assert gr(st=None) == NULL and gr(gx=None) == NULL and gr(ent=None) == NULL
    assert gr(ti=None) == NULL and gr(tok=None) == NULL and gr(top=0) == NULL
    assert gr(gx=P + 1) == ALIGN and gr(gt=P + 2) == ALIGN and gr(gx=P + 2, dt=2) == ALIGN
    assert gr(rows=0) == 0


def test_native_path_refuses_host_tensors():
    """There is no CPU fallback."""
    from if_i_could_turn_back_time_amd import cache_append, cache_attention, token_logprobs
    c = KVCache.new(2, 1, 64, device="cpu")
    x = torch.zeros(1, 1, 64, dtype=torch.float16)
    i = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        cache_append(c, x, x, i, i[0])
    with pytest.raises(ValueError, match="GPU"):
        cache_attention(x, c, i, i[0])
    with pytest.raises(ValueError, match="GPU"):
        token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long))
    k, v = c.read(i[0], 40)
    assert k.shape == v.shape == (1, 40, 64) and not k.any()
    for kw in (dict(page=40), dict(head_dim=24), dict(head_dim=512)):
        with pytest.raises(ValueError):
            KVCache.new(**{**dict(pages=1, heads=1, head_dim=64, device="cpu"), **kw})
