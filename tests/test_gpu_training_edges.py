"""Calls at the edges of what the embedding, the norms around a block and the head's log probabilities
take: nothing to do, rows without a gradient, rows in pieces, gradients far apart, the least values."""
import pytest
import torch
from torch import nn

from if_i_could_turn_back_time_amd import (PackedWeight, QuantLinear, _capi as C, head_logprobs,
                                           residual_norm, token_embedding)
from test_gpu_head import assert_close, exact, some
from test_gpu_step import Net, _batch, _trained

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# ------------------------------------------------------------------ rows without a gradient
def _head(fmt, block, scale=1.0, V=300, K=256):
    w = torch.randn(V, K, generator=torch.Generator().manual_seed(V)) / 8
    w[0] *= scale
    return PackedWeight.quantize(w, fmt, fwht_block=block, device="cuda")


@pytest.mark.parametrize("M", [16, 60])
@pytest.mark.parametrize("fmt, block, scale, dt", [
    ("gf4", 128, 1.0, torch.float16), ("gf4", 128, 1.0, torch.bfloat16), ("e2m1", 128, 1.0, torch.float16),
    ("gf4", 0, 1.0, torch.float32), ("e2m1", 0, 1.0, torch.float32), ("e2m1", 0, 1.0, torch.bfloat16),
    ("e2m1", 0, 2.0 ** -40, torch.bfloat16)])
def test_padding_under_packed_heads(fmt, block, scale, dt, M):
    """A row without a gradient gets none under every head, whatever its hidden states hold."""
    head = _head(fmt, block, scale)
    g = torch.Generator().manual_seed(M)
    x = (torch.randint(-4, 5, (M, 256), generator=g) / 4).to(dt).cuda()
    t = torch.randint(300, (M,), generator=g).cuda()
    gl, ge = torch.randn(2, M, generator=g).cuda()
    t[7], gl[9], gl[10] = -100, 0, 0
    ge[[7, 9, 10]] = 0
    for with_entropy in (False, True):
        def grads(x):
            x = x.clone().requires_grad_(True)
            r = head_logprobs(x, head, t)
            of, by = (r.logprob, gl) if not with_entropy else ((r.logprob, r.entropy), (gl, ge))
            return torch.autograd.grad(of, x, by)[0]
        want = grads(x)
        bad = x.clone()
        bad[7], bad[9, 3], bad[10, 4] = float("nan"), float("inf"), float("nan")
        got = grads(bad)
        assert (got[[7, 9, 10]] == 0).all()
        assert torch.equal(got, want) and want[8].any()
    # an entropy's gradient alone is one, though the row has no token
    x = x.clone().requires_grad_(True)
    ge[7] = 1
    got, = torch.autograd.grad(head_logprobs(x, head, t).entropy, x, ge)
    assert got[7].any() and not got[9].any()


# ------------------------------------------------------------------ nothing to do
@pytest.mark.parametrize("V", [9, 262143, 262144, 300000])
def test_embedding_of_no_tokens(V):
    """An empty batch's gradient is 0, on both sides of the limits of the small sort."""
    for dt in (torch.bfloat16, torch.float32):
        w = torch.randn(V, 5, device="cuda").to(dt).requires_grad_(True)
        out = token_embedding(torch.empty(0, 3, dtype=torch.int64, device="cuda"), w)
        assert out.shape == (0, 3, 5)
        gw, = torch.autograd.grad(out, w, torch.empty_like(out))
        assert gw.shape == w.shape and gw.dtype == dt and not gw.any()


# ------------------------------------------------------------------ launches of 2^32 threads
def test_padding_most_rows():
    """As many rows as fb_pad_rows takes, of a width that has a workgroup for each."""
    rows, K, ld = 1 << 24, 4097, 4104
    torch.cuda.empty_cache()
    src = torch.randint(1, 30000, (K,), dtype=torch.int16, device="cuda")
    dst = torch.empty(rows, ld, dtype=torch.int16, device="cuda")
    dst[::4099] = -1
    dst[-1] = -1
    rc = C.lib().fb_pad_rows(src.data_ptr(), 0, rows, K, dst.data_ptr(), ld,
                             torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0
    want = torch.cat([src, torch.zeros(ld - K, dtype=torch.int16, device="cuda")])
    for r in range(0, rows, 1 << 18):
        assert bool((dst[r:r + (1 << 18)] == want).all()), r
    del dst
    torch.cuda.empty_cache()
