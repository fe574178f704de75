"""Attention over the 8-bit cache and its neighbours where waits, scales, masks and bounds meet:
long runs of rows, block scales far apart, bounds that are too small, rows of no sequence."""
import numpy as np
import pytest
import torch

from if_i_could_turn_back_time_amd import KVCache, cache_append, cache_attention
from test_gpu_cache import Case

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _i32(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ weights of long runs of rows
@pytest.mark.parametrize("D,group,n", [(64, 64, 2500), (128, 64, 2100), (256, 40, 1700)])
def test_weights_of_long_runs(D, group, n):
    """Every workgroup walks its rows in six stages of LDS or more, and q (40 MB and more) does not
    stay in the L2: a stage read before its rows have arrived shows.  The reference is fp64.  A
    weight is off by exp(2 d) - 1 for d = (D + 24) u * (a score's sum of magnitudes) and by 24 u (1 +
    that sum) for the exponential; a token's sum of at most 2^10 fp32 additions in a row adds 2^10 u
    of it."""
    heads, page = 2, 64
    g = torch.Generator(device=DEV).manual_seed(D)
    cache = KVCache.new(-(-n // page), heads, D, page, DEV)
    table = torch.arange(cache.k.shape[0], dtype=torch.int32, device=DEV)[None]
    kv = torch.randn(2, n, heads, D, device=DEV, generator=g).bfloat16()
    cu, lens = _i32(0, n), _i32(n)
    cache_append(cache, kv[0], kv[1], table, _i32(0), cu)
    q = torch.randn(n, heads * group, D, device=DEV, generator=g).bfloat16()
    k, _ = cache.read(table[0], n)
    want = torch.zeros(heads, n, dtype=torch.float64, device=DEV)
    err = torch.zeros_like(want)
    seen = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
    for h in range(heads):
        kh = k[h].double()
        for j in range(h * group, (h + 1) * group):
            qj = q[:, j].double()
            p = (qj @ kh.t() * D ** -0.5).masked_fill(~seen, -torch.inf).softmax(-1)
            mags = (qj.abs() @ kh.abs().t() * D ** -0.5).masked_fill(~seen, 0).amax(-1)
            want[h] += p.sum(0)
            err[h] += (torch.expm1(2 * (D + 24) * U * mags) + 24 * U * (1 + mags)) @ p
    first = None
    for _ in range(4):
        w = torch.zeros(1, heads, n, device=DEV)
        cache_attention(q, cache, table, lens, cu, weights=w, max_len=n)
        assert bool(((w[0].double() - want).abs() <= err + 2.0 ** 10 * U * want).all())
        first = w if first is None else first
        assert torch.equal(first, w)


# ------------------------------------------------------------------ tiny scales, unwritten blocks
@pytest.mark.parametrize("fill", [0, 255])
@pytest.mark.parametrize("scale", [1e-9, 1e-30])
@pytest.mark.parametrize("new,group", [(1, 4), (5, 2), (5, 20)])
def test_tiny_scale_beside_unwritten_blocks(new, group, scale, fill):
    """Five tokens held: the rest of their chunk are blocks that hold any scale, and what is masked
    there must not come up.  A block of zero keys has the least scale of all."""
    def spoil(x):
        x[:, 0, 1] = 0
    c = Case([0], 2, 64, 64, parts=1)
    c.append([0], [5], 1.0, spoil)
    c.lens = [5]
    used = c.cache.k_scale[c.table[0].long(), :, :1].clone()
    c.cache.k_scale.fill_(fill)
    c.cache.k_scale[c.table[0].long(), :, :1] = used
    w = torch.zeros(1, 2, 128, device=DEV)
    c.attend([new], group, scale=scale, weights=w)
