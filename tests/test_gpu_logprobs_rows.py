"""Token log probabilities of more rows than a grid has workgroups in one direction, and of logits
far from 0."""
import numpy as np
import pytest
import torch

from if_i_could_turn_back_time_amd import token_logprobs
from oracle import cache_oracle as O
from test_gpu_logprobs import DEV, U, _check, _rel

pytestmark = pytest.mark.gpu


def test_many_rows():
    """2^23 + 5 rows of two logits, with the gradient: against the formula in fp64, to 16 units in
    fp32's last place of the sizes that enter."""
    rows, u = 2 ** 23 + 5, 2.0 ** -24
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, 2, device="cuda", generator=g).requires_grad_(True)
    tok = torch.randint(2, (rows,), device="cuda", generator=g)
    r = token_logprobs(x, tok, top=1)
    r.logprob.sum().backward()
    with torch.no_grad():
        d = x.double()
        lse = d.logsumexp(-1)
        own = d.gather(1, tok[:, None])[:, 0]
        size = 1 + d.abs().amax(-1)
        assert bool(((r.logprob.double() - (own - lse)).abs() <= 16 * u * size).all())
        best, ids = d.max(-1)
        assert torch.equal(r.top_ids[:, 0], ids)
        assert bool(((r.top_logprobs[:, 0].double() - (best - lse)).abs() <= 16 * u * size).all())
        p = (d - lse[:, None]).exp()
        want = torch.nn.functional.one_hot(tok, 2).double() - p
        assert bool(((x.grad.double() - want).abs() <= 32 * u * size[:, None]).all())
        entropy = -(p * (d - lse[:, None])).sum(-1)
        assert bool(((r.entropy.double() - entropy).abs() <= 32 * u * size).all())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [43, 3001, 70001])
def test_masks_of_any_size(dt, V):
    """Forbidden tokens given as large negative numbers: alone at first in a thread's walk, and with
    an ordinary logit behind them."""
    g = torch.Generator().manual_seed(V)
    masks = [-1e8, -1e9, -1e10, -3e10, -1e12, -7e13, -1e15, -1e20, -3e25, -1e29, -1e30, -3.38e38]
    x = torch.randn(len(masks), V, generator=g)
    for i, mask in enumerate(masks):
        x[i, torch.rand(V, generator=g) < 0.9] = mask * (1 + 0.01 * torch.rand((), generator=g))
        x[i, :V // 2] = mask
        x[i, -1] = 1.0
    x = x.to(dt)
    tok = torch.randint(V, (len(masks),), generator=g)
    tok[::2] = V - 1
    _check(x, tok, 5, token_logprobs(x.to(DEV), tok.to(DEV), top=5))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [43, 5003])
def test_logits_of_any_size(dt, V):
    """Rows of logits from 1e7 to 1e38 and around such values, with the gradient."""
    g = torch.Generator().manual_seed(V + 1)
    sizes = [1e7, 1e8, 1e9, 1e10, 1e12, 1e20, 1e29, 1e30, 1e37]
    rows = [s * torch.randn(V, generator=g) for s in sizes]
    rows += [c + torch.randn(V, generator=g) for s in sizes for c in (s, -s)]
    x = torch.stack(rows).clamp(-3e38, 3e38).to(dt)
    tok = torch.randint(V, (len(rows),), generator=g)
    tok[::2] = x[::2].float().argmax(1)
    xd = x.to(DEV).requires_grad_(True)
    r = token_logprobs(xd, tok.to(DEV), top=3)
    _check(x, tok, 3, type(r)(*(a.detach() for a in r)))
    (r.logprob + 0.5 * r.entropy).sum().backward()
    ulp = 2.0 ** -24 if dt == torch.float32 else 2.0 ** -8
    for i in range(len(rows)):
        lp, ent, tl, ti, p, logp = O.logprobs(x[i].double().numpy(), int(tok[i]), 3)
        want = O.logprobs_grad(p, logp, ent, int(tok[i]), 1.0, 0.5)
        span = np.where(p > 0, np.abs(logp), 0.0) + ent
        bound = (2 * _rel(V) + 16 * U * (1 + span)) * p * (1 + 0.5 * span) + 16 * U * np.abs(want)
        bound = bound + ulp * (np.abs(want) + bound) + 2.0 ** -126
        got = xd.grad[i].double().cpu().numpy()
        assert (np.abs(got - want) <= bound).all(), (i, np.abs(got - want).max())
