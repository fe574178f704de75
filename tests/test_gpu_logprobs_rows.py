"""Token log probabilities of more rows than a grid has workgroups in one direction."""
import pytest
import torch

from if_i_could_turn_back_time_amd import token_logprobs

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
