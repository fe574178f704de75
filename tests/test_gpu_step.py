"""A training step's operators together: the embedding, the norms around blocks of packed layers with their
gates, and the log probabilities under a head that is the embedding's own table, against the same in torch
operations; captured and replayed."""
import pytest
import torch
from torch import nn

from if_i_could_turn_back_time_amd import (QuantLinear, head_logprobs, residual_norm,
                                           token_embedding)

pytestmark = pytest.mark.gpu
VOCAB, WIDTH, LAYERS = 700, 128, 2


class Net(nn.Module):
    """Blocks of two packed layers between sandwich norms, a gate for each channel; embedding and head
    tied."""

    def __init__(self, plain=False):
        super().__init__()
        torch.manual_seed(4)
        self.table = nn.Parameter((torch.randn(VOCAB, WIDTH) / WIDTH ** 0.5).bfloat16().cuda())
        self.gains = nn.ParameterList(nn.Parameter(1 + 0.1 * torch.randn(WIDTH).cuda())
                                      for _ in range(2 * LAYERS + 1))
        self.gates = nn.ParameterList(nn.Parameter(0.5 * torch.randn(WIDTH).cuda())
                                      for _ in range(LAYERS))
        self.up = nn.ModuleList(QuantLinear(nn.Linear(WIDTH, 256, bias=False), fmt="e2m1").cuda()
                                for _ in range(LAYERS))
        self.down = nn.ModuleList(QuantLinear(nn.Linear(256, WIDTH, bias=False), fmt="e2m1").cuda()
                                  for _ in range(LAYERS))
        self.plain = plain

    def embed(self, tokens):
        if not self.plain:
            return token_embedding(tokens, self.table, WIDTH ** 0.5)
        there = ((tokens >= 0) & (tokens < VOCAB))[..., None]
        return (torch.where(there, self.table[tokens.clamp(0, VOCAB - 1)].float(), 0.0)
                * WIDTH ** 0.5).bfloat16()

    def seam(self, x, branch, i):
        if branch is None:
            args = dict(branch=None, gate=None, branch_weight=None)
        else:
            args = dict(branch=branch, gate=self.gates[i - 1], branch_weight=self.gains[LAYERS + i])
        if not self.plain:
            return residual_norm(x, self.gains[i], scale=0.7, **args)
        h = x.float()
        if branch is not None:
            b = branch.float()
            b = b * torch.rsqrt(b.square().mean(-1, keepdim=True) + 1e-6) * args["branch_weight"]
            h = h + 0.7 * args["gate"] * b
        n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * self.gains[i]
        return h.bfloat16(), n.bfloat16()

    def forward(self, tokens, following):
        x, branch = self.embed(tokens), None
        for i in range(LAYERS):
            x, y = self.seam(x, branch, i)
            branch = self.down[i](nn.functional.silu(self.up[i](y)))
        x, y = self.seam(x, branch, LAYERS)
        if not self.plain:
            r = head_logprobs(y, self.table, following)
            return r.logprob, r.entropy
        logp = torch.log_softmax(y.flatten(0, 1).float() @ self.table.float().T, -1)
        logp = logp.view(*following.shape, VOCAB)
        there = (following >= 0) & (following < VOCAB)
        lp = logp.gather(-1, following.clamp(0, VOCAB - 1)[..., None])[..., 0]
        return torch.where(there, lp, 0.0), -(logp.exp() * logp).sum(-1)


def _batch(seed):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(VOCAB, (3, 50), generator=g)
    tokens[1, 40:] = -100
    following = torch.roll(tokens, -1, 1)
    following[:, -1] = -100
    return tokens.cuda(), following.cuda()




def _trained(net):
    for p in net.parameters():
        p.requires_grad_(not any(p is q for m in net.modules() if isinstance(m, QuantLinear)
                                 for q in m.parameters()))
    return [p for p in net.parameters() if p.requires_grad]


def test_step_against_torch():
    tokens, following = _batch(0)
    got = []
    for plain in (False, True):
        net = Net(plain)
        params = _trained(net)
        lp, ent = net(tokens, following)
        loss = -lp.sum() / 100 - 0.01 * ent.mean()
        got.append((lp.detach(), ent.detach(), *torch.autograd.grad(loss, params)))
    for i, (a, b) in enumerate(zip(*got)):
        a, b = a.double(), b.double()
        # a dozen roundings to bf16 on the way, in both: each moves a vector by 2^-9 of its length on
        # average at most, and the two runs by twice that
        assert (a - b).norm() <= 24 * 2.0 ** -8 * b.norm(), i


def test_captured_step_replays():
    net = Net()
    params = _trained(net)
    tokens, following = _batch(0)

    def step():
        lp, ent = net(tokens, following)
        loss = -lp.sum() / 100 - 0.01 * ent.mean()
        return (loss.detach(), *torch.autograd.grad(loss, params))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    for seed in (1, 2, 3):
        for t, new in zip((tokens, following), _batch(seed)):
            t.copy_(new)
        with torch.no_grad():
            net.gates[0].mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_steps_at_once_on_two_streams():
    """Two steps side by side, each on its own stream, give what they give alone."""
    net = Net()
    params = _trained(net)
    batches = [_batch(s) for s in (5, 6)]

    def step(batch):
        lp, ent = net(*batch)
        return (lp.detach(), *torch.autograd.grad(-lp.sum() - ent.sum(), params))

    alone = [step(b) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    for _ in range(3):
        got = []
        for b, s in zip(batches, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step(b))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
