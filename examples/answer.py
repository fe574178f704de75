"""A small decoder of packed linear layers that answers, from its prompts to the scores of what it
said: the cache, the attention over it, its eviction and the log probabilities used together.

    python examples/answer.py [--sequences 4] [--prompt 300] [--new 64] [--keep 128]

Weights are random, so the answers mean nothing; what the calls do to them does.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from if_i_could_turn_back_time_amd import (KVCache, cache_append, cache_attention,  # noqa: E402
                                           cache_evict, quantize_module, token_logprobs)


class Norm(nn.Module):
    def __init__(self, width: int):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(width))

    def forward(self, x):
        x32 = x.float()
        x32 = x32 * torch.rsqrt(x32.square().mean(-1, keepdim=True) + 1e-6)
        return (x32 * self.weight).to(x.dtype)


def rotated(x, pos):
    """x [tokens, heads, D] turned by its tokens' places."""
    half = x.shape[-1] // 2
    f = 10000.0 ** (-torch.arange(half, device=x.device) / half)
    a = (pos[:, None] * f)[:, None]
    u, v = x.float().chunk(2, -1)
    return torch.cat([u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()], -1).to(x.dtype)


class Block(nn.Module):
    def __init__(self, width: int, heads: int, cached: int, head_dim: int):
        super().__init__()
        self.split = [heads, cached, cached]
        self.D = head_dim
        self.norm, self.norm2 = Norm(width), Norm(width)
        self.qkv = nn.Linear(width, sum(self.split) * head_dim, bias=False)
        self.out = nn.Linear(heads * head_dim, width, bias=False)
        self.up = nn.Linear(width, 4 * width, bias=False)
        self.down = nn.Linear(2 * width, width, bias=False)

    def forward(self, x, pos, cache, seqs, weights):
        """``seqs``: the sequences' table, what they held before, with these tokens, and the
        further arguments of the calls."""
        table, before, after, cu, more = seqs
        q, k, v = self.qkv(self.norm(x)).unflatten(-1, (-1, self.D)).split(self.split, 1)
        cache_append(cache, rotated(k, pos), v, table, before, cu, max_new=more["max_new"])
        y = cache_attention(rotated(q, pos), cache, table, after, cu, weights=weights, **more)
        x = x + self.out(y.flatten(1))
        a, b = self.up(self.norm2(x)).chunk(2, -1)
        return x + self.down(nn.functional.silu(a) * b)


class Decoder(nn.Module):
    def __init__(self, vocab: int = 2000, width: int = 512, layers: int = 2, heads: int = 8,
                 cached: int = 2, head_dim: int = 64):
        super().__init__()
        self.embed = nn.Embedding(vocab, width)
        self.blocks = nn.ModuleList(Block(width, heads, cached, head_dim) for _ in range(layers))
        self.norm = Norm(width)
        self.head = nn.Linear(width, vocab, bias=False)
        self.cached, self.head_dim = cached, head_dim

    def hidden(self, tokens, pos, caches, seqs, weights):
        x = self.embed(tokens)
        for block, cache, w in zip(self.blocks, caches, weights):
            x = block(x, pos, cache, seqs, w)
        return x

    def logits(self, hidden):
        return self.head(self.norm(hidden))


class Answers:
    """Sequences that a model is answering: a pool of pages a layer, two tables of them (a
    sequence moves to the other when it is cut), and what every token was attended to."""

    def __init__(self, model: Decoder, sequences: int, longest: int, page: int = 64):
        dev = model.head.codes.device
        self.model, self.longest = model, longest
        per = -(-longest // page)
        self.table, self.spare = torch.randperm(
            2 * sequences * per, device=dev).int().view(2, sequences, per)
        self.caches = [KVCache.new(2 * sequences * per, model.cached, model.head_dim, page, dev)
                       for _ in model.blocks]
        self.weights = [torch.zeros(sequences, model.cached, longest, device=dev)
                        for _ in model.blocks]
        self.held = torch.zeros(sequences, dtype=torch.int32, device=dev)  # cached tokens
        self.pos = torch.zeros(sequences, dtype=torch.int64, device=dev)   # tokens so far
        self.token = torch.zeros(sequences, dtype=torch.int64, device=dev)
        self.logprob = torch.zeros(sequences, device=dev)

    def _said(self, logits):
        """Takes the likeliest token."""
        r = token_logprobs(logits, self.token, top=1)
        self.token.copy_(r.top_ids[:, 0])
        self.logprob.copy_(r.top_logprobs[:, 0])

    def read(self, prompts: list[torch.Tensor]):
        """Takes the sequences' prompts in one pass; their hidden states."""
        dev = self.held.device
        n = torch.tensor([len(p) for p in prompts])
        cu = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).int().to(dev)
        pos = torch.cat([torch.arange(len(p)) for p in prompts]).to(dev)
        most, n = int(n.max()), n.to(dev)
        seqs = (self.table, self.held, self.held + n.int(), cu,
                {"max_new": most, "max_len": most})
        hidden = self.model.hidden(torch.cat(prompts).to(dev), pos, self.caches, seqs,
                                   self.weights)
        self.held += n.int()
        self.pos += n
        self._said(self.model.logits(hidden[cu[1:].long() - 1]))
        return hidden

    def cut(self, keep: int, recent: int):
        """Leaves every sequence its ``recent`` last tokens and, up to ``keep``, those that were
        attended to most, for each layer and cached head by itself."""
        for cache, weights in zip(self.caches, self.weights):
            r = cache_evict(cache, self.table, self.held, weights, keep, recent, self.spare,
                            max_len=self.longest)
            weights.zero_()
            weights[..., :keep] = r.weights
        self.held.copy_(r.lens)
        old = self.table.clone()
        self.table.copy_(self.spare)
        self.spare.copy_(old)

    def step(self):
        """One more token of every sequence; in place, so that it can be captured."""
        seqs = (self.table, self.held, self.held + 1, None,
                {"max_new": 1, "max_len": self.longest})
        hidden = self.model.hidden(self.token, self.pos, self.caches, seqs, self.weights)
        self._said(self.model.logits(hidden))
        self.held += 1
        self.pos += 1

    def captured_step(self):
        """:meth:`step` as a HIP graph, with the state as it was before; call ``replay()``."""
        state = [self.held, self.pos, self.token, self.logprob, *self.weights]
        state += [x.view(torch.uint8) for cache in self.caches for x in cache]
        was = [x.clone() for x in state]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.step()
        for x, y in zip(state, was):
            x.copy_(y)
        return graph


@torch.no_grad()
def answer(model: Decoder, prompts: list[torch.Tensor], new: int, keep: int, recent: int,
           graph: bool = True):
    """``new`` tokens for each prompt with their log probabilities; beside the prompts no more
    than ``keep`` tokens a sequence are held when they begin."""
    longest = max(max(len(p) for p in prompts), keep) + new
    a = Answers(model, len(prompts), longest)
    a.read(prompts)
    a.cut(keep, recent)
    said = [(a.token.clone(), a.logprob.clone())]
    step = a.captured_step().replay if graph else a.step
    for _ in range(new - 1):
        step()
        said.append((a.token.clone(), a.logprob.clone()))
    tokens, logprobs = (torch.stack(x, 1) for x in zip(*said))
    return tokens, logprobs, a


def tune(model: Decoder, texts: list[torch.Tensor], steps: int, rate: float = 0.05):
    """Makes ``texts`` likelier by the last norm's gains (the packed layers are frozen, the
    gradient goes through the head's): the losses of the steps."""
    with torch.no_grad():
        a = Answers(model, len(texts), max(len(t) for t in texts))
        hidden = a.read(texts)
    following = torch.cat([torch.cat([t[1:], t.new_full((1,), -100)]) for t in texts])
    following = following.to(hidden.device)  # the last of a text has none
    gains = torch.optim.SGD([model.norm.weight], lr=rate)
    losses = []
    for _ in range(steps):
        r = token_logprobs(model.logits(hidden), following)
        loss = -r.logprob.sum() / (following >= 0).sum()
        gains.zero_grad()
        loss.backward()
        gains.step()
        losses.append(float(loss.detach()))
    return losses


def build(seed: int = 0, **sizes) -> Decoder:
    """A decoder with random weights, its linear layers packed as E2M1."""
    torch.manual_seed(seed)
    model = quantize_module(Decoder(**sizes), 4, fmt="e2m1").cuda()
    model.embed.bfloat16()
    return model


def main(argv=None) -> int:
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("sequences", 4), ("prompt", 300), ("new", 64), ("keep", 128),
                        ("recent", 32)):
        p.add_argument("--" + name, type=int, default=value)
    a = p.parse_args(argv)
    model = build()
    lengths = [max(1, a.prompt - 37 * i) for i in range(a.sequences)]
    prompts = [torch.randint(model.embed.num_embeddings, (n,)) for n in lengths]
    tokens, logprobs, state = answer(model, prompts, a.new, a.keep, a.recent)
    for n, held, t, lp in zip(lengths, state.held.tolist(), tokens, logprobs):
        print(f"prompt of {n}: {held} tokens held, {t[:8].tolist()} ..., "
              f"mean log probability {lp.mean():.3f}")
    print("loss of the prompts:", *(f"{x:.4f}" for x in tune(model, prompts, 5)))
    return 0


if __name__ == "__main__":
    sys.exit(main())
