"""The example decoder: cache, attention, eviction and log probabilities used together."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "answer.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("answer", _PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture(scope="module")
def model(example):
    return example.build(vocab=777, width=256, heads=4, cached=2, head_dim=64)


def _prompts(*lengths):
    g = torch.Generator().manual_seed(3)
    return [torch.randint(777, (n,), generator=g) for n in lengths]


@pytest.mark.parametrize("lengths, keep", [((70, 33, 1), 40), ((130,), 256)])
def test_graph_answers_as_eager(example, model, lengths, keep):
    torch.manual_seed(0)
    a = example.answer(model, _prompts(*lengths), 9, keep, 8, graph=False)
    torch.manual_seed(0)
    b = example.answer(model, _prompts(*lengths), 9, keep, 8, graph=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.isfinite(a[1]).all() and (a[1] <= 0).all()
    assert (a[0] >= 0).all() and (a[0] < 777).all()
    held = torch.tensor([min(n, keep) + 8 for n in lengths])
    assert torch.equal(b[2].held.cpu(), held.int())
    assert torch.equal(b[2].pos.cpu(), torch.tensor(lengths) + 8)


def test_weights_add_up(example, model):
    """Every row's attention weights of a query head sum to 1, whatever was read and cut."""
    a = example.Answers(model, 2, 100)
    with torch.no_grad():
        a.read(_prompts(90, 50))
    heads = model.blocks[0].split[0] // model.cached
    for w in a.weights:
        got = w.double().sum(-1).cpu()
        want = heads * torch.tensor([90.0, 50.0]).double()[:, None]
        # sums of up to 360 rows of weights, each rounded to 16 bits at most
        assert ((got - want).abs() <= want * 2.0 ** -8).all()


def test_tuning_lowers_the_loss(example):
    model = example.build(seed=1, vocab=500, width=256, heads=4, cached=1, head_dim=32)
    losses = example.tune(model, _texts(500), 6)
    assert all(b < a for a, b in zip(losses, losses[1:]))


def test_tuning_gradient(example):
    """The gains' gradient against torch's log_softmax over the same logits, in fp32."""
    model = example.build(seed=1, vocab=500, width=256, heads=4, cached=1, head_dim=32)
    texts = _texts(500)
    with torch.no_grad():
        hidden = example.Answers(model, len(texts), 64).read(texts)
    target = torch.randint(500, (len(hidden),), device="cuda")
    grads = []
    for plain in (False, True):
        model.norm.weight.grad = None
        logits = model.logits(hidden)
        logits.retain_grad()
        if plain:
            lp = torch.log_softmax(logits.double(), -1).gather(1, target[:, None])
        else:
            lp = example.token_logprobs(logits, target).logprob
        (-lp.mean()).backward()
        grads.append(logits.grad.double())
    # both are rounded to bf16 once: half a unit in the last place each, and one for the sums
    assert ((grads[0] - grads[1]).abs() <= 2.0 ** -7 * grads[1].abs() + 1e-9).all()


def _texts(vocab):
    g = torch.Generator().manual_seed(5)
    return [torch.randint(vocab, (n,), generator=g) for n in (60, 31)]
