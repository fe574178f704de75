"""The embedding and its gradient against sums in 64 bits."""
import pytest
import torch

from if_i_could_turn_back_time_amd import token_embedding

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _tiny(dt):
    """Half a step at the bottom of the type's range."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def check(tokens, V, K, dt, scale=1.0, weight=None, g=None):
    gen = torch.Generator().manual_seed(V + K)
    w = torch.randn(V, K, generator=gen).to(dt).cuda() if weight is None else weight
    w = w.detach().requires_grad_(True)
    t = tokens.cuda()
    out = token_embedding(t, w, scale)
    half = torch.finfo(dt).eps / 2
    flat = t.reshape(-1).long()
    there = (flat >= 0) & (flat < V)
    safe = flat.clamp(0, V - 1)
    want = torch.where(there[:, None], w.detach().double()[safe] * scale, 0.0)
    assert out.shape == (*tokens.shape, K) and out.dtype == dt
    # one product in fp32, one rounding to the type
    tol = want.abs() * (half + 2.0 ** -23) + _tiny(dt)
    assert ((out.detach().double().reshape(-1, K) - want).abs() <= tol).all()
    if g is None:
        g = torch.randn(out.shape, generator=gen).to(dt).cuda()
    gw, = torch.autograd.grad(out, w, g)
    again, = torch.autograd.grad(token_embedding(t, w, scale), w, g)
    rows = torch.where(there[:, None], g.double().reshape(-1, K), 0.0)
    want = torch.zeros(V, K, dtype=torch.float64, device="cuda").index_add_(0, safe, rows) * scale
    total = torch.zeros(V, K, dtype=torch.float64, device="cuda").index_add_(0, safe, rows.abs())
    n = torch.zeros(V, device="cuda", dtype=torch.float64).index_add_(0, safe, there.double())
    # n - 1 additions of a row's n terms, each off by half a step of a partial sum, then the scale
    tol = (n[:, None] + 2) * 2.0 ** -24 * total * abs(scale) + half * want.abs() + _tiny(dt)
    assert gw.shape == w.shape and gw.dtype == dt
    assert ((gw.double() - want).abs() <= tol).all()
    assert (gw[n == 0] == 0).all()
    assert torch.equal(gw, again)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows, V, K", [
    (1, 1, 1), (1, 5, 8), (4, 1000, 513), (31, 7, 3), (32, 7, 16), (33, 2, 24), (64, 3, 100),
    (200, 63, 7), (200, 64, 9), (1000, 65, 33), (1000, 4097, 64), (4096, 300, 2049), (777, 50, 4096)])
def test_sizes(rows, V, K, dt):
    g = torch.Generator().manual_seed(rows)
    check(torch.randint(V, (rows,), generator=g), V, K, dt, 0.75)


@pytest.mark.parametrize("rows, V", [(16384, 1000), (16385, 1000), (20000, 70000), (100, 300000),
                                     (100001, 3), (70000, 17000000)])
def test_sorts(rows, V):
    """One workgroup's sort and the passes over memory, on both sides of their limits."""
    g = torch.Generator().manual_seed(V)
    check(torch.randint(V, (rows,), generator=g), V, 8 if V < 1 << 20 else 1, torch.bfloat16)


@pytest.mark.parametrize("rows", [1, 31, 32, 64, 65, 4096, 40000])
@pytest.mark.parametrize("kind", ["one", "padding", "most", "sorted", "outside"])
def test_runs(rows, kind):
    V, K, g = 100, 40, torch.Generator().manual_seed(5)
    t = torch.randint(V, (rows,), generator=g)
    if kind == "one":
        t[:] = 42
    elif kind == "padding":
        t[:] = -100
    elif kind == "most":  # one token has nine of ten places
        t[torch.rand(rows, generator=g) < 0.9] = V - 1
    elif kind == "sorted":
        t = t.sort().values
    else:
        t[::3], t[1::3] = V, -1
        t[::5] = 2 ** 40 + 3
    check(t, V, K, torch.float16, -2.0)


def test_shapes_types_and_strides():
    g = torch.Generator().manual_seed(0)
    t = torch.randint(50, (3, 5, 7), generator=g)
    check(t, 50, 24, torch.float32)
    check(t.int(), 50, 24, torch.bfloat16)
    check(t.transpose(0, 2), 50, 24, torch.float16)
    check(t[0, 0, 0], 50, 24, torch.float16)
    wide = torch.randn(50, 100, generator=g).bfloat16().cuda()
    check(t, 50, 33, torch.bfloat16, weight=wide[:, 7:40])
    check(t, 50, 25, torch.bfloat16, weight=wide[:, ::4])
    gr = torch.randn(3, 5, 7, 48, generator=g).bfloat16().cuda()
    check(t, 50, 24, torch.bfloat16, g=gr[..., ::2])
    check(t, 50, 24, torch.bfloat16, g=gr[..., 1:25])
    check(t, 50, 24, torch.bfloat16, g=gr[:1, :1, :1, :24].expand(3, 5, 7, 24))


def test_offsets_beyond_32_bits():
    V, K = 1_100_000, 2048
    w = torch.zeros(V, K, device="cuda", dtype=torch.bfloat16)
    t = torch.tensor([V - 1, 5, V - 2, V - 1, 1048577, 524289], device="cuda")
    w[t] = torch.randn(6, K, device="cuda").bfloat16()
    w.requires_grad_(True)
    out = token_embedding(t, w)
    assert torch.equal(out, w.detach()[t])
    g = torch.randint(-8, 9, (6, K), device="cuda").bfloat16()
    gw, = torch.autograd.grad(out, w, g)
    assert torch.equal(gw[t], torch.stack([g[0] + g[3], g[1], g[2], g[0] + g[3], g[4], g[5]]))
    gw[t] = 0
    assert not gw.view(torch.int16).any()


def test_no_tokens():
    w = torch.randn(9, 4, device="cuda", requires_grad=True)
    out = token_embedding(torch.empty(2, 0, dtype=torch.int64, device="cuda"), w)
    assert out.shape == (2, 0, 4)
    gw, = torch.autograd.grad(out.sum(), w)
    assert torch.equal(gw, torch.zeros_like(w))


def test_values_pass_through():
    """Infinities and NaN reach their rows, and only them."""
    w = torch.randn(9, 40, device="cuda").bfloat16()
    w[3, 5], w[4] = float("inf"), float("nan")
    t = torch.tensor([3, 1, 4, -100], device="cuda")
    out = token_embedding(t, w, 2.0)
    assert torch.equal(out[0], 2 * w[3]) and out[2].isnan().all()
    assert torch.equal(out[1], 2 * w[1]) and (out[3] == 0).all()
    w.requires_grad_(True)
    g = torch.ones(4, 40, device="cuda").bfloat16()
    g[3], g[1, 0] = float("nan"), float("inf")
    gw, = torch.autograd.grad(token_embedding(t, w), w, g)
    assert gw[1, 0] == float("inf") and (gw[1, 1:] == 1).all() and (gw[[0, 2, 5, 6, 7, 8]] == 0).all()


def test_captured_and_on_another_stream():
    w = torch.randn(500, 64, device="cuda", requires_grad=True)
    t = torch.randint(500, (4, 50), device="cuda")
    g = torch.randn(4, 50, 64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        out = token_embedding(t, w, 1.5)
        return out.detach(), torch.autograd.grad(out, w, g)[0]

    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(3):
        t.copy_(torch.randint(-1, 501, (4, 50), device="cuda"))
        g.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_refusals():
    w = torch.randn(9, 4, device="cuda", requires_grad=True)
    t = torch.tensor([1, 2], device="cuda")
    for call in [lambda: token_embedding(t.cpu(), w), lambda: token_embedding(t, w.cpu()),
                 lambda: token_embedding(t.float(), w), lambda: token_embedding(t, w[0]),
                 lambda: token_embedding(t, w.double()), lambda: token_embedding(t, w[:0]),
                 lambda: token_embedding(t, w, float("inf"))]:
        with pytest.raises((ValueError, RuntimeError)):
            call()
    gw, = torch.autograd.grad(token_embedding(t, w).sum(), w)  # the calls before left nothing behind
    assert float(gw.sum()) == 8
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(token_embedding(t, w).square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda w: token_embedding(t, w), (w,))


def test_capture_beside_an_eager_graph_is_refused():
    """An eager graph of the leaf that is still alive would lead the backward pass out of the capture."""
    w = torch.randn(9, 4, device="cuda", requires_grad=True)
    t = torch.tensor([1, 2], device="cuda")
    alive = token_embedding(t, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph, stream=side):
            token_embedding(t, w)
    torch.cuda.synchronize()
    gw, = torch.autograd.grad(alive.sum(), w)
    assert float(gw.sum()) == 8
