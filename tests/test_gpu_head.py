"""Log probabilities under a head without its logits, against the same from logits in 64 bits."""
import pytest
import torch

from if_i_could_turn_back_time_amd import PackedWeight, QuantLinear, head_logprobs, token_logprobs

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float16, torch.bfloat16]


def exact(x, w, tokens, gl=None, ge=None):
    """logprob, entropy, grad_x, grad_w, and what bounds the gradients' terms."""
    l = x.double() @ w.double().T
    logp = torch.log_softmax(l, -1)
    p = logp.exp()
    ent = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    there = (tokens >= 0) & (tokens < w.shape[0])
    at = tokens.long().clamp(0, w.shape[0] - 1)[:, None]
    lp = torch.where(there, logp.gather(1, at)[:, 0], 0.0)
    if gl is None:
        return lp, ent
    gl = torch.where(there, gl, 0.0).double()[:, None]
    ge = ge.double()[:, None]
    G = -p * (gl + ge * (logp + ent[:, None]))
    G.scatter_add_(1, at, gl)
    return lp, ent, G @ w.double(), G.T @ x.double(), G


def some(M, V, K, dt, seed=0, padded=True):
    """Hidden states and weights that are small multiples of 1/4, so that logits are exact in fp32."""
    g = torch.Generator().manual_seed(seed + M + V + K)
    x = torch.randint(-4, 5, (M, K), generator=g).to(dt) / 4
    w = torch.randint(-2, 3, (V, K), generator=g).to(dt) / (4 if K < 100 else 16)
    t = torch.randint(V, (M,), generator=g)
    if padded:
        t[1::5] = -100
        t[4::11] = V
    gl, ge = torch.randn(2, M, generator=g)
    return [v.cuda() for v in (x, w, t, gl, ge)]


def assert_close(got, want, lp_tol=512 * U):
    # exact logits; exponentials are off by 2 U, differences of logits (less than 64) by 64 U, sums
    # over the vocabulary add at most 32 values a thread and then join: below 256 U for log z in all;
    # the entropy divides two such sums
    for a, b in zip(got, want):
        assert ((a.double() - b).abs() <= lp_tol * (2 + b.abs())).all()


def check(M, V, K, dt, seed=0):
    x, w, t, gl, ge = some(M, V, K, dt, seed)
    x.requires_grad_(True), w.requires_grad_(True)
    r = head_logprobs(x, w, t)
    lp, ent, gx, gw, G = exact(x.detach(), w.detach(), t, gl, ge)
    assert r.logprob.dtype == r.entropy.dtype == torch.float32
    assert_close((r.logprob.detach(), r.entropy.detach()), (lp, ent))
    got = torch.autograd.grad((r.logprob, r.entropy), (x, w), (gl, ge))
    again = head_logprobs(x, w, t)
    again = torch.autograd.grad((again.logprob, again.entropy), (x, w), (gl, ge))
    half = torch.finfo(dt).eps / 2
    # each value of G: 1024 U of its row's terms, then half a step; sums of V (or M) products; the result
    own = 1024 * U * (gl.abs() + 16 * ge.abs()).double()[:, None] * (G.abs() + torch.softmax(
        x.detach().double() @ w.detach().double().T, -1))
    off = half * G.abs() + own
    small = 2.0 ** -38 * (gl.abs() + 24 * ge.abs()).double()  # fp16: below G's smallest step
    dx = off @ w.detach().double().abs() + small[:, None] * w.detach().double().abs().sum(0)
    dw = off.T @ x.detach().double().abs() + small.max() * x.detach().double().abs().sum(0)
    dx += V * U * (G.abs() @ w.detach().double().abs())
    dw += M * U * (G.abs().T @ x.detach().double().abs())
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    for a, b, d, c in zip(got, (gx, gw), (dx, dw), again):
        assert a.shape == b.shape and a.dtype == dt
        err = (a.double() - b).abs()
        assert (err <= d * (1 + half) + half * b.abs() + tiny).all(), float((err / b.abs().max()).max())
        assert torch.equal(a, c)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M", [1, 15, 16, 17, 64, 65, 128, 129, 257, 600])
def test_rows(M, dt):
    check(M, 300, 72, dt)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 4, 63, 127, 128, 129, 255, 256, 257, 1001, 5000])
def test_vocabularies(V, dt):
    check(33, V, 40, dt)
    check(150, V, 64, dt)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("K", [1, 3, 8, 16, 31, 63, 64, 65, 120, 128, 129, 200, 264, 600])
def test_widths(K, dt):
    check(20, 200, K, dt)
    check(140, 170, K, dt)


@pytest.mark.parametrize("M, V, K", [(1000, 20000, 256), (300, 40000, 520), (2050, 9000, 1032),
                                     (5000, 700, 264), (4, 100000, 128), (70, 60000, 264)])
def test_large(M, V, K):
    """Tiles of every size, the contraction in parts, several rounds of workgroups."""
    check(M, V, K, torch.bfloat16)


@pytest.mark.parametrize("M", [1, 16, 40, 64, 100])
@pytest.mark.parametrize("V, K", [(3000, 64), (3000, 200), (3000, 328), (1800, 1096), (34000, 200)])
def test_few_rows(M, V, K):
    """Tiles that begin at different columns, of which the last may be less than a stage."""
    check(M, V, K, torch.float16 if K == 328 else torch.bfloat16)


def test_pieces():
    """More rows than are reduced, and more of G than is held, at once; a sort over memory."""
    check(20000, 30000, 64, torch.bfloat16)


def test_offsets_beyond_32_bits():
    """A weight of more than 4 GiB, all of it 0 but its last rows."""
    V, K, M, last = 1_100_000, 2048, 20, 300
    w = torch.zeros(V, K, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(3)
    w[-last:] = (torch.randint(-2, 3, (last, K), generator=g) / 32).bfloat16().cuda()
    x = (torch.randint(-4, 5, (M, K), generator=g) / 4).bfloat16().cuda()
    t = torch.randint(V - last, V, (M,), generator=g).cuda()
    t[::4] = torch.randint(V - last, (5,), generator=g).cuda()
    gl, ge = torch.randn(2, M, generator=g).cuda()
    w.requires_grad_(True), x.requires_grad_(True)
    r = head_logprobs(x, w, t)
    gx, gw = torch.autograd.grad((r.logprob, r.entropy), (x, w), (gl, ge))
    xd, wd = x.detach().double(), w.detach()[-last:].double()
    l = xd @ wd.T
    top = l.amax(-1, keepdim=True).clamp(min=0)
    z = (l - top).exp().sum(-1, keepdim=True) + (V - last) * (-top).exp()
    lse = top + z.log()
    p, p0 = (l - lse).exp(), (-lse).exp()
    ent = (-(p * (l - lse)).sum(-1, keepdim=True) + (V - last) * p0 * lse)
    own = t >= V - last
    at = (t - (V - last)).clamp(min=0)[:, None]
    lp = torch.where(own, l.gather(1, at)[:, 0], 0.0) - lse[:, 0]
    assert_close((r.logprob.detach(), r.entropy.detach()), (lp, ent[:, 0]))
    gl, ge = gl.double()[:, None], ge.double()[:, None]
    G = -p * (gl + ge * (l - lse + ent))
    G.scatter_add_(1, at, torch.where(own[:, None], gl, 0.0))
    G0 = -p0 * (gl - ge * (lse - ent))
    half = 2.0 ** -8
    size = (G.abs() + 1e-3 * (gl.abs() + 24 * ge.abs())).T @ xd.abs()
    assert ((gw[-last:].double() - G.T @ xd).abs() <= half * (2 * size + (G.T @ xd).abs())).all()
    rest = (G0.T @ xd)[0]
    there = torch.zeros(V - last, dtype=torch.bool, device="cuda")
    there[t[~own]] = True
    size = (G0.abs().T @ xd.abs())[0]
    for rows in (slice(0, 3), slice(524286, 524290), slice(1048574, 1048578), slice(V - last - 3, V - last)):
        err = (gw[rows].double() - rest).abs()
        assert ((err <= half * 2 * size + 1e-30) | there[rows][:, None]).all()
    # a token in the part of zeros: its row has the given token's value too
    for i in torch.nonzero(~own)[:, 0].tolist():
        want = rest + gl[i] * xd[i]
        assert ((gw[t[i]].double() - want).abs() <= half * 2 * (size + gl[i].abs() * xd[i].abs())).all()
    want = G @ wd
    assert ((gx.double() - want).abs() <= half * 2.1 * (G.abs() @ wd.abs()) + 1e-6).all()


def test_only_some_gradients():
    for need in ((True, False), (False, True)):
        x, w, t, gl, ge = some(40, 90, 24, torch.bfloat16)
        full = [v.clone().requires_grad_(True) for v in (x, w)]
        want = torch.autograd.grad(head_logprobs(*full, t).logprob, full, gl)
        x.requires_grad_(need[0]), w.requires_grad_(need[1])
        r = head_logprobs(x, w, t)
        got, = torch.autograd.grad(r.logprob, x if need[0] else w, gl)
        assert torch.equal(got, want[0] if need[0] else want[1])
        r = head_logprobs(x, w, t)
        only, = torch.autograd.grad(r.entropy, x if need[0] else w, ge)
        assert torch.isfinite(only).all() and not torch.equal(got, only)


def test_shapes_strides_and_alignment():
    g = torch.Generator().manual_seed(1)
    w = (torch.randint(-2, 3, (50, 160), generator=g) / 4).bfloat16().cuda()
    x = (torch.randint(-4, 5, (3, 5, 160), generator=g) / 4).bfloat16().cuda()
    t = torch.randint(50, (3, 5), generator=g).cuda()
    for cut in (slice(0, 64), slice(1, 65), slice(8, 72), slice(3, 70), slice(0, 160, 2)):
        for xs, ts in ((x, t), (x.transpose(0, 1), t.T), (x[1:2, 2:3].expand(3, 5, 160), t)):
            a, b = xs[..., cut].detach().requires_grad_(True), w[:, cut].detach().requires_grad_(True)
            r = head_logprobs(a, b, ts.int())
            assert r.logprob.shape == ts.shape
            flat = a.detach().reshape(15, -1)
            want = exact(flat, b.detach(), ts.reshape(-1))
            assert_close((r.logprob.reshape(-1), r.entropy.reshape(-1)), want)
            ga, gb = torch.autograd.grad(r.logprob.sum(), (a, b))
            ref = [flat.contiguous().requires_grad_(True), b.detach().contiguous().requires_grad_(True)]
            ra, rb = torch.autograd.grad(head_logprobs(*ref, ts.reshape(-1)).logprob.sum(), ref)
            assert torch.equal(ga.reshape(15, -1), ra) and torch.equal(gb, rb)
    one = head_logprobs(x[0, 0], w, t[0, 0])
    assert one.logprob.shape == ()


def test_no_rows():
    x = torch.empty(0, 16, device="cuda").half().requires_grad_(True)
    w = torch.ones(9, 16, device="cuda").half().requires_grad_(True)
    r = head_logprobs(x, w, torch.empty(0, dtype=torch.int64, device="cuda"))
    gx, gw = torch.autograd.grad(r.logprob.sum(), (x, w))
    assert r.logprob.shape == (0,) and gx.shape == (0, 16) and torch.equal(gw, torch.zeros_like(w))


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_without_gradient(dt):
    """Padding gives nothing to the weights whatever its hidden states hold, and gets nothing."""
    x, w, t, gl, ge = some(50, 70, 40, dt, padded=False)
    t[7], gl[9], gl[10] = -100, 0, 0
    clean = [v.clone().requires_grad_(True) for v in (x, w)]
    want = torch.autograd.grad(head_logprobs(*clean, t).logprob, clean, gl)
    x[7], x[9, 3], x[10, 4] = float("nan"), float("inf"), float("nan")
    x.requires_grad_(True), w.requires_grad_(True)
    r = head_logprobs(x, w, t)
    got = torch.autograd.grad(r.logprob, (x, w), gl)
    assert torch.equal(got[1], want[1])
    assert torch.equal(got[0], want[0]) and (got[0][[7, 9, 10]] == 0).all()
    assert r.logprob[7] == 0 and r.logprob[9].isnan() and r.entropy[7].isnan()
    assert torch.isfinite(r.logprob[:9]).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_of_very_different_gradients(dt):
    """Gradients 2^40 apart keep their rows' own precision (fp16: as far as its range goes)."""
    x, w, t, gl, _ = some(40, 60, 32, dt, padded=False)
    up = torch.ones(40, device="cuda")
    up[::2] = 2.0 ** (-40 if dt == torch.bfloat16 else -8)
    x.requires_grad_(True)
    small, = torch.autograd.grad(head_logprobs(x, w, t).logprob, x, gl * up)
    plain, = torch.autograd.grad(head_logprobs(x, w, t).logprob, x, gl)
    want = plain.double() * up.double()[:, None]
    info = torch.finfo(dt)
    # the same products but for a power of two, rounded again
    assert ((small.double() - want).abs() <= info.eps * want.abs() + info.smallest_normal * info.eps).all()


def test_large_logits():
    """Distances between logits that leave one token, and logits far from 0."""
    w = torch.zeros(300, 16, device="cuda").bfloat16()
    w[:, 0] = 1024
    w[17, 1] = 4
    x = torch.zeros(3, 16, device="cuda").bfloat16()
    x[:, 0] = torch.tensor([1024.0, -1024.0, 0.0])
    x[:, 1] = torch.tensor([64.0, 64.0, 256.0])
    t = torch.tensor([17, 3, 17], device="cuda")
    r = head_logprobs(x, w, t)
    lp, ent = exact(x, w, t)
    assert_close((r.logprob, r.entropy), (lp, ent))


def test_against_differences():
    """Gradients along a direction against a central difference in 64 bits."""
    x, w, t, gl, ge = some(12, 40, 24, torch.bfloat16)
    leaves = [v.clone().requires_grad_(True) for v in (x, w)]
    r = head_logprobs(*leaves, t)
    grads = torch.autograd.grad((r.logprob, r.entropy), leaves, (gl, ge))
    for i in range(2):
        e, f = torch.randn(leaves[i].shape, device="cuda", dtype=torch.float64), []
        for s in (1e-5, -1e-5):
            v = [x.double(), w.double()]
            v[i] = v[i] + s * e
            lp, ent = exact(*v, t)
            f.append(float((lp * gl).sum() + (ent * ge).sum()))
        along = float((grads[i].double() * e).sum())
        # G and the gradient are rounded to 2^-8 of their size, errors add up as the terms do
        terms = exact(x, w, t, gl, ge)[4].abs()
        size = (terms @ w.double().abs()) if i == 0 else (terms.T @ x.double().abs())
        assert abs((f[0] - f[1]) / 2e-5 - along) <= 2.0 ** -8 * 2.1 * float((size * e.abs()).sum())


def test_captured_and_on_another_stream():
    x, w, t, gl, ge = some(150, 500, 72, torch.bfloat16)
    x.requires_grad_(True), w.requires_grad_(True)

    def step():
        r = head_logprobs(x, w, t)
        return (r.logprob.detach(), r.entropy.detach(),
                *torch.autograd.grad((r.logprob, r.entropy), (x, w), (gl, ge)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(3):
        fresh = some(150, 500, 72, torch.bfloat16, seed=i + 1)
        with torch.no_grad():
            for a, b in zip((x, w, t, gl, ge), fresh):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_capture_beside_an_eager_graph_is_refused():
    x, w, t, gl, _ = some(20, 50, 24, torch.bfloat16)
    w.requires_grad_(True)
    alive = head_logprobs(x, w, t).logprob
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph, stream=side):
            head_logprobs(x, w, t)
    torch.cuda.synchronize()
    assert torch.isfinite(torch.autograd.grad(alive, w, gl)[0]).all()


# ------------------------------------------------------------------ packed heads
def packed_case(fmt, V, K, block=0):
    g = torch.Generator().manual_seed(V)
    w = torch.randn(V, K, generator=g) / 8
    return PackedWeight.quantize(w, fmt, fwht_block=block, device="cuda")


@pytest.mark.parametrize("fmt, block, dt", [("e2m1", 0, torch.bfloat16), ("e2m1", 0, torch.float16),
                                            ("e2m1", 0, torch.float32), ("gf4", 0, torch.float16),
                                            ("gf4", 0, torch.bfloat16), ("gf4", 128, torch.float16)])
@pytest.mark.parametrize("M", [1, 16, 17, 200])
def test_packed(fmt, block, dt, M):
    V, K = 777, 256
    pw = packed_case(fmt, V, K, block)
    w = pw.dequant_device(torch.float32).double()
    g = torch.Generator().manual_seed(M)
    x = (torch.randint(-4, 5, (M, K), generator=g) / 4).to(dt).cuda().requires_grad_(True)
    t = torch.randint(-1, V, (M,), generator=g).cuda()
    gl, ge = torch.randn(2, M, generator=g).cuda()
    r = head_logprobs(x, pw, t)
    xd = x.detach().double()
    if block:  # the weight is rotated; the activation's rotation is rounded to fp16
        h = torch.ones(1, 1, dtype=torch.float64, device="cuda")
        while h.shape[0] < block:
            h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
        rot = torch.block_diag(*[h / block ** 0.5] * (K // block))
        w = w @ rot
    lp, ent, gx, _, G = exact(xd, w, t, gl, ge)
    terms = xd.abs() @ w.abs().T
    # logits: K sums in fp32 of products that may be rounded once (a rotation: of fp16 values)
    off = float((terms * (K * U + (2.0 ** -10 if block else 0))).max())
    for a, b in ((r.logprob, lp), (r.entropy, ent)):
        assert ((a.double() - b).abs() <= 4 * off * (1 + b.abs()) + 512 * U * (2 + b.abs())).all()
    got, = torch.autograd.grad((r.logprob, r.entropy), x, (gl, ge))
    assert got.dtype == dt and got.shape == x.shape
    half = torch.finfo(dt).eps / 2
    size = (gl.abs() + 24 * ge.abs()).double()[:, None]
    allowed = half * gx.abs() + (4 * off + 1024 * U) * size * w.abs().max() * 2 + 2.0 ** -24
    assert ((got.double() - gx).abs() <= allowed).all()


def test_packed_head_is_the_layer():
    """A QuantLinear head in pieces of rows, against its logits."""
    q = QuantLinear(torch.nn.Linear(200, 1000, bias=False), fmt="e2m1").cuda()
    x = torch.randn(2, 70, 200, device="cuda").bfloat16()
    t = torch.randint(1000, (2, 70), device="cuda")
    r = head_logprobs(x, q, t)
    w = q.dequantized_weight().cuda()
    want = token_logprobs(x.float() @ w.float().T, t)
    assert ((r.logprob - want.logprob).abs() <= 1e-4).all()  # logits of a few units, 200 terms in fp32
    assert r.logprob.shape == (2, 70)


def test_refusals():
    x, w = torch.randn(3, 16, device="cuda").half(), torch.randn(9, 16, device="cuda").half()
    t = torch.tensor([1, 2, 3], device="cuda")
    biased = QuantLinear(torch.nn.Linear(128, 16), fmt="e2m1").cuda()
    pw = packed_case("e2m1", 32, 128)
    wide = torch.randn(3, 128, device="cuda")
    for args in [(x.cpu(), w, t), (x, w.cpu(), t), (x, w, t.cpu()), (x.float(), w.float(), t),
                 (x.bfloat16(), w, t), (x, w[0], t), (x, w[:, :8], t), (x, w, t[:2]), (x, w, t.float()),
                 (x, w[:0], t), (wide, biased, t), (x, pw, t), (wide, pw, t[:1]),
                 (wide.double(), pw, t)]:
        with pytest.raises((ValueError, RuntimeError)):
            head_logprobs(*args)
    y = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(head_logprobs(y, w, t).logprob.square().sum(), y, create_graph=True)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda x: head_logprobs(x, w, t)[0], (x,))
