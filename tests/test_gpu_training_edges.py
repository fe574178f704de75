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


# ------------------------------------------------------------------ gradients far apart
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("most", [32.0, 1024.0])
@pytest.mark.parametrize("less", [12, 16, 20])
def test_weight_gradient_of_small_gradients(less, most, entropy):
    """fp16: rows whose gradients are 2^-12 to 2^-20 of the largest give their tokens' rows of the weight
    what they give alone.  Two kinds of rows, with the tokens of one vocabulary's half each: the other
    half's have probabilities of exp(-128), which are 0 in fp32."""
    V, K, M = 64, 40, 48
    g = torch.Generator().manual_seed(less)
    x = torch.randn(M, K, generator=g).half()
    w = torch.zeros(V, K).half()
    x[:, 0], w[:, 0] = 8, 8
    x[1::2, 0], w[V // 2:, 0] = -8, -8
    t = torch.randint(V // 2, (M,), generator=g)
    t[1::2] += V // 2
    gl = (0.5 + torch.rand(M, generator=g)) * most
    ge = (0.5 + torch.rand(M, generator=g)) * most / 32 if entropy else torch.zeros(M)
    gl[1::2] *= 2.0 ** -less
    ge[1::2] *= 2.0 ** -less
    x, w, t, gl, ge = (v.cuda() for v in (x, w, t, gl, ge))
    x.requires_grad_(True), w.requires_grad_(True)
    r = head_logprobs(x, w, t)
    _, gw = torch.autograd.grad((r.logprob, r.entropy) if entropy else r.logprob, (x, w),
                                (gl, ge) if entropy else gl)
    _, _, _, want, G = exact(x.detach(), w.detach(), t, gl, ge)
    half, info = 2.0 ** -11, torch.finfo(torch.float16)
    # Each G: p is 1/32 in both (logits that are equal, exactly), off by a few steps of fp32 where the
    # entropy comes in, then half a step of fp16; its products with x in sums of M; the result's rounding,
    # of half its least step where it is small.
    own = 64 * U * (G.abs() + (gl.abs() + 16 * ge.abs()).double()[:, None] / 32)
    own[::2, V // 2:] = 0
    own[1::2, :V // 2] = 0
    off = (half * G.abs() + own + M * U * G.abs()).T @ x.detach().double().abs()
    allowed = off * (1 + half) + half * want.abs() + info.smallest_normal * info.eps / 2
    err = (gw.double() - want).abs()
    assert (err <= allowed).all(), float((err / allowed).max())
    # and in sum: roundings are as likely up as down, so their sums are far below that bound
    for part in (slice(0, V // 2), slice(V // 2, V)):
        e, n = err[part][:, 1:].norm(), want[part][:, 1:].norm()
        floor = info.smallest_normal * info.eps / 2 * (V // 2 * K) ** 0.5
        assert e <= 2 * half * n + floor, float(e / n)


def test_weight_gradient_of_rows_of_all_sizes():
    """fp16: hidden states from 2^-12 to 2^12 under gradients that take it back: every row counts alike."""
    V, K, M = 128, 24, 64
    g = torch.Generator().manual_seed(6)
    x = torch.randn(M, K, generator=g)
    size = torch.randint(-12, 13, (M, 1), generator=g)
    x = torch.ldexp(x, size).half()
    w = torch.zeros(V, K).half()
    t = torch.randperm(V, generator=g)[:M]
    gl = torch.ldexp(1 + torch.rand(M, generator=g), -size[:, 0])
    x, w, t, gl = (v.cuda() for v in (x, w, t, gl))
    w.requires_grad_(True)
    gw, = torch.autograd.grad(head_logprobs(x, w, t).logprob, w, gl)
    *_, want, G = exact(x, w.detach(), t, gl, 0 * gl)
    half = 2.0 ** -11
    off = ((half + (64 + M) * U) * G.abs()).T @ x.double().abs()
    info = torch.finfo(torch.float16)
    allowed = off * (1 + half) + half * want.abs() + info.smallest_normal * info.eps / 2
    assert ((gw.double() - want).abs() <= allowed).all()


@pytest.mark.parametrize("M", [1023, 1024, 1025, 3000])
def test_weight_gradient_scales_of_many_rows(M):
    """fp16: one row's gradient far above the others', wherever it is."""
    V, K = 96, 40
    for at in (0, 300, M - 1):
        g = torch.Generator().manual_seed(M + at)
        x, w = torch.randn(M, K, generator=g).half(), torch.zeros(V, K).half()
        t = torch.randint(V - 1, (M,), generator=g)
        x[:, 0], w[:, 0] = 0, 0
        x[at, 0], w[V - 1, 0], t[at] = 64, 8, V - 1  # the row's own token alone: exp(-512) for others
        gl = torch.randn(M, generator=g)
        gl[at] = 2.0 ** 18
        x, w, t, gl = (v.cuda() for v in (x, w, t, gl))
        w.requires_grad_(True)
        gw, = torch.autograd.grad(head_logprobs(x, w, t).logprob, w, gl)
        *_, want, G = exact(x, w.detach(), t, gl, 0 * gl)
        # as in test_weight_gradient_of_small_gradients; p is 1/96 of the other rows, to fp32
        half, info = 2.0 ** -11, torch.finfo(torch.float16)
        G[at] = 0  # 1 - p, which is 0 in fp32 too
        off = ((half + (64 + M) * U) * G.abs() + 64 * U / V * gl.abs()[:, None] * (gl.abs()[:, None] < 100)
               ).T @ x.double().abs()
        allowed = off * (1 + half) + half * want.abs() + info.smallest_normal * info.eps / 2
        assert ((gw.double() - want).abs() <= allowed).all()


# ------------------------------------------------------------------ fp32 hidden states
@pytest.mark.parametrize("M", [5, 40])
@pytest.mark.parametrize("fmt", ["e2m1", "gf4"])
@pytest.mark.parametrize("entropy", [False, True])
def test_packed_head_keeps_fp32(fmt, M, entropy):
    """The gradient of fp32 hidden states is in fp32 terms throughout."""
    V, K = 64, 256
    head = _head(fmt, 0, V=V, K=K)
    w = head.dequant_device(torch.float32).double()
    g = torch.Generator().manual_seed(M)
    x = (torch.randint(-4, 5, (M, K), generator=g) / 4).cuda().requires_grad_(True)
    t = torch.randint(V, (M,), generator=g).cuda()
    gl, ge = torch.randn(2, M, generator=g).cuda()
    if not entropy:
        ge = 0 * ge
    r = head_logprobs(x, head, t)
    got, = torch.autograd.grad((r.logprob, r.entropy) if entropy else r.logprob, x,
                               (gl, ge) if entropy else gl)
    xd = x.detach().double()
    _, ent, gx, _, G = exact(xd, w, t, gl, ge)
    logp = torch.log_softmax(xd @ w.T, -1)
    p = logp.exp()
    gl, ge = gl.abs().double()[:, None], ge.abs().double()[:, None]
    # logits: K sums of terms (exact for E2M1, whose steps are few); the exponent of 2 below 16, three
    # roundings of it and those of the sum: 2^-18, and as much of p; the entropy 2^-15
    logit = K * U * (xd.abs() @ w.abs().T) if fmt == "gf4" else torch.zeros_like(p)
    dp = 2.0 ** -18 + 2 * logit.amax(-1, keepdim=True)
    dh = 2.0 ** -15 + 16 * logit.amax(-1, keepdim=True)
    own = p * (dp * (gl + ge * (logp.abs() + ent[:, None] + 1)) + dh * ge) + 4 * U * G.abs()
    # the products' terms are exact in three 16-bit parts, 3 V of which are summed
    allowed = own @ w.abs() + 4 * V * U * (G.abs() @ w.abs()) + 2 * U * gx.abs()
    assert got.dtype == torch.float32
    err = (got.double() - gx).abs()
    assert (err <= allowed).all(), float((err / allowed).max())


# ------------------------------------------------------------------ pieces
def _check_packed(head, w, x, t, gl, ge, terms=1, size=None):
    """Results and gradient of hidden states whose logits are exact in fp32.  size: of w's terms."""
    size = w.abs() if size is None else size
    r = head_logprobs(x, head, t)
    got, = torch.autograd.grad((r.logprob, r.entropy), x, (gl, ge))
    lp, ent, gx, _, G = exact(x.detach(), w, t, gl, ge)
    assert_close((r.logprob.detach(), r.entropy.detach()), (lp, ent))
    p = torch.softmax(x.detach().double() @ w.T, -1)
    dt = x.dtype
    half = torch.finfo(dt).eps / 2
    n = int((p > 2.0 ** -149).sum(-1).max())  # terms of a sum that are not 0 in fp32
    own = 1024 * U * (gl.abs() + 16 * ge.abs()).double()[:, None] * (G.abs() + p)
    off = (half * G.abs() + own + terms * n * U * G.abs()) @ size
    small = 2.0 ** -38 * (gl.abs() + 24 * ge.abs()).double()[:, None] * size.sum(0)
    assert got.dtype == dt and got.shape == x.shape
    err = (got.double() - gx).abs()
    assert (err <= off * (1 + half) + half * gx.abs() + small).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_packed_head_in_pieces_of_rows(dt):
    """More rows than have their logits at once (2,672 of 50,000), of a width that is padded to 256."""
    M, V, K = 2800, 50000, 200
    torch.manual_seed(9)
    head = QuantLinear(nn.Linear(K, V, bias=False), fmt="e2m1").cuda()
    w = head.dequantized_weight().cuda().double()
    g = torch.Generator().manual_seed(2)
    x = (torch.randint(-4, 5, (M, K), generator=g) / 4).to(dt).cuda().requires_grad_(True)
    t = torch.randint(-1, V, (M,), generator=g).cuda()
    gl, ge = torch.randn(2, M, generator=g).cuda()
    _check_packed(head, w, x, t, gl, ge, terms=3)


def test_rotated_head_in_pieces_of_rows():
    """A last piece of rows may take more workspace than a whole one (5,441 rows of 1,000 x 256, 8,192)."""
    V, K, M = 1000, 256, 8192 + 5441
    head = _head("gf4", 128, V=V, K=K)
    g = torch.Generator().manual_seed(1)
    x = (torch.randint(-4, 5, (M, K), generator=g) / 4).half().cuda()
    t = torch.randint(V, (M,), generator=g).cuda()
    gl = torch.randn(M, generator=g).cuda()

    def grads(rows):
        a = x[rows].clone().requires_grad_(True)
        return torch.autograd.grad(head_logprobs(a, head, t[rows]).logprob, a, gl[rows])[0]

    got = grads(slice(None))
    for rows in (slice(0, 8192), slice(8192, None)):  # the pieces by themselves: the same calls
        assert torch.equal(got[rows], grads(rows))
    assert got.abs().amax(-1).min() > 0


# ------------------------------------------------------------------ large vocabularies
@pytest.mark.parametrize("block, dt", [(4, torch.float16), (0, torch.bfloat16), (0, torch.float32)])
def test_packed_head_of_a_large_vocabulary(block, dt):
    """More tokens than fb_grad_x takes, in pieces of rows too.  Few of the tokens can come up, some on
    both sides of the first piece's end: the others' logits are 128 below, their probabilities 0."""
    V, K, M = (1 << 18) + 56, 128, 600
    g = torch.Generator().manual_seed(3)
    w = torch.randn(V, K, generator=g) / 8
    some_tokens = torch.cat([torch.arange(20), torch.arange((1 << 18) - 10, (1 << 18) + 10),
                             torch.arange(V - 20, V)])
    w[:, :4] = 0
    w[:, 0] = -8
    w[some_tokens, 0] = 8
    head = PackedWeight.quantize(w, "e2m1", fwht_block=block, device="cuda")
    w = head.dequant_device(torch.float32).double()
    size = w.abs()
    if block:  # a rotation of 4 halves: exact
        h = torch.tensor([[1, 1, 1, 1], [1, -1, 1, -1], [1, 1, -1, -1], [1, -1, -1, 1]]).double() / 2
        rot = torch.block_diag(*[h] * (K // 4)).cuda()
        w, size = w @ rot, 2 * size @ rot.abs()  # and its sums are rounded
    assert torch.equal(w[some_tokens.cuda(), 0], torch.full((60,), 8.0, device="cuda").double())
    x = torch.randint(-4, 5, (M, K), generator=g) / 4
    x[:, :4] = 0
    x[:, 0] = 8
    x = x.to(dt).cuda().requires_grad_(True)
    t = some_tokens[torch.randint(len(some_tokens), (M,), generator=g)].cuda()
    gl, ge = torch.randn(2, M, generator=g).cuda()
    _check_packed(head, w, x, t, gl, ge, terms=3, size=size)


# ------------------------------------------------------------------ the least values
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("e", [-60, -63, -64, -70, -74])
def test_norms_of_the_least_values(e, dt):
    """Rows whose squares are below fp32's normal numbers are normalised as others are, without an eps."""
    M, d = 7, 256
    g = torch.Generator().manual_seed(-e)
    sign = 1 - 2 * torch.randint(2, (3, M, d), generator=g)
    x, b, gy = (torch.ldexp(s.double(), torch.tensor(n)).to(dt).cuda()
                for s, n in zip(sign, (e, e, 0)))
    w = torch.ones(d, device="cuda", dtype=dt)
    x.requires_grad_(True)
    r = residual_norm(x, w, eps=0.0)
    # every square is 2^(2 e), which fp32 has: 1 in size
    assert ((r.normed.double() - sign[0].cuda()).abs() <= 2.0 ** -20).all()
    gx, = torch.autograd.grad(r.normed, x, gy)
    n = sign[0].cuda().double()
    want = (gy.double() - n * (gy.double() * n).mean(-1, keepdim=True)) * 2.0 ** -e
    # a few roundings in fp32, and the type's
    assert ((gx.double() - want).abs() <= (torch.finfo(dt).eps + 2.0 ** -18) * 2.0 ** -e).all()
    r = residual_norm(torch.zeros_like(x), w, b, branch_weight=w, eps=0.0)
    assert ((r.stream.double() - sign[1].cuda()).abs() <= 2.0 ** -20).all()


# ------------------------------------------------------------------ a step whose loss is the entropy
def test_step_of_the_entropy_against_torch():
    tokens, following = _batch(4)
    got = []
    for plain in (False, True):
        net = Net(plain)
        params = _trained(net)
        _, ent = net(tokens, following)
        got.append(torch.autograd.grad(ent.sum() / 100, params))
    for i, (a, b) in enumerate(zip(*got)):
        a, b = a.double(), b.double()
        # a dozen roundings to bf16 on the way in both, each of 2^-9 of a vector's length at most on average
        assert b.norm() > 0 and (a - b).norm() <= 24 * 2.0 ** -9 * b.norm(), i


# ------------------------------------------------------------------ the entropy's gradient alone
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M, V, K", [(200, 8000, 256), (33, 3000, 120)])
def test_gradient_of_the_entropy_alone(M, V, K, dt):
    """Its large values lie at other tokens than the given one, whose rounding alone is made up for: what
    the logits' gradient loses in 16 bits is there in the results, and no more."""
    x, w, t, _, ge = some(M, V, K, dt, padded=False)
    x.requires_grad_(True), w.requires_grad_(True)
    got = torch.autograd.grad(head_logprobs(x, w, t).entropy, (x, w), ge)
    _, _, gx, gw, G = exact(x.detach(), w.detach(), t, 0 * ge, ge)
    up = torch.ldexp(torch.ones_like(G[:, :1]), 14 - G.abs().amax(-1, keepdim=True).log2().ceil().int())
    lost = (G * up).to(dt).double() / up - G
    for a, b, e in zip(got, (gx, gw), (lost @ w.detach().double(), lost.T @ x.detach().double())):
        # two sets of roundings, and a quarter for those that fall to the other side
        assert (a.double() - b).norm() <= 1.25 * ((b.to(dt).double() - b).norm() + e.norm())


# ------------------------------------------------------------------ captured, and in part
@pytest.mark.parametrize("fmt, block, dt", [("e2m1", 0, torch.bfloat16), ("e2m1", 0, torch.float32),
                                            ("gf4", 128, torch.float16)])
@pytest.mark.parametrize("M", [12, 90])
def test_captured_packed_heads(fmt, block, dt, M):
    """Every way to a packed head's gradient, replayed with new data, padding among it."""
    head = _head(fmt, block)
    g = torch.Generator().manual_seed(M)

    def batch():
        t = torch.randint(-2, 300, (M,), generator=g)
        return ((torch.randint(-4, 5, (M, 256), generator=g) / 4).to(dt).cuda(), t.cuda(),
                *torch.randn(2, M, generator=g).cuda())

    x, t, gl, ge = batch()
    x.requires_grad_(True)

    def step():
        r = head_logprobs(x, head, t)
        return (r.logprob.detach(), r.entropy.detach(),
                *torch.autograd.grad((r.logprob, r.entropy), x, (gl, ge)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        fresh = batch()
        with torch.no_grad():
            for a, b in zip((x, t, gl, ge), fresh):
                a.copy_(b)
            ge[:3] = 0
            if i == 2:
                x[t < 0] = float("nan")
                ge[t < 0] = 0
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
        assert torch.equal(got[1].nan_to_num(-1), want[1].nan_to_num(-1))
        assert torch.isfinite(got[2]).all() and (i != 2 or bool((got[2][t < 0] == 0).all()))


def test_one_gradient_in_fp16():
    """The hidden states' gradient is the same bits with the weight's and without it, and the other way."""
    x, w, t, gl, ge = some(60, 90, 24, torch.float16)
    gl[::3] *= 2.0 ** -18
    full = [v.clone().requires_grad_(True) for v in (x, w)]
    r = head_logprobs(*full, t)
    want = torch.autograd.grad((r.logprob, r.entropy), full, (gl, 0.1 * ge))
    for i in range(2):
        one = [x.clone(), w.clone()]
        one[i].requires_grad_(True)
        r = head_logprobs(*one, t)
        got, = torch.autograd.grad((r.logprob, r.entropy), one[i], (gl, 0.1 * ge))
        assert torch.equal(got, want[i])


def test_fp16_without_any_gradient():
    """Incoming gradients of 0, and of the largest numbers, in fp16."""
    x, w, t, gl, _ = some(20, 30, 16, torch.float16, padded=False)
    x.requires_grad_(True), w.requires_grad_(True)
    for g in torch.autograd.grad(head_logprobs(x, w, t).logprob, (x, w), 0 * gl):
        assert (g == 0).all()
    gx, gw = torch.autograd.grad(head_logprobs(x, w, t).logprob, (x, w), 2.0 ** 100 * (1 + gl.abs()))
    assert not gx.isnan().any() and not gw.isnan().any() and gx.isinf().any() and gw.isinf().any()
