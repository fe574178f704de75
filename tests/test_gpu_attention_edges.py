"""Attention over the 8-bit cache and its neighbours where waits, scales, masks and bounds meet:
long runs of rows, block scales far apart, bounds that are too small, rows of no sequence."""
import numpy as np
import pytest
import torch

from if_i_could_turn_back_time_amd import (KVCache, cache_append, cache_attention,
                                           cache_evict, token_logprobs)
from oracle import cache_oracle as O
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


# ------------------------------------------------------------------ value scales far apart
def _scaled(lens, heads, D, dt, gains, low, seed=0):
    """Sequences whose value blocks (32 tokens) are gains[block % len] times as large; keys of the
    blocks in ``low`` have a channel that makes their scores small where q's first is 8."""
    c = Case([0] * len(lens), heads, D, 64, dt, parts=1, seed=seed)
    per = -(-max(lens) // 64)
    c.table = torch.arange(len(lens) * per, dtype=torch.int32, device=DEV).view(len(lens), per)
    c.cache = KVCache.new(len(lens) * per, heads, D, 64, DEV)
    for x in c.cache:
        x.view(torch.uint8).fill_(0x7F)  # NaN codes, a scale of 1, where nobody writes
    for start in range(0, max(lens), 32):
        count = [max(0, min(32, n - start)) for n in lens]

        def spoil(x, block=start // 32):
            x[:, 0] = x[:, 0].clamp(-2, 2)
            x[:, 0, :, 0] = -float(low.get(block % len(gains), 0))
            x[:, 1] *= gains[block % len(gains)]
        c.append([min(start, n) for n in lens], count, 1.0, spoil)
    c.lens = list(lens)
    return c


def _strict(c, new, group, qdt, **kw):
    """Attention within a bound that knows no value beyond its weight: each weight is off by 2^-11 of
    itself, or by 2^-32 of the row's largest but no more than itself; sums are fp32 (as in
    test_gpu_cache.py)."""
    T, Hq = sum(new), c.heads * group
    q = torch.randn(T, Hq, c.D, generator=c.g).clamp(-2, 2)
    q[..., 0] = 8
    q = q.to(qdt)
    out = cache_attention(q.to(DEV), c.cache, c.table, _i32(*c.lens),
                          _i32(0, *np.cumsum(new)), **kw)
    q, out = q.double().numpy(), out.double().cpu().numpy()
    ulp, least = (2.0 ** -11, 2.0 ** -25) if qdt == torch.float16 else (2.0 ** -8, 2.0 ** -134)
    at = 0
    for b, n in enumerate(new):
        for h in range(c.heads):
            k, v = c.k[b][h].values(), c.v[b][h].values()
            t = len(k)
            for j in range(h * group, (h + 1) * group):
                o, _, p, mags, pv = O.attention(q[at:at + n, j], k, v, c.D ** -0.5)
                d = (c.D + 24) * U * mags
                rel = np.expm1(2 * d) + 8 * U * mags + 2.0 ** -11 + t * U
                bound = rel[:, None] * pv + np.minimum(p, 2.0 ** -32) @ np.abs(v)
                bound = bound + ulp * (np.abs(o) + bound) + least
                got = out[at:at + n, j]
                bad = ~(np.abs(got - o) <= bound)
                assert not bad.any(), (b, h, j, np.argwhere(bad)[:4], got[bad][:4], o[bad][:4])
        at += n


GAINS = {
    "a large block behind": ([1.0, 2.0 ** 40], {}),
    "one whose weight is nothing": ([2.0 ** 40, 1.0, 1.0, 1.0], {0: 40}),
    "one whose weight is little": ([1.0, 2.0 ** 40, 1.0], {1: 20}),
    "within a unit": ([1.0, 2.0 ** 7, 2.0 ** -15, 2.0 ** -8], {1: 5}),
    "just beyond it": ([1.0, 2.0 ** 8, 2.0 ** -15, 1.0, 2.0 ** -16], {}),
    "up and down": ([2.0 ** -30, 2.0 ** 20, 2.0 ** -10, 0.0, 2.0 ** 25, 2.0 ** -35], {1: 60, 4: 60}),
}


@pytest.mark.parametrize("which", list(GAINS))
@pytest.mark.parametrize("lens,new,heads,group,D", [
    ([100, 290], [1, 1], 2, 4, 64), ([70, 131], [4, 3], 1, 3, 128), ([65, 200], [1, 2], 1, 5, 48),
    ([333], [16], 1, 1, 256), ([700], [2], 1, 8, 128), ([130, 97], [70, 97], 2, 2, 64),
    ([300, 33], [250, 33], 1, 3, 128), ([150], [120], 1, 1, 80), ([170], [140], 1, 2, 256)])
def test_value_scales_far_apart(which, lens, new, heads, group, D):
    """The values of a block with another scale cost no other token's weight a bit, whether the
    block comes before or behind, in the same tile or for rows that do not see it."""
    print(which, lens, new, heads, group, D, flush=True)
    gains, low = GAINS[which]
    c = _scaled(lens, heads, D, torch.float32, gains, low)
    _strict(c, new, group, torch.bfloat16)


@pytest.mark.parametrize("new,group", [([1], 4), ([3], 4), ([120], 2)])
def test_fp16_values_far_apart(new, group):
    """The extremes of fp16 side by side, with fp16 queries."""
    c = _scaled([190], 2, 128, torch.float16, [1e-3, 1.5e4, 1e-3, 1e-5], {1: 60})
    _strict(c, new, group, torch.float16)


@pytest.mark.parametrize("new", [[1], [40]])
def test_value_scales_far_apart_in_parts(new):
    """A long cache, so that parts and waves with units of their own are joined."""
    gains = [1.0] * 40 + [2.0 ** 35] + [2.0 ** -12] * 30 + [2.0 ** -30]
    c = _scaled([5000], 1, 64, torch.float32, gains, {40: 60})
    _strict(c, new, 2, torch.bfloat16)


# ------------------------------------------------------------------ bounds and rows of no sequence
def _poison(*shapes):
    """Leaves NaN in the memory that the allocator hands out next."""
    x = [torch.full(shape, float("nan"), dtype=dt, device=DEV) for shape, dt in shapes]
    del x


@pytest.mark.parametrize("new,group,lens", [([1, 1], 4, [900, 333]), ([50, 21], 4, [900, 333]),
                                            ([20], 1, [40]), ([3], 20, [2000])])
def test_max_new_of_nothing(new, group, lens):
    """max_new too small, 0 as well, changes speed only."""
    c = Case(lens, 2, 128, 64)
    T = sum(new)
    for kw in ({"max_new": 0}, {"max_new": 0, "max_len": 0}):
        _poison(((T, 2 * group, 128), torch.bfloat16), ((T, 2 * group), torch.float32))
        c.attend(new, group, **kw)


@pytest.mark.parametrize("new,group,lens,kw", [
    ([1, 1], 4, [900, 333], {}), ([1, 1, 1], 2, [40, 7, 90], {"max_new": 1}), ([60, 21], 4, [900, 333], {}),
    ([150, 0, 130], 1, [1500, 10, 700], {"max_new": 150, "max_len": 1500}), ([0, 0], 2, [5, 6], {}),
    ([300], 8, [300], {"max_new": 300})])
@pytest.mark.parametrize("before,behind", [(0, 7), (3, 0), (2, 150)])
def test_rows_of_no_sequence(new, group, lens, kw, before, behind):
    """A padded batch: the rows that are no sequence's get 0 and -inf, the others what they get
    without them, bit for bit where the work is split alike."""
    heads, D, T = 2, 64, sum(new)
    c = Case(lens, heads, D, 64)
    q = torch.randn(before + T + behind, heads * group, D, generator=c.g).bfloat16().to(DEV)
    cu = _i32(0, *np.cumsum(new))
    inner = q[before:before + T]
    kw = {"max_new": max(new), **kw}
    want, want_lse = cache_attention(inner, c.cache, c.table, _i32(*lens), cu, return_lse=True, **kw)
    for _ in range(3):
        _poison((q.shape, q.dtype), (q.shape[:2], torch.float32))
        out, lse = cache_attention(q, c.cache, c.table, _i32(*lens), cu + before, return_lse=True,
                                   **kw)
        assert torch.equal(out[before:before + T], want)
        assert torch.equal(lse[before:before + T], want_lse)
        for rows in (slice(0, before), slice(before + T, None)):
            assert bool((out[rows] == 0).all()) and bool((lse[rows] == -torch.inf).all())


# ------------------------------------------------------------------ reading the cache back
def test_read_is_exact():
    """Every code at every scale whose products fp32 holds, as numpy's ldexp has it."""
    cache = KVCache.new(250, 1, 16, 32, DEV)
    codes = torch.arange(512, device=DEV).to(torch.uint8).view(32, 16)
    cache.k.view(torch.uint8)[:] = codes
    cache.v.view(torch.uint8)[:] = codes.view(2, 16, 16).transpose(1, 2)
    cache.k_scale[:, 0, 0] = torch.arange(250, device=DEV).to(torch.uint8)
    cache.v_scale.copy_(cache.k_scale)
    k, v = cache.read(torch.arange(250, device=DEV, dtype=torch.int32), 250 * 32)
    with np.errstate(over="ignore", under="ignore"):
        want = np.ldexp(codes.view(torch.float8_e4m3fn).float().cpu().numpy()[None],
                        np.arange(-127, 123)[:, None, None])
    for got in (k, v):
        np.testing.assert_array_equal(got.view(250, 32, 16).cpu().numpy(), want)


# ------------------------------------------------------------------ eviction across scales
@pytest.mark.parametrize("D", [64, 80, 256])
@pytest.mark.parametrize("big", [2.0 ** 28, 2.0 ** 100, 3e38])
def test_evict_zeros_from_large_blocks(D, big):
    """Tokens of zeros, of tiny values and of NaN leave blocks of large ones for blocks of their own."""
    n, heads, page = 200, 2, 64

    def spoil(x):
        x.clamp_(-1, 1)
        x *= big
        x[::2] = 0                    # zeros in blocks of large values
        x[64:96] = 0                  # and a block of them
        x[96:128:2] = 1e-30
        x[130, 0, 0, 3] = x[132, 1, 1, 5] = float("nan")
    c = Case([0], heads, D, page, torch.float32, parts=1)
    need = -(-n // page)
    c.cache = KVCache.new(2 * need, heads, D, page, DEV)
    c.table = torch.arange(need, dtype=torch.int32, device=DEV)[None]
    c.append([0], [n], 1.0, spoil)
    c.lens = [n]
    c.check_codes()
    w = torch.zeros(1, heads, n, device=DEV)
    w[..., ::2] = 1  # the even ones stay
    new_table = torch.arange(need, 2 * need, dtype=torch.int32, device=DEV)[None]
    r = cache_evict(c.cache, c.table, _i32(n), w, 105, 9, new_table, max_len=n)
    k, v = c.cache.read(new_table[0], 105)
    for h in range(heads):
        ids = r.kept[0, h].cpu().numpy()
        np.testing.assert_array_equal(ids, O.evict(w[0, h].cpu().numpy(), 105, 9))
        for got, old in ((k[h], c.k[0][h]), (v[h], c.v[0][h])):
            cut = O.Tokens(D)
            cut.append(old.values()[ids])
            np.testing.assert_array_equal(got.double().cpu().numpy(), cut.values())


# ------------------------------------------------------------------ appending no more than max_new
@pytest.mark.parametrize("max_new", [0, 1, 2, 31, 33, 40])
def test_append_writes_no_more_than_max_new(max_new):
    """Of 40 tokens a sequence the first max_new come into the cache and into the scales."""
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(80, 2, 64, device=DEV, generator=g) * torch.linspace(1, 90, 80, device=DEV)[:, None, None]
    table, start = _i32(0, 1, 2, 3, 4, 5).view(2, 3), _i32(30, 7)
    got, want = (KVCache.new(6, 2, 64, 32, DEV) for _ in range(2))
    cache_append(got, x, x, table, start, _i32(0, 40, 80), max_new=max_new)
    n = min(max_new, 40)
    y = torch.cat([x[:n], x[40:40 + n]])
    cache_append(want, y, y, table, start, _i32(0, n, 2 * n))
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ------------------------------------------------------------------ weights beside a row of NaN
@pytest.mark.parametrize("new,group,D", [(4, 2, 64), (3, 4, 128), (9, 4, 64), (60, 2, 128), (150, 1, 256),
                                         (90, 20, 64)])
def test_weights_beside_a_row_of_nan(new, group, D):
    """A query of NaN makes NaN of the weights of the tokens that it sees, and of no others: those
    get what the later rows give them."""
    n, heads, bad = 400, 2, new // 2
    c = Case([n], heads, D, 64)
    q = torch.randn(new, heads * group, D, generator=c.g).bfloat16().to(DEV)
    cu, lens = _i32(0, new), _i32(n)
    spoilt = q.clone()
    spoilt[bad, :, 1] = float("nan")
    w, later = (torch.zeros(1, heads, n, device=DEV) for _ in range(2))
    cache_attention(spoilt, c.cache, c.table, lens, cu, weights=w, max_len=n)
    cache_attention(q[bad + 1:], c.cache, c.table, lens, _i32(0, new - bad - 1), weights=later, max_len=n)
    seen = n - new + bad + 1
    assert bool(w[..., :seen].isnan().all())
    # the same rows' weights, summed in another order: at most 2^12 of them
    got, want = w[0, :, seen:].double(), later[0, :, seen:].double()
    assert bool(((got - want).abs() <= 2.0 ** 13 * U * want).all())


# ------------------------------------------------------------------ values near fp32's range
@pytest.mark.parametrize("lens,new,group", [([6000], [1], 4), ([5000, 300], [1, 1], 1), ([4000], [3], 8),
                                            ([3000], [40], 2), ([6000, 2500], [30, 41], 2)])
def test_large_values_in_parts(lens, new, group):
    """Values of 2^120 to 2^126, all of one sign: no sum over a part or over the parts may overflow."""
    c = _scaled(lens, 2, 64, torch.float32, [2.0 ** 122, 2.0 ** 124], {})
    for side in c.v:
        assert all(np.abs(v.values()).max() < 2.0 ** 127 for v in side)
    c.cache.v.view(torch.uint8).bitwise_and_(0x7F)
    for side in c.v:
        for v in side:
            v.codes = np.abs(v.codes)
    _strict(c, new, group, torch.bfloat16)


# ------------------------------------------------------------------ what torch knows of these calls
def test_in_place_writes_raise_versions():
    c = Case([90], 2, 64, 64)
    lens = _i32(90)
    w = torch.zeros(1, 2, 128, device=DEV)
    p = torch.ones(1, 2, 128, device=DEV, requires_grad=True)
    product = w * p  # keeps w
    before = [x._version for x in c.cache]
    q = torch.randn(1, 4, 64, device=DEV, dtype=torch.bfloat16)
    cache_attention(q, c.cache, c.table, lens)
    assert [x._version for x in c.cache] == before
    cache_attention(q, c.cache, c.table, lens, weights=w, max_len=90)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        product.sum().backward()
    assert [x._version for x in c.cache] == before
    cache_append(c.cache, q[:, :2], q[:, 2:], c.table, lens)
    assert all(x._version > v for x, v in zip(c.cache, before))
    before = [x._version for x in c.cache]
    spare = _i32(*[i for i in range(5) if i not in c.table[0].tolist()][:1])[None]
    cache_evict(c.cache, c.table, lens, w, 40, 8, spare, max_len=90)
    assert all(x._version > v for x, v in zip(c.cache, before))
    with torch.inference_mode():
        cache = KVCache.new(2, 2, 64, 64, DEV)
    cache_append(cache, q[:, :2], q[:, 2:], _i32(0, 1)[None], _i32(0))  # has no version, and works
    assert bool((cache.k_scale[0, :, 0] > 0).all())


def _calls():
    c = Case([90], 2, 64, 64)
    lens = _i32(90)
    spare = _i32(*[i for i in range(5) if i not in c.table[0].tolist()][:1])[None]
    w = torch.rand(1, 2, 128, device=DEV)
    tok = torch.zeros(1, dtype=torch.long, device=DEV)
    q = torch.randn(1, 4, 64, device=DEV, dtype=torch.bfloat16)
    return q, (lambda q: cache_attention(q, c.cache, c.table, lens),
               lambda q: cache_append(c.cache, q[:, :2], q[:, 2:], c.table, lens) or q,
               lambda q: cache_evict(c.cache, c.table, lens, w, 40, 8, spare, max_len=90).weights,
               lambda q: token_logprobs(q.flatten(1), tok).logprob)


@pytest.mark.parametrize("which", range(4))
def test_recording_is_refused(which):
    """A trace would hold what the call gave once, a recorded graph an empty buffer."""
    from torch.fx.experimental.proxy_tensor import make_fx
    q, calls = _calls()
    call = calls[which]
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, (q,), check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(call)(q)
    call(q)


@pytest.mark.parametrize("which", range(4))
def test_fake_tensors_are_refused(which):
    from torch._subclasses.fake_tensor import FakeTensorMode
    q, calls = _calls()
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises((RuntimeError, ValueError)):
        calls[which](q)


# ------------------------------------------------------------------ scores far from 0
@pytest.mark.parametrize("size", [1e8, 1e9, 1e10, 1e12, 1e20])
@pytest.mark.parametrize("new,group,lens", [(1, 4, 300), (3, 4, 70), (60, 2, 300), (1, 2, 4000)])
def test_scores_of_any_size(new, group, lens, size):
    """Scores so large that fp32 holds them to many units: the weights are those of one token or of a
    few, and the outputs lie between the least and the largest value that a row sees."""
    c = Case([0], 2, 64, 64, torch.bfloat16, parts=1)
    c.table = torch.arange(-(-lens // 64), dtype=torch.int32, device=DEV)[None]
    c.cache = KVCache.new(c.table.shape[1], 2, 64, 64, DEV)

    def spoil(x):
        x[:, 0] *= size
    c.append([0], [lens], 1.0, spoil)
    q = torch.randn(new, 2 * group, 64, generator=c.g).bfloat16().to(DEV)
    w = torch.zeros(1, 2, lens, device=DEV)
    out, lse = cache_attention(q, c.cache, c.table, _i32(lens), _i32(0, new), weights=w, max_len=lens,
                               return_lse=True)
    assert bool(((w >= 0) & (w <= new * group * 1.01)).all())
    out = out.double().cpu().numpy()
    assert bool(lse.isfinite().all())
    for h in range(2):
        v = c.v[0][h].values()
        for i in range(new):
            seen = v[:lens - new + 1 + i]
            lo, hi = seen.min(0), seen.max(0)
            slack = 2.0 ** -7 * np.maximum(np.abs(lo), np.abs(hi))  # rounding to 16 bits, and of sums
            got = out[i, h * group:(h + 1) * group]
            assert (got >= lo - slack).all() and (got <= hi + slack).all()
