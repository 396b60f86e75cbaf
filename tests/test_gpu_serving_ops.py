"""The serving operators on the GPU against their 64-bit definitions (tests/serving_reference.py).

Tolerances: an output is off by at most half a step of its type relative to its value, and by
what the fp32 arithmetic before the rounding can add; the reference gives the second for each
element.  What a cache holds is compared bit for bit.
"""
import math

import pytest

import serving_reference as ref
from serving_reference import U, half_step

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def ops():
    from kernelcodegen_amd import ops as o
    return o


def within(got, want, slack):
    """|got - want| <= half a step of the wanted value (and of what the slack adds to it) + slack, everywhere."""
    h = half_step(got.dtype)
    got, tiny = got.double().cpu(), torch.finfo(got.dtype).tiny
    bound = h * want.abs() + (1 + h) * slack + tiny
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), "%d of %d outside, worst by %.3g of its bound" % (
        int(bad.sum()), bad.numel(), float(((got - want).abs() / bound).nan_to_num(math.inf).max()))


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(seed, *shape, dtype=F32):
    return torch.randn(shape, generator=gen(seed)).to(dtype)


# ---- norm and rotation --------------------------------------------------------------------------

# batch, tokens, query heads, key heads, D, rotated elements
NORM_SHAPES = [(1, 1, 1, 1, 64, 64), (1, 1, 32, 8, 128, 128), (2, 3, 5, 5, 128, 64), (3, 7, 8, 1, 64, 32),
               (1, 130, 12, 4, 64, 16), (2, 65, 3, 2, 128, 32), (1, 4100, 3, 1, 128, 128), (1, 9, 40, 40, 128, 112)]


def norm_inputs(shape, dtype, seed, far=100):
    b, s, hq, hk, d, rot = shape
    q, k = normal(seed, b, s, hq, d, dtype=dtype), normal(seed + 1, b, s, hk, d, dtype=dtype)
    q[:, :, 0] *= 30
    wq, wk = ((1 + 0.3 * normal(seed + i, d)).to(dtype) for i in (2, 3))
    pos = torch.randint(0, far, (b, s), generator=gen(seed + 4)).to(torch.int32)
    freq = (1e4 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))).float()
    return q, k, wq, wk, pos, freq


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_norm_rope(dev, shape, interleaved, dtype):
    q, k, wq, wk, pos, freq = norm_inputs(shape, dtype, 11)
    got = ops().qk_norm_rope(*(t.to(dev) for t in (q, k, wq, wk, pos, freq)), eps=1e-5, interleaved=interleaved)
    for g, x, w in zip(got, (q, k), (wq, wk)):
        want, size = ref.norm_rope(x, w, pos, freq, 1e-5, interleaved)
        # a row's sum (D / 8 products in a lane, then lanes), its root and quotient, two products, the angle's
        # rounding (half a turn: pi u), sine and cosine, and a product and a sum
        within(g, want, 32 * U * size)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_norm_rope_backward(dev, shape, interleaved, dtype):
    q, k, wq, wk, pos, freq = norm_inputs(shape, dtype, 21)
    dq, dk = normal(31, *q.shape, dtype=dtype), normal(32, *k.shape, dtype=dtype)
    gq, gk, gwq, gwk = ops().qk_norm_rope_backward(*(t.to(dev) for t in (dq, dk, q, k, wq, wk, pos, freq)), eps=1e-5,
                                                   interleaved=interleaved)
    for dx, dw, dy, x, w in ((gq, gwq, dq, q, wq), (gk, gwk, dk, k, wk)):
        want, want_w, size, size_w = ref.norm_rope_backward(dy, x, w, pos, freq, 1e-5, interleaved)
        within(dx, want, U * size)
        within(dw, want_w, U * size_w)


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_gradient_is_the_slope(dev, interleaved):
    """Differences of the forward kernel along a direction, against the gradient's product with it."""
    shape = (1, 3, 2, 1, 64, 32)
    q, k, wq, wk, pos, freq = norm_inputs(shape, F32, 41)
    dq, dk = normal(51, *q.shape), normal(52, *k.shape)
    o = ops()
    to = lambda *ts: [t.to(dev) for t in ts]  # noqa: E731
    g = o.qk_norm_rope_backward(*to(dq, dk, q, k, wq, wk, pos, freq), eps=1e-5, interleaved=interleaved)
    point = [q, k, wq, wk]
    for i, x in enumerate(point):
        way = normal(60 + i, *x.shape) * x.abs().clamp(min=0.1)
        h = 2.0 ** -7

        def f(step):
            moved = [t + step * way if j == i else t for j, t in enumerate(point)]
            yq, yk = o.qk_norm_rope(*to(*moved, pos, freq), eps=1e-5, interleaved=interleaved)
            return float((yq.cpu().double() * dq.double()).sum() + (yk.cpu().double() * dk.double()).sum()), yq, yk
        (hi, yq, yk), (lo, _, _) = f(h), f(-h)
        slope = (hi - lo) / (2 * h)
        want = float((g[i].cpu().double() * way.double()).sum())
        # fp32 noise of two values over 2h, and the third derivative: the definition's own difference shows it
        def exact(step):
            moved = [(t.double() + step * way.double()) if j == i else t.double() for j, t in enumerate(point)]
            return sum(float((ref.norm_rope(a, b, pos, freq, 1e-5, interleaved)[0] * c.double()).sum())
                       for a, b, c in ((moved[0], moved[2], dq), (moved[1], moved[3], dk)))
        curve = abs((exact(h) - exact(-h)) / (2 * h) - want)
        noise = 33 * U * float((yq.cpu().abs().double() * 2 * dq.abs().double()).sum()
                               + (yk.cpu().abs().double() * 2 * dk.abs().double()).sum() + 40) / h
        assert abs(slope - want) <= noise + curve + 64 * U * float((g[i].cpu().abs().double() * way.abs().double()).sum())
        assert curve < 0.05 * max(abs(want), 1.0)


def test_norm_rope_far_positions_and_strides(dev):
    """Positions beyond what fp32 angles resolve, negative ones, and every layout a user may hold."""
    b, s, hq, hk, d = 2, 5, 4, 2, 128
    freq = (1e6 ** (-torch.arange(64, dtype=torch.float64) / 64)).float()
    pos = torch.tensor([[0, 1, -1, 2 ** 31 - 1, 1000003], [-2 ** 31, 77, 131071, 524287, 16777217]], dtype=torch.int32)
    wq, wk = normal(1, d), normal(2, d)
    o = ops()
    fused = normal(3, b, s, hq + 2 * hk, d).to(dev)
    views = [(fused[:, :, :hq], fused[:, :, hq:hq + hk]),
             (fused[:, :, :hq].transpose(1, 2).contiguous().transpose(1, 2), fused[:, :, hq:hq + hk]),  # [B,H,S,D]
             (fused[:1, :, :hq].expand(b, s, hq, d), fused[:, :, hq:hq + 1].expand(b, s, hk, d))]  # broadcast
    odd = torch.empty(b * s * (hq + hk) * (d + 1) + 3, device=dev)  # rows of no alignment
    oq = odd[1:1 + b * s * hq * (d + 1)].view(b, s, hq, d + 1)[..., :d].copy_(views[0][0])
    ok = odd[2 + b * s * hq * (d + 1):][:b * s * hk * (d + 1)].view(b, s, hk, d + 1)[..., :d].copy_(views[0][1])
    views.append((oq, ok))
    for q, k in views:
        layouts = [None, (torch.empty(b, hq, s, d, device=dev).transpose(1, 2), torch.empty(s, b, hk, d, device=dev).transpose(0, 1)),
                   (torch.empty(b, s, hq, d + 1, device=dev)[..., 1:], torch.empty(b, s, hk, d, device=dev))]
        for out in layouts:
            got = o.qk_norm_rope(q, k, wq.to(dev), wk.to(dev), pos.to(dev), freq.to(dev), out=out)
            if out is not None:
                assert got[0] is out[0] and got[1] is out[1]
            for g, x, w in zip(got, (q, k), (wq, wk)):
                want, size = ref.norm_rope(x.cpu(), w, pos, freq, 1e-6, False)
                within(g, want, 32 * U * size)
        dq, dk = normal(5, b, hq, s, d).to(dev).transpose(1, 2), normal(6, b, s, hk, d).to(dev)
        g = o.qk_norm_rope_backward(dq, dk, q, k, wq.to(dev), wk.to(dev), pos.to(dev), freq.to(dev))
        for dx, dw, dy, x, w in ((g[0], g[2], dq, q, wq), (g[1], g[3], dk, k, wk)):
            want, want_w, size, size_w = ref.norm_rope_backward(dy.cpu(), x.cpu(), w, pos, freq, 1e-6, False)
            within(dx, want, U * size)
            within(dw, want_w, U * size_w)


def test_norm_rope_of_packed_tokens(dev):
    """[tokens,H,D] is [1,tokens,H,D], also on another stream than the tensors' own."""
    q, k, wq, wk, pos, freq = (t.to(dev) for t in norm_inputs((1, 37, 4, 2, 64, 32), BF16, 91))
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    o = ops()
    whole = o.qk_norm_rope(q, k, wq, wk, pos, freq) + o.qk_norm_rope_backward(dq, dk, q, k, wq, wk, pos, freq)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        packed = o.qk_norm_rope(q[0], k[0], wq, wk, pos[0], freq) + o.qk_norm_rope_backward(
            dq[0], dk[0], q[0], k[0], wq, wk, pos[0], freq)
        torch.cuda.current_stream().synchronize()
    for a, b in zip(whole, packed):
        assert b.dim() == min(a.dim(), 3) and torch.equal(a.reshape(b.shape), b)


def test_norm_rope_tiny_rows_without_eps(dev):
    """eps 0 counts as the smallest normal number: rows of zeros give zeros, rows whose squares vanish stay finite."""
    q, k, wq, wk, pos, freq = norm_inputs((1, 2, 2, 1, 64, 64), F32, 95)
    q[0, 0] = 0
    q[0, 1] *= 1e-25
    got = ops().qk_norm_rope(*(t.to(dev) for t in (q, k, wq, wk, pos, freq)), eps=0.0)
    for g, x, w in zip(got, (q, k), (wq, wk)):
        want, size = ref.norm_rope(x, w, pos, freq, torch.finfo(F32).tiny, False)
        within(g, want, 32 * U * size)


def test_norm_rope_in_place_zero_rows_and_nonfinite(dev):
    q, k, wq, wk, pos, freq = norm_inputs((1, 6, 3, 2, 64, 64), BF16, 71)
    q[0, 0, 0] = 0
    q[0, 1, 1, 5] = math.inf
    k[0, 2, 1, 7] = math.nan
    args = [t.to(dev) for t in (q, k, wq, wk, pos, freq)]
    apart = ops().qk_norm_rope(*args)
    assert torch.equal(apart[0][0, 0, 0], torch.zeros(64, dtype=BF16, device=dev))
    # only the row that holds them is touched by what is not finite
    assert torch.isfinite(apart[0].float()).all(-1).sum() == 6 * 3 - 1
    assert torch.isfinite(apart[1].float()).all(-1).sum() == 6 * 2 - 1
    ops().qk_norm_rope(*args, out=(args[0], args[1]))
    for a, b in zip(apart, args):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_infinity_behind_the_rotated_elements(dev, interleaved):
    """An element that is not rotated mixes with no other: beside an infinity the formula's zeros stay zeros,
    and the gradients of other weights stay numbers."""
    q, k, wq, wk, pos, freq = norm_inputs((1, 3, 2, 1, 64, 32), F32, 97)
    dq, dk = normal(98, *q.shape), normal(99, *k.shape)
    at = 41
    q[0, 1, 1, at] = math.inf
    args = [t.to(dev) for t in (q, k, wq, wk, pos, freq)]
    got = ops().qk_norm_rope(*args, interleaved=interleaved)[0].cpu()
    want, _ = ref.norm_rope(q, wq, pos, freq, 1e-6, interleaved)
    assert want.isnan().sum() == 1 and torch.equal(got.isnan(), want.isnan())
    assert (got[0, 1, 1].nan_to_num() == 0).all()
    q[0, 1, 1, at], dq[0, 1, 1, at] = 1.0, math.inf
    args[0] = q.to(dev)
    dw = ops().qk_norm_rope_backward(dq.to(dev), dk.to(dev), *args, interleaved=interleaved)[2].cpu()
    _, want, _, bound = ref.norm_rope_backward(dq, q, wq, pos, freq, 1e-6, interleaved)
    rest = torch.arange(64) != at
    assert want[rest].isfinite().all() and want[at].isinf() and dw[at] == want[at]
    within(dw[rest], want[rest], U * bound[rest])


@pytest.mark.parametrize("dtype, tokens", [(BF16, 16384), (F32, 8192)])
def test_norm_rope_outputs_past_the_caches(dev, dtype, tokens):
    """Outputs of 256 MiB and more are stored past the caches: the same bits as in parts, and the definition's values."""
    hq, hk, d = 48, 16, 128
    assert tokens * (hq + hk) * d * dtype.itemsize >= 1 << 28
    g = torch.Generator(device=dev).manual_seed(5)
    q, k = (torch.randn(1, tokens, h, d, generator=g, device=dev, dtype=dtype) for h in (hq, hk))
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g, device=dev)).to(dtype)
    pos = torch.randint(0, 100, (1, tokens), generator=g, device=dev, dtype=torch.int32)
    freq = (1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().to(dev)
    got = ops().qk_norm_rope(q, k, wq, wk, pos, freq)
    cut = tokens // 2 - 1
    parts = [ops().qk_norm_rope(q[:, at], k[:, at], wq, wk, pos[:, at], freq) for at in (slice(0, cut), slice(cut, None))]
    for i, g in enumerate(got):
        assert torch.equal(g, torch.cat([p[i] for p in parts], 1))
    some = torch.tensor([0, 1, cut, tokens - 2, tokens - 1])
    for g, x, w in zip(got, (q, k), (wq, wk)):
        want, size = ref.norm_rope(x[:, some].cpu(), w.cpu(), pos[:, some].cpu(), freq.cpu(), 1e-6, False)
        within(g[:, some], want, 32 * U * size)  # as in test_norm_rope


def test_norm_rope_backward_repeats_bit_for_bit(dev):
    q, k, wq, wk, pos, freq = (t.to(dev) for t in norm_inputs((2, 700, 6, 2, 128, 128), BF16, 81))
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    first = ops().qk_norm_rope_backward(dq, dk, q, k, wq, wk, pos, freq)
    for _ in range(3):
        for a, b in zip(first, ops().qk_norm_rope_backward(dq, dk, q, k, wq, wk, pos, freq)):
            assert torch.equal(a, b)


# ---- cache --------------------------------------------------------------------------------------


def filled_cache(dev, pages, heads, page, dim, dtype, seed=0):
    """A cache whose bytes are known: k and v differ, exponents are ordinary."""
    o = ops()
    if dtype == BF16:
        return o.KvCache(*(normal(seed + i, pages, heads, page, dim, dtype=BF16).to(dev) for i in (1, 2)))
    k, v = (torch.randint(0, 256, (pages, heads, page, dim), generator=gen(seed + i), dtype=torch.uint8) for i in (1, 2))
    k[(k & 127) == 127] = 3
    v[(v & 127) == 127] = 5
    kx, vx = (torch.randint(118, 123, (pages, heads, page), generator=gen(seed + i), dtype=torch.uint8) for i in (3, 4))
    return o.KvCache(k.to(dev).view(E4M3), v.to(dev).view(E4M3), kx.to(dev), vx.to(dev))


def raw(t):
    return t.view(torch.uint8) if t.dtype == E4M3 else t.view(torch.int16) if t.dtype == BF16 else t


def cache_values(cache):
    """k and v of a cache in float64 on the CPU."""
    if cache.k.dtype == BF16:
        return cache.k.cpu().double(), cache.v.cpu().double()
    return (ref.dequantise(raw(cache.k).cpu(), cache.k_exp.cpu()), ref.dequantise(raw(cache.v).cpu(), cache.v_exp.cpu()))


def expected_write(cache, k, v, slots):
    """What the cache has to hold after the write, as raw tensors on the CPU: token by token, the last one wins."""
    held = [raw(cache.k).cpu().clone(), raw(cache.v).cpu().clone()]
    exps = [None, None] if cache.k_exp is None else [cache.k_exp.cpu().clone(), cache.v_exp.cpu().clone()]
    pages, heads, page, dim = cache.k.shape
    for part, x in enumerate((k, v)):
        x = x.cpu().reshape(-1, heads, dim)
        new, e = (x.to(BF16).view(torch.int16), None) if cache.k_exp is None else ref.quantise(x)
        for t, slot in enumerate(slots.reshape(-1).tolist()):
            if 0 <= slot < pages * page:
                held[part][slot // page, :, slot % page] = new[t]
                if e is not None:
                    exps[part][slot // page, :, slot % page] = e[t]
    return held, exps


def assert_cache_holds(cache, want):
    held, exps = want
    for got, w in zip((cache.k, cache.v), held):
        g = raw(got).cpu()
        if got.dtype == E4M3:  # the sign of a NaN is not compared
            g = torch.where((g & 127) == 127, torch.full_like(g, 127), g)
        assert torch.equal(g, w)
    for got, w in zip((cache.k_exp, cache.v_exp), exps):
        assert w is None or torch.equal(got.cpu(), w)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("tokens, heads, page, dim", [(1, 1, 16, 64), (5, 3, 16, 128), (61, 8, 32, 64), (300, 2, 256, 128),
                                                      (4100, 1, 64, 64), (4099, 3, 128, 128)])
def test_cache_write_and_read(dev, tokens, heads, page, dim, kind, dtype):
    pages = -(-tokens // page) + 2
    cache = filled_cache(dev, pages, heads, page, dim, kind)
    k = normal(1, tokens, heads, dim) * torch.exp(3 * normal(2, tokens, heads, 1))
    v = normal(3, tokens, heads, dim) * torch.exp(3 * normal(4, tokens, heads, 1))
    k, v = k.to(dtype), v.to(dtype)
    slots = torch.randperm(pages * page, generator=gen(5))[:tokens].to(torch.int32)
    slots[::7] = -1
    want = expected_write(cache, k, v, slots)
    ops().kv_cache_write(cache, k.to(dev), v.to(dev), slots.to(dev))
    assert_cache_holds(cache, want)
    slots[::5] = pages * page  # past the end: zeros
    for out_dtype in (F32, BF16):
        got = ops().kv_cache_read(cache, slots.to(dev), out_dtype=out_dtype)
        live = (slots >= 0) & (slots < pages * page)
        at = slots[live].long()
        for g, values in zip(got, cache_values(cache)):
            assert not g.cpu()[~live].any()
            rows = values[at // page, :, at % page]
            assert torch.equal(g.cpu()[live].double(), rows.to(out_dtype).double())  # bf16 numbers: exact in both


def test_cache_write_edges(dev):
    """Rows of zeros, the borders of the exponent, ties, subnormals, the largest numbers, NaN and infinities."""
    dim = 64
    x = torch.zeros(24, 1, dim)
    x[1, 0, 3] = 448.0
    x[2, 0, 3] = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9))
    x[3, 0, :] = torch.arange(dim) * 0.0078125  # ties between neighbours
    x[4, 0, :] = torch.tensor([1.0625, 1.1875, -1.0625, 2.125] * 16)
    x[4, 0, 0] = 448
    x[5, 0, :] = torch.logspace(-9, 2.6, dim)
    x[6, 0, :] = 3.4028234e38
    x[7, 0, 1] = 1e-45
    x[8, 0, :] = torch.logspace(-45, -36, dim)
    x[9, 0, 4], x[9, 0, 5] = math.nan, 2.0
    x[10, 0, 4], x[10, 0, 5] = math.inf, -3.0
    x[11, 0, 4], x[11, 0, 6] = -math.inf, math.nan
    x[12, 0, :] = math.nan
    x[13, 0, :] = 2.0 ** -119 * 448
    x[14, 0, :] = 2.0 ** -126 * 448
    x[15, 0, :] = 2.0 ** -127 * 448
    x[16, 0, :] = -0.0
    x[17:, 0] = normal(9, 7, dim) * torch.tensor([1e-38, 1e-30, 1e-3, 1, 1e3, 1e30, 1e37])[:, None]
    for kind in (E4M3, BF16):
        cache = filled_cache(dev, 3, 1, 16, dim, kind)
        slots = torch.arange(24, dtype=torch.int32)
        if kind == BF16:
            x = torch.where(torch.isnan(x), torch.zeros_like(x), x)  # which NaN is not compared
        want = expected_write(cache, x, -x, slots)
        ops().kv_cache_write(cache, x.to(dev), (-x).to(dev), slots.to(dev))
        assert_cache_holds(cache, want)


@pytest.mark.parametrize("tokens", [2, 300, 4200])
def test_cache_write_same_slot_twice(dev, tokens):
    """Of tokens with one slot the last is written, whatever the workgroups' order; slots out of the cache are left out."""
    cache = filled_cache(dev, 4, 2, 16, 128, E4M3)
    k, v = normal(1, tokens, 2, 128, dtype=BF16), normal(2, tokens, 2, 128, dtype=BF16)
    slots = torch.randint(-3, 70, (tokens,), generator=gen(3)).to(torch.int32)
    slots[-1] = slots[0]
    slots[tokens // 2] = -2 ** 31
    slots[tokens // 3] = 2 ** 31 - 1
    want = expected_write(cache, k, v, slots)
    for _ in range(3):
        ops().kv_cache_write(cache, k.to(dev), v.to(dev), slots.to(dev))
        assert_cache_holds(cache, want)


@pytest.mark.parametrize("kind", [E4M3, BF16])
@pytest.mark.parametrize("tokens, heads, dim", [(6500, 2, 64), (8192 + 300, 1, 128), (2 * 8192 + 1, 2, 64)])
def test_cache_write_of_long_prompts(dev, tokens, heads, dim, kind):
    """Four tokens to a workgroup, and calls that are cut into launches of 8192 tokens: slots named twice inside a
    workgroup, inside a launch, and in two launches hold the last token."""
    cache = filled_cache(dev, 500, heads, 16, dim, kind)
    k, v = normal(1, tokens, heads, dim, dtype=BF16), normal(2, tokens, heads, dim, dtype=BF16)
    slots = torch.randint(-3, 8003, (tokens,), generator=gen(3)).to(torch.int32)
    slots[1::50] = slots[0::50][:slots[1::50].numel()]  # neighbours
    slots[-1] = slots[0]
    if tokens > 8192:
        slots[8191], slots[8192] = 77, 77  # on both sides of a launch's end
        late = slots[8192:]
        assert torch.isin(slots[:8192], late[late >= 0]).any()
    want = expected_write(cache, k, v, slots)
    for _ in range(2):
        ops().kv_cache_write(cache, k.to(dev), v.to(dev), slots.to(dev))
        assert_cache_holds(cache, want)


@pytest.mark.parametrize("kind, out_dtype", [(E4M3, BF16), (BF16, F32), (BF16, BF16)])
def test_cache_read_of_long_prompts(dev, kind, out_dtype):
    """Outputs of up to 32 MiB and larger ones, which are stored past the caches, are the cache's values alike."""
    heads, dim, page = 8, 128, 64
    most = (32 << 20) // (2 * heads * dim * out_dtype.itemsize)
    cache = filled_cache(dev, 40, heads, page, dim, kind)
    values = [t.to(out_dtype) for t in cache_values(cache)]
    slots = torch.randint(-1, 40 * page, (most + 1,), generator=gen(4)).to(torch.int32)
    live = (slots >= 0)[:, None, None]
    at = slots.clamp(min=0).long()
    for tokens in (most, most + 1):
        got = ops().kv_cache_read(cache, slots[:tokens].to(dev), out_dtype=out_dtype)
        for g, v in zip(got, values):
            assert torch.equal(g.cpu(), torch.where(live, v[at // page, :, at % page], 0)[:tokens])


def test_cache_layouts(dev):
    """Parts of a fused projection, [B,H,S,D] memory, unaligned rows, [B,S] slots."""
    b, s, heads, dim = 3, 5, 2, 64
    o = ops()
    fused = normal(1, b, s, 3 * heads, dim, dtype=BF16).to(dev)
    odd = torch.empty(b * s * heads * (dim + 1) + 1, dtype=BF16, device=dev)[1:].view(b, s, heads, dim + 1)[..., :dim]
    odd.copy_(fused[:, :, :heads])
    bhsd = fused[:, :, heads:2 * heads].transpose(1, 2).contiguous().transpose(1, 2)
    for k, v in ((fused[:, :, heads:2 * heads], fused[:, :, 2 * heads:]), (odd, bhsd),
                 (fused[:1, :, :heads].expand(b, s, heads, dim), bhsd)):
        for kind in (BF16, E4M3):
            cache = filled_cache(dev, 3, heads, 16, dim, kind)
            slots = torch.randperm(48, generator=gen(2))[:b * s].to(torch.int32).view(b, s)
            want = expected_write(cache, k, v, slots)
            o.kv_cache_write(cache, k, v, slots.to(dev))
            assert_cache_holds(cache, want)
            outs = (torch.zeros(b, heads, s, dim, dtype=BF16, device=dev).transpose(1, 2),
                    torch.zeros(b, s, heads, dim + 1, dtype=BF16, device=dev)[..., 1:])
            got = o.kv_cache_read(cache, slots.to(dev), out=outs)
            for g, values in zip(got, cache_values(cache)):
                at = slots.long()
                assert torch.equal(g.cpu().double(), values[at // 16, :, at % 16])


# ---- attention over the cache ---------------------------------------------------------------------


def check_fmha(dev, cache, q, table, context, drafts, tree, scale, out_dtype, **how):
    """Runs and compares every row; rows that are not asked for have to stay as they were."""
    before = torch.full(q.shape, 7.0, dtype=out_dtype)
    out = before.to(dev)
    i32 = lambda t: None if t is None else torch.tensor(t, dtype=torch.int32, device=dev)  # noqa: E731
    k, v = how.pop("values", None) or cache_values(cache)
    got = ops().fmha_cache(q.to(dev), cache, table.to(dev), i32(context), draft_lens=i32(drafts),
                           tree_mask=None if tree is None else tree.to(dev), scale=scale, out=out, **how)
    want, arith, weight = ref.fmha_cache(q, k, v, table, context, drafts, tree, scale, before)
    # fp32 output: weights split over three bf16 numbers, off by 2^-24; bf16 output: rounded once
    off = 2.0 ** -24 if out_dtype == F32 else 2.0 ** -8
    # second-order terms of numerator and denominator both off by `off`
    within(got, want, arith + off * (1 + 4 * off) * weight)
    return got


def make_table(batch, per, pages, seed):
    return torch.randperm(pages, generator=gen(seed))[:batch * per].view(batch, per).to(torch.int32)


def random_trees(batch, n, seed):
    g = gen(seed)
    m = torch.zeros(batch, n, dtype=torch.int64)
    for b in range(batch):
        for i in range(n):
            word = 1 << i
            if i:
                word |= int(m[b, int(torch.randint(0, i, (1,), generator=g))]) & (2 ** 64 - 1)
            m[b, i] = word - 2 ** 64 if word >= 2 ** 63 else word
    return m


# batch, N, query heads, cache heads, D, page, contexts
FMHA_SHAPES = [(1, 1, 1, 1, 64, 16, [0]), (1, 1, 8, 8, 128, 16, [1]), (2, 1, 8, 1, 128, 16, [15, 16]),
               (3, 1, 4, 2, 64, 32, [31, 32, 33]), (4, 3, 6, 2, 128, 64, [0, 63, 127, 200]),
               (2, 13, 12, 4, 64, 16, [130, 7]), (1, 64, 5, 5, 128, 128, [250]), (2, 33, 7, 1, 64, 256, [600, 3]),
               (1, 2, 32, 2, 128, 16, [1111]), (3, 5, 32, 32, 64, 16, [65, 64, 0]), (1, 40, 16, 2, 128, 32, [97]),
               (1, 1, 4, 1, 128, 16, [5003]), (2, 17, 28, 4, 64, 16, [2050, 1])]


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("shape", FMHA_SHAPES)
def test_fmha_cache(dev, shape, kind, out_dtype):
    B, N, Hq, Hk, D, page, context = shape
    per = -(-(max(context) + N) // page)
    cache = filled_cache(dev, B * per + 2, Hk, page, D, kind, seed=N)
    q = normal(7, B, N, Hq, D, dtype=BF16)
    table = make_table(B, per, B * per + 2, 8)
    check_fmha(dev, cache, q, table, context, None, None, D ** -0.5, out_dtype)
    if N > 1:
        drafts = [max(0, N - 3 * b) for b in range(B)]
        check_fmha(dev, cache, q, table, context, drafts, random_trees(B, N, 9), D ** -0.5, out_dtype)


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0])
def test_fmha_cache_scales(dev, scale, kind):
    cache = filled_cache(dev, 12, 2, 16, 64, kind)
    q = normal(1, 2, 3, 4, 64, dtype=BF16)
    check_fmha(dev, cache, q, make_table(2, 6, 12, 2), [80, 11], None, None, scale, F32)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_fmha_cache_lengths_and_tables_not_to_be_trusted(dev, kind):
    """Lengths below zero and beyond the table, pages outside the cache: not seen, and not read."""
    cache = filled_cache(dev, 8, 2, 16, 128, kind)
    q = normal(1, 6, 4, 4, 128, dtype=BF16)
    table = torch.tensor([[0, 1, 2], [3, -1, 4], [5, 8, 2 ** 31 - 1], [-2 ** 31, -7, 99], [6, 7, 0], [1, 1, 1]],
                         dtype=torch.int32)
    context = [2 ** 31 - 1, 40, 20, 41, -5, 47]
    for drafts in (None, [4, 9, -3, 2, 3, 4]):
        for out_dtype in (BF16, F32):
            check_fmha(dev, cache, q, table, context, drafts, None, 0.1, out_dtype)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_fmha_cache_rows_that_see_nothing(dev, kind):
    cache = filled_cache(dev, 4, 1, 16, 64, kind)
    q = normal(1, 2, 3, 2, 64, dtype=BF16)
    tree = torch.tensor([[0, 1, -1], [0, 0, 4]], dtype=torch.int64)
    got = check_fmha(dev, cache, q, make_table(2, 2, 4, 1), [0, 0], None, tree, 0.125, F32)
    assert not got[0, 0].any() and not got[1, :2].any() and got[1, 2].any()
    # bits of drafted tokens that are not there count for nothing
    got = check_fmha(dev, cache, q, make_table(2, 2, 4, 1), [0, 0], [1, 2], tree, 0.125, F32)
    assert not got[1, :2].any()


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("D", [64, 128])
def test_fmha_cache_unseen_keys_have_no_influence(dev, D, kind, poison):
    """Not-finite keys and values behind the last key, and in drafts that a query does not see."""
    B, N, heads, page = 2, 5, 2, 16
    cache = filled_cache(dev, 10, heads, page, D, kind)
    table = make_table(B, 5, 10, 3)
    context = [37, 64]
    bad = torch.tensor(poison if kind == BF16 else math.nan).to(kind)
    trees = torch.tensor([[1, 3, 5, 13, 17], [1, 2, 4, 8, 16]], dtype=torch.int64)
    clean_k, clean_v = cache_values(cache)
    for b in range(B):
        for key in list(range(context[b] + N, 80)) + [context[b] + 2]:  # the tail, and the third draft
            p, o = int(table[b, key // page]), key % page
            for t in (cache.k, cache.v):
                raw(t)[p, :, o] = raw(bad.view(1))[0].to(dev)
    q = normal(1, B, N, 4, D, dtype=BF16)
    sees = [[n for n in range(N) if (int(trees[b, n]) >> 2) & 1] for b in range(B)]
    assert sees == [[2, 3], [2]]
    out = ops().fmha_cache(q.to(dev), cache, table.to(dev), torch.tensor(context, dtype=torch.int32, device=dev),
                           tree_mask=trees.to(dev), scale=0.1, out_dtype=F32).cpu()
    want, arith, weight = ref.fmha_cache(q, clean_k, clean_v, table, context, None, trees, 0.1, out)
    for b in range(B):
        for n in range(N):
            if n in sees[b]:
                assert not torch.isfinite(out[b, n]).any()
            else:
                within(out[b, n], want[b, n], arith[b, n] + 2.0 ** -24 * 2 * weight[b, n])


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_fmha_cache_one_value_not_finite(dev, kind):
    """A single value that is not finite reaches the outputs of its own column, in the rows that see it."""
    cache = filled_cache(dev, 6, 1, 16, 128, kind)
    table = make_table(2, 3, 6, 3)
    context = [20, 3]
    bad = torch.tensor(math.inf if kind == BF16 else math.nan).to(kind)
    for b, key, column in ((0, 2, 77), (1, 4, 5)):  # a key of the context; the second draft
        raw(cache.v)[int(table[b, key // 16]), 0, key % 16, column] = raw(bad.view(1))[0].to(dev)
    q = normal(1, 2, 3, 2, 128, dtype=BF16)
    trees = torch.tensor([[1, 3, 5], [1, 3, 5]], dtype=torch.int64)
    out = ops().fmha_cache(q.to(dev), cache, table.to(dev), torch.tensor(context, dtype=torch.int32, device=dev),
                           tree_mask=trees.to(dev), scale=0.1).cpu().float()
    finite = torch.ones(2, 3, 2, 128, dtype=torch.bool)
    finite[0, :, :, 77] = False
    finite[1, 1, :, 5] = False
    assert torch.equal(torch.isfinite(out), finite)


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("context, N, D", [(200, 1, 64), (200, 9, 128), (1500, 2, 128)])
def test_fmha_cache_values_of_infinity(dev, context, N, D, out_dtype):
    """Weights are positive: an infinity among the values that every query sees is the output of its column, infinities
    of both signs in a column give NaN, and the other columns are what they are without them."""
    page, width = 16, 100
    cache = filled_cache(dev, width, 2, page, D, BF16)
    table = make_table(1, width, width, 3)
    clean = cache_values(cache)

    def put(key, column, value):
        cache.v[int(table[0, key // page]), :, key % page, column] = value
    put(5, 7, math.inf)
    put(40, 9, -math.inf)
    put(33, 11, math.inf)
    put(150, 11, -math.inf)
    put(context - 1, 50, math.inf)  # in a chunk that reaches beyond the context
    q = normal(1, 1, N, 8, D, dtype=BF16)
    got = ops().fmha_cache(q.to(dev), cache, table.to(dev), torch.tensor([context], dtype=torch.int32, device=dev), scale=0.1,
                           out_dtype=out_dtype).cpu()
    want, arith, weight = ref.fmha_cache(q, *clean, table, [context], None, None, 0.1, torch.zeros(q.shape))
    assert (got[..., 7] == math.inf).all() and (got[..., 9] == -math.inf).all() and (got[..., 50] == math.inf).all()
    assert got[..., 11].isnan().all()
    rest = torch.ones(D, dtype=torch.bool)
    rest[[7, 9, 11, 50]] = False
    off = 2.0 ** -24 if out_dtype == F32 else 2.0 ** -8  # as in check_fmha
    within(got[..., rest], want[..., rest], (arith + off * (1 + 4 * off) * weight)[..., rest])


def test_fmha_cache_large_scores(dev):
    """Scores far apart and rising along the keys: the running maximum moves in every tile."""
    cache = filled_cache(dev, 40, 1, 16, 64, BF16)
    table = torch.arange(40, dtype=torch.int32).view(1, 40)
    ramp = torch.linspace(-1, 1, 640).view(40, 1, 16, 1)
    q = normal(1, 1, 2, 8, 64, dtype=BF16).abs()
    for sign in (1, -1):
        cache.k.copy_((sign * ramp * torch.ones(64) * 8).to(BF16))
        check_fmha(dev, cache, q, table, [638], None, None, 1.0, F32)
        check_fmha(dev, cache, q, table, [638], None, None, 30.0, F32)


@pytest.mark.parametrize("B, longest", [(65, 3000), (130, 700), (1100, 300)])
def test_fmha_cache_many_sequences(dev, B, longest):
    """More sequences than lanes: empty ones, ones without drafts, a few long ones among short ones."""
    N, Hq, Hk, D, page = 2, 2, 1, 64, 16
    g = gen(B)
    context = torch.randint(0, 40, (B,), generator=g)
    context[::9] = 0
    context[3], context[B // 2], context[B - 1] = longest, longest // 2, longest - 17
    drafts = torch.randint(0, N + 1, (B,), generator=g)
    drafts[3] = drafts[B - 1] = N
    per = -(-(longest + N) // page)
    cache = filled_cache(dev, per + 50, Hk, page, D, BF16)
    table = torch.randint(0, per + 50, (B, per), generator=g).to(torch.int32)
    q = normal(1, B, N, Hq, D, dtype=BF16)
    for workspace in (None, torch.empty(200000, dtype=torch.uint8, device=dev)):
        check_fmha(dev, cache, q, table, context.tolist(), drafts.tolist(), None, 0.125, F32, workspace=workspace)


def marked_workspace(cache, table, N, Hq, size=None):
    """A workspace of the preferred (or the given) size whose bytes show whether partial results were stored."""
    B, width = table.shape
    need = ops().fmha_cache_workspace_bytes(cache, width, B, N, Hq)
    assert need > 0
    return torch.full((need if size is None else size,), 0xa5, dtype=torch.uint8, device=cache.device)


def was_cut(workspace, cache):
    """The first row of the first slot is stored if any sequence was cut."""
    return bool((workspace[:4 * cache.dim] != 0xa5).any())


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("B, longest", [(65, 900), (130, 700), (1024, 500), (1100, 1000), (2100, 600)])
def test_fmha_cache_many_sequences_of_which_some_are_cut(dev, B, longest, out_dtype):
    """More sequences than lanes, and more than one pass of the launch that finds their units takes: the long ones, on
    both sides of a pass's end, are cut and joined, among empty ones, short ones and ones without drafts."""
    N, Hq, Hk, D, page = 2, 2, 1, 64, 16
    g = gen(B)
    context = torch.randint(0, 40, (B,), generator=g)
    context[::9] = 0
    drafts = torch.randint(0, N + 1, (B,), generator=g)
    far = [b for b in (3, 64, 999, 1022, 1023, 1024, 1025, 1099, 2047, 2048, 2099) if b < B] + [B - 1]
    for i, b in enumerate(far):
        context[b], drafts[b] = longest - 37 * i, N
    context[5], drafts[5] = longest, 0
    width = 60  # more room than any of them needs
    cache = filled_cache(dev, 90, Hk, page, D, BF16)
    table = torch.randint(0, 90, (B, width), generator=g).to(torch.int32)
    q = normal(1, B, N, Hq, D, dtype=BF16)
    need = ops().fmha_cache_workspace_bytes(cache, width, B, N, Hq)
    got = []
    for size in (need, need, need // 3):
        workspace = marked_workspace(cache, table, N, Hq, size)
        got.append(check_fmha(dev, cache, q, table, context.tolist(), drafts.tolist(), None, 0.125, out_dtype,
                              workspace=workspace))
        assert was_cut(workspace, cache)
    assert torch.equal(got[0], got[1])


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("B, N, Hq, Hk, D", [(24, 3, 8, 8, 64), (64, 1, 8, 8, 128), (9, 5, 24, 8, 128)])
def test_fmha_cache_cut_batches(dev, B, N, Hq, Hk, D, kind, out_dtype):
    """Batches of up to 64 sequences that are not few for the chip: every wave finds its unit, and a joining workgroup
    takes several rows, the last one fewer."""
    page, width = 16, 80
    context = [37 * (b * 7 % B) * 32 // B % 1250 for b in range(B)]
    context[1], context[B - 1] = 1250, 0
    drafts = [max(0, N - b % 4) for b in range(B)] if N > 1 else [b % 5 and 1 for b in range(B)]
    drafts[1] = N
    cache = filled_cache(dev, 200, Hk, page, D, kind, seed=B)
    table = torch.randint(0, 200, (B, width), generator=gen(B)).to(torch.int32)
    q = normal(7, B, N, Hq, D, dtype=BF16)
    workspace = marked_workspace(cache, table, N, Hq)
    check_fmha(dev, cache, q, table, context, drafts, random_trees(B, N, 9), D ** -0.5, out_dtype, workspace=workspace)
    assert was_cut(workspace, cache)


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("N, Hq, D", [(1, 8, 128), (9, 16, 128), (1, 8, 64), (20, 16, 64)])
def test_fmha_cache_tables_with_room_beyond_the_caches(dev, N, Hq, D, kind, out_dtype):
    """Keys and values are requested past the caches where all tables together have room for more than 192 MiB."""
    B, Hk, page = 3, 8, 16
    width = (192 << 20) // (B * page * Hk * D * 2 * kind.itemsize) + 1
    cache = filled_cache(dev, 70, Hk, page, D, kind, seed=N)
    table = torch.randint(0, 70, (B, width), generator=gen(N)).to(torch.int32)
    q = normal(7, B, N, Hq, D, dtype=BF16)
    workspace = marked_workspace(cache, table, N, Hq)
    for context in ([700, 15, 1201], [33, 0, 64]):
        check_fmha(dev, cache, q, table, context, None, None, D ** -0.5, out_dtype, workspace=workspace)
    assert was_cut(workspace, cache)


def test_fmha_cache_no_queries_at_all(dev):
    for B in (3, 100):
        cache = filled_cache(dev, 64, 2, 16, 128, E4M3)
        q = normal(1, B, 2, 4, 128, dtype=BF16)
        table = torch.zeros(B, 64, dtype=torch.int32)
        check_fmha(dev, cache, q, table, [900] * B, [0] * B, None, 1.0, BF16)


@pytest.mark.parametrize("power", [-90, 60])
def test_fmha_cache_exponents_far_from_one(dev, power):
    """V's powers of two go through the weights: rows of very small and very large values, and both together."""
    cache = filled_cache(dev, 8, 1, 16, 64, E4M3)
    cache.v_exp.add_(power)
    cache.v_exp[::2] -= 7
    q = normal(1, 1, 3, 2, 64, dtype=BF16)
    for out_dtype in (BF16, F32):
        check_fmha(dev, cache, q, make_table(1, 8, 8, 2), [120], None, None, 0.1, out_dtype)
    # K's: scores of 2^power times the queries' 2^-power
    cache = filled_cache(dev, 8, 1, 16, 64, E4M3)
    cache.k_exp.add_(power)
    check_fmha(dev, cache, (q.float() * 2.0 ** -power).to(BF16), make_table(1, 8, 8, 2), [120], None, None, 0.1, F32)


def test_fmha_cache_query_layouts(dev):
    """Queries inside a fused projection, in [B,H,N,D] memory and of no alignment; outputs likewise; no workspace."""
    B, N, Hq, Hk, D = 2, 3, 6, 2, 128
    cache = filled_cache(dev, 80, Hk, 16, D, E4M3)
    table = make_table(B, 40, 80, 1)
    args = (cache, table.to(dev), torch.tensor([600, 333], dtype=torch.int32, device=dev))
    fused = normal(1, B, N, Hq + 4, D, dtype=BF16).to(dev)
    want = ops().fmha_cache(fused[:, :, :Hq].contiguous(), *args, scale=0.1)
    k, v = cache_values(cache)
    exact, arith, weight = ref.fmha_cache(fused[:, :, :Hq].cpu(), k, v, table, [600, 333], None, None, 0.1, want.cpu())
    within(want, exact, arith + 2.0 ** -8 * 1.02 * weight)
    for q in (fused[:, :, :Hq], fused[:, :, :Hq].transpose(1, 2).contiguous().transpose(1, 2),
              torch.zeros(B * N * Hq * (D + 1) + 1, dtype=BF16, device=dev)[1:].view(B, N, Hq, D + 1)[..., :D].copy_(fused[:, :, :Hq])):
        for out in (None, torch.empty(B, Hq, N, D, dtype=BF16, device=dev).transpose(1, 2),
                    torch.empty(B, N, Hq, D + 1, dtype=BF16, device=dev)[..., 1:]):
            assert torch.equal(ops().fmha_cache(q, *args, scale=0.1, out=out), want)
    # with less workspace, or none that can be used, the call splits less
    for size in (0, 16, 1 << 14, 1 << 16):
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        within(ops().fmha_cache(fused[:, :, :Hq], *args, scale=0.1, workspace=ws), exact, arith + 2.0 ** -8 * 1.02 * weight)


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_fmha_cache_layouts_and_workspaces_of_cut_sequences(dev, kind, out_dtype):
    """Outputs in every layout through the joining launch; smaller workspaces split less, down to not at all."""
    B, N, Hq, Hk, D, page = 2, 3, 6, 2, 128, 16
    cache = filled_cache(dev, 200, Hk, page, D, kind)
    table, context = make_table(B, 100, 200, 1), [1500, 903]
    fused = normal(1, B, N, Hq + 4, D, dtype=BF16).to(dev)
    q = fused[:, :, :Hq]
    workspace = marked_workspace(cache, table, N, Hq)
    want = check_fmha(dev, cache, q.cpu(), table, context, None, None, 0.1, out_dtype, workspace=workspace)
    assert was_cut(workspace, cache)
    args = (cache, table.to(dev), torch.tensor(context, dtype=torch.int32, device=dev))
    assert torch.equal(ops().fmha_cache(q, *args, scale=0.1, out_dtype=out_dtype), want)  # its own workspace
    odd = torch.zeros(B * N * Hq * (D + 1) + 1, dtype=BF16, device=dev)[1:].view(B, N, Hq, D + 1)[..., :D].copy_(q)
    outs = (torch.empty(B, Hq, N, D, dtype=out_dtype, device=dev).transpose(1, 2),
            torch.empty(B, N, Hq, D + 1, dtype=out_dtype, device=dev)[..., 1:],
            torch.empty(N, B, Hq + 1, D, dtype=out_dtype, device=dev).transpose(0, 1)[:, :, 1:])
    for x in (q, odd):
        for out in outs:
            out.fill_(-1)
            assert torch.equal(ops().fmha_cache(x, *args, scale=0.1, out=out), want)
    need = workspace.numel()
    cut = []
    for size in (0, 16, need // 16, need // 8, need - 1, need + 100):
        workspace = marked_workspace(cache, table, N, Hq, size)
        check_fmha(dev, cache, q.cpu(), table, context, None, None, 0.1, out_dtype, workspace=workspace)
        cut.append(was_cut(workspace, cache))
    assert cut[:2] == [False, False] and cut[2:] == [True] * 4


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_fmha_cache_large_scores_across_units(dev, kind):
    """Scores that rise (or fall) along keys which several workgroups share: the units' maxima are far apart."""
    page, pages = 16, 60
    cache = filled_cache(dev, pages, 1, page, 64, kind)
    table = torch.arange(pages, dtype=torch.int32).view(1, pages)
    ramp = torch.linspace(-1, 1, pages * page).view(pages, 1, page, 1)
    q = normal(1, 1, 2, 8, 64, dtype=BF16).abs()
    slots = torch.arange(pages * page, dtype=torch.int32, device=dev)
    v = normal(2, pages * page, 1, 64, dtype=BF16).to(dev)
    for sign in (1, -1):
        k = (sign * ramp * torch.ones(64) * 8).to(BF16).reshape(-1, 1, 64).to(dev)
        ops().kv_cache_write(cache, k, v, slots)
        for scale in (1.0, 30.0):
            workspace = marked_workspace(cache, table, 2, 8)
            check_fmha(dev, cache, q, table, [957], None, None, scale, F32, workspace=workspace)
            assert was_cut(workspace, cache)


def test_cache_beyond_32_bits(dev):
    """A cache of 2^32 elements and more: its last pages are written, read and attended to."""
    heads, page, dim = 8, 256, 128
    pages = (1 << 32) // (heads * page * dim) + 5
    o = ops()
    cache = o.KvCache.empty(pages, heads, page, dim, device=dev)
    assert cache.k.numel() > 1 << 32
    tokens = 2 * page - 9
    at = (pages - 2) * page + torch.arange(tokens, dtype=torch.int32)
    low = torch.arange(tokens, dtype=torch.int32) + page  # where an address cut to 32 bits might land
    k, v = normal(1, tokens, heads, dim, dtype=BF16).to(dev), normal(2, tokens, heads, dim, dtype=BF16).to(dev)
    o.kv_cache_write(cache, -v, -k, low.to(dev))
    o.kv_cache_write(cache, k, v, at.to(dev))
    codes, exps = ref.quantise(k.cpu())
    assert torch.equal(raw(cache.k)[pages - 2:].cpu().transpose(1, 2).reshape(-1, heads, dim)[:tokens], codes)
    got_k, got_v = o.kv_cache_read(cache, at.to(dev), out_dtype=F32)
    want_k = ref.dequantise(codes, exps)
    want_v = ref.dequantise(*ref.quantise(v.cpu()))
    assert torch.equal(got_k.cpu().double(), want_k) and torch.equal(got_v.cpu().double(), want_v)
    q = normal(3, 1, 2, 16, dim, dtype=BF16)
    table = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32)
    got = o.fmha_cache(q.to(dev), cache, table.to(dev), torch.tensor([tokens - 2], dtype=torch.int32, device=dev),
                       scale=0.09, out_dtype=F32)
    small = torch.zeros(2, heads, page, dim, dtype=torch.float64), torch.zeros(2, heads, page, dim, dtype=torch.float64)
    for to, x in zip(small, (want_k, want_v)):
        for t in range(tokens):
            to[t // page, :, t % page] = x[t]
    want, arith, weight = ref.fmha_cache(q, *small, torch.tensor([[0, 1]]), [tokens - 2], None, None, 0.09, got.cpu())
    within(got, want, arith + 2.0 ** -24 * 2 * weight)


# ---- together -----------------------------------------------------------------------------------


def serving_step(o, cache, qkv, weights, pos, freq, slots, table, context, drafts, tree, Hq, Hk, out):
    """What one decoding step of a layer runs."""
    q, k = o.qk_norm_rope(qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], *weights, pos, freq)
    o.kv_cache_write(cache, k, qkv[:, :, Hq + Hk:], slots)
    o.fmha_cache(q, cache, table, context, draft_lens=drafts, tree_mask=tree, scale=q.shape[-1] ** -0.5, out=out)


def step_inputs(dev, seed, B=3, N=4, Hq=8, Hk=2, D=128, page=16, context=(70, 0, 129)):
    per = 10
    table = make_table(B, per, 32, 4)
    slots = torch.full((B, N), -1, dtype=torch.int32)
    for b in range(B):
        for n in range(N):
            key = context[b] + n
            slots[b, n] = int(table[b, key // page]) * page + key % page
    pos = torch.tensor(context)[:, None] + torch.arange(N)
    freq = 1e4 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    host = dict(qkv=normal(seed, B, N, Hq + 2 * Hk, D, dtype=BF16), wq=(1 + 0.1 * normal(seed + 1, D)).to(BF16),
                wk=(1 + 0.1 * normal(seed + 2, D)).to(BF16), pos=pos.to(torch.int32), freq=freq.float(), slots=slots,
                table=table, context=torch.tensor(context, dtype=torch.int32),
                drafts=torch.tensor([4, 3, 1], dtype=torch.int32), tree=random_trees(B, N, 5))
    return host, {n: t.to(dev) for n, t in host.items()}


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_a_decoding_step(dev, kind):
    o = ops()
    cache = filled_cache(dev, 32, 2, 16, 128, kind)
    host, d = step_inputs(dev, 100)
    out = torch.full((3, 4, 8, 128), 7.0, dtype=BF16, device=dev)
    before_k, before_v = raw(cache.k).cpu().clone(), raw(cache.v).cpu().clone()
    serving_step(o, cache, d["qkv"], (d["wq"], d["wk"]), d["pos"], d["freq"], d["slots"], d["table"], d["context"],
                 d["drafts"], d["tree"], 8, 2, out)
    q, k = o.qk_norm_rope(d["qkv"][:, :, :8], d["qkv"][:, :, 8:10], d["wq"], d["wk"], d["pos"], d["freq"])
    for g, x, w in ((q, host["qkv"][:, :, :8], host["wq"]), (k, host["qkv"][:, :, 8:10], host["wk"])):
        want, size = ref.norm_rope(x, w, host["pos"], host["freq"], 1e-6, False)
        within(g, want, 32 * U * size)
    # everything but the new slots is as it was
    touched = torch.zeros(32 * 16, dtype=torch.bool)
    touched[host["slots"].reshape(-1).long()] = True
    touched = touched.view(32, 1, 16, 1)
    for now, then in ((cache.k, before_k), (cache.v, before_v)):
        assert torch.equal(raw(now).cpu()[~touched.expand_as(then)], then[~touched.expand_as(then)])
    got_k, _ = o.kv_cache_read(cache, d["slots"], out_dtype=BF16)
    if kind == BF16:
        assert torch.equal(got_k, k)
    kk, vv = cache_values(cache)
    want, arith, weight = ref.fmha_cache(q.cpu(), kk, vv, host["table"], host["context"], host["drafts"], host["tree"],
                                         128 ** -0.5, torch.full(out.shape, 7.0))
    within(out, want, arith + 2.0 ** -8 * 1.02 * weight)


def test_drafts_agree_with_attention_over_whole_sequences(dev):
    """A chain over a bf16 cache is the causal attention of the same tokens; so is a prefill on what is read back."""
    o = ops()
    B, S, H, D, N = 2, 96, 4, 128, 32
    q, k, v = (normal(i, B, S, H, D, dtype=BF16).to(dev) for i in (1, 2, 3))
    cache = filled_cache(dev, 14, H, 16, D, BF16)
    table = make_table(B, 7, 14, 4)
    key = torch.arange(S)
    slots = (table[:, key // 16] * 16 + (key % 16)).to(torch.int32).to(dev)
    o.kv_cache_write(cache, k, v, slots)
    bhsd = [t.transpose(1, 2).contiguous() for t in (q, k, v)]
    whole = o.fmha(*bhsd, scale=D ** -0.5, causal=True, out_dtype=F32).transpose(1, 2)
    part = o.fmha_cache(q[:, S - N:], cache, table.to(dev), torch.full((B,), S - N, dtype=torch.int32, device=dev),
                        scale=D ** -0.5, out_dtype=F32)
    kk, vv = cache_values(cache)
    want, arith, weight = ref.fmha_cache(q[:, S - N:].cpu(), kk, vv, table, [S - N] * B, None, None, D ** -0.5,
                                         torch.zeros(B, N, H, D))
    within(part, want, arith + 2.0 ** -24 * 2 * weight)
    assert ((whole[:, S - N:].cpu().double() - want).abs() <= 2.0 ** -8 * 1.2 * weight + arith).all()
    outs = tuple(torch.empty(B, H, S, D, dtype=BF16, device=dev) for _ in range(2))
    o.kv_cache_read(cache, slots, out=tuple(t.transpose(1, 2) for t in outs))
    assert torch.equal(outs[0], bhsd[1]) and torch.equal(outs[1], bhsd[2])
    assert torch.equal(o.fmha(bhsd[0], *outs, scale=D ** -0.5, causal=True, out_dtype=F32).transpose(1, 2), whole)


def test_a_prompt_continues_a_cached_prefix(dev):
    """More new tokens than one call takes, grouped heads: written and attended to in chains of up to 64."""
    o = ops()
    B, H, Hk, D, page, new = 2, 8, 2, 64, 16, 150
    prefix, width = [70, 33], 14
    cache = filled_cache(dev, 30, Hk, page, D, BF16)
    table = make_table(B, width, 30, 4)
    q, k, v = (normal(i, B, new, h, D, dtype=BF16).to(dev) for i, h in ((1, H), (2, Hk), (3, Hk)))
    key = torch.tensor(prefix)[:, None] + torch.arange(new)
    slots = (table.gather(1, key // page) * page + key % page).to(torch.int32).to(dev)
    parts = []
    for at in range(0, new, 64):
        now = slice(at, at + 64)
        o.kv_cache_write(cache, k[:, now], v[:, now], slots[:, now].contiguous())
        context = torch.tensor([p + at for p in prefix], dtype=torch.int32, device=dev)
        parts.append(o.fmha_cache(q[:, now], cache, table.to(dev), context, scale=D ** -0.5, out_dtype=F32))
    want, arith, weight = ref.fmha_cache(q.cpu(), *cache_values(cache), table, prefix, None, None, D ** -0.5,
                                         torch.zeros(q.shape))
    within(torch.cat(parts, 1), want, arith + 2.0 ** -24 * 2 * weight)


def test_captured_steps_replay(dev):
    """Two captured steps and the backward pass, replayed with eager work between and with inputs that change."""
    o = ops()
    cache = filled_cache(dev, 32, 2, 16, 128, E4M3)
    twin = filled_cache(dev, 32, 2, 16, 128, E4M3)
    _, d = step_inputs(dev, 200)
    outs = [torch.zeros(3, 4, 8, 128, dtype=BF16, device=dev) for _ in range(2)]

    def step(c, out):
        serving_step(o, c, d["qkv"], (d["wq"], d["wk"]), d["pos"], d["freq"], d["slots"], d["table"], d["context"],
                     d["drafts"], d["tree"], 8, 2, out)

    def back():
        return o.qk_norm_rope_backward(d["qkv"][:, :, :8], d["qkv"][:, :, 8:10], d["qkv"][:, :, :8],
                                       d["qkv"][:, :, 8:10], d["wq"], d["wk"], d["pos"], d["freq"])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(cache, outs[0])
        back()
    side.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        step(cache, outs[0])
        grads = back()
    with torch.cuda.graph(graphs[1]):
        step(cache, outs[1])
    for round_ in range(4):
        d["qkv"].copy_(normal(300 + round_, *d["qkv"].shape, dtype=BF16))
        d["context"].copy_(torch.tensor([70 - round_, round_, 129 - 3 * round_], dtype=torch.int32))
        outs[0].fill_(-1)
        graphs[0].replay()
        graphs[1].replay()
        eager = torch.full_like(outs[0], -1.0)
        torch.cuda.synchronize()
        step(twin, eager)
        assert torch.equal(raw(cache.k), raw(twin.k)) and torch.equal(cache.v_exp, twin.v_exp)
        assert torch.equal(outs[0], eager)
        for a, b in zip(grads, back()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("B", [3, 70])
def test_captured_attention_of_cut_sequences_replays(dev, B):
    """Two captured calls with the launches that find units and join them, in workspaces of the capture's own,
    replayed with eager work between and with lengths, tables and keys that change."""
    o = ops()
    N, Hq, Hk, D, page, width = 2, 8, 2, 64, 16, 64
    cache = filled_cache(dev, 100, Hk, page, D, BF16)
    q = normal(1, B, N, Hq, D, dtype=BF16).to(dev)
    table = torch.randint(0, 100, (B, width), generator=gen(2)).to(torch.int32).to(dev)
    context = torch.full((B,), 900, dtype=torch.int32, device=dev)
    drafts = torch.full((B,), N, dtype=torch.int32, device=dev)
    assert o.fmha_cache_workspace_bytes(cache, width, B, N, Hq) > 0
    outs = [torch.zeros(B, N, Hq, D, dtype=t, device=dev) for t in (BF16, F32)]

    def call(out):
        return o.fmha_cache(q, cache, table, context, draft_lens=drafts, scale=0.125, out=out)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for out in outs:
            call(out)
    side.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in outs]
    for graph, out in zip(graphs, outs):
        with torch.cuda.graph(graph):
            call(out)
    g = gen(3)
    for round_ in range(4):
        q.copy_(normal(10 + round_, *q.shape, dtype=BF16))
        cache.k.copy_(normal(20 + round_, *cache.k.shape, dtype=BF16))
        lengths = torch.randint(0, 60, (B,), generator=g).to(torch.int32)
        lengths[round_ % B], lengths[-1] = 1000 - 100 * round_, 1022
        context.copy_(lengths)
        drafts.copy_(torch.randint(0, N + 1, (B,), generator=g).to(torch.int32))
        drafts[-1] = N
        table.copy_(torch.randint(0, 100, (B, width), generator=g).to(torch.int32))
        for out in outs:
            out.fill_(-1)
        for graph in graphs + graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert torch.equal(out, call(torch.full_like(out, -1)))
        workspace = marked_workspace(cache, table, N, Hq)
        got = check_fmha(dev, cache, q.cpu(), table.cpu(), lengths.tolist(), drafts.tolist(), None, 0.125, F32,
                         workspace=workspace)
        assert was_cut(workspace, cache)
        live = (torch.arange(N, device=dev) < drafts[:, None])[..., None, None]
        assert torch.equal(torch.where(live, got, -1.0), outs[1])


def test_two_streams_at_once(dev):
    """Calls that overlap on two streams do not share anything."""
    o = ops()
    caches = [filled_cache(dev, 300, 2, 16, 128, E4M3, seed=10 * i) for i in range(2)]
    table = make_table(1, 300, 300, 1).to(dev)
    context = torch.tensor([4790], dtype=torch.int32, device=dev)
    q = normal(1, 1, 4, 8, 128, dtype=BF16).to(dev)
    alone = [o.fmha_cache(q, c, table, context, scale=0.1) for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(o.fmha_cache(q, caches[i], table, context, scale=0.1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, alone[i]) for g in got[i])


def test_refusals_of_the_python_layer(dev):
    o = ops()
    _, d = step_inputs(dev, 1)
    q, k, v = d["qkv"][:, :, :8], d["qkv"][:, :, 8:10], d["qkv"][:, :, 10:]
    cache = filled_cache(dev, 32, 2, 16, 128, E4M3)
    norm = dict(q=q, k=k, q_weight=d["wq"], k_weight=d["wk"], positions=d["pos"], inv_freq=d["freq"])

    def refused(fn, base, **change):
        with pytest.raises((ValueError, __import__("kernelcodegen_amd").lib.KcgError)):
            fn(**{**base, **change})
    for change in (dict(q=q.half()), dict(k=k.float()), dict(q=q.cpu()), dict(k=k[:, :2]), dict(k=k[..., :64]),
                   dict(q=q.transpose(2, 3)), dict(q_weight=d["wq"].float()), dict(k_weight=d["wk"][:64]),
                   dict(positions=d["pos"].long()), dict(positions=d["pos"][:2]), dict(positions=d["pos"].cpu()),
                   dict(inv_freq=d["freq"].double()), dict(inv_freq=d["freq"][:5]), dict(inv_freq=d["freq"][:0]),
                   dict(eps=-1.0), dict(out=(q, q)), dict(q=q[:0], k=k[:0], positions=d["pos"][:0]),
                   dict(out=(torch.empty(1, 4, 8, 128, dtype=BF16, device=dev).expand(3, 4, 8, 128), k))):
        refused(o.qk_norm_rope, norm, **change)
    refused(o.qk_norm_rope_backward, dict(norm, dq=q, dk=k), dq=q.float())
    refused(o.qk_norm_rope_backward, dict(norm, dq=q, dk=k), dk=k[:, :, :1])
    refused(o.qk_norm_rope_backward, dict(norm, dq=q, dk=k), workspace=torch.empty(16, device=dev))
    write = dict(cache=cache, k=k, v=v, slots=d["slots"])
    for change in (dict(cache=None), dict(k=k.half()), dict(v=v.float()), dict(k=q, v=q), dict(slots=d["slots"].long()),
                   dict(slots=d["slots"][:2]), dict(slots=d["slots"].cpu()), dict(k=k[:0], v=v[:0], slots=d["slots"][:0])):
        refused(o.kv_cache_write, write, **change)
    read = dict(cache=cache, slots=d["slots"])
    for change in (dict(out_dtype=torch.float16), dict(slots=d["slots"].float()), dict(out=(k, q)), dict(slots=d["slots"][:0]),
                   dict(out=(k, v[:, :, :1].expand(3, 4, 2, 128)))):
        refused(o.kv_cache_read, read, **change)
    attend = dict(q=q, cache=cache, block_table=d["table"], context_lens=d["context"])
    for change in (dict(q=q.float()), dict(q=q[:, :, :3]), dict(q=q[..., :64]), dict(block_table=d["table"].long()),
                   dict(block_table=d["table"][:2]), dict(block_table=d["table"][:, :0]), dict(context_lens=d["context"][:2]),
                   dict(draft_lens=d["drafts"].long()), dict(tree_mask=d["tree"].int()), dict(tree_mask=d["tree"][:, :2]),
                   dict(out_dtype=torch.float16), dict(out=torch.empty(3, 4, 8, 128, device=dev), out_dtype=BF16),
                   dict(scale=math.nan), dict(q=q[:, :1].expand(3, 65, 8, 128)), dict(cache=cache.k)):
        refused(o.fmha_cache, attend, **change)
    for bad in ((cache.k, cache.v), (cache.k, cache.v, cache.k_exp, cache.k_exp[:3]), (cache.k.float(), cache.v.float()),
                (cache.k, raw(cache.v), cache.k_exp, cache.v_exp), (q[:, :, :2], q[:, :, :2])):
        with pytest.raises(ValueError):
            o.KvCache(*bad)
    # a cache whose geometry the library does not take is refused at its first use
    small = torch.zeros(4, 2, 8, 128, dtype=BF16, device=dev)
    refused(o.kv_cache_read, dict(cache=o.KvCache(small, small.clone()), slots=d["slots"]))
