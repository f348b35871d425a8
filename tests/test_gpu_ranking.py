"""The ranking operators (alsmi.ranking) against their definitions in 64 bits (oracle.ranking_oracle).

Tolerances.  Codes, scales, item lists and selected scores are exact.  A score is a sum of `width`
exact products (up to three bf16 parts per fp32 activation) in fp32: each of at most 3 * width
additions is off by at most one ulp (2^-23) of a partial sum, which is at most sum |a_k t_k|; the
output type rounds once by half a step.  An adjusted score passes at most eight roundings (three
parameters to fp32, division or product, product and sum of the penalty, two biases) relative to the
largest magnitude met, then the output's half step."""
import numpy as np
import pytest
import torch

from alsmi import ranking as rk
from oracle import ranking_oracle as ro

pytestmark = pytest.mark.gpu

F32, F64, F16, BF16 = torch.float32, torch.float64, torch.float16, torch.bfloat16
NAN, INF = float('nan'), float('inf')


def gpu(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.detach().to(F64).cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def strided(t, pad=3, offset=1):
    """The same values in rows `pad` elements further apart, starting `offset` elements into the
    memory."""
    n, m = t.shape
    flat = torch.full((offset + n * (m + pad),), 7.0, dtype=t.dtype, device=t.device)
    view = flat[offset:].view(n, m + pad)[:, :m]
    view.copy_(t)
    return view, flat


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------ quantise
SHAPES = [(1, 1), (3, 8), (5, 31), (4, 32), (7, 33), (300, 10), (17, 64), (9, 100), (130, 128),
          (2, 1000), (3, 2047), (2, 2049), (1, 9000)]


@pytest.mark.parametrize('dtype', [F32, F64, F16, BF16])
@pytest.mark.parametrize('shape', SHAPES)
def test_quantize_matches_definition(shape, dtype):
    rng = np.random.default_rng(shape[0] * 1000 + shape[1])
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal((shape[0], 1)) * 3)
    x[rng.random(shape) < 0.05] = 0.0
    xd = gpu(x).to(dtype)
    want_c, want_s = ro.mx4_quantize(host(xd))
    for source in (xd, strided(xd)[0], strided(xd, 5, 2)[0]):
        t = rk.mx4_quantize(source)
        assert t.shape == shape and t.width == shape[1]
        np.testing.assert_array_equal(t.scales.cpu().numpy(), want_s)
        np.testing.assert_array_equal(t.codes.cpu().numpy(), want_c)
    assert t.nbytes == 17 * shape[0] * ((shape[1] + 31) // 32)


@pytest.mark.parametrize('dtype', [F32, F64, F16, BF16])
def test_quantize_ties_extremes_and_non_finite(dtype):
    """Every midpoint and its neighbours at scales from the smallest to the largest the type
    has, blocks of zeros, and blocks with infinities and NaN beside ordinary ones."""
    info = torch.finfo(dtype)
    edge = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    rows = []
    lo, hi = int(np.floor(np.log2(info.tiny))), int(np.floor(np.log2(info.max)))
    for e in {lo - 2, lo, lo + 3, -20, 0, 7, hi - 3, hi - 2}:
        with np.errstate(over='ignore'):
            base = np.ldexp(np.concatenate((edge, edge * (1 + info.eps), edge * (1 - info.eps / 2),
                                            [4.0, 6.0, 7.0, 0.0, 0.5, 1.0, 7.9, 4.5, 3.0, 2.0, 1.5])),
                            e)
        rows += [base, -base, base[::-1]]
    x = torch.tensor(np.array(rows), dtype=F64).to(dtype)
    extra = torch.zeros(8, 32, dtype=dtype)
    extra[1] = -0.0
    extra[2, 5], extra[3, 31], extra[4, 0] = INF, -INF, NAN
    extra[5] = info.max
    extra[6] = info.smallest_normal / 4
    extra[7, 9] = info.smallest_normal * info.eps  # the smallest denormal
    x = torch.cat((x, extra))
    x = torch.cat((x, x.flip(0)), dim=1)  # two blocks a row
    want_c, want_s = ro.mx4_quantize(host(x))
    t = rk.mx4_quantize(x.cuda())
    np.testing.assert_array_equal(t.scales.cpu().numpy(), want_s)
    np.testing.assert_array_equal(t.codes.cpu().numpy(), want_c)
    np.testing.assert_array_equal(host(rk.mx4_dequantize(t, F64)),
                                  ro.mx4_values(want_c, want_s, 64))


def test_quantize_fp64_is_not_rounded_twice():
    """Values within 1e-12 of a midpoint, which fp32 could not tell from it."""
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    row = np.concatenate((mid * (1 + 1e-12), mid * (1 - 1e-12), mid, [4.0]))
    x = np.stack((row, -row, row * 2.0 ** 300, row * 2.0 ** -300))
    want_c, want_s = ro.mx4_quantize(x)
    t = rk.mx4_quantize(gpu(x))
    np.testing.assert_array_equal(t.scales.cpu().numpy(), want_s)
    np.testing.assert_array_equal(t.codes.cpu().numpy(), want_c)


@pytest.mark.parametrize('dtype', [F32, F64, F16, BF16])
@pytest.mark.parametrize('n,width', [(1, 1), (256, 40), (5, 33), (3, 2080), (40, 256)])
def test_dequantize_every_code_and_scale(n, width, dtype):
    rng = np.random.default_rng(width)
    b = (width + 31) // 32
    codes = rng.integers(0, 256, (n, 16 * b), dtype=np.uint8)
    scales = rng.integers(0, 256, (n, b), dtype=np.uint8)
    scales.ravel()[:4] = np.array([0, 255, 254, 127], dtype=np.uint8)[:scales.size]
    t = rk.Mx4Table(gpu(codes), gpu(scales), width)
    want = torch.from_numpy(ro.mx4_values(codes, scales, width)).to(dtype)
    np.testing.assert_array_equal(host(rk.mx4_dequantize(t, dtype)), host(want))
    ids = rng.integers(-2, n + 2, 50).astype(np.int32)
    ids[:3] = (-2 ** 31, 2 ** 31 - 1, n - 1)
    picked = torch.full((50, width), NAN, dtype=dtype)
    ok = (ids >= 0) & (ids < n)
    picked[torch.from_numpy(ok)] = want[torch.from_numpy(ids[ok].astype(np.int64))]
    out, flat = strided(torch.zeros(50, width, dtype=dtype, device='cuda'))
    rk.mx4_dequantize(t, dtype, rows=gpu(ids), out=out)
    np.testing.assert_array_equal(host(out), host(picked))
    gaps = flat[1:].view(50, width + 3)[:, width:]
    assert bool((gaps == 7).all()) and float(flat[0]) == 7


# -------------------------------------------------------------------------------------- scores
def check_scores(got, a, values, out_dtype, parts=3):
    ref = a @ values.T
    with np.errstate(invalid='ignore'):
        mag = np.abs(a) @ np.abs(values).T
    tol = parts * a.shape[1] * 2.0 ** -23 * mag + half_step(out_dtype) * np.abs(ref)
    tol += torch.finfo(out_dtype).smallest_normal  # fp16 results below its normal range
    bad = ~(np.abs(got - ref) <= tol)
    nan = np.isnan(ref)
    assert (np.isnan(got) == nan).all()
    assert not (bad & ~nan).any(), (np.abs(got - ref) / mag).max()


SCORES = [(1, 1, 1), (1, 17, 31), (3, 100, 32), (16, 65, 33), (17, 50, 64), (40, 37, 65),
          (70, 130, 96), (5, 63, 128), (64, 64, 128), (33, 70, 129), (100, 200, 160),
          (130, 257, 512), (2, 300, 1000), (1, 1, 4097), (20, 500, 640), (150, 260, 1024),
          (300, 520, 300)]


@pytest.mark.parametrize('kind', ['f32', 'bf16', 'f16', 'mx4'])
@pytest.mark.parametrize('m,n,width', SCORES)
def test_scores_match_definition(m, n, width, kind):
    rng = np.random.default_rng(m + 10 * n + 100 * width)
    codes, scales = ro.mx4_quantize(rng.standard_normal((n, width)) *
                                    np.exp(rng.standard_normal((n, 1))))
    values = ro.mx4_values(codes, scales, width)
    table = rk.Mx4Table(gpu(codes), gpu(scales), width)
    a = gpu(rng.standard_normal((m, width)))
    if kind == 'mx4':
        ca, sa = ro.mx4_quantize(host(a))
        at, av = rk.Mx4Table(gpu(ca), gpu(sa), width), ro.mx4_values(ca, sa, width)
    else:
        at = a.to({'f32': F32, 'bf16': BF16, 'f16': F16}[kind])
        av = host(at)
    for out_dtype in (F32, BF16, F16):
        check_scores(host(rk.mx4_scores(at, table, out_dtype=out_dtype)), av, values, out_dtype)
    got = rk.mx4_scores(at, table)
    assert got.dtype == (F32 if kind == 'mx4' else at.dtype)
    # rows by id, some of them missing; strided activations and output
    ids = rng.integers(-1, m + 1, m + 3).astype(np.int32)
    picked = np.full((m + 3, width), np.nan)
    ok = (ids >= 0) & (ids < m)
    picked[ok] = av[ids[ok]]
    source = at if kind == 'mx4' else strided(at)[0]
    out, flat = strided(torch.zeros(m + 3, n, device='cuda'), 5, 3)
    rk.mx4_scores(source, table, rows=gpu(ids), out=out)
    check_scores(host(out), picked, values, F32)
    assert bool((flat[3:].view(m + 3, n + 5)[:, n:] == 7).all()) and bool((flat[:3] == 7).all())


@pytest.mark.parametrize('kind', ['f32', 'bf16', 'f16', 'mx4'])
@pytest.mark.parametrize('m,n,width', [(1, 300001, 64), (3, 540000, 130), (20, 140000, 132),
                                       (1, 70001, 200), (257, 9001, 128), (2048, 2049, 192),
                                       (513, 2000, 2080), (300, 6001, 300), (1000, 2100, 1100),
                                       (129, 8300, 135), (4000, 3333, 520), (70, 16385, 512),
                                       (40, 30001, 256), (90, 9000, 250), (1020, 16300, 700),
                                       (40, 25000, 1100), (3, 140000, 300), (300, 60000, 300),
                                       (18, 70000, 1030)])
def test_scores_large(m, n, width, kind):
    """Sizes that take the long-walk and one-step forms; a strip of items against the definition,
    the rest against another order of the same items."""
    g = torch.Generator(device='cuda')
    g.manual_seed(m + n)
    table = rk.mx4_quantize(torch.randn(n, width, generator=g, device='cuda'))
    a = torch.randn(m, width, generator=g, device='cuda')
    at = rk.mx4_quantize(a) if kind == 'mx4' else a.to({'f32': F32, 'bf16': BF16, 'f16': F16}[kind])
    av = host(rk.mx4_dequantize(at)) if kind == 'mx4' else host(at)
    got = rk.mx4_scores(at, table, out_dtype=F32)
    half = rk.mx4_scores(at, table, out_dtype=BF16)
    assert torch.equal(half, got.to(BF16))  # rounded once, from the same sums
    strip = torch.cat((torch.arange(0, min(n, 64)), torch.arange(n // 2, n // 2 + 40) % n,
                       torch.arange(max(0, n - 70), n))).cuda()
    values = ro.mx4_values(table.codes[strip].cpu().numpy(), table.scales[strip].cpu().numpy(), width)
    check_scores(host(got[:, strip]), av, values, F32)
    back = rk.Mx4Table(table.codes.flip(0).contiguous(), table.scales.flip(0).contiguous(), width)
    assert torch.equal(rk.mx4_scores(at, back, out_dtype=F32).flip(1), got)


@pytest.mark.parametrize('kind', ['f32', 'bf16', 'f16', 'mx4'])
@pytest.mark.parametrize('m,n,width', [(200, 9001, 300), (300, 70000, 544), (17, 40000, 700),
                                       (1010, 16250, 544), (50, 24999, 1030)])
def test_scores_of_picked_rows_large(m, n, width, kind):
    """Rows by id, some missing, out of strided activations into a strided output, at sizes of the
    tiled forms; blocks that are no number reach their items alone."""
    g = torch.Generator(device='cuda')
    g.manual_seed(m)
    table = rk.mx4_quantize(torch.randn(n, width, generator=g, device='cuda'))
    table.scales[5, -1] = 255
    table.scales[n - 1, 0] = 255
    a = torch.randn(3 * m, width, generator=g, device='cuda')
    at = rk.mx4_quantize(a) if kind == 'mx4' else strided(
        a.to({'f32': F32, 'bf16': BF16, 'f16': F16}[kind]), 1, 1)[0]
    ids = torch.randint(0, 3 * m, (m,), generator=g, device='cuda').to(torch.int32)
    ids[3], ids[m - 1] = -1, 3 * m
    out, flat = strided(torch.zeros(m, n, device='cuda'), 3, 1)
    rk.mx4_scores(at, table, rows=ids, out=out)
    assert bool((flat[1:].view(m, n + 3)[:, n:] == 7).all())
    none = torch.zeros(m, dtype=torch.bool, device='cuda')
    none[3] = none[m - 1] = True
    nan = torch.isnan(out)
    want = torch.zeros_like(nan)
    want[none] = True
    want[:, 5] = want[:, n - 1] = True
    assert torch.equal(nan, want)
    values = rk.mx4_dequantize(at) if kind == 'mx4' else at.float()
    picked = values[ids.long().clamp(0, 3 * m - 1)]
    cols = torch.randint(6, n - 1, (50,), generator=g, device='cuda')
    check_scores(host(out[~none][:, cols]), host(picked[~none]),
                 host(rk.mx4_dequantize(table, rows=cols.to(torch.int32))), F32)


@pytest.mark.parametrize('kind', ['f32', 'bf16', 'f16', 'mx4'])
@pytest.mark.parametrize('width', [40, 200])
def test_scores_with_infinities_nan_and_extreme_scales(width, kind):
    """A block that is no number makes its item's scores NaN and no other's; infinite and NaN
    activations stay in their rows; elements behind the width are never looked at."""
    rng = np.random.default_rng(width)
    n, m = 40, 20
    codes, scales = ro.mx4_quantize(rng.standard_normal((n, width)))
    codes |= (codes & 0x77 == 0).astype(np.uint8) * 0x11  # no zeros: 0 * inf is NaN
    codes |= ((codes & 0x07) == 0).astype(np.uint8)
    codes |= ((codes & 0x70) == 0).astype(np.uint8) * 0x10
    scales[3, 1] = 255
    scales[5] = 0
    scales[6] = 200
    values = ro.mx4_values(codes, scales, width)
    table = rk.Mx4Table(gpu(codes), gpu(scales), width)
    a = rng.standard_normal((m, width))
    if kind == 'mx4':
        ca, sa = ro.mx4_quantize(a)
        sa[4, 0] = 255
        sa[7] = 1
        at, av = rk.Mx4Table(gpu(ca), gpu(sa), width), ro.mx4_values(ca, sa, width)
    else:
        dtype = {'f32': F32, 'bf16': BF16, 'f16': F16}[kind]
        a[2, 0], a[4, width - 1], a[9, 33] = np.inf, np.nan, -np.inf
        if kind == 'f32':
            a[11] *= 1e-38
            a[12] *= 1e30
        full = torch.full((m, width + 8), NAN, dtype=dtype, device='cuda')
        full[:, :width] = gpu(a)
        at = full[:, :width]
        av = host(at)
    got = host(rk.mx4_scores(at, table, out_dtype=F32))
    with np.errstate(invalid='ignore', over='ignore'):
        ref = (av[:, None, :] * values[None]).sum(-1)
        mag = np.abs(av[:, None, :] * values[None]).sum(-1)
    # Finite operands whose products leave fp32's range: +inf and -inf may meet in an fp32 sum
    # (2^73 from the scale times 1e30 = 2^99.7), so only "not finite or within the tolerance" holds
    past = np.isfinite(mag) & (mag > np.finfo(np.float32).max)
    assert not past[np.arange(m) != 12].any()
    inf = np.isinf(ref)
    assert (np.isnan(got) == np.isnan(ref))[~past].all()
    assert (got[inf] == ref[inf]).all()
    ok = np.isfinite(ref) & ~past
    # An activation's last part is cut at bf16's smallest number, 2^-133, so each product may lose
    # that times the table's element; products below fp32's normal range are off by 2^-149 at most.
    with np.errstate(invalid='ignore'):
        lost = 2.0 ** -133 * np.abs(values).max(1) + 3 * 2.0 ** -149
        tol = width * (3 * 2.0 ** -23 * mag + lost)
        worst = np.argwhere(ok & ~(np.abs(got - ref) <= tol))
    assert worst.size == 0, [(i, j, got[i, j], ref[i, j], tol[i, j]) for i, j in worst[:8]]


def test_scores_of_nothing():
    table = rk.mx4_quantize(torch.randn(5, 40, device='cuda'))
    none = rk.mx4_quantize(torch.randn(0, 40, device='cuda'))
    assert len(none) == 0
    assert rk.mx4_scores(torch.zeros(0, 40, device='cuda'), table).shape == (0, 5)
    assert rk.mx4_scores(torch.zeros(2, 40, device='cuda'), none).shape == (2, 0)
    assert rk.mx4_dequantize(none).shape == (0, 40)


# -------------------------------------------------------------------------------------- adjust
def lists(rng, rows, items, mean, low=-3, high=3):
    n = rng.poisson(mean, rows)
    n[rng.random(rows) < 0.2] = 0
    ptr = np.concatenate(([0], np.cumsum(n))).astype(np.int64)
    ids = rng.integers(low, max(items // 3, 1) + high, int(ptr[-1])).astype(np.int32)
    return ptr, ids


ADJUST = [(1, 1), (3, 31), (2, 64), (4, 1000), (5, 2048), (3, 2049), (2, 5003), (33, 300)]


def adjust_case(rng, n, m, what):
    kw, want = {}, {}
    if 'history' in what or 'exclude' in what:
        h = lists(rng, n, m, 40)
        kw['history'], want['history'] = tuple(map(gpu, h)), h
    if 'exclude' in what:
        kw['exclude'] = want['exclude'] = True
    if 'history' in what:
        for name, v in (('repetition', 1.3), ('frequency', 0.25), ('presence', -0.5)):
            if 'tensors' in what:
                v = (v * rng.uniform(0.5, 2, n)).astype(np.float32)
                kw[name], want[name] = gpu(v), v
            else:
                kw[name] = want[name] = v
    if 'rows' in what:
        r = rng.integers(-1, n + 2, n).astype(np.int32)
        kw['history_rows'], want['history_rows'] = gpu(r), r
    if 'bias' in what:
        want['item_bias'] = rng.standard_normal(m).astype(np.float32)
        kw['item_bias'] = gpu(want['item_bias'])
        p, i = lists(rng, n, m, 9)
        v = rng.standard_normal(i.size).astype(np.float32)
        kw['row_bias'], want['row_bias'] = (gpu(p), gpu(i), gpu(v)), (p, i, v)
    if 'mask' in what:
        allowed = rng.random((4, m)) < 0.6
        allowed[1] = False
        words = rk.pack_mask(allowed)
        r = rng.integers(-1, 5, n).astype(np.int32)
        kw['mask'], want['mask'] = gpu(words), words
        kw['mask_rows'], want['mask_rows'] = gpu(r), r
    return kw, want


@pytest.mark.parametrize('dtype', [F32, F64, F16, BF16])
@pytest.mark.parametrize('what', ['', 'history', 'history tensors rows', 'exclude', 'exclude rows mask',
                                  'bias', 'mask', 'history tensors bias mask'])
@pytest.mark.parametrize('n,m', ADJUST)
def test_adjust_matches_definition(n, m, what, dtype):
    rng = np.random.default_rng(n * 10007 + m)
    s = gpu(rng.standard_normal((n, m)) * 3).to(dtype)
    kw, want = adjust_case(rng, n, m, what)
    ref, mag = ro.adjust_scores(host(s), **want)
    eps = half_step(F64 if dtype == F64 else F32)
    tol = 8 * eps * mag + half_step(dtype) * np.where(np.isfinite(ref), np.abs(ref), 0)
    tol += torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    inf = np.isinf(ref)

    def check(got):
        got = host(got)
        assert (got[inf] == ref[inf]).all()
        assert (np.abs(got[~inf] - ref[~inf]) <= tol[~inf]).all()
    kept = s.clone()
    check(rk.adjust_scores(s, **kw))
    assert torch.equal(s, kept)
    # strided in, strided out, nothing written between the rows
    source, _ = strided(s)
    out, flat = strided(torch.zeros_like(s), 4, 2)
    check(rk.adjust_scores(source, out=out, **kw))
    assert bool((flat[2:].view(n, m + 4)[:, m:] == 7).all()) and bool((flat[:2] == 7).all())
    # in place, contiguous and strided
    again = s.clone()
    assert rk.adjust_scores(again, out=again, **kw) is again
    check(again)
    inner, flat = strided(s)
    check(rk.adjust_scores(inner, out=inner, **kw))
    assert bool((flat[1:].view(n, m + 3)[:, m:] == 7).all())


def test_adjust_non_finite_scores():
    """NaN and infinities stay where nothing takes them out, and go where the mask or the
    exclusion does; the type's lowest value is an ordinary score."""
    m = 40
    for dtype in (F32, F16, BF16, F64):
        low = torch.finfo(dtype).min
        s = torch.zeros(2, m, dtype=dtype, device='cuda')
        s[:, 0], s[:, 1], s[:, 2], s[:, 3] = NAN, INF, -INF, low
        s[:, 10], s[:, 11], s[:, 12] = NAN, INF, -INF
        allowed = np.ones((2, m), dtype=bool)
        allowed[1, 10:13] = False
        h = (gpu(np.array([0, 3, 6], dtype=np.int64)), gpu(np.array([0, 1, 2] * 2, dtype=np.int32)))
        got = rk.adjust_scores(s, history=h, repetition=2.0, frequency=1.0, presence=1.0,
                               mask=gpu(rk.pack_mask(allowed)))
        assert bool(torch.isnan(got[:, 0]).all())
        assert bool((got[:, 1] == INF).all()) and bool((got[:, 2] == -INF).all())
        assert bool((got[:, 3] == low).all())
        assert bool(torch.isnan(got[0, 10])) and float(got[0, 11]) == INF
        assert bool((got[1, 10:13] == -INF).all())
        out = rk.adjust_scores(s, history=h, exclude=True)
        assert bool((out[:, :3] == -INF).all()) and bool(torch.isnan(out[:, 10]).all())


def test_adjust_many_occurrences_and_long_lists():
    """One item 100 000 times, lists longer than a workgroup's turn, the last of equal bias
    entries, pointers that leave the list."""
    m, n = 5000, 3
    rng = np.random.default_rng(5)
    ids = np.concatenate((np.full(100000, 17), rng.integers(0, m, 30000), [-1, m, 2 ** 31 - 1]))
    ptr = np.array([0, 100000, ids.size, ids.size], dtype=np.int64)
    h = (gpu(ptr), gpu(ids.astype(np.int32)))
    s = torch.zeros(n, m, dtype=F32, device='cuda')
    got = host(rk.adjust_scores(s, history=h, frequency=1.0))
    for r in range(n):
        part = ids[ptr[r]:ptr[r + 1]]
        want = -np.bincount(part[(part >= 0) & (part < m)], minlength=m).astype(np.float64)
        np.testing.assert_array_equal(got[r], want)
    values = rng.standard_normal(ids.size).astype(np.float32)
    got = host(rk.adjust_scores(s, row_bias=h + (gpu(values),)))
    assert got[0, 17] == values[99999]
    wide = (gpu(np.array([-5, 4, 2, 10 ** 12], dtype=np.int64)), h[1][:6].contiguous())
    got = host(rk.adjust_scores(s, history=wide, frequency=1.0))
    assert got[0, 17] == -4 and (got[1] == 0).all() and got[2, 17] == -4


# ---------------------------------------------------------------------------------------- topk
def check_topk(s, k, **kw):
    items, best = rk.topk_rows(s, k, **kw)
    raw = s.contiguous().cpu()
    view = raw.view(torch.int16).numpy().view(np.float16) if s.dtype == BF16 else raw.numpy()
    want = ro.topk_rows(view, k)
    np.testing.assert_array_equal(items.cpu().numpy(), want)
    picked = torch.gather(raw, 1, torch.from_numpy(want.astype(np.int64)))
    assert best.dtype == s.dtype
    np.testing.assert_array_equal(host(best), host(picked))


TOPK = [(1, 1, 1), (3, 5, 5), (2, 64, 7), (2, 1024, 1024), (2, 4096, 10), (2, 4097, 1), (3, 4097, 1024),
        (1, 50000, 1024), (5, 10000, 100), (1, 300000, 64), (2, 8191, 300), (40, 3000, 33),
        (1, 1000003, 10), (300, 257, 20), (2, 20000, 512), (9, 26744, 10)]


@pytest.mark.parametrize('dtype', [F32, F64, F16, BF16])
@pytest.mark.parametrize('n,m,k', TOPK)
def test_topk_matches_definition(n, m, k, dtype):
    g = torch.Generator(device='cuda')
    g.manual_seed(n + 7 * m + k)
    s = torch.randn(n, m, generator=g, device='cuda').to(dtype)
    check_topk(s, k)
    check_topk(strided(s)[0], k)
    # sorted rows: the best all in one place
    check_topk(torch.sort(s, dim=1, descending=True).values.contiguous(), k)
    check_topk(torch.sort(s, dim=1).values.contiguous(), k)


@pytest.mark.parametrize('dtype', [F32, F64, F16, BF16])
@pytest.mark.parametrize('m,k', [(50, 50), (4096, 1024), (9000, 10), (9000, 1000), (60000, 257)])
def test_topk_ties_and_special_values(m, k, dtype):
    """All scores equal, all -inf, a few different ones, -inf except for fewer than k, NaN of
    both signs, both zeros, denormals."""
    g = torch.Generator(device='cuda')
    g.manual_seed(m + k)
    rows = [torch.full((m,), 1.5), torch.full((m,), -INF), torch.zeros(m),
            torch.randint(0, 3, (m,), generator=g, device='cuda').cpu().float(),
            torch.full((m,), -INF), torch.randn(m), torch.randn(m) * 0]
    rows[4][torch.randperm(m)[:max(1, k // 2)]] = 2.0
    rows[5][torch.randperm(m)[:10]] = NAN
    rows[5][torch.randperm(m)[:10]] = INF
    s = torch.stack(rows).to(dtype)
    s[5, m // 3] = -s[5, m // 3].abs()
    s[5, m // 2] = torch.copysign(torch.tensor(NAN), torch.tensor(-1.0)).to(dtype)
    s[6, 1::3] = -0.0
    s[6, 2::3] = torch.finfo(dtype).smallest_normal / 2
    check_topk(s.cuda(), k)


def test_topk_batches():
    s = torch.randn(50, 9000, device='cuda')
    check_topk(s, 20, max_workspace_bytes=20000)
    check_topk(strided(s)[0], 20, max_workspace_bytes=1)


# ------------------------------------------------------------------------------- used together
def chain(state, k):
    t = rk.mx4_quantize(state['items'])
    s = rk.mx4_scores(state['users'], t, rows=state['ids'])
    s = rk.adjust_scores(s, history=state['history'], history_rows=state['ids'], exclude=True,
                         item_bias=state['bias'], mask=state['mask'])
    return rk.topk_rows(s, k) + (s,)


def chain_state(rng, n=30, m=5000, width=50, sel=17):
    allowed = rng.random(m) < 0.7
    return {'items': gpu(rng.standard_normal((m, width)), F32),
            'users': gpu(rng.standard_normal((n, width)), F32),
            'ids': gpu(rng.integers(0, n, sel).astype(np.int32)),
            'history': tuple(map(gpu, lists(rng, n, m, 60, 0, 0))),
            'bias': gpu(rng.standard_normal(m).astype(np.float32)),
            'mask': gpu(rk.pack_mask(allowed))}


def test_catalogue_in_four_bits_to_lists():
    """Quantise, score, adjust, select, against the same steps in 64 bits: every listed score is
    its item's score, nothing that is taken out is listed, nothing better is missing."""
    st = chain_state(np.random.default_rng(3))
    items, best, _ = (host(t) for t in chain(st, 25))
    codes, scales = ro.mx4_quantize(host(st['items']))
    values = ro.mx4_values(codes, scales, 50)
    ids = host(st['ids'])
    users = host(st['users'])[ids]
    ref, _ = ro.adjust_scores(users @ values.T, tuple(host(t) for t in st['history']), ids,
                              exclude=True, item_bias=host(st['bias']), mask=host(st['mask']))
    mag = np.abs(users) @ np.abs(values).T + np.abs(host(st['bias']))
    tol = (3 * 50 + 2) * 2.0 ** -23 * mag
    pick = lambda x: np.take_along_axis(x, items.astype(np.int64), axis=1)
    assert np.isfinite(best).all()
    assert (np.abs(best - pick(ref)) <= pick(tol)).all()
    rest = ref.copy()
    np.put_along_axis(rest, items.astype(np.int64), -np.inf, axis=1)
    assert (rest.max(1) <= best[:, -1] + tol.max(1)).all()


def test_chain_captured_and_replayed():
    """The chain in a graph, replayed with other inputs in the same memory, with eager work between
    the replays."""
    rng = np.random.default_rng(4)
    st = chain_state(rng)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(st, 25)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(st, 25)
    for step in range(4):
        st['items'].copy_(gpu(rng.standard_normal((5000, 50)), F32))
        st['ids'].copy_(gpu(rng.integers(0, 30, 17).astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        want = chain(st, 25)
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    rng = np.random.default_rng(6)
    states = [chain_state(rng) for _ in range(2)]
    want = [chain(s, 25) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(5):
        got = []
        for s, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                got.append(chain(s, 25))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


@pytest.mark.parametrize('rank,m', [(3, 40), (20, 700), (64, 2000), (100, 333)])
@pytest.mark.parametrize('dtype', ['float32', 'float64'])
def test_score_items_is_the_block_that_is_ranked(rank, m, dtype):
    from alsmi import device as dev
    device = dev.require_gpu()
    rng = np.random.default_rng(rank)
    U, V = rng.standard_normal((rank, 50)), rng.standard_normal((rank, m))
    Ud, Vd = dev.factors_to_device(U, dtype, device), dev.factors_to_device(V, dtype, device)
    users = rng.integers(0, 50, 70).astype(np.int32)
    s = dev.score_items(rank, gpu(users), Ud, Vd)
    Uq, Vq = dev.factors_to_host(Ud, rank), dev.factors_to_host(Vd, rank)
    mag = np.abs(Uq[:, users]).T @ np.abs(Vq)
    # fp32: the fp16 split keeps 2^-20 of each product, the sums add 3 * 128 roundings
    tol = (2.0 ** -20 + 3 * 128 * 2.0 ** -24 if dtype == 'float32' else 130 * 2.0 ** -53) * mag
    assert (np.abs(host(s) - Uq[:, users].T @ Vq) <= tol).all()
    items, best = rk.topk_rows(s, 10)
    want_items, want = dev.topk_items(rank, gpu(users), Ud, Vd, 10)
    assert torch.equal(items, want_items) and torch.equal(best, want)


@pytest.mark.parametrize('dtype', ['float32', 'float64'])
def test_recommend_with_exclusion_bias_mask_and_quantised_items(dtype, monkeypatch):
    import pickle
    from alsmi import ALS
    import scipy.sparse as sps
    rng = np.random.default_rng(11)
    n, m, k = 60, 500, 12
    R = sps.random(n, m, 0.08, format='csr', random_state=1, data_rvs=lambda s: rng.integers(1, 6, s))
    R = sps.vstack([R, sps.csr_matrix((1, m))], format='csr')      # a user without ratings
    rows, cols = R.nonzero()
    als = ALS(8, random_state=0, max_iter=3, dtype=dtype).fit((rows, cols), R)
    triplets = ALS(8, random_state=0, max_iter=3, dtype=dtype).fit(
        (rows.astype(np.int32), cols.astype(np.int32)), np.asarray(R[rows, cols]).ravel(), shape=R.shape)
    users = np.concatenate((rng.integers(0, n + 1, 30), [n, -1]))
    bias = rng.standard_normal(m).astype(np.float32)
    one, each = rng.random(m) < 0.5, rng.random((users.size, m)) < 0.3
    each[3] = False
    each[4, 7:] = False
    dense = als.user_feats.T @ als.item_feats
    codes, scales = ro.mx4_quantize(als.item_feats.T)
    coarse = als.user_feats.T @ ro.mx4_values(codes, scales, 8).T
    seen = R.toarray() != 0
    for kw in (dict(exclude_seen=True), dict(item_bias=bias), dict(allowed=one), dict(allowed=each),
               dict(exclude_seen=True, item_bias=bias, allowed=each), dict(catalogue='mx4'),
               dict(exclude_seen=True, item_bias=bias, allowed=one, catalogue='mx4')):
        want = (coarse if kw.get('catalogue') == 'mx4' else dense)[users].copy()
        if 'item_bias' in kw:
            want += bias
        if kw.get('exclude_seen'):
            want[seen[users]] = -np.inf
        if 'allowed' in kw:
            want[~np.broadcast_to(kw['allowed'], want.shape)] = -np.inf
        tol = 1e-10 if dtype == 'float64' and 'catalogue' not in kw else 2e-5
        for model, block in ((als, None), (triplets, None), (als, 7)):
            if block:  # several blocks of users
                monkeypatch.setattr('alsmi.als._BLOCK_SCORES', block * m)
            items, scores = model.recommend(users, k, **kw)
            monkeypatch.undo()
            got = np.take_along_axis(want, items.astype(np.int64), axis=1)
            out = np.isinf(scores)
            assert (np.isinf(got) == out).all()
            assert np.abs(scores[~out] - got[~out]).max() <= tol
            rest = want.copy()
            np.put_along_axis(rest, items.astype(np.int64), -np.inf, axis=1)
            assert (rest.max(1) <= scores[:, -1] + tol).all()
            assert all(np.unique(r).size == k for r in items)
    # nothing on offer: the smallest ids, all at -inf
    items, scores = als.recommend([0], 3, allowed=np.zeros(m, bool))
    assert list(items[0]) == [0, 1, 2] and np.isinf(scores).all()
    copy = pickle.loads(pickle.dumps(als))
    a, b = copy.recommend(users, k, catalogue='mx4'), als.recommend(users, k, catalogue='mx4')
    assert (a[0] == b[0]).all() and (a[1] == b[1]).all()
    # a new rating is seen, and the changed user is scored with the new factors
    best = int(als.recommend([0], 1, exclude_seen=True)[0][0, 0])
    als.update_user(0, best, 5.0)
    assert best not in als.recommend([0], k, exclude_seen=True)[0]
    with pytest.raises(ValueError):
        als.recommend([0], m + 1, exclude_seen=True)


# ------------------------------------------------------------------------- the ends of the range
def test_topk_of_rows_of_the_lowest_key():
    """Rows of the one score that ranks below all others (every bit set), of as many items as an
    index has room for: the last two differ from "no score" by their index alone."""
    for n, k in ((128, 127), (128, 65), (1024, 1023), (16384, 1024), (32768, 1024), (65536, 700)):
        for dtype, whole in ((F32, torch.int32), (BF16, torch.int16), (F64, torch.int64)):
            s = torch.full((2, n), -1, dtype=whole, device='cuda').view(dtype)
            s[1, n - 1], s[1, n // 2] = 1.0, 2.0
            items, best = rk.topk_rows(s, k)
            assert torch.equal(items[0].cpu(), torch.arange(k, dtype=torch.int32))
            want = torch.tensor([n // 2, n - 1] + [i for i in range(k) if i != n // 2][:k - 2])
            assert torch.equal(items[1].cpu(), want.to(torch.int32))
            assert bool((best[0].view(whole) == -1).all()) and best[1, :2].tolist() == [2.0, 1.0]


@pytest.mark.parametrize('n,m,k', [(2 ** 23 + 5, 3, 2), (2 ** 21 + 3, 66, 65), (70001, 1000, 64),
                                   (70001, 1024, 1)])
def test_topk_of_very_many_short_rows(n, m, k):
    """More rows than one launch has room for."""
    g = torch.Generator(device='cuda')
    g.manual_seed(m)
    s = torch.randint(-40, 40, (n, m), generator=g, device='cuda', dtype=torch.int8).to(BF16)
    items, best = rk.topk_rows(s, k)
    for lo, hi in ((0, 1000), (2 ** 21 - 500, 2 ** 21 + 500), (n - 1000, n)):
        want, order = torch.sort(s[lo:hi], dim=1, descending=True, stable=True)
        assert torch.equal(items[lo:hi], order[:, :k].to(torch.int32))
        assert torch.equal(best[lo:hi], want[:, :k])
    assert torch.equal(best, s.gather(1, items.to(torch.int64)))
    assert bool((best[:, :-1] >= best[:, 1:]).all()) if k > 1 else True


def test_adjust_very_many_short_rows():
    n, m = 2 ** 23 + 9, 3
    g = torch.Generator(device='cuda')
    g.manual_seed(3)
    s = torch.rand(n, m, generator=g, device='cuda')
    ids = torch.randint(-1, m, (n,), generator=g, device='cuda', dtype=torch.int32)
    ptr = torch.arange(n + 1, device='cuda')
    mask_rows = torch.randint(-1, 2, (n,), generator=g, device='cuda', dtype=torch.int32)
    mask = gpu(rk.pack_mask(np.array([[1, 1, 0], [1, 0, 1]], dtype=bool)))
    got = rk.adjust_scores(s, history=(ptr, ids), exclude=True, mask=mask, mask_rows=mask_rows)
    gone = torch.arange(m, device='cuda') == ids[:, None]
    gone[:, 2] |= mask_rows == 0
    gone[:, 1] |= mask_rows == 1
    assert torch.equal(got, s.masked_fill(gone, -INF))


@pytest.mark.parametrize('kind', ['f32', 'f16', 'mx4'])
def test_scores_of_very_many_rows(kind):
    n, m, width = 2 ** 22 + 70, 3, 5
    g = torch.Generator(device='cuda')
    g.manual_seed(4)
    table = rk.mx4_quantize(torch.randn(m, width, generator=g, device='cuda'))
    a = torch.randn(n, width, generator=g, device='cuda')
    at = rk.mx4_quantize(a) if kind == 'mx4' else a.to({'f32': F32, 'f16': F16}[kind])
    av = rk.mx4_dequantize(at, F64) if kind == 'mx4' else at.to(F64)
    values = rk.mx4_dequantize(table, F64)
    order = torch.randperm(n, generator=g, device='cuda').to(torch.int32)
    order[n - 3] = n
    for rows in (None, order):
        got = rk.mx4_scores(at, table, rows=rows, out_dtype=F32).to(F64)
        if rows is not None:
            assert bool(torch.isnan(got[n - 3]).all())
            got[n - 3] = 0
            rows[n - 3] = 0
        x = av if rows is None else av[rows.to(torch.int64)]
        if rows is not None:
            x[n - 3] = 0
        tol = 3 * width * 2.0 ** -23 * (x.abs() @ values.abs().T) + 2.0 ** -126
        assert bool(((got - x @ values.T).abs() <= tol).all())


@pytest.mark.parametrize('kind,m', [('f32', 700), ('f16', 1100)])
def test_scores_of_very_long_rows(kind, m):
    """Activations whose parts are split in more than one batch of rows; the first rows against the
    definition, all against their own values for one item picked out of the batch."""
    n, width = 2800, 65536
    g = torch.Generator(device='cuda')
    g.manual_seed(m)
    table = rk.mx4_quantize(torch.randn(n, width, generator=g, device='cuda'))
    a = torch.randn(m, width, generator=g, device='cuda').to({'f32': F32, 'f16': F16}[kind])
    got = rk.mx4_scores(a, table, out_dtype=F32).to(F64)
    values = rk.mx4_dequantize(table, F64)
    x = a.to(F64)
    tol = 3 * width * 2.0 ** -23 * (x.abs() @ values.abs().T)
    assert bool(((got - x @ values.T).abs() <= tol).all())


@pytest.mark.parametrize('kind', ['f32', 'bf16', 'mx4'])
@pytest.mark.parametrize('m,n,width', [(300, 20000, 544), (300, 9000, 64), (2, 9000, 300)])
def test_scores_of_codes_at_any_word(m, n, width, kind):
    """Codes aligned to four bytes and no more."""
    g = torch.Generator(device='cuda')
    g.manual_seed(width)

    def shifted(t):
        flat = torch.empty(t.codes.numel() + 4, dtype=torch.uint8, device='cuda')
        flat[4:] = t.codes.view(-1)
        return rk.Mx4Table(flat[4:].view(t.codes.shape), t.scales, t.width)
    table = rk.mx4_quantize(torch.randn(n, width, generator=g, device='cuda'))
    a = torch.randn(m, width, generator=g, device='cuda')
    at = shifted(rk.mx4_quantize(a)) if kind == 'mx4' else a.to({'f32': F32, 'bf16': BF16}[kind])
    av = host(rk.mx4_dequantize(at)) if kind == 'mx4' else host(at)
    got = rk.mx4_scores(at, shifted(table), out_dtype=F32)
    check_scores(host(got), av, host(rk.mx4_dequantize(table)), F32)


def test_offsets_past_32_bits():
    """Blocks of scores of more than 2^31 elements, a table of more than 2^32 bytes of codes: their last
    rows are those of the same rows by themselves."""
    g = torch.Generator(device='cuda')
    g.manual_seed(1)
    n, m = 70000, 32768
    table = rk.mx4_quantize(torch.randn(m, 32, generator=g, device='cuda'))
    a = torch.randn(n, 32, generator=g, device='cuda').to(BF16)
    s = rk.mx4_scores(a, table)
    tail = rk.mx4_scores(a[-200:], table)
    assert torch.equal(s[-200:], tail)
    ids = torch.randint(0, m, (n * 4,), generator=g, device='cuda', dtype=torch.int32)
    ptr = torch.arange(0, 4 * n + 1, 4, device='cuda')
    rk.adjust_scores(s, history=(ptr, ids), exclude=True, out=s)
    rk.adjust_scores(tail, history=(ptr[-201:].clone(), ids), exclude=True, out=tail)
    assert torch.equal(s[-200:], tail)
    for k in (10, 100):
        items, best = rk.topk_rows(s, k)
        items1, best1 = rk.topk_rows(tail, k)
        assert torch.equal(items[-200:], items1) and torch.equal(best[-200:], best1)
    del s, tail
    n, width = 262144 + 100, 32800
    x = torch.zeros(n, width, dtype=BF16, device='cuda')
    x[-100:] = torch.randn(100, width, generator=g, device='cuda')
    table, last = rk.mx4_quantize(x), rk.mx4_quantize(x[-100:])
    assert torch.equal(table.codes[-100:], last.codes)
    assert torch.equal(table.scales[-100:], last.scales)
    ids = torch.arange(n - 100, n, device='cuda', dtype=torch.int32)
    assert torch.equal(rk.mx4_dequantize(table, BF16, rows=ids), rk.mx4_dequantize(last, BF16))
    rk.mx4_dequantize(table, BF16, out=x)
    assert torch.equal(x[-100:], rk.mx4_dequantize(last, BF16))
    a, values = host(x[-3:]), host(x[-100:])
    check_scores(host(rk.mx4_scores(x[-3:], table, out_dtype=F32)[:, -100:]), a, values, F32)
    check_scores(host(rk.mx4_scores(table, last, rows=ids[-3:])), a, values, F32)
    many = torch.cat((ids, ids, ids))
    check_scores(host(rk.mx4_scores(table, last, rows=many)), np.tile(values, (3, 1)), values, F32)


@pytest.mark.parametrize('n,m,k,limit', [(4, 5000000, 10, 3), (4, 1000000, 64, 3), (502, 100000, 1000, 400)])
def test_topk_of_a_last_batch_of_fewer_rows(n, m, k, limit):
    """A rest of the rows, which is cut into more parts than a full batch; the workspace is not left."""
    g = torch.Generator(device='cuda')
    g.manual_seed(n)
    s = torch.randn(n, m, generator=g, device='cuda')
    need = rk._lib.load().alsmi_topk_rows_workspace_bytes
    items, best = rk.topk_rows(s, k, max_workspace_bytes=limit * need(0, 1, m, k))
    want, order = torch.sort(s, dim=1, descending=True, stable=True)
    assert torch.equal(best, want[:, :k]) and torch.equal(items, order[:, :k].to(torch.int32))
    del want, order
    for rows in (1, 2, 100, 102, 128, 129, n):
        if rows > n:
            continue
        size = need(0, rows, m, k)
        ws = torch.full((size + 4096,), 77, dtype=torch.uint8, device='cuda')
        rk._call(s.device, 'alsmi_topk_rows', 0, rows, m, s.data_ptr(), m, k, items.data_ptr(),
                 best.data_ptr(), ws.data_ptr())
        assert bool((ws[size:] == 77).all())


@pytest.mark.parametrize('dtype', [F32, F64, F16, BF16])
@pytest.mark.parametrize('n,m', [(600, 30011), (1100, 8193), (3, 70000), (130, 40000)])
def test_topk_of_ordered_rows(n, m, dtype):
    """Rows in which every key beats the ones before it, none does, all are equal, hardly any is
    there, or they come in runs: the most and the fewest candidates a walk can meet."""
    g = torch.Generator(device='cuda')
    g.manual_seed(n)
    up = torch.arange(m, device='cuda', dtype=F32) / 3 - 5000
    few = torch.full((m,), -INF, device='cuda')
    few[m - 30:] = torch.randn(30, generator=g, device='cuda')
    rows = [up, -up, torch.zeros_like(up), few, few.flip(0), up % 97, -(up % 8192), up.abs(),
            torch.randn(m, generator=g, device='cuda'),
            torch.randint(-3, 3, (m,), generator=g, device='cuda').to(F32)]
    rows = torch.stack([r.to(dtype) for r in rows])
    # an order of the whole block by the order of its ten rows
    which = torch.arange(n, device='cuda') % len(rows)
    s = rows[which]
    want, order = torch.sort(rows + 0.0, dim=1, descending=True, stable=True)  # (+0 and -0 as one)
    s = s + 0.0
    for k in (1, 24, 25, 64, 65, 300, 1000, 1024):
        items, best = rk.topk_rows(s, k)
        assert torch.equal(items, order[:, :k].to(torch.int32)[which])
        assert torch.equal(best, want[:, :k][which])


def test_every_form_captured_and_replayed():
    """Calls of each form in a graph of their own, replayed on other inputs in the same memory with
    eager work between the replays."""
    g = torch.Generator(device='cuda')
    g.manual_seed(9)
    rand = lambda *shape: torch.randn(*shape, generator=g, device='cuda')
    forms = []
    for m, n, width in ((1, 3000, 64), (40, 3000, 200), (5, 3000, 900), (300, 9000, 520),
                        (1020, 16300, 520), (50, 700, 300)):
        table = rk.mx4_quantize(rand(n, width))
        for dtype in (F32, BF16):
            a = rand(m, width).to(dtype)
            forms.append((a, lambda a=a, t=table: rk.mx4_scores(a, t, out_dtype=F32)))
        a = rand(m, width)
        forms.append((a, lambda a=a, t=table: rk.mx4_scores(rk.mx4_quantize(a), t)))
    for n, m, k in ((1, 50000, 10), (2, 900, 7), (1, 50000, 60), (3, 70000, 500), (700, 20000, 100),
                    (1, 1000000, 1024)):
        s = rand(n, m)
        forms.append((s, lambda s=s, k=k: rk.topk_rows(s, k)))
    ptr = torch.arange(0, 401, 100, device='cuda')
    ids = torch.randint(0, 9000, (400,), generator=g, device='cuda').to(torch.int32)
    s = rand(4, 9000)
    forms.append((s, lambda s=s: rk.adjust_scores(s, history=(ptr, ids), repetition=1.5, presence=0.5,
                                                  row_bias=(ptr, ids, s[0, :400].clone()))))
    forms.append((s, lambda s=s: rk.mx4_dequantize(rk.mx4_quantize(s))))
    graphs = []
    for source, call in forms:
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out if isinstance(out, tuple) else (out,)))
    for step in range(3):
        for source, _ in forms:
            source.copy_(torch.randn(source.shape, generator=g, device='cuda'))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, call), (_, out) in zip(forms, graphs):
            want = call()
            for a, b in zip(out, want if isinstance(want, tuple) else (want,)):
                assert torch.equal(a, b)


@pytest.mark.parametrize('rank,m', [(3, 40), (20, 700), (64, 2000), (100, 333)])
@pytest.mark.parametrize('dtype', ['float32', 'float64'])
def test_score_items_of_users_the_table_does_not_have(rank, m, dtype):
    """Rows of NaN for them, and the other rows as without them (the smallest user has the largest
    factors, so rows read in place of the missing ones would show in the scale too)."""
    from alsmi import device as dev
    device = dev.require_gpu()
    rng = np.random.default_rng(rank)
    U, V = rng.standard_normal((rank, 50)), rng.standard_normal((rank, m))
    U[:, 0] *= 1e6
    Ud, Vd = dev.factors_to_device(U, dtype, device), dev.factors_to_device(V, dtype, device)
    users = rng.integers(1, 50, 150).astype(np.int32)
    none = rng.random(150) < 0.2
    users[none] = rng.choice([-1, 50, 51, -2 ** 31, 2 ** 31 - 1], none.sum())
    got = dev.score_items(rank, gpu(users), Ud, Vd)
    assert torch.equal(torch.isnan(got), gpu(none)[:, None].expand(-1, m))
    want = dev.score_items(rank, gpu(users[~none]), Ud, Vd)
    assert torch.equal(got[gpu(~none)], want)
    assert bool(torch.isnan(dev.score_items(rank, gpu(users[none][:1]), Ud, Vd)).all())


def test_tables_of_more_rows_than_a_launch_has_room_for():
    """As many rows as a call takes, of one element: 2^24 workgroups of 256 threads and more.  Every row
    is one of the same thirteen, which a small table quantises too."""
    n, period = 2 ** 31 - 1, 13
    small = torch.linspace(-6.5, 7.0, period, device='cuda')[:, None]
    few = rk.mx4_quantize(small)
    want = rk.mx4_dequantize(few)
    ids = torch.arange(n, dtype=torch.int32, device='cuda').remainder_(period)
    whole = n - n % period

    def check(got, rest):
        assert bool((got[:whole].view(-1, period) == want.view(1, period)).all())
        assert torch.equal(got[whole:], want[:rest])
    x = torch.empty(n, 1, device='cuda')
    step = 1 << 28
    for lo in range(0, n, step):
        x[lo:lo + step, 0] = small[:, 0].index_select(0, ids[lo:lo + step])
    table = rk.mx4_quantize(x)
    assert torch.equal(table.codes[-period:], few.codes.roll(-(n % period), 0))
    assert torch.equal(table.scales[-period:], few.scales.roll(-(n % period), 0))
    x.fill_(NAN)
    rk.mx4_dequantize(table, out=x)
    check(x, n % period)
    del table
    x.fill_(NAN)
    rk.mx4_dequantize(few, rows=ids, out=x)
    check(x, n % period)
    del x, ids
    torch.cuda.empty_cache()  # (54 GB at most)


@pytest.mark.parametrize('kind', ['bf16', 'mx4'])
def test_scores_of_more_items_than_a_launch_has_room_for(kind):
    """2^29 items of a few rows' product, in the form whose workgroups take 32 of them each.  All
    elements of an item are alike, so its score is known; the scores are small whole numbers."""
    n, width = 2 ** 29 + 5, 257
    blocks = (width + 31) // 32
    codes = torch.empty(n, 16 * blocks, dtype=torch.uint8, device='cuda')
    # items in the order 1, 1.5, -2, 0, 4, 1, ...; two codes a byte, +0 behind the width
    lut = torch.tensor([0x22, 0x33, 0xcc, 0x00, 0x66], dtype=torch.uint8, device='cuda')
    value = torch.tensor([1.0, 1.5, -2.0, 0.0, 4.0], device='cuda')
    whole = n - n % 5
    codes[:whole].view(-1, 5, 16 * blocks).copy_(lut.view(1, 5, 1))
    codes[whole:] = lut[:n % 5, None]
    codes[:, width // 2] &= 0x0f
    codes[:, width // 2 + 1:] = 0
    scales = torch.full((n, blocks), 127, dtype=torch.uint8, device='cuda')
    table = rk.Mx4Table(codes, scales, width)
    a = torch.zeros(2, width, dtype=BF16, device='cuda')
    a[0, ::8], a[1, 256], a[1, 0] = 0.5, 2.0, 1.0
    at = rk.mx4_quantize(a) if kind == 'mx4' else a
    got = rk.mx4_scores(at, table, out_dtype=BF16)
    for r, total in ((0, 16.5), (1, 3.0)):
        want = (value * total).to(BF16)
        assert bool((got[r, :whole].view(-1, 5) == want).all())
        assert torch.equal(got[r, whole:], want[:n % 5])
    del table, codes, scales, got
    torch.cuda.empty_cache()  # (85 GB)


def test_item_bias_in_the_precision_of_fp64_scores():
    """Biases that fp32 cannot hold, added in 64 bits: sums of few binary digits, so exact."""
    rng = np.random.default_rng(8)
    for n, m in ((1, 1), (3, 31), (5, 2049), (7, 5000)):
        s = rng.integers(-8, 8, (n, m)) / 8
        bias = rng.integers(-8, 8, m) / 8 + rng.integers(-8, 8, m) * 2.0 ** -40
        got = rk.adjust_scores(gpu(s), item_bias=gpu(bias))
        np.testing.assert_array_equal(host(got), s + bias)
        # an element into its memory, and in fp32 as before
        flat = gpu(np.concatenate(([7.0], bias)))
        np.testing.assert_array_equal(host(rk.adjust_scores(gpu(s), item_bias=flat[1:])), s + bias)
        single = bias.astype(np.float32)
        got = rk.adjust_scores(gpu(s), item_bias=gpu(single))
        np.testing.assert_array_equal(host(got), s + single.astype(np.float64))


def test_recommend_adds_a_bias_in_the_precision_of_the_model():
    """Items of equal factors whose biases differ by 1e-12 of them."""
    from alsmi import ALS
    m = 300
    als = ALS(rank=2)
    als.user_feats, als.item_feats = np.ones((2, 3)), np.ones((2, m))
    bias = 1.0 + 1e-12 * np.random.default_rng(0).permutation(m)
    items, scores = als.recommend([0, 2], 20, item_bias=bias)
    want = np.argsort(-bias)[:20]
    assert (items == want).all() and np.abs(scores - (2 + bias[want])).max() < 1e-14
    items, scores = als.recommend([0], 20, item_bias=bias, catalogue='mx4')
    assert np.abs(scores - 3.0).max() < 1e-6


def test_adjust_into_a_view_and_into_columns_beside():
    s = torch.randn(5, 3000, device='cuda')
    bias = torch.randn(3000, device='cuda')
    want = s + bias
    both = torch.full((5, 6000), 7.0, device='cuda')
    both[:, :3000] = s
    rk.adjust_scores(both[:, :3000], item_bias=bias, out=both[:, 3000:])
    assert torch.equal(both[:, 3000:], want) and torch.equal(both[:, :3000], s)
    rk.adjust_scores(both[:, :3000], item_bias=bias, out=both[:, :3000])
    assert torch.equal(both[:, :3000], want)


def test_score_items_over_its_operands_is_refused():
    from alsmi import device as dev
    U, V = torch.ones(6, 16, device='cuda'), torch.ones(8, 16, device='cuda')
    users = torch.zeros(3, dtype=torch.int32, device='cuda')
    flat = torch.zeros(64, device='cuda')
    for args in ((users, U, V, U.view(-1)[72:].view(3, 8)), (users, U, V, V.view(-1)[:24].view(3, 8)),
                 (flat[20:23].view(torch.int32), U, V, flat[:24].view(3, 8))):
        with pytest.raises(ValueError, match='overlap'):
            dev.score_items(3, *args[:3], out=args[3])
    out = flat[24:48].view(3, 8)
    assert dev.score_items(3, flat[20:23].view(torch.int32), U, V, out=out) is out
    assert bool((out == 16).all()) and bool((flat[:24] == 0).all()) and bool((flat[48:] == 0).all())


# ------------------------------------------------------------ sums that are exact, so bit for bit
FORMS = [  # rows, items, width: one for each form of the product, in the order of their rules
    (1, 100, 20), (40, 100, 20), (1, 100, 60), (40, 70, 60), (3, 100, 128), (70, 130, 100),
    (5, 300, 250), (70, 300, 250), (2, 300, 1000), (3, 100000, 300), (20, 500, 640), (40, 90000, 300),
    (100, 16400, 300), (130, 16400, 300), (300, 9001, 544), (1020, 16300, 700), (64, 33000, 1030),
    (129, 8300, 2080)]


def exact_table(g, n, width, codes):
    """Rows of random codes out of `codes` and scales of 1, 2 and 4, codes of 0 behind the width."""
    blocks = (width + 31) // 32
    pick = torch.tensor(codes, dtype=torch.uint8, device='cuda')
    nibble = pick[torch.randint(0, len(codes), (n, 32 * blocks), generator=g, device='cuda')]
    nibble[:, width:] = 0
    scales = torch.randint(127, 130, (n, blocks), generator=g, device='cuda', dtype=torch.uint8)
    return rk.Mx4Table((nibble[:, 0::2] | nibble[:, 1::2] << 4).contiguous(), scales, width)


def table_values(table, dtype=F64):
    """What codes and scales stand for, by the table of sixteen values."""
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype,
                       device='cuda')
    both = torch.stack((table.codes & 15, table.codes >> 4), dim=-1).flatten(1)[:, :table.width]
    unit = torch.exp2(table.scales.to(dtype) - 127).repeat_interleave(32, dim=1)[:, :table.width]
    return lut[both.to(torch.int32)] * unit


@pytest.mark.parametrize('kind', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('m,n,width', FORMS + [(700, 2800, 65536)])
def test_every_part_of_an_activation_counts(m, n, width, kind):
    """One activation a row that is not zero, with as many significant bits as its type has (the last of
    them set), and table elements that are powers of two: a score is one product and exact, so the
    last bit of the last bf16 part has to be there.  The rows' elements lie all over the width."""
    g = torch.Generator(device='cuda')
    g.manual_seed(m + 3 * n + width)
    table = exact_table(g, n, width, [1, 2, 4, 6, 9, 10, 12, 14])
    dtype, bits = {'f32': (F32, 24), 'bf16': (BF16, 8), 'f16': (F16, 11)}[kind]
    rows = torch.arange(m, device='cuda')
    ends = torch.tensor([0, width - 1, width // 2], device='cuda')
    for turn in range(2 if m * width > 1 << 22 else 8):  # few rows meet few places of the width
        at = torch.randint(0, width, (m,), generator=g, device='cuda')
        at[:min(m, 3)] = ends.roll(turn)[:min(m, 3)]
        value = torch.randint(2 ** (bits - 2), 2 ** (bits - 1), (m,), generator=g, device='cuda') * 2 + 1
        value = value * (1 - 2 * torch.randint(0, 2, (m,), generator=g, device='cuda'))
        value = value.to(F64) * 2.0 ** -(bits // 2)
        a = torch.zeros(m, width, dtype=dtype, device='cuda')
        a[rows, at] = value.to(dtype)
        byte = table.codes[:, at // 2]
        nibble = torch.where(at % 2 == 1, byte >> 4, byte & 15).to(torch.int32)
        power = torch.exp2(torch.tensor([0., -1, 0, 0, 1, 0, 2, 0], device='cuda')[nibble & 7].to(F64) +
                           table.scales[:, at // 32].to(F64) - 127)
        want = (power * (1.0 - 2.0 * (nibble >> 3).to(F64))).t() * value[:, None]
        assert torch.equal(rk.mx4_scores(a, table, out_dtype=F32).to(F64), want)


@pytest.mark.parametrize('kind', ['f32', 'bf16', 'f16', 'mx4'])
@pytest.mark.parametrize('m,n,width', FORMS + [(700, 2800, 65536), (1100, 2800, 65536), (130, 65536, 300),
                                               (2048, 2049, 1024), (512, 5000, 4096), (300, 8200, 992)])
def test_every_element_of_a_row_counts(m, n, width, kind):
    """Small whole activations (at most 3, or codes of at most 2) against any codes (at most 24): a sum is a
    whole number of halves, at most 65536 * 72 * 2 of them, or of quarters, at most 65536 * 48 * 4.  Both
    are below 2^24, so fp32 sums in any order are exact and a left out element shows."""
    g = torch.Generator(device='cuda')
    g.manual_seed(m + n + 5 * width)
    table = exact_table(g, n, width, list(range(16)))
    if kind == 'mx4':
        a = exact_table(g, m, width, [0, 1, 2, 4, 9, 10, 12])
        a.scales.fill_(127)
        values = table_values(a)
    else:
        a = torch.randint(-3, 4, (m, width), generator=g, device='cuda')
        values = a.to(F64)
        a = a.to({'f32': F32, 'bf16': BF16, 'f16': F16}[kind])
    got = rk.mx4_scores(a, table, out_dtype=F32)
    for lo in range(0, n, 20000):  # (fp64 products in parts: tables of 90000 items are 200 MB)
        part = rk.Mx4Table(table.codes[lo:lo + 20000], table.scales[lo:lo + 20000], width)
        assert torch.equal(got[:, lo:lo + 20000].to(F64), values @ table_values(part).t())


@pytest.mark.parametrize('dtype', [F32, F64, F16, BF16])
@pytest.mark.parametrize('n,m,k', [(1, 1000000, 1024), (3, 400000, 1000), (1, 10000000, 1024), (7, 300000, 513)])
def test_topk_through_a_middle_level(n, m, k, dtype):
    """More kept keys than one workgroup takes, so that a level in between reads keys and writes keys, into the
    second half of the workspace; the workspace is not left."""
    g = torch.Generator(device='cuda')
    g.manual_seed(m + k)
    s = torch.randn(n, m, generator=g, device='cuda', dtype=F64).to(dtype) + 0.0
    few = torch.randint(-2, 3, (n, m), generator=g, device='cuda').to(dtype)
    hardly = torch.full((n, m), -INF, dtype=dtype, device='cuda')
    hardly[:, m // 3::m // 700] = s[:, m // 3::m // 700]
    up = torch.sort(s, dim=1).values.contiguous()
    code = rk._CODES[dtype]
    size = rk._lib.load().alsmi_topk_rows_workspace_bytes(code, n, m, k)
    for rows in (s, few, hardly, up, up.flip(1).contiguous()):
        want, order = torch.sort(rows, dim=1, descending=True, stable=True)
        items, best = rk.topk_rows(rows, k)
        assert torch.equal(best, want[:, :k]) and torch.equal(items, order[:, :k].to(torch.int32))
        ws = torch.full((size + 4096,), 77, dtype=torch.uint8, device='cuda')
        items.zero_()
        rk._call(rows.device, 'alsmi_topk_rows', code, n, m, rows.data_ptr(), m, k, items.data_ptr(),
                 best.data_ptr(), ws.data_ptr())
        assert torch.equal(items, order[:, :k].to(torch.int32)) and bool((ws[size:] == 77).all())


def test_the_ends_of_the_exact_range():
    """Elements of the two largest scales (exact in fp64, infinities from 2^128 on in fp32, bf16 and beside
    float activations) and the smallest activations whose last bit is not cut off."""
    codes = torch.tensor([[2, 3, 4, 5, 6, 7, 1, 0]], dtype=torch.uint8, device='cuda').repeat(3, 4)
    codes = (codes[:, 0::2] | codes[:, 1::2] << 4).contiguous()
    table = rk.Mx4Table(codes, gpu(np.array([[252], [253], [254]], dtype=np.uint8)), 32)
    grid = np.tile([1, 1.5, 2, 3, 4, 6, 0.5, 0], 4)
    value = grid * 2.0 ** np.array([[125.0], [126], [127]])
    np.testing.assert_array_equal(host(rk.mx4_dequantize(table, F64)), value)
    capped = np.where(value >= 2.0 ** 128, INF, value)
    for dtype in (F32, BF16):
        np.testing.assert_array_equal(host(rk.mx4_dequantize(table, dtype)), capped)
    one = torch.eye(32, device='cuda')[:7] * 0.25  # each element of an item by itself
    got = host(rk.mx4_scores(one, table))
    np.testing.assert_array_equal(got[:, 0], 0.25 * value[0, :7])
    assert np.isnan(got[:, 1:]).all()  # (a zero beside an infinity)
    both = host(rk.mx4_scores(rk.mx4_quantize(one), table))  # both in 4 bits: nothing is widened
    np.testing.assert_array_equal(both, 0.25 * value[:, :7].T)
    small = rk.Mx4Table(codes[:1].contiguous(), gpu(np.array([[130]], dtype=np.uint8)), 32)
    a = torch.zeros(2, 32, device='cuda')
    a[0, 0], a[1, 0] = (2.0 ** 24 - 1) * 2.0 ** -133, (2.0 ** 24 - 1) * 2.0 ** -134
    got = host(rk.mx4_scores(a, small))
    assert got[0, 0] == 8 * (2.0 ** 24 - 1) * 2.0 ** -133
    assert got[1, 0] == 8 * (2.0 ** 24 - 2) * 2.0 ** -134


def test_refit_releases_the_quantised_items():
    """The table in 4 bits, and the factor table that it was made from, go with the factors they belong to."""
    import weakref
    from alsmi import ALS
    rng = np.random.default_rng(1)
    pairs = rng.integers(0, 30, 200), rng.integers(0, 40, 200)
    als = ALS(4, random_state=0, max_iter=1).fit(pairs, rng.random(200) + 1, shape=(30, 40))
    als.recommend([0], 3, catalogue='mx4')
    old = weakref.ref(als._mx4[0])
    als.fit(pairs, rng.random(200) + 1, shape=(30, 40))
    assert als._mx4 is None and old() is None
    items, scores = als.recommend([0], 40, catalogue='mx4')
    codes, scales = ro.mx4_quantize(als.item_feats.T)
    want = (als.user_feats.T @ ro.mx4_values(codes, scales, 4).T)[0]
    assert np.abs(scores[0] - want[items[0]]).max() < 1e-5


@pytest.mark.parametrize('dtype', ['float32', 'float64'])
def test_score_items_captured_and_replayed(dtype):
    """In a graph with the steps behind it, replayed on other factors and users, with eager calls of other
    users between the replays (each call clears and fills a scale of its own)."""
    from alsmi import device as dev
    rng = np.random.default_rng(3)
    rank, n, m = 20, 400, 3000
    draw = lambda k, size: gpu(rng.standard_normal((k, 32)) * (np.arange(32) < rank) * size).to(
        F32 if dtype == 'float32' else F64)
    U, V = draw(n, 1.0), draw(m, 1.0)
    users = gpu(rng.integers(0, n, 90).astype(np.int32))

    def call():
        s = dev.score_items(rank, users, U, V)
        return (s,) + rk.topk_rows(s, 12)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for size in (1e-3, 1e5, 1.0):
        U.copy_(draw(n, size))
        V.copy_(draw(m, size * 10))
        users.copy_(gpu(rng.integers(-1, n + 1, 90).astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, call()):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) if a.is_floating_point() else \
                torch.equal(a, b)
        dev.score_items(rank, users[:5].clone(), U * 100, V)
