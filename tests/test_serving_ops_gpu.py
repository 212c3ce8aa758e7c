"""The serving operators (e4m3 norm and product, paged append and attention)
against 64-bit restatements, at the sizes, strides and masks where they can go
wrong; then a decoder layer of them, in order."""
import ctypes as C
import math

import pytest
import torch

from fluxvla_b200 import _lib, ops, pack
from tests import serving_ref as R

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3 = torch.float8_e4m3fn
BF16_HALF = 2.0 ** -8      # half a step, relative
DEV = 'cuda'
MODES = {'gemma': _lib.NORM_GEMMA_RMS, 'ada': _lib.NORM_ADA_RMS,
         'rms': _lib.NORM_RMS, 'none': _lib.NORM_NONE}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dt=F32):
    return torch.randn(*shape, generator=g, device=DEV).to(dt)


def values(q):
    return q.to(F32).to(F64)


# ---------------------------------------------------------------- norm_fp8
def norm_inputs(g, rows, dim, mode, xt, dt):
    x = randn(g, rows, dim) * (1 + 20 * (torch.rand(
        dim, generator=g, device=DEV) > 0.97))
    x = x.to(xt)
    kw = {}
    if dt is not None:
        kw['delta'] = randn(g, rows, dim, dt=dt)
    if mode == 'gemma':
        kw['w'] = randn(g, dim, dt=BF16) * 0.3
    if mode == 'ada':
        kw['mod'] = randn(g, 2 * dim) * 0.3
    return x, kw


def check_norm(mode, x, kw, q, s, res=None):
    """Codes, scales and residual are those of the formula: nothing is rounded
    before them to fewer than 64 bits, so nothing may differ."""
    h, q_ref, s_ref = R.norm_fp8(MODES[mode], x, **kw)
    if 'delta' in kw:
        assert torch.equal(res, h)
    assert torch.equal(s, s_ref)
    assert torch.equal(values(q), q_ref)


@pytest.mark.parametrize('mode', list(MODES))
@pytest.mark.parametrize('xt,dt', [(F32, BF16), (BF16, BF16), (F32, None),
                                   (BF16, F32)])
@pytest.mark.parametrize('rows,dim', [(1, 1), (1, 2048), (3, 127), (5, 129),
                                      (64, 1024), (2, 1152), (7, 4304),
                                      (2, 8192), (3, 16384), (130, 64)])
def test_norm_fp8(mode, xt, dt, rows, dim):
    g = gen(rows * 131 + dim)
    x, kw = norm_inputs(g, rows, dim, mode, xt, dt)
    q = torch.empty(rows, dim, dtype=E4M3, device=DEV)
    s = torch.empty(rows, -(-dim // 128), device=DEV)
    res = torch.empty_like(x) if dt is not None else None
    ops.norm_fp8(MODES[mode], x, q, s, res=res, **kw)
    check_norm(mode, x, kw, q, s, res)


def test_norm_fp8_strides_in_place_and_beyond_the_norm_limit():
    g = gen(1)
    # views into wider buffers, odd offsets: value-by-value path; the columns
    # around the views stay as they were
    big = randn(g, 6, 301)
    wide_q = torch.full((6, 305), 7, dtype=torch.uint8, device=DEV)
    wide_s = torch.full((6, 5), 9.0, device=DEV)
    x = big[:, 1:301]
    kw = dict(delta=randn(g, 6, 300, dt=BF16), w=randn(g, 300, dt=BF16))
    before = big.clone()
    ref = before[:, 1:301]
    q, s = wide_q.view(E4M3)[:, 3:303], wide_s[:, 1:4]
    ops.norm_fp8(_lib.NORM_GEMMA_RMS, x, q, s, res=x, **kw)
    check_norm('gemma', ref, kw, q, s, x)
    assert torch.equal(big[:, 0], before[:, 0])
    assert (wide_q[:, :3] == 7).all() and (wide_q[:, 303:] == 7).all()
    assert (wide_s[:, 0] == 9).all() and (wide_s[:, 4] == 9).all()
    # without a norm a row may be longer than the norms' limit
    x = randn(g, 2, 20000, dt=BF16)
    q = torch.empty(2, 20000, dtype=E4M3, device=DEV)
    s = torch.empty(2, 157, device=DEV)
    ops.norm_fp8(_lib.NORM_NONE, x, q, s)
    check_norm('none', x, {}, q, s)


@pytest.mark.parametrize('mode', list(MODES))
@pytest.mark.parametrize('rows,dim', [(3, 8), (2, 255), (5, 1025), (3, 4099),
                                      (2, 16383)])
def test_norm_fp8_unaligned_rows_and_weights(mode, rows, dim):
    """Views that start off 16 bytes, in place, weights too; what lies around
    them stays."""
    g = gen(dim)
    x, kw = norm_inputs(g, rows, dim, mode, BF16, BF16)
    if 'w' in kw:
        kw['w'] = torch.cat([kw['w'][:1], kw['w']])[1:]
    if 'mod' in kw:
        kw['mod'] = torch.cat([kw['mod'][:1], kw['mod']])[1:]
    wide = torch.full((rows, dim + 5), 3.0, dtype=BF16, device=DEV)
    wide[:, 3:3 + dim] = x
    wide_q = torch.full((rows, dim + 7), 7, dtype=torch.uint8, device=DEV)
    q, s = wide_q.view(E4M3)[:, 5:5 + dim], torch.empty(rows, -(-dim // 128), device=DEV)
    h = wide[:, 3:3 + dim]
    ops.norm_fp8(MODES[mode], h, q, s, res=h, **kw)
    check_norm(mode, x, kw, q, s, h)
    assert (wide[:, :3] == 3).all() and (wide[:, 3 + dim:] == 3).all()
    assert (wide_q[:, :5] == 7).all() and (wide_q[:, 5 + dim:] == 7).all()


@pytest.mark.parametrize('dim', [128, 131])
def test_norm_fp8_sum_is_formed_in_f32(dim):
    """1 + 2^-8 + 2^-31 is 1 + 2^-8 in f32, which goes to the even bf16, 1."""
    g = gen(28)
    x = torch.ones(64, dim, dtype=BF16, device=DEV)
    delta = 2.0 ** -8 + randn(g, 64, dim) * 2.0 ** -31
    delta[0] = 2.0 ** -8 + 2.0 ** -31
    for x, delta in ((x, delta), (randn(g, 64, dim, dt=BF16), randn(g, 64, dim)),
                     (randn(g, 64, dim), randn(g, 64, dim, dt=BF16))):
        res = torch.empty_like(x)
        q = torch.empty(64, dim, dtype=E4M3, device=DEV)
        s = torch.empty(64, -(-dim // 128), device=DEV)
        ops.norm_fp8(_lib.NORM_NONE, x, q, s, delta=delta, res=res)
        assert torch.equal(res, (x.float() + delta.float()).to(x.dtype))
        check_norm('none', res, {}, q, s)


def test_norm_fp8_values_on_the_borders_between_codes():
    """Every border of the format, times a scale that is not a power of two,
    and its neighbours: the even code, and the codes on either side."""
    grid = R.e4m3_grid().float().to(DEV)
    mid = (grid[1:] + grid[:-1]) / 2
    for unit in (1.0, 3.0, 2.0 ** -20 * 5):
        row = torch.zeros(5, 128, device=DEV)
        flat = torch.cat([mid, torch.nextafter(mid, mid * 2),
                          torch.nextafter(mid, mid * 0)]) * unit
        # one slot in each group holds the largest value, which sets the scale
        body = torch.zeros(row.shape[0] * 127, device=DEV)
        body[:flat.numel()] = flat
        row[:, 1:] = body.view(-1, 127)
        row[:, 0] = -448.0 * unit
        q = torch.empty(row.shape, dtype=E4M3, device=DEV)
        s = torch.empty(row.shape[0], 1, device=DEV)
        ops.norm_fp8(_lib.NORM_NONE, row, q, s)
        check_norm('none', row, {}, q, s)


def test_norm_fp8_codes_of_every_bf16_quotient():
    """Every significand of a value under every one of the group's largest, over
    the exponents that the codes reach."""
    m = (128 + torch.arange(128, device=DEV)).double()
    rows = []
    for e in range(0, 19):
        body = (m * 2.0 ** -e).expand(128, 128).clone()
        body[:, 1::2] *= -1
        body = body.clamp(-m[:, None], m[:, None])
        body[:, 0] = m
        rows.append(body)
    x = torch.cat(rows).to(BF16)
    q = torch.empty(x.shape, dtype=E4M3, device=DEV)
    s = torch.empty(x.shape[0], 1, device=DEV)
    ops.norm_fp8(_lib.NORM_NONE, x, q, s)
    check_norm('none', x, {}, q, s)


@pytest.mark.parametrize('size', [1.0, 2.0 ** -40, 2.0 ** 100])
def test_norm_fp8_codes_near_borders_of_any_scale(size):
    """32-bit values at most three steps from a border times the scale."""
    g = gen(15)
    grid = R.e4m3_grid().to(DEV)
    grid = grid[grid >= 0]
    mid = ((grid[1:] + grid[:-1]) / 2)[:126]
    top = (1 + torch.rand(2000, generator=g, device=DEV)) * size
    s_ref = (top.double() / 448).float()
    y = (mid * s_ref.double()[:, None]).float()
    steps = torch.randint(-3, 4, y.shape, generator=g, device=DEV, dtype=torch.int32)
    y = (y.view(torch.int32) + steps).view(F32)
    x = torch.zeros(2000, 128, device=DEV)
    x[:, 1:1 + y.shape[1]] = y.clamp(max=top[:, None])
    x[:, 0] = -top
    q = torch.empty(x.shape, dtype=E4M3, device=DEV)
    s = torch.empty(2000, 1, device=DEV)
    ops.norm_fp8(_lib.NORM_NONE, x, q, s)
    check_norm('none', x, {}, q, s)


def test_norm_fp8_zero_tiny_nan_and_infinite_rows():
    x = torch.zeros(5, 256, device=DEV)
    x[1] = 1e-30                      # below the smallest scale
    x[2, 5] = math.nan
    x[2, 6:] = 2.0
    x[3, 200] = math.inf
    x[3, :128] = 1.0
    x[4] = 3e38
    q = torch.empty(5, 256, dtype=E4M3, device=DEV)
    s = torch.empty(5, 2, device=DEV)
    ops.norm_fp8(_lib.NORM_NONE, x, q, s)
    v = values(q) * s.to(F64).repeat_interleave(128, 1)
    assert (v[0] == 0).all() and (v[1] == 0).all()
    assert torch.isnan(v[2, 5]) and torch.isfinite(v[2, 6:]).all()
    assert (v[2, 6:128] - 2).abs().max() <= 2.0 ** -23   # the scale's rounding
    assert torch.isfinite(v[3, :128]).all() and torch.isnan(v[3, 128:]).all()
    assert ((v[4] / 3e38 - 1).abs() <= 2.0 ** -22).all()
    # a zero row through a norm: zeros, not NaN
    w = torch.zeros(256, dtype=BF16, device=DEV)
    ops.norm_fp8(_lib.NORM_GEMMA_RMS, x[:1], q[:1], s[:1], w=w)
    assert (values(q[:1]) == 0).all()


@pytest.mark.parametrize('mode', ['gemma', 'ada', 'rms'])
@pytest.mark.parametrize('size,eps', [(1e38, 1e-6), (1e-18, 1e-6), (1e-30, 0.0),
                                      (3e-39, 0.0), (1e30, 0.0)])
def test_norm_fp8_at_the_ends_of_the_range(mode, size, eps):
    """Rows whose norm factor 32 bits hold badly or not at all."""
    g = gen(9)
    x, kw = norm_inputs(g, 4, 300, mode, F32, None)
    x = (x.double() / x.abs().max() * size).float()
    q = torch.empty(4, 300, dtype=E4M3, device=DEV)
    s = torch.empty(4, 3, device=DEV)
    ops.norm_fp8(MODES[mode], x, q, s, eps=eps, **kw)
    _, q_ref, s_ref = R.norm_fp8(MODES[mode], x, eps=eps, **kw)
    assert torch.equal(s, s_ref) and torch.equal(values(q), q_ref)


def test_norm_fp8_shifts_that_cancel_the_normed_values():
    """Groups whose values are all small against the normed values and shifts
    that they are the sums of: whole rows, and a last group of one column."""
    x = torch.ones(3, 300, device=DEV)
    x[1] = 7.0
    x[2, ::2] = -1.0
    mod = torch.zeros(600, device=DEV)
    mod[300:] = -1.0
    cases = [(x, mod)]
    g = gen(21)
    for dim in (1, 129, 257):
        x = randn(g, 1, dim).expand(4, dim).contiguous()
        mod = randn(g, 2 * dim) * 0.3
        z = x[0].double() * torch.rsqrt(x[0].double().square().mean() + 1e-6)
        mod[-1] = -(z * (1 + mod[:dim].double()))[-1].float()
        cases.append((x, mod))
    for x, mod in cases:
        rows, dim = x.shape
        q = torch.empty(rows, dim, dtype=E4M3, device=DEV)
        s = torch.empty(rows, -(-dim // 128), device=DEV)
        ops.norm_fp8(_lib.NORM_ADA_RMS, x, q, s, mod=mod)
        h, m = x.to(F64), mod.to(F64)
        z = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * (1 + m[:dim])
        y = z + m[dim:]
        # a few roundings of 64 bits, of the terms
        err = 2.0 ** -50 * (z.abs() + m[dim:].abs())
        for i in range(s.shape[1]):
            c = slice(128 * i, 128 * i + 128)
            scale = s[:, i:i + 1].to(F64)
            top = y[:, c].abs().amax(1, keepdim=True).clamp(min=2.0 ** -60)
            # the scale's rounding to f32
            near = err[:, c].amax(1, keepdim=True) + 2.0 ** -24 * top
            assert ((448 * scale - top).abs() <= near).all()
            # half a step of e4m3 (relative 2^-4, or of the smallest step)
            half = 2.0 ** -4 * y[:, c].abs() + 2.0 ** -10 * scale
            assert ((values(q[:, c]) * scale - y[:, c]).abs() <= half + near).all()


@pytest.mark.parametrize('mode', ['gemma', 'ada'])
@pytest.mark.parametrize('xt', [F32, BF16])
def test_norm_fp8_weights_up_to_the_end_of_the_range(mode, xt):
    """Values that 32 bits do not hold, though their scales and codes do: past
    the largest, and normed ones below the smallest under large weights."""
    g = gen(22)
    rows, dim = 64, 640
    x = randn(g, rows, dim)
    size = 20 + 18.5 * torch.rand(dim, generator=g, device=DEV)
    w = randn(g, dim).sign() * 10.0 ** size
    w[:128] = 3e38
    x[:, 128:256] *= 1e-42
    w[128:256] = 1e38
    w[512:] *= 1e-30
    if mode == 'gemma':
        kw = dict(w=w.to(BF16))
    else:
        shift = randn(g, dim) * 10.0 ** (-3 + 40 * torch.rand(dim, generator=g, device=DEV))
        shift[128:256] = 0
        kw = dict(mod=torch.cat([w, shift]))
    x = x.to(xt)
    q = torch.empty(rows, dim, dtype=E4M3, device=DEV)
    s = torch.empty(rows, 5, device=DEV)
    ops.norm_fp8(MODES[mode], x, q, s, **kw)
    assert torch.isfinite(s).all()
    check_norm(mode, x, kw, q, s)


@pytest.mark.parametrize('mode', ['gemma', 'ada', 'rms'])
@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf])
def test_norm_fp8_rows_that_are_not_finite(mode, bad):
    g = gen(25)
    x, kw = norm_inputs(g, 5, 300, mode, F32, None)
    x[2, 200] = bad
    q = torch.empty(5, 300, dtype=E4M3, device=DEV)
    s = torch.empty(5, 3, device=DEV)
    ops.norm_fp8(MODES[mode], x, q, s, **kw)
    rest = torch.arange(5, device=DEV) != 2
    check_norm(mode, x[rest], kw, q[rest], s[rest])
    v = values(q[2]) * s[2].to(F64).repeat_interleave(128)[:300]
    others = torch.arange(300, device=DEV) != 200
    assert torch.isnan(v[200])
    if bad != bad:
        assert torch.isnan(v).all()
    elif mode == 'ada':
        # the shift, to half a step (or half the smallest step of its group)
        shift = kw['mod'][300:].to(F64)
        top = torch.nn.functional.pad(shift.abs(), (0, 84)).view(3, 128).amax(1)
        low = top.repeat_interleave(128)[:300] / 448 * 2.0 ** -10
        err = (v - shift).abs() - (2.0 ** -4 * shift.abs() + low) * (1 + 2.0 ** -20)
        assert (err[others] <= 0).all()
    else:
        assert (v[others] == 0).all()


@pytest.mark.parametrize('dt', [F32, BF16])
def test_norm_fp8_many_codes(dt):
    """Over a million values, and groups whose largest value is a multiple of 7:
    scales that make values meet borders exactly."""
    g = gen(10)
    x = randn(g, 1024, 1024, dt=dt)
    big = torch.tensor([3.5, 7.0, 8.75, 14.0], device=DEV)
    x[:512, ::128] = big[torch.arange(512, device=DEV) % 4, None].to(dt)
    q = torch.empty(1024, 1024, dtype=E4M3, device=DEV)
    s = torch.empty(1024, 8, device=DEV)
    ops.norm_fp8(_lib.NORM_NONE, x, q, s)
    check_norm('none', x, {}, q, s)
    w = randn(g, 1024, dt=BF16) * 0.1
    ops.norm_fp8(_lib.NORM_GEMMA_RMS, x, q, s, w=w)
    check_norm('gemma', x, dict(w=w), q, s)


# ---------------------------------------------------------------- gemm_fp8
def gemm_inputs(g, m, n, k):
    x = randn(g, m, k)
    a = torch.empty(m, k, dtype=E4M3, device=DEV)
    sa = torch.empty(m, -(-k // 128), device=DEV)
    ops.norm_fp8(_lib.NORM_NONE, x, a, sa)
    b, sb = pack.quantize_blocks(randn(g, n, k) * k ** -0.5)
    return a, sa, b, sb


def check_gemm(out, a, sa, b, sb, epilogue):
    """Each product of two e4m3 values is exact in f32; a group of 128 and the
    sum over groups add at most 128 + groups roundings (2^-23 of the partial
    sum where additions truncate), the two scales one each."""
    c, mag = R.gemm_fp8(a, sa, b, sb)
    err = mag * (128 + sa.shape[1] + 8 + 4) * 2.0 ** -23
    if epilogue == _lib.EPI_GEGLU:
        gate, up = c[:, 0::2], c[:, 1::2]
        eg, eu = err[:, 0::2], err[:, 1::2]
        ref = R.gelu(gate) * up
        # |gelu'| <= 1.13; exp and the division add a few f32 roundings
        err = 1.13 * eg * (up.abs() + eu) + R.gelu(gate).abs() * eu
        err = err + 2.0 ** -18 * (ref.abs() + gate.abs() * up.abs() * 2.0 ** -6)
    else:
        ref = c
    if out.dtype == BF16:
        err = err + BF16_HALF * (ref.abs() + err)
    bad = (out.to(F64) - ref).abs() > err
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


EPIS = {'bf16': _lib.EPI_BF16, 'f32': _lib.EPI_F32_STORE,
        'geglu': _lib.EPI_GEGLU}


@pytest.mark.parametrize('epi', list(EPIS))
@pytest.mark.parametrize('m,n,k', [
    (1, 2, 1), (1, 128, 128), (1, 2560, 2048), (3, 130, 144), (16, 256, 300),
    (17, 1152, 4304), (33, 254, 1000), (51, 1024, 4096), (64, 2048, 16384),
    (65, 128, 256), (100, 514, 640), (128, 256, 128), (129, 130, 272),
    (300, 1152, 1152), (816, 2560, 2048), (257, 4098, 1040),
    (1500, 4100, 272), (2049, 8194, 1000), (8, 384, 5000), (4000, 2, 16),
    (7, 20002, 528), (70, 38000, 130)])
def test_gemm_fp8(epi, m, n, k):
    g = gen(m + 3 * n + 7 * k)
    kp = -(-k // 16) * 16          # rows of 16-byte multiples
    a, sa, b, sb = gemm_inputs(g, m, n, kp)
    a, b = a[:, :k], b[:, :k]      # and a width that is none
    cols = n // 2 if epi == 'geglu' else n
    wide = torch.full((m + 2, cols + 8), 5.0, device=DEV,
                      dtype=F32 if epi == 'f32' else BF16)
    out = wide[1:m + 1, :cols]
    ops.gemm_fp8(a, sa, b, sb, out, epilogue=EPIS[epi])
    check_gemm(out, a, sa, b, sb, EPIS[epi])
    assert (wide[0] == 5).all() and (wide[m + 1] == 5).all()
    assert (wide[:, cols:] == 5).all()
    again = torch.empty_like(out)
    ops.gemm_fp8(a, sa, b, sb, again, epilogue=EPIS[epi])
    assert torch.equal(again, out)
    assert ops.device_status() == 0


@pytest.mark.parametrize('m,n', [(9, 64), (9, 62), (300, 130), (4096, 8192),
                                 (4096, 8190)])
def test_gemm_fp8_geglu_of_gates_far_from_zero(m, n):
    """gelu is 0 far below zero, whatever it is multiplied by, and the gate
    itself far above it."""
    k = 16
    size = torch.tensor([20.0, 1e3, 1e6, 1e12, 1e19, 3e19, 1e25, 1e30, 1e37],
                        device=DEV)
    sa = size[torch.arange(m, device=DEV) % 9][:, None].contiguous()
    sb = torch.ones(-(-n // 128), 1, device=DEV)
    a, b = torch.zeros(m, k, device=DEV), torch.zeros(n, k, device=DEV)
    a[:, 0] = 1.0
    b[1::2, 0] = torch.where(torch.arange(n // 2, device=DEV) % 2 == 0, 1.0, -4.0)
    out = torch.full((m, n // 2), 5.0, dtype=BF16, device=DEV)
    b[0::2, 0] = -1.0
    ops.gemm_fp8(a.to(E4M3), sa, b.to(E4M3), sb, out, epilogue=_lib.EPI_GEGLU)
    assert (out == 0).all()
    b[0::2, 0] = 1.0
    ops.gemm_fp8(a.to(E4M3), sa, b.to(E4M3), sb, out, epilogue=_lib.EPI_GEGLU)
    # the gate, to a few roundings of 32 bits, times up
    c = sa.to(F64) * b[:, 0].to(F64)
    want = c[:, 0::2] * c[:, 1::2]
    held = want.abs() < 3e38
    err = (BF16_HALF + 2.0 ** -20) * want.abs()
    assert ((out.to(F64) - want).abs() <= err)[held].all()
    assert torch.isinf(out[want.abs() > 3.5e38]).all()


def test_gemm_fp8_nan_stays_in_its_row_and_column():
    g = gen(5)
    a, sa, b, sb = gemm_inputs(g, 70, 192, 256)
    a.view(torch.uint8)[3, 9] = 0x7f
    b.view(torch.uint8)[100, 200] = 0x7f
    out = torch.empty(70, 192, device=DEV)
    ops.gemm_fp8(a, sa, b, sb, out, epilogue=_lib.EPI_F32_STORE)
    nan = torch.zeros(70, 192, dtype=torch.bool, device=DEV)
    nan[3], nan[:, 100] = True, True
    assert torch.equal(torch.isnan(out), nan)


@pytest.mark.parametrize('m,n', [(70, 192), (900, 16384)])
def test_gemm_fp8_infinite_scales_stay_in_their_rows(m, n):
    """As norm_fp8 gives them for a group with an infinity."""
    g = gen(29)
    x = randn(g, m, 304)
    x[3, 140] = math.inf
    a = torch.empty(m, 304, dtype=E4M3, device=DEV)
    sa = torch.empty(m, 3, device=DEV)
    ops.norm_fp8(_lib.NORM_NONE, x, a, sa)
    inf = torch.zeros(m, 3, dtype=torch.bool, device=DEV)
    inf[3, 1] = True
    assert torch.equal(torch.isinf(sa), inf)
    b, sb = pack.quantize_blocks(randn(g, n, 304))
    out = torch.empty(m, n, device=DEV)
    ops.gemm_fp8(a, sa, b, sb, out, epilogue=_lib.EPI_F32_STORE)
    nan = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    nan[3] = True
    assert torch.equal(~torch.isfinite(out), nan)


# ------------------------------------------------------------ paged_append
def rope(max_pos, dim):
    return pack.rope_table(max_pos, dim, device=DEV)


@pytest.mark.parametrize('tokens,heads,kv,dim,page', [
    (1, 8, 1, 256, 16), (51, 8, 1, 256, 48), (7, 4, 2, 64, 1),
    (33, 6, 3, 128, 100), (5, 2, 1, 72, 8), (9, 3, 3, 10, 4), (2, 0, 2, 128, 32)])
@pytest.mark.parametrize('interleaved', [False, True])
def test_paged_append(tokens, heads, kv, dim, page, interleaved):
    g = gen(tokens * 7 + dim)
    qkv = randn(g, tokens, (heads + 2 * kv) * dim + 8, dt=BF16)[:, :-8]
    rows = qkv.unflatten(1, (heads + 2 * kv, dim))
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:tokens]
    slots = slots.to(torch.int32)
    if tokens > 4:
        slots[2] = -1
        slots[4] = -100
    pos = torch.randint(0, 500, (tokens,), generator=g, device=DEV,
                        dtype=torch.int32)
    table = rope(500, dim)
    kc = randn(g, pages, page, kv, dim, dt=BF16)
    vc = randn(g, pages, page, kv, dim, dt=BF16)
    kc0, vc0 = kc.clone(), vc.clone()
    q_out = torch.empty(tokens, heads, dim, dtype=BF16, device=DEV)
    if heads:
        ops.paged_append(q, k, v, slots, kc, vc, q_out=q_out, positions=pos,
                         rope_cs=table, rope_interleaved=interleaved)
    else:
        ops.paged_append(None, k, v, slots, kc, vc, positions=pos,
                         rope_cs=table, rope_interleaved=interleaved)

    def near(got, x):
        # two products and a sum in f32, then one rounding to bf16
        ref = R.rotate(x, pos, table, interleaved)
        amp = R.rotate(x.abs(), pos, table.abs() * torch.tensor(
            [1.0, -1.0], device=DEV), interleaved).abs() + x.abs().to(F64)
        err = BF16_HALF * ref.abs() + 2.0 ** -22 * amp
        assert ((got.to(F64) - ref).abs() <= err).all()

    if heads:
        near(q_out, q)
    keep = slots >= 0
    at = slots[keep].long()
    flat_k, flat_v = kc.flatten(0, 1), vc.flatten(0, 1)
    full = torch.zeros(tokens, kv, dim, dtype=BF16, device=DEV)
    full[keep] = flat_k[at]
    ref_k = R.rotate(k, pos, table, interleaved)
    amp = 2 * k.abs().to(F64).amax(-1, keepdim=True)
    err = (BF16_HALF * ref_k.abs() + 2.0 ** -22 * amp)[keep]
    assert ((full[keep].to(F64) - ref_k[keep]).abs() <= err).all()
    assert torch.equal(flat_v[at], v[keep])
    # every other row of the caches is as it was
    rest = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    rest[at] = False
    assert torch.equal(flat_k[rest], kc0.flatten(0, 1)[rest])
    assert torch.equal(flat_v[rest], vc0.flatten(0, 1)[rest])
    assert ops.device_status() == 0


def test_paged_append_in_place_without_rotation_and_head_major_cache():
    g = gen(3)
    q = randn(g, 6, 2, 64, dt=BF16)
    k, v = randn(g, 6, 2, 64, dt=BF16), randn(g, 6, 2, 64, dt=BF16)
    slots = torch.arange(6, dtype=torch.int32, device=DEV) * 3
    # pages laid out head by head, and one key cache row wider than its values
    kc = torch.zeros(3, 2, 8, 80, dtype=BF16, device=DEV)[..., :64].transpose(1, 2)
    vc = torch.zeros(3, 2, 8, 64, dtype=BF16, device=DEV).transpose(1, 2)
    q0 = q.clone()
    ops.paged_append(q, k, v, slots, kc, vc, q_out=q)
    assert torch.equal(q, q0)
    idx = slots.long()
    assert torch.equal(kc[idx // 8, idx % 8], k)
    assert torch.equal(vc[idx // 8, idx % 8], v)
    pos = torch.arange(6, dtype=torch.int32, device=DEV)
    ops.paged_append(q, k, v, slots, kc, vc, q_out=q, positions=pos,
                     rope_cs=rope(8, 64))
    ref = R.rotate(q0, pos, rope(8, 64), False)
    assert ((q.to(F64) - ref).abs() <= BF16_HALF * ref.abs() + 2.0 ** -20 *
            q0.abs().amax()).all()


def test_paged_append_rows_outside_the_cache_or_the_table():
    """Nothing is written for them, and the status word says so once."""
    g = gen(4)
    k, v = randn(g, 4, 1, 64, dt=BF16), randn(g, 4, 1, 64, dt=BF16)
    q = randn(g, 4, 2, 64, dt=BF16)
    kc = torch.zeros(2, 4, 1, 64, dtype=BF16, device=DEV)
    vc = torch.zeros_like(kc)
    q_out = torch.full_like(q, 3.0)
    slots = torch.tensor([0, 8, 2, -1], dtype=torch.int32, device=DEV)
    pos = torch.tensor([1, 1, 16, -1], dtype=torch.int32, device=DEV)
    ops.paged_append(q, k, v, slots, kc, vc, q_out=q_out, positions=pos,
                     rope_cs=rope(16, 64))
    assert ops.device_status(reset=True) == _lib.FVB_ERR_INVALID_ARG
    flat = vc.flatten(0, 1)
    assert torch.equal(flat[0], v[0]) and (flat[1:] == 0).all()
    assert (q_out[1:] == 3).all() and not (q_out[0] == 3).any()
    # padding alone is no error
    ops.paged_append(q[3:], k[3:], v[3:], slots[3:], kc, vc, q_out=q_out[3:],
                     positions=pos[3:], rope_cs=rope(16, 64))
    assert ops.device_status() == 0 and (q_out[3] == 3).all()


# --------------------------------------------------------- paged_attention
def workspace(heads, kv, dim):
    n = ops.paged_attention_workspace_bytes(heads, kv, dim)
    return torch.zeros(n, dtype=torch.uint8, device=DEV)


def paged_inputs(g, lens, heads, kv, dim, page, head_major=False, width=None):
    """A cache whose unused rows and table entries would be noticed."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + 2
    width = width or max(need + [1])
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), width), -7, dtype=torch.int32, device=DEV)
    shape = (total, kv, page, dim) if head_major else (total, page, kv, dim)
    kc = torch.full(shape, math.nan, dtype=BF16, device=DEV)
    vc = torch.full(shape, math.nan, dtype=BF16, device=DEV)
    if head_major:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    at = 0
    for b, n in enumerate(lens):
        pages = perm[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = pages
        for c in (kc, vc):
            rows = torch.full((need[b] * page, kv, dim), math.nan, dtype=BF16,
                              device=DEV)
            rows[:n] = randn(g, n, kv, dim, dt=BF16)
            c[pages.long()] = rows.view(need[b], page, kv, dim)
    q = randn(g, len(lens), heads, dim, dt=BF16)
    return q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


def check_attention(out, lse, q, kc, vc, table, lens, scale):
    """Scores: dim products and sums in f32 (2^-23 each of the magnitudes);
    a weight is off by that and by 2^-15 (exp2, two bf16 halves, the running
    rescales); the output by the weights' error, twice for the quotient, and
    its own rounding."""
    ref, ref_lse, mag, qk = R.attention(q, kc, vc, table, lens, scale)
    es = qk * (q.shape[2] + 4) * 2.0 ** -23
    err = (2 * es + 2.0 ** -15)[..., None] * mag * 2
    err = err + BF16_HALF * (ref.abs() + err)
    assert ((out.to(F64) - ref).abs() <= err).all()
    empty = lens <= 0
    assert (out[empty] == 0).all() and (lse[empty] == -math.inf).all()
    d = (lse.to(F64) - ref_lse)[~empty].abs()
    assert (d <= es[~empty] + 2.0 ** -15 + 2.0 ** -23 * ref_lse[~empty].abs()).all()


@pytest.mark.parametrize('heads,kv,dim,page', [
    (8, 1, 256, 16), (8, 1, 256, 48), (1, 1, 64, 1), (4, 4, 128, 8),
    (12, 4, 64, 100), (32, 2, 128, 64), (40, 1, 256, 7), (5, 1, 256, 256),
    (16, 1, 256, 32), (18, 2, 64, 16)])
def test_paged_attention(heads, kv, dim, page):
    g = gen(heads * 1000 + dim + page)
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 0, 300, 867, 5]
    args = paged_inputs(g, lens, heads, kv, dim, page, head_major=kv > 1)
    ws = workspace(heads, kv, dim)
    out = torch.empty_like(args[0])
    lse = torch.empty(len(lens), heads, device=DEV)
    for _ in range(2):
        out.fill_(7.0)
        lse.fill_(7.0)
        ops.paged_attention(*args, out, scale=dim ** -0.5, lse=lse,
                            workspace=ws)
        check_attention(out, lse, *args, dim ** -0.5)
        assert ops.device_status() == 0


@pytest.mark.parametrize('lens', [
    [1], [64], [65], [816], [9000], [40000], [0, 0, 0], [0, 20000, 0],
    [1] * 400, [3000 + 17 * i for i in range(9)],
    [100000 // (i + 1) for i in range(40)]])
def test_paged_attention_lengths(lens):
    """One short sequence, one that every CTA shares, many that share a CTA,
    and lengths that differ by orders of magnitude."""
    g = gen(len(lens) + lens[0])
    args = paged_inputs(g, lens, 8, 1, 128, 64)
    ws = workspace(8, 1, 128)
    out = torch.empty_like(args[0])
    lse = torch.empty(len(lens), 8, device=DEV)
    ops.paged_attention(*args, out, scale=0.2, lse=lse, workspace=ws)
    check_attention(out, lse, *args, 0.2)
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    ops.paged_attention(*args, again, scale=0.2, lse=lse2, workspace=ws)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_paged_attention_views_large_scores_and_no_lse():
    g = gen(11)
    lens = [130, 7, 1000]
    q, kc, vc, table, ln = paged_inputs(g, lens, 4, 2, 64, 16, width=90)
    wide = randn(g, 3, 4 * 64 + 6, dt=BF16)
    q = wide[:, 2:258].unflatten(1, (4, 64))
    outw = torch.full((3, 8, 64), 9.0, dtype=BF16, device=DEV)
    out = outw[:, 2:6]
    scale = 30.0       # weights of 0 and 1 nearly everywhere
    ws = workspace(4, 2, 64)
    ops.paged_attention(q, kc, vc, table[:, :70], ln, out, scale=scale,
                        workspace=ws)
    lse = torch.empty(3, 4, device=DEV)
    out2 = torch.empty(3, 4, 64, dtype=BF16, device=DEV)
    ops.paged_attention(q, kc, vc, table, ln, out2, scale=scale, lse=lse,
                        workspace=ws)
    assert torch.equal(out, out2)
    check_attention(out2, lse, q, kc, vc, table, ln, scale)
    assert (outw[:, :2] == 9).all() and (outw[:, 6:] == 9).all()


def test_single_rows_heads_and_pages_of_any_stride():
    """A dimension of size 1 has no stride that could be misaligned."""
    g = gen(16)
    pool = randn(g, 64 * 16 + 7, dt=BF16)
    kc = pool[:1024].as_strided((1, 16, 1, 64), (3, 64, 5, 1))
    vc = pool[:1024].as_strided((1, 16, 1, 64), (1, 64, 7, 1))
    q = randn(g, 64, dt=BF16).as_strided((1, 1, 64), (13, 11, 1))
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    ln = torch.tensor([13], dtype=torch.int32, device=DEV)
    out = torch.empty(64, dtype=BF16, device=DEV).as_strided((1, 1, 64), (3, 1, 1))
    lse = torch.empty(1, 1, device=DEV)
    ops.paged_attention(q, kc, vc, table, ln, out, scale=0.2, lse=lse,
                        workspace=workspace(1, 1, 64))
    check_attention(out, lse, q, kc, vc, table, ln, 0.2)
    # one kv head seen as four (a stride of 0): read row by row
    kc4, vc4 = kc.expand(1, 16, 4, 64), vc.expand(1, 16, 4, 64)
    q4 = randn(g, 1, 8, 64, dt=BF16)
    out, lse = torch.empty_like(q4), torch.empty(1, 8, device=DEV)
    ops.paged_attention(q4, kc4, vc4, table, ln, out, scale=0.2, lse=lse,
                        workspace=workspace(8, 4, 64))
    check_attention(out, lse, q4, kc4, vc4, table, ln, 0.2)


@pytest.mark.parametrize('page', [16, 7, 1])
def test_single_rows_heads_and_pages_of_any_stride_in_c(page):
    """The same through the C entry, which is given every stride."""
    g = gen(27)
    pages = 1 if page > 1 else 9
    n = page * pages
    kc, vc = (randn(g, pages, page, 1, 64, dt=BF16) for _ in range(2))
    q, out = randn(g, 1, 1, 64, dt=BF16), torch.empty(1, 1, 64, dtype=BF16, device=DEV)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    ln = torch.tensor([n], dtype=torch.int32, device=DEV)
    lse, ws = torch.empty(1, 1, device=DEV), workspace(1, 1, 64)
    a = _lib.PagedAttnArgs(
        q=q.data_ptr(), q_row_stride=13, q_head_stride=-5, k_cache=kc.data_ptr(),
        kc_page_stride=page * 64 if pages > 1 else 3,
        kc_row_stride=64 if page > 1 else 5, kc_head_stride=7,
        v_cache=vc.data_ptr(), vc_page_stride=page * 64 if pages > 1 else -1,
        vc_row_stride=64 if page > 1 else 1, vc_head_stride=9, n_pages=pages,
        page_size=page, page_table=table.data_ptr(), ld_table=pages,
        max_pages=pages, seq_lens=ln.data_ptr(), out=out.data_ptr(),
        out_row_stride=1, out_head_stride=2, lse=lse.data_ptr(), lse_row_stride=1,
        batch=1, heads=1, kv_heads=1, head_dim=64, scale=0.2,
        workspace=ws.data_ptr(), workspace_bytes=ws.numel())
    st = torch.cuda.current_stream().cuda_stream
    assert _lib.lib().fvb_paged_attention(C.byref(a), C.c_void_p(st)) == 0
    check_attention(out, lse, q, kc, vc, table, ln, 0.2)


def test_calls_on_two_streams_and_graphs_that_share_a_workspace():
    g = gen(17)
    a = paged_inputs(g, [4000, 10, 900], 8, 1, 128, 16)
    b = paged_inputs(g, [77] * 50, 16, 2, 64, 7)
    outs = [torch.empty_like(a[0]), torch.empty_like(b[0])]
    lses = [torch.empty(3, 8, device=DEV), torch.empty(50, 16, device=DEV)]
    wss = [workspace(8, 1, 128), workspace(16, 2, 64)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, args in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                ops.paged_attention(*args, outs[i], scale=0.1, lse=lses[i],
                                    workspace=wss[i])
    torch.cuda.synchronize()
    for i, args in enumerate((a, b)):
        check_attention(outs[i], lses[i], *args, 0.1)
    # two graphs on one workspace, replayed one after the other
    ws = torch.zeros(max(w.numel() for w in wss), dtype=torch.uint8, device=DEV)
    graphs = []
    for i, args in enumerate((a, b)):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=streams[0]):
            ops.paged_attention(*args, outs[i], scale=0.1, lse=lses[i], workspace=ws)
    for o in outs:
        o.fill_(5.0)
    for _ in range(10):
        graphs[0].replay()
        graphs[1].replay()
    torch.cuda.synchronize()
    for i, args in enumerate((a, b)):
        check_attention(outs[i], lses[i], *args, 0.1)
    assert ops.device_status() == 0


def test_paged_attention_bad_lengths_and_pages_are_reported():
    g = gen(12)
    q, kc, vc, table, ln = paged_inputs(g, [20, 33, 40], 2, 1, 64, 16)
    kc.nan_to_num_(0.5)
    vc.nan_to_num_(0.5)
    ws = workspace(2, 1, 64)
    out = torch.empty_like(q)
    lse = torch.empty(3, 2, device=DEV)
    good = torch.empty_like(q)
    ops.paged_attention(q, kc, vc, table, ln, good, scale=0.1, workspace=ws)
    bad_len = ln.clone()
    bad_len[0], bad_len[2] = -3, 1000     # taken as 0 and as 48 keys
    ops.paged_attention(q, kc, vc, table, bad_len, out, scale=0.1, lse=lse,
                        workspace=ws)
    assert ops.device_status(reset=True) == _lib.FVB_ERR_INVALID_ARG
    assert (out[0] == 0).all() and torch.equal(out[1], good[1])
    bad = table.clone()
    bad[1, 1] = kc.shape[0]
    ops.paged_attention(q, kc, vc, bad, ln, out, scale=0.1, workspace=ws)
    assert ops.device_status(reset=True) == _lib.FVB_ERR_INVALID_ARG
    assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    ops.paged_attention(q, kc, vc, table, ln, out, scale=0.1, workspace=ws)
    assert ops.device_status() == 0 and torch.equal(out, good)


@pytest.mark.parametrize('pages,columns', [(0, 0), (0, 3), (2, 0)])
@pytest.mark.parametrize('batch', [1, 300])
def test_empty_caches_and_tables(pages, columns, batch):
    """No page, no column: empty sequences as anywhere else, others reported."""
    g = gen(26)
    q = randn(g, batch, 2, 64, dt=BF16)
    cache = torch.empty(pages, 16, 1, 64, dtype=BF16, device=DEV)
    table = torch.zeros(batch, columns, dtype=torch.int32, device=DEV)
    ws = workspace(2, 1, 64)
    for n, status in ((0, 0), (5, _lib.FVB_ERR_INVALID_ARG)):
        lens = torch.full((batch,), n, dtype=torch.int32, device=DEV)
        out, lse = torch.full_like(q, 5.0), torch.zeros(batch, 2, device=DEV)
        ops.paged_attention(q, cache, cache, table, lens, out, scale=1.0, lse=lse,
                            workspace=ws)
        assert (out == 0).all() and (lse == -math.inf).all()
        assert ops.device_status(reset=True) == status
    # padding alone, and a slot that is not there
    k = randn(g, batch, 1, 64, dt=BF16)
    if pages == 0:
        for slot, status in ((-1, 0), (0, _lib.FVB_ERR_INVALID_ARG)):
            slots = torch.full((batch,), slot, dtype=torch.int32, device=DEV)
            got = torch.zeros_like(q)
            ops.paged_append(q, k, k, slots, cache, cache.clone(), q_out=got)
            assert torch.equal(got, q if slot < 0 else torch.zeros_like(q))
            assert ops.device_status(reset=True) == status


@pytest.mark.parametrize('dim,page', [(64, 16), (128, 7), (256, 32)])
@pytest.mark.parametrize('n', [200, 6000])
def test_paged_attention_values_that_are_not_finite(dim, page, n):
    """They stay in their head, or in their dimension of it."""
    g = gen(23)
    q, kc, vc, table, ln = paged_inputs(g, [40] + [n] * 6, 4, 2, dim, page)
    ws = workspace(4, 2, dim)
    good, good_lse = torch.empty_like(q), torch.empty(7, 4, device=DEV)
    ops.paged_attention(q, kc, vc, table, ln, good, scale=0.125, lse=good_lse,
                        workspace=ws)

    def row(cache, seq, key):
        return cache[int(table[seq, key // page]), key % page]

    row(kc, 1, 150)[1, 3] = math.nan
    row(vc, 2, 17)[0, 5] = math.inf
    row(vc, 3, 17)[0, 6] = -math.inf
    row(vc, 3, 33)[0, 7] = math.nan
    q[4, 2, 0] = math.nan
    row(kc, 5, 199)[0, 0] = math.inf       # scores of +infinity or -infinity
    q[5, 0, 0], q[5, 1, 0] = 1.0, -1.0
    q[6] = q[6].abs() + 0.5                # scores of -infinity, all of them
    for key in range(n):
        row(kc, 6, key)[1] = -math.inf
    out, lse = torch.empty_like(q), torch.empty(7, 4, device=DEV)
    ops.paged_attention(q, kc, vc, table, ln, out, scale=0.125, lse=lse, workspace=ws)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[1, 2:] = True
    bad[2, :2, 5] = True
    bad[3, :2, 6:8] = True
    bad[4, 2] = True
    bad[5, 0] = True
    assert torch.equal(~torch.isfinite(out), bad)
    assert torch.equal(torch.isnan(lse), bad.all(-1))
    assert (out[6, 2:] == 0).all() and (lse[6, 2:] == -math.inf).all()
    # one key fewer
    assert torch.isfinite(out[5, 1]).all() and lse[5, 1] != good_lse[5, 1]
    same = ~bad
    same[5, 1] = same[6] = False           # other queries
    assert torch.equal(out[same], good[same])
    assert torch.equal(lse[same.any(-1)], good_lse[same.any(-1)])


def test_paged_attention_offsets_beyond_32_bits():
    """Pages more than 2^32 bytes and 2^31 elements apart."""
    g = gen(13)
    page, dim = 16, 64
    step = (1 << 30) + 16 * dim * 2                 # elements between pages
    pool = torch.empty(2 * step + page * dim, dtype=BF16, device=DEV)
    kc = pool.as_strided((3, page, 1, dim), (step, dim, dim, 1))
    vc = torch.empty(3, page, 1, dim, dtype=BF16, device=DEV)
    k, v = randn(g, 48, 1, dim, dt=BF16), randn(g, 48, 1, dim, dt=BF16)
    slots = torch.arange(48, dtype=torch.int32, device=DEV)
    ops.paged_append(None, k, v, slots, kc, vc)
    assert torch.equal(kc.reshape(48, 1, dim), k)
    q = randn(g, 1, 4, dim, dt=BF16)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    ln = torch.tensor([45], dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    lse = torch.empty(1, 4, device=DEV)
    ops.paged_attention(q, kc, vc, table, ln, out, scale=0.125, lse=lse,
                        workspace=workspace(4, 1, dim))
    check_attention(out, lse, q, kc, vc, table, ln, 0.125)


def test_shapes_that_share_a_workspace_and_captured_calls():
    """One workspace over several shapes; a captured append + attention whose
    lengths grow between replays; another stream."""
    g = gen(14)
    ws = torch.zeros(max(ops.paged_attention_workspace_bytes(40, 1, 256),
                         ops.paged_attention_workspace_bytes(8, 1, 64)),
                     dtype=torch.uint8, device=DEV)
    for lens, heads, kv, dim in (([5000, 3], 40, 1, 256), ([700] * 90, 8, 1, 64),
                                 ([5000, 3], 8, 2, 128)):
        args = paged_inputs(g, lens, heads, kv, dim, 32)
        out = torch.empty_like(args[0])
        lse = torch.empty(len(lens), heads, device=DEV)
        ops.paged_attention(*args, out, scale=0.1, lse=lse, workspace=ws)
        check_attention(out, lse, *args, 0.1)

    lens = [100, 63, 2000]
    q, kc, vc, table, ln = paged_inputs(g, [n + 40 for n in lens], 8, 1, 256, 16)
    kc.nan_to_num_(0.25)
    vc.nan_to_num_(0.25)
    ln.copy_(torch.tensor(lens, device=DEV))
    x = randn(g, 3, 10, 256, dt=BF16)
    rows = torch.arange(3, device=DEV)
    slots = torch.empty(3, dtype=torch.int32, device=DEV)
    pos = torch.empty(3, dtype=torch.int32, device=DEV)
    cs = rope(4096, 256)
    out = torch.empty_like(q)
    lse = torch.empty(3, 8, device=DEV)

    def step():
        ops.paged_append(x[:, :8], x[:, 8:9], x[:, 9:], slots, kc, vc, q_out=q,
                         positions=pos, rope_cs=cs)
        ops.paged_attention(q, kc, vc, table, ln, out, scale=0.0625, lse=lse,
                            workspace=ws)

    def place(at):
        pos.copy_(at)
        ln.copy_(at + 1)
        page = table[rows, (at // 16).long()]
        slots.copy_(page * 16 + at % 16)

    at = torch.tensor(lens, dtype=torch.int32, device=DEV)
    place(at)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        check_attention(out, lse, q, kc, vc, table, ln, 0.0625)
        with torch.cuda.graph(graph, stream=side):
            step()
    for i in range(30):
        at += 1
        place(at)
        x.copy_(randn(g, 3, 10, 256, dt=BF16))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_attention(out, lse, q, kc, vc, table, ln, 0.0625)
        assert torch.equal(vc[table[rows, (at // 16).long()].long(), (at % 16).long()],
                           x[:, 9:])
    assert ops.device_status() == 0


# ------------------------------------------------------- the run of them all
@pytest.mark.parametrize('tokens', [1, 5, 70])
def test_decoder_layer_of_one_token_per_request(tokens):
    """norm -> qkv -> append -> attention -> codes -> o -> residual + norm ->
    gate/up -> codes -> down, each step against its formula on what the step
    before it gave."""
    g = gen(20 + tokens)
    width, heads, dim, mlp, page = 512, 4, 128, 1024, 16
    qkv_w, qkv_s = pack.quantize_blocks(randn(g, (heads + 2) * dim, width) * 0.05)
    o_w, o_s = pack.quantize_blocks(randn(g, width, heads * dim) * 0.05)
    gu_w, gu_s = pack.quantize_blocks(pack.pack_geglu(
        randn(g, mlp, width) * 0.05, randn(g, mlp, width) * 0.05))
    dn_w, dn_s = pack.quantize_blocks(randn(g, width, mlp) * 0.05)
    w1, w2 = randn(g, width, dt=BF16) * 0.1, randn(g, width, dt=BF16) * 0.1
    lens = [(37 * i) % 200 + 1 for i in range(tokens)]      # new token included
    _, kc, vc, table, ln = paged_inputs(g, lens, heads, 1, dim, page)
    at = ln - 1
    rows = torch.arange(tokens, device=DEV)
    slots = (table[rows, (at // page).long()] * page + at % page).to(torch.int32)
    cs = rope(256, dim)
    x = randn(g, tokens, width)
    ws = workspace(heads, 1, dim)

    def codes(mode, x, **kw):
        q = torch.empty(x.shape, dtype=E4M3, device=DEV)
        s = torch.empty(x.shape[0], -(-x.shape[1] // 128), device=DEV)
        res = torch.empty_like(x) if 'delta' in kw else None
        ops.norm_fp8(MODES[mode], x, q, s, res=res, **kw)
        check_norm(mode, x, kw, q, s, res)
        return q, s, res

    def product(a, sa, b, sb, epi='bf16'):
        n = b.shape[0] // 2 if epi == 'geglu' else b.shape[0]
        out = torch.empty(tokens, n, dtype=F32 if epi == 'f32' else BF16, device=DEV)
        ops.gemm_fp8(a, sa, b, sb, out, epilogue=EPIS[epi])
        check_gemm(out, a, sa, b, sb, EPIS[epi])
        return out

    a, sa, _ = codes('gemma', x, w=w1)
    qkv = product(a, sa, qkv_w, qkv_s).unflatten(1, (heads + 2, dim))
    q = torch.empty(tokens, heads, dim, dtype=BF16, device=DEV)
    ops.paged_append(qkv[:, :heads], qkv[:, heads:heads + 1], qkv[:, heads + 1:],
                     slots, kc, vc, q_out=q, positions=at, rope_cs=cs)
    ref = R.rotate(qkv[:, :heads], at, cs, False)
    assert ((q.to(F64) - ref).abs() <= BF16_HALF * ref.abs() + 2.0 ** -20 *
            qkv.abs().amax()).all()
    o = torch.empty_like(q)
    lse = torch.empty(tokens, heads, device=DEV)
    ops.paged_attention(q, kc, vc, table, ln, o, scale=dim ** -0.5, lse=lse,
                        workspace=ws)
    check_attention(o, lse, q, kc, vc, table, ln, dim ** -0.5)
    a, sa, _ = codes('none', o.flatten(1))
    a, sa, x2 = codes('gemma', x, w=w2, delta=product(a, sa, o_w, o_s))
    h = product(a, sa, gu_w, gu_s, 'geglu')
    a, sa, _ = codes('none', h)
    y = x2 + product(a, sa, dn_w, dn_s, 'f32')
    assert torch.isfinite(y).all() and ops.device_status() == 0


class Layer:
    """The operators of a decoder layer on buffers of its own, one call after
    the other; ``sync`` waits for the GPU after each."""

    def __init__(self, tokens, seed):
        g = gen(seed)
        self.tokens, self.g = tokens, g
        self.heads, self.dim, page, width, mlp = 8, 128, 16, 1024, 2048

        def weight(n, k, geglu=False):
            w = randn(g, n, k) * k ** -0.5
            if geglu:
                w = pack.pack_geglu(w[:n // 2], w[n // 2:])
            return pack.quantize_blocks(w)

        def codes(n):
            return (torch.empty(tokens, n, dtype=E4M3, device=DEV),
                    torch.empty(tokens, n // 128, device=DEV))

        self.qkv_w = weight((self.heads + 2) * self.dim, width)
        self.o_w = weight(width, self.heads * self.dim)
        self.gu_w, self.dn_w = weight(2 * mlp, width, True), weight(width, mlp)
        self.w1, self.w2 = (randn(g, width, dt=BF16) * 0.1 for _ in range(2))
        lens = [(37 * i) % 500 + 1 for i in range(tokens)]
        _, self.kc, self.vc, self.table, _ = paged_inputs(
            g, lens, self.heads, 1, self.dim, page)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.cs = rope(512, self.dim)
        self.x = torch.empty(tokens, width, device=DEV)
        self.c = [codes(width), codes(self.heads * self.dim), codes(width), codes(mlp)]
        self.qkv = torch.empty(tokens, (self.heads + 2) * self.dim, dtype=BF16, device=DEV)
        self.q, self.att = (torch.empty(tokens, self.heads, self.dim, dtype=BF16, device=DEV)
                            for _ in range(2))
        self.o, self.down = (torch.empty(tokens, width, dtype=BF16, device=DEV)
                             for _ in range(2))
        self.h = torch.empty(tokens, mlp, dtype=BF16, device=DEV)
        self.lse = torch.empty(tokens, self.heads, device=DEV)
        self.ws = workspace(self.heads, 1, self.dim)
        self.at, self.slots = torch.empty_like(self.lens), torch.empty_like(self.lens)

    def inputs(self):
        """A new residual row and a new place in the cache for each token."""
        self.x.copy_(randn(self.g, *self.x.shape))
        at = (torch.rand(self.tokens, generator=self.g, device=DEV) * self.lens).int()
        rows = torch.arange(self.tokens, device=DEV)
        self.at.copy_(at)
        self.slots.copy_(self.table[rows, (at // 16).long()] * 16 + at % 16)

    def run(self, sync=False):
        heads, wait = self.heads, torch.cuda.synchronize if sync else lambda: None
        rows = self.qkv.unflatten(1, (heads + 2, self.dim))
        (a, sa), (b, sb), (c, sc), (d, sd) = self.c
        for call in (
                lambda: ops.norm_fp8(_lib.NORM_GEMMA_RMS, self.x, a, sa, w=self.w1),
                lambda: ops.gemm_fp8(a, sa, *self.qkv_w, self.qkv),
                lambda: ops.paged_append(
                    rows[:, :heads], rows[:, heads:heads + 1], rows[:, heads + 1:],
                    self.slots, self.kc, self.vc, q_out=self.q, positions=self.at,
                    rope_cs=self.cs),
                lambda: ops.paged_attention(
                    self.q, self.kc, self.vc, self.table, self.lens, self.att,
                    scale=self.dim ** -0.5, lse=self.lse, workspace=self.ws),
                lambda: ops.norm_fp8(_lib.NORM_NONE, self.att.flatten(1), b, sb),
                lambda: ops.gemm_fp8(b, sb, *self.o_w, self.o),
                lambda: ops.norm_fp8(_lib.NORM_GEMMA_RMS, self.x, c, sc, w=self.w2,
                                     delta=self.o, res=self.x),
                lambda: ops.gemm_fp8(c, sc, *self.gu_w, self.h, epilogue=_lib.EPI_GEGLU),
                lambda: ops.norm_fp8(_lib.NORM_NONE, self.h, d, sd),
                lambda: ops.gemm_fp8(d, sd, *self.dn_w, self.down)):
            call()
            wait()

    def state(self):
        # bytes: the unused rows of the caches are NaN
        return [t.clone().view(torch.uint8) for t in (
            self.x, self.down, self.h, self.o, self.att, self.lse, self.q, self.kc, self.vc,
            *(t for pair in self.c for t in pair))]


@pytest.mark.parametrize('tokens', [1, 16, 200])
def test_layers_back_to_back_equal_layers_call_by_call(tokens):
    """Each kernel may start while the one before it still writes what it reads
    (codes, scales, queries, cache rows): ten layers of new inputs without a
    wait, eager and captured, against the same with a wait after every call."""
    steps, step, eager, graphed = 10, *(Layer(tokens, 40) for _ in range(3))
    want, got = [], []
    for _ in range(steps):
        step.inputs()
        step.run(sync=True)
        want.append(step.state())
    torch.cuda.synchronize()
    for _ in range(steps):
        eager.inputs()
        eager.run()
        got.append(eager.state())
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    # captured: two layers in a row on the same inputs
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        graphed.run()
        graphed.run()
    step, twice = Layer(tokens, 40), []
    for _ in range(steps):
        step.inputs()
        step.run(sync=True)
        step.run(sync=True)
        twice.append(step.state())
    for a in twice:
        graphed.inputs()
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(a, graphed.state()))
    assert ops.device_status() == 0


def test_operators_on_streams_of_their_own():
    """Products of both kernels, norms and attention side by side, in an order
    that changes, give what each gives alone."""
    g = gen(30)
    jobs = []
    for m, n, k, epi in ((816, 8192, 2048, 'geglu'), (64, 2048, 4096, 'f32'),
                         (1, 2560, 2048, 'bf16'), (768, 1152, 4304, 'bf16'),
                         (2000, 4096, 1024, 'bf16')):
        args = gemm_inputs(g, m, n, k)
        out = torch.empty(m, n // 2 if epi == 'geglu' else n, device=DEV,
                          dtype=F32 if epi == 'f32' else BF16)
        jobs.append((lambda args=args, out=out, epi=epi: ops.gemm_fp8(
            *args, out, epilogue=EPIS[epi]), [out]))
    for lens, heads, kv, dim, page in (([3000] * 20, 8, 1, 128, 16),
                                       ([9000], 8, 2, 64, 7),
                                       (list(range(100, 164)), 16, 1, 256, 32)):
        args = paged_inputs(g, lens, heads, kv, dim, page)
        out, lse = torch.empty_like(args[0]), torch.empty(len(lens), heads, device=DEV)
        ws = workspace(heads, kv, dim)
        jobs.append((lambda args=args, out=out, lse=lse, ws=ws: ops.paged_attention(
            *args, out, scale=0.1, lse=lse, workspace=ws), [out, lse]))
    x = randn(g, 2000, 2048)
    q = torch.empty(2000, 2048, dtype=E4M3, device=DEV)
    s = torch.empty(2000, 16, device=DEV)
    jobs.append((lambda: ops.norm_fp8(_lib.NORM_RMS, x, q, s), [q.view(torch.uint8), s]))
    want = []
    for call, outs in jobs:
        call()
        want.append([t.clone() for t in outs])
        for t in outs:
            t.fill_(3)
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for i in range(60):
        for j in range(len(jobs)):
            j = (j * 4 + i) % len(jobs)          # 9 jobs: 4 is prime to them
            with torch.cuda.stream(streams[j]):
                jobs[j][0]()
    torch.cuda.synchronize()
    for (_, outs), ref in zip(jobs, want):
        assert all(torch.equal(a, b) for a, b in zip(outs, ref))
    assert ops.device_status() == 0
