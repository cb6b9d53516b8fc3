"""GPU tests of what lies between two linear layers: products with an epilogue, 8-bit checkpoints of activations and the
gradients taken from them, against the definitions in 64 bits."""

import math

import pytest
import torch

from msamp import _backend
from msamp.common.dtype import Dtypes
from msamp.common.tensor import BlockTensor, ScalingMeta, ScalingTensor
from msamp.operators.activation import Activation
from msamp.operators.gemm import Gemm
from oracle import activation as oact

pytestmark = pytest.mark.gpu

DTYPES = (torch.float32, torch.float16, torch.bfloat16)
ROUNDING = {dtype: torch.finfo(dtype).eps / 2 for dtype in DTYPES}    # half a unit in the last place
SMALLEST = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}    # of a type, denormal


def gen(seed):
    return torch.Generator().manual_seed(seed)


def allowed(dtype, want, error):
    """A value within `error` of `want`, rounded once to dtype."""
    return error + ROUNDING[dtype] * (want.abs() + error) + SMALLEST[dtype] / 2


def assert_within(got, want, bound, what):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    off = (got - want).abs()
    ok = (off <= bound) | torch.isnan(want) | (got == want)
    assert bool(ok.all()), (what, int((~ok).sum()), float((off / bound)[~ok].max()), int((~ok).flatten().nonzero()[0]))


# ---- checkpoints ---------------------------------------------------------------------------------------------------
def activations(rows, cols, dtype, seed, scale=1.0):
    x = torch.randn(rows, cols, generator=gen(seed)) * scale
    x.view(-1)[::37] *= 25.0
    return x.to(dtype)


def assert_packed(packed, x):
    codes, exponents = oact.pack(x)
    assert torch.equal(packed.exponent.cpu(), exponents)
    # (a NaN has one code, whatever its sign)
    nan = (codes & 0x7f) == 0x7f
    assert torch.equal((packed.value.cpu() & 0x7f) == 0x7f, nan)
    assert torch.equal(packed.value.cpu()[~nan], codes[~nan])


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cols', [(1, 1), (1, 31), (3, 32), (2, 33), (7, 77), (5, 128), (129, 8), (33, 1000), (64, 4301), (257, 4096)])
def test_checkpoint_has_the_codes_of_its_definition(dtype, rows, cols):
    x = activations(rows, cols, dtype, rows * 1000 + cols)
    packed = BlockTensor.pack(x.cuda())
    assert packed.shape == x.shape and packed.nbytes == packed.value.numel() + packed.exponent.numel()
    assert_packed(packed, x)
    want = oact.unpack(packed.value.cpu(), packed.exponent.cpu(), cols)
    for out in DTYPES:
        assert torch.equal(packed.to(out).cpu(), want.to(out)), out


@pytest.mark.parametrize('dtype', DTYPES)
def test_checkpoint_at_the_edges_of_its_formats(dtype):
    """Block maxima at and next to 448 * 2^E, zeros, denormals, the type's largest and smallest values, ties, infinities and NaN."""
    top = torch.finfo(dtype).max
    edge = torch.tensor([448.0, 449.0, 447.0, 1.75, 1.7500001, 1.751, 0.0, -0.0, 1e-30, 1e-40, 2.0**-126, 2.0**-149, top, top / 2, 2.0**-24])
    x = torch.randn(edge.numel() * 2, 96, generator=gen(3))
    x = x / x.abs().amax(1, keepdim=True)
    x = x * edge.repeat(2).unsqueeze(1)
    x[:, 5] = edge.repeat(2)
    x[:, 40] = -edge.repeat(2)
    x = x.to(dtype)
    x[3, 7], x[4, 8], x[5, 9] = math.inf, -math.inf, math.nan
    x[6, :32] = math.inf
    x[7, 32:64] = math.nan
    x[8, 64:] = torch.arange(32).to(dtype) * (1 + 1 / 16)    # middles of two codes
    packed = BlockTensor.pack(x.cuda())
    assert_packed(packed, x)
    want = oact.unpack(packed.value.cpu(), packed.exponent.cpu(), 96).to(dtype)
    got = packed.to(dtype).cpu()
    assert torch.equal(torch.nan_to_num(got, nan=77.0), torch.nan_to_num(want, nan=77.0))
    assert torch.isnan(got[3, 7]) and torch.isnan(got[4, 8]) and torch.isnan(got[5, 9]) and bool(torch.isnan(got[6, :32]).all())
    finite = torch.isfinite(x.float())
    block = oact.blocks(torch.where(finite, x.double(), torch.zeros_like(x, dtype=torch.float64))).abs().amax(2).repeat_interleave(32, 1)
    # half a step of three bits below the value's binade, at least half a step of the block's smallest codes
    off = (oact.unpack(packed.value.cpu(), packed.exponent.cpu(), 96) - x.double()).abs()
    bound = torch.maximum(x.double().abs() / 16, torch.maximum(block / 448 * 2.0**-9, torch.tensor(2.0**-136, dtype=torch.float64)))
    assert bool((off <= bound)[finite].all())


def test_checkpoint_of_any_order_in_memory():
    x = torch.randn(6, 40, 3, 70, generator=gen(5)).cuda()
    for view in (x, x[:, 3:, :, :64], x[..., 5:], x.transpose(1, 2), x.transpose(2, 3), x[::2], x[0, 0, 0], x[0, 0, 0, 3], x[..., ::2],
                 x[:1].expand(4, 40, 3, 70), x[0, :, 0, 2:66], x[0, :1, 0, 1:2].expand(5, 9)):
        packed = BlockTensor.pack(view)
        flat = view.reshape(-1, view.shape[-1]) if view.dim() else view.reshape(1, 1)
        assert packed.shape == view.shape
        assert_packed(packed, flat.cpu())
        assert packed.float().shape == view.shape
    for shape in ((0, ), (0, 5), (5, 0), (2, 0, 3)):
        packed = BlockTensor.pack(torch.empty(shape, device='cuda'))
        assert packed.float().shape == shape and packed.numel() == 0


def test_checkpoint_refusals():
    x = torch.randn(4, 64, device='cuda')
    with pytest.raises(TypeError):
        BlockTensor.pack([1.0])
    with pytest.raises(TypeError):
        BlockTensor.pack(x.double())
    with pytest.raises(TypeError):
        BlockTensor.pack(x.int())
    with pytest.raises(ValueError):
        BlockTensor.pack(x.cpu())
    packed = BlockTensor.pack(x)
    with pytest.raises(TypeError):
        packed.to(torch.int32)
    with pytest.raises(ValueError):
        BlockTensor(packed.value, packed.exponent, (4, 65))
    with pytest.raises(ValueError):
        BlockTensor(packed.value, packed.exponent[:, :1], (4, 64))
    with pytest.raises(TypeError):
        BlockTensor(packed.value.int(), packed.exponent, (4, 64))


# ---- products with an epilogue ------------------------------------------------------------------------------------
def whole_codes(rows, cols, seed, most=3):
    """A ScalingTensor of small whole numbers times a power of two: products of them are summed without rounding."""
    x = torch.randint(-most, most + 1, (rows, cols), generator=gen(seed)).float()
    meta = ScalingMeta(Dtypes.kfloat8_e4m3, scale_inv=torch.tensor(2.0**-5, device='cuda'))
    return x, ScalingTensor(x.to(torch.float8_e4m3fn).view(torch.uint8).cuda(), meta)


def epilogue_error(z, gate, y, residual):
    """Of the float32 epilogue: an activation is within 1e-6 of |z| (its exponential's argument is rounded to 2^-24 of itself, two
    approximations within an ulp or two, Phi within 2.1e-7), every product and sum behind it within 2^-24 of its result."""
    g = 1.0 if gate is None else gate.double().abs()
    r = 0.0 if residual is None else residual.double().abs()
    return 1e-6 * z.abs() * g + 2.0**-23 * (y.abs() + r)


def check_product(n, m, k, dtype, name, bias, gate, residual, seed, checkpoint=False, wide=False, most=3):
    x, xs = whole_codes(n, k, seed, most)
    w, ws = whole_codes(m, k, seed + 1, most)
    z = x.double() @ w.double().t() * 2.0**-10
    b = g = r = None
    if bias:
        b = (torch.randint(-64, 65, (m, ), generator=gen(seed + 2)).float() / 64).to(dtype)
        z = z + b.double()
    y = oact.value(z, name)
    def beside(s):
        t = torch.randn(n, 2 * m + 3 if wide else m, generator=gen(s)).to(dtype)
        return (t[:, m + 1:2 * m + 1], t.cuda()[:, m + 1:2 * m + 1]) if wide else (t, t.cuda())
    if gate:
        g, g_gpu = beside(seed + 3)
        y = y * g.double()
    if residual:
        r, r_gpu = beside(seed + 4)
        y = y + r.double()
    got = Gemm.fp8_gemm_fused(ws, xs, Dtypes.dtype_to_qtype[dtype], bias=None if b is None else b.cuda(), activation=name,
                              gate=g_gpu if gate else None, residual=r_gpu if residual else None, checkpoint=checkpoint)
    if checkpoint:
        got, z8, g8 = got
        assert z8.shape == (n, m)
        assert_packed(z8, z.float())
        assert (g8 is None) == (g is None)
        if g8 is not None:
            assert_packed(g8, g)
    assert got.dtype == dtype
    assert_within(got, y, allowed(dtype, y, epilogue_error(z, g, y, r)), (n, m, k, dtype, name))


@pytest.mark.parametrize('name', oact.NAMES)
@pytest.mark.parametrize('dtype', DTYPES)
def test_fused_product_of_few_rows(dtype, name):
    check_product(1, 96, 256, dtype, name, True, True, True, 11)
    check_product(5, 100, 200, dtype, name, False, True, False, 12, checkpoint=True, wide=True)
    check_product(48, 65, 1040, dtype, name, True, False, True, 13, checkpoint=True)


@pytest.mark.parametrize('n', [1, 2, 15, 16, 17, 31, 33, 63, 64, 65])
@pytest.mark.parametrize('m,k', [(1, 1), (7, 15), (31, 16), (32, 17), (33, 127), (257, 128), (300, 129), (1000, 1200)])
def test_fused_product_of_odd_sizes(n, m, k):
    check_product(n, m, k, torch.bfloat16, 'silu', True, True, False, n * m + k, checkpoint=m % 2 == 1, wide=n % 2 == 1)


# (a compute unit, one tile or several; two slices of K and one; a ragged last slice; few rounds of large tiles)
@pytest.mark.parametrize('n,m,k', [(65, 128, 128), (129, 257, 64), (200, 136, 384), (128, 128, 4096), (300, 72, 1040), (1024, 1032, 2064),
                                   (2560, 4360, 272), (2500, 4101, 384), (4100, 8200, 128), (2048, 4104, 77), (2100, 4128, 200), (150, 512, 1033)])
@pytest.mark.parametrize('dtype', DTYPES)
def test_fused_product_of_tiles(n, m, k, dtype):
    check_product(n, m, k, dtype, 'gelu_tanh', True, True, True, n + m + k, checkpoint=True, wide=m % 8 != 0, most=1)


@pytest.mark.parametrize('name', oact.NAMES)
def test_fused_product_of_large_tiles(name):
    """Every activation in the 256 x 256-tile kernel, whole tiles and ragged ones, with every part of the epilogue and with one."""
    check_product(2304, 8192, 256, torch.bfloat16, name, True, True, True, 3, checkpoint=True, most=1)
    check_product(2400, 8256, 400, torch.float16, name, False, False, False, 4, checkpoint=True, most=1)
    check_product(2400, 8256, 400, torch.bfloat16, name, False, name != 'relu', True, 5, most=1)


def test_fused_product_keeps_infinities_and_nan_apart():
    """A NaN code in one row of x, an infinite gate value and an infinite residual reach the outputs that they are part of and no others."""
    for n in (3, 200):
        x, xs = whole_codes(n, 256, 21)
        w, ws = whole_codes(64, 256, 22)
        xs.value[1, 7] = 0x7f
        gate = torch.ones(n, 64, device='cuda', dtype=torch.bfloat16)
        residual = torch.zeros(n, 64, device='cuda', dtype=torch.bfloat16)
        gate[2, 5], residual[0, 9] = math.inf, -math.inf
        out, z8, g8 = Gemm.fp8_gemm_fused(ws, xs, Dtypes.kbfloat16, activation='gelu', gate=gate, residual=residual, checkpoint=True)
        assert bool(torch.isnan(out[1]).all()) and bool(torch.isnan(z8.float()[1]).all())
        assert out[0, 9] == -math.inf and not bool(torch.isfinite(out[2, 5])) and bool(torch.isnan(g8.float()[2, 5]))
        out[1], out[0, 9], out[2, 5] = 0, 0, 0
        assert bool(torch.isfinite(out).all())


def test_fused_product_in_place_of_its_residual_and_on_another_stream():
    x, xs = whole_codes(130, 512, 31)
    w, ws = whole_codes(96, 512, 32)
    residual = torch.randn(130, 96, device='cuda').bfloat16()
    want = Gemm.fp8_gemm_fused(ws, xs, Dtypes.kbfloat16, activation='silu', residual=residual)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = Gemm.fp8_gemm_fused(ws, xs, Dtypes.kbfloat16, activation='silu', residual=residual)
    side.synchronize()
    assert torch.equal(got, want)


def test_fused_product_refusals():
    x, xs = whole_codes(4, 64, 41)
    w, ws = whole_codes(8, 64, 42)
    q = Dtypes.kbfloat16
    out = Gemm.fp8_gemm_fused(ws, xs, q)
    with pytest.raises(ValueError):
        Gemm.fp8_gemm_fused(ws, xs, q, activation='swish')
    with pytest.raises(TypeError):
        Gemm.fp8_gemm_fused(ws.value, xs, q)
    with pytest.raises(TypeError):
        Gemm.fp8_gemm_fused(ws, ScalingTensor(xs.value, ScalingMeta(Dtypes.kfloat8_e5m2)), q)
    with pytest.raises(ValueError):
        Gemm.fp8_gemm_fused(ws, whole_codes(4, 65, 1)[1], q)
    with pytest.raises(ValueError):
        Gemm.fp8_gemm_fused(ws, xs, q, gate=out[:, :4])
    with pytest.raises(TypeError):
        Gemm.fp8_gemm_fused(ws, xs, q, gate=out.float())
    with pytest.raises(ValueError):
        Gemm.fp8_gemm_fused(ws, xs, q, residual=out.cpu())
    with pytest.raises(ValueError):
        Gemm.fp8_gemm_fused(ws, xs, q, bias=out[0, :4])
    with pytest.raises(ValueError):
        Gemm.fp8_gemm_fused(whole_codes(8, 0, 1)[1], whole_codes(4, 0, 1)[1], q)
    empty = Gemm.fp8_gemm_fused(ws, whole_codes(0, 64, 1)[1], q, checkpoint=True)
    assert empty[0].shape == (0, 8) and empty[1].shape == (0, 8)


# ---- gradients -----------------------------------------------------------------------------------------------------
def held(rows, cols, seed, scale=1.0):
    """A checkpoint and the values that it holds."""
    packed = BlockTensor.pack(activations(rows, cols, torch.float32, seed, scale).cuda())
    return packed, oact.unpack(packed.value.cpu(), packed.exponent.cpu(), cols)


def slope_error(z):
    """Of the float32 derivatives: as an activation's, and where they subtract from one (1 - s, held to 2^-24) up to |z|^3 of that."""
    return 1e-6 * (1.0 + z.abs()**3)


def check_gradients(rows, cols, dtype, name, gated, bias_dtype, seed, stride=0):
    z8, z = held(rows, cols, seed)
    g8, g = held(rows, cols, seed + 1) if gated else (None, None)
    dy = torch.randn(rows, cols + stride, generator=gen(seed + 2)).to(dtype)
    dy_gpu = dy.cuda()[:, stride:]
    dy = dy[:, stride:]
    dz, dg, db = Activation.backward(dy_gpu, z8, name, gate=g8, bias_dtype=bias_dtype)
    want_dz, want_dg, want_db = oact.gradients(dy, z, name, g)
    part = dy.double().abs() * (1.0 if g is None else g.abs())
    error = part * slope_error(z) + 2.0**-22 * want_dz.abs()
    assert dz.dtype == dtype and dz.is_contiguous()
    assert_within(dz, want_dz, allowed(dtype, want_dz, error), ('dz', rows, cols, dtype, name))
    if gated:
        assert_within(dg, want_dg, allowed(dtype, want_dg, dy.double().abs() * z.abs() * 1e-6 + 2.0**-23 * want_dg.abs()), ('dgate', rows, cols))
    assert (dg is None) == (g is None) and (db is None) == (bias_dtype is None)
    if db is not None:
        assert db.dtype == bias_dtype
        # a sum of n float32 numbers in any order: n roundings of at most the sum of the magnitudes; here no chain is longer than 256
        bound = error.sum(0) + 256 * 2.0**-24 * want_dz.abs().sum(0)
        assert_within(db, want_db, allowed(bias_dtype, want_db, bound), ('dbias', rows, cols))


@pytest.mark.parametrize('name', oact.NAMES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('gated', [False, True])
def test_gradients_are_those_of_the_formula(dtype, name, gated):
    check_gradients(37, 96, dtype, name, gated, None, 51)
    check_gradients(130, 77, dtype, name, gated, torch.float32, 52, stride=1)
    check_gradients(64, 256, dtype, name, gated, dtype, 53, stride=8)


@pytest.mark.parametrize('rows,cols', [(1, 1), (1, 32), (2, 31), (300, 8), (1000, 33), (5000, 16), (17, 5000), (4097, 520), (70, 16384)])
def test_gradients_of_odd_sizes(rows, cols):
    for bias_dtype in (None, torch.float32):
        check_gradients(rows, cols, torch.bfloat16, 'silu', True, bias_dtype, rows + cols)


@pytest.mark.parametrize('name', oact.NAMES[2:])
def test_gradients_are_what_differences_say(name):
    """The loss sum(dy * act(z) * gate), in 64 bits, moved by h either way in every z and gate: its central difference is off by
    h^2 / 6 of a third derivative (below 10 for all of these) and by 2^-53 of the loss' parts over h."""
    z8, z = held(20, 64, 61)
    g8, g = held(20, 64, 62)
    dy = torch.randn(20, 64, generator=gen(63))
    dz, dg, _ = Activation.backward(dy.cuda(), z8, name, gate=g8)
    h = 1e-5
    part = lambda z, g: dy.double() * oact.value(z, name) * g    # noqa: E731
    want_z = (part(z + h, g) - part(z - h, g)) / (2 * h)
    want_g = (part(z, g + h) - part(z, g - h)) / (2 * h)
    scale = dy.double().abs() * (1 + g.abs()) * (1 + z.abs())
    bound = scale * (slope_error(z) + 10 * h * h + 2.0**-50 / h) + 2.0**-22 * want_z.abs()
    assert_within(dz, want_z, bound, 'dz')
    assert_within(dg, want_g, bound + 2.0**-22 * want_g.abs(), 'dgate')


def test_gradients_repeat_to_the_bit_and_pass_nan_on():
    z8, z = held(3000, 264, 71)
    dy = torch.randn(3000, 264, device='cuda').bfloat16()
    first = Activation.backward(dy, z8, 'gelu', bias_dtype=torch.float32)
    for _ in range(3):
        again = Activation.backward(dy, z8, 'gelu', bias_dtype=torch.float32)
        assert torch.equal(first[0], again[0]) and torch.equal(first[2], again[2])
    dy[5, 7] = math.nan
    x = torch.randn(3000, 264, device='cuda')
    x[9, 11] = math.inf
    for name in oact.NAMES[1:]:
        dz, _, db = Activation.backward(dy, BlockTensor.pack(x), name, bias_dtype=torch.float32)
        assert bool(torch.isnan(dz[5, 7])) and bool(torch.isnan(dz[9, 11])) and int(torch.isnan(dz).sum()) == 2
        assert bool(torch.isnan(db[7])) and bool(torch.isnan(db[11])) and int(torch.isnan(db).sum()) == 2


@pytest.mark.parametrize('qtype', [Dtypes.kfloat8_e5m2, Dtypes.kfloat8_e4m3])
@pytest.mark.parametrize('dtype,rows,cols', [(torch.bfloat16, 130, 96), (torch.float16, 33, 77), (torch.float32, 1, 5), (torch.bfloat16, 2000, 520)])
@pytest.mark.parametrize('gated', [False, True])
def test_gradients_cast_as_the_gated_cast_does(qtype, dtype, rows, cols, gated):
    fmt, top, least, bits = (torch.float8_e4m3fn, 448.0, -6, 3) if qtype == Dtypes.kfloat8_e4m3 else (torch.float8_e5m2, 57344.0, -14, 2)
    z8, z = held(rows, cols, 81)
    g8, g = held(rows, cols, 82) if gated else (None, None)
    dy = (torch.randn(rows, cols, generator=gen(83)) * 1e-3).to(dtype)
    want_dz, want_dg, want_db = oact.gradients(dy, z, 'gelu', g)
    error = dy.double().abs() * (1.0 if g is None else g.abs()) * slope_error(z) + 2.0**-22 * want_dz.abs()
    amax = float(want_dz.abs().max())
    meta = ScalingMeta(qtype, window_size=4)
    for full in (False, True):
        if full:    # delayed: the scale is the meta's, whatever the gradient; half of the largest values leave the format
            meta.amax_counter.fill_(4)
            meta.scale.fill_(2.0**math.ceil(math.log2(top / amax)))
            meta.amax.zero_()
            meta.amax[0] = amax / 2
        dz, dg, db = Activation.backward_cast(dy.cuda(), z8, 'gelu', meta, gate=g8, bias_dtype=torch.float32)
        scale = float(meta.scale)
        if not full:
            assert scale == 2.0**math.floor(math.log2(top / amax))
        assert abs(float(meta.amax[0]) - amax) <= 1e-5 * amax
        assert float(meta.scale_inv) == 1.0 / scale and dz.meta is meta and dz.value.shape == (rows, cols)
        v = (want_dz * scale).clamp(-top, top)
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0**least))) - bits)
        got = dz.value.cpu().view(fmt).double()
        assert_within(got, v, step / 2 * 1.0001 + error * scale, (qtype, full))
        if gated:
            assert_within(dg, want_dg, allowed(dtype, want_dg, dy.double().abs() * z.abs() * 1e-6 + 2.0**-23 * want_dg.abs()), 'dgate')
        assert_within(db, want_db, error.sum(0) + 256 * 2.0**-24 * want_dz.abs().sum(0) + 2.0**-24 * want_db.abs(), 'dbias')
    # a larger maximum that is there already stays
    meta.amax[0] = 2 * amax
    Activation.backward_cast(dy.cuda(), z8, 'gelu', meta, gate=g8)
    assert float(meta.amax[0]) == torch.tensor(2 * amax).float().item()


def test_gradient_refusals():
    z8, z = held(4, 64, 91)
    dy = torch.randn(4, 64, device='cuda')
    meta = ScalingMeta(Dtypes.kfloat8_e5m2, window_size=16)
    with pytest.raises(ValueError):
        Activation.backward(dy, z8, 'tanh')
    with pytest.raises(TypeError):
        Activation.backward(dy, z8.float(), 'gelu')
    with pytest.raises(ValueError):
        Activation.backward(dy[:3], z8, 'gelu')
    with pytest.raises(ValueError):
        Activation.backward(dy.cpu(), z8, 'gelu')
    with pytest.raises(TypeError):
        Activation.backward(dy.double(), z8, 'gelu')
    with pytest.raises(TypeError):
        Activation.backward(dy, z8, 'gelu', bias_dtype=torch.int32)
    with pytest.raises(ValueError):
        Activation.backward(dy, z8, 'gelu', gate=held(4, 32, 1)[0])
    with pytest.raises(ValueError):
        Activation.backward_cast(dy, z8, 'gelu', ScalingMeta(Dtypes.kfloat8_e5m2))
    with pytest.raises(ValueError):
        Activation.backward_cast(dy, z8, 'gelu', ScalingMeta(Dtypes.kfloat16, window_size=16))
    with pytest.raises(ValueError):
        Activation.backward_cast(torch.empty(0, 64, device='cuda'), held(4, 64, 1)[0], 'gelu', meta)
    empty = BlockTensor.pack(torch.empty(0, 64, device='cuda'))
    dz, dg, db = Activation.backward(torch.empty(0, 64, device='cuda'), empty, 'gelu', gate=empty, bias_dtype=torch.float32)
    assert dz.shape == (0, 64) and dg.shape == (0, 64) and bool((db == 0).all())


# ---- every code, long tensors, tiles of two sizes -----------------------------------------------------------------------
@pytest.mark.parametrize('name', oact.NAMES)
@pytest.mark.parametrize('gated', [False, True])
def test_gradients_at_every_code(name, gated):
    """All 256 codes under exponents from the least to where every activation is through with bending: with a bias gradient and without."""
    exponents = [1, 50, *range(90, 140)]
    rows, cols = len(exponents), 256
    z8 = BlockTensor.pack(torch.zeros(rows, cols, device='cuda'))
    z8.value.copy_(torch.arange(256, dtype=torch.uint8).repeat(rows, 1))
    z8.exponent.copy_(torch.tensor(exponents, dtype=torch.uint8)[:, None].expand(rows, cols // 32))
    z = oact.unpack(z8.value.cpu(), z8.exponent.cpu(), cols)
    g8, g = held(rows, cols, 91) if gated else (None, None)
    dy = torch.randn(rows, cols, generator=gen(92))
    want_dz, want_dg, _ = oact.gradients(dy, z, name, g)
    z = z.nan_to_num()    # (for the bounds)
    # beyond 16 every slope is within 2e-6 of 0 or 1, and what is left of it is held to 1e-5 of itself
    error = dy.double().abs() * (1.0 if g is None else g.abs()) * torch.where(z.abs() > 16.0, 1e-6, slope_error(z.clamp(-16.0, 16.0)))
    for bias_dtype in (None, torch.float32):
        dz, dg, db = Activation.backward(dy.cuda(), z8, name, gate=g8, bias_dtype=bias_dtype)
        assert_within(dz, want_dz, allowed(torch.float32, want_dz, error + 2.0**-22 * want_dz.abs()), (name, gated, bias_dtype))
        if gated:
            assert_within(dg, want_dg, allowed(torch.float32, want_dg, dy.double().abs() * z.abs() * 1e-6 + 2.0**-23 * want_dg.abs()), (name, 'dgate'))
        if db is not None:    # (the columns of the two NaN codes and no others; without an activation the slope is 1 whatever z is)
            assert torch.isnan(db).nonzero().flatten().tolist() == ([] if name is None else [127, 255])


@pytest.mark.parametrize('n,m,k,dtype', [(4289, 4096, 4096, torch.bfloat16), (12605, 4304, 1200, torch.float16), (3342, 11000, 1040, torch.float16),
                                         (4400, 4101, 2064, torch.bfloat16)])
def test_fused_product_in_tiles_of_two_sizes(n, m, k, dtype):
    """A little more than whole rounds of large tiles: the last rows go to small ones, with their part of every operand."""
    x, xs = whole_codes(n, k, 101, 1)
    w, ws = whole_codes(m, k, 102, 1)
    z = (x.cuda().double() @ w.cuda().double().t() * 2.0**-10).cpu()
    gate, residual = torch.randn(n, m, generator=gen(103)).to(dtype), torch.randn(n, m, generator=gen(104)).to(dtype)
    got, z8, g8 = Gemm.fp8_gemm_fused(ws, xs, Dtypes.dtype_to_qtype[dtype], activation='silu', gate=gate.cuda(), residual=residual.cuda(),
                                      checkpoint=True)
    y = oact.value(z, 'silu') * gate.double() + residual.double()
    assert_within(got, y, allowed(dtype, y, epilogue_error(z, gate, y, residual)), (n, m, k))
    assert_packed(z8, z.float())
    assert_packed(g8, gate)


def same_blocks(t, rows):
    """Every block of `rows` rows of t holds what the first one does, and the rest the first part of it."""
    whole = t.shape[0] // rows * rows
    blocks = t[:whole].view(-1, rows, *t.shape[1:])
    return bool((blocks == blocks[:1]).all()) and torch.equal(t[whole:], t[:t.shape[0] - whole])


def test_operands_past_4_gib():
    """Offsets of more than 32 bits into x, and then into everything else: blocks of 1024 rows over and over."""
    block, n = 1024, (1 << 20) + 300
    x, xs = whole_codes(block, 4112, 111, 1)
    w, ws = whole_codes(256, 4112, 112, 1)
    long = ScalingTensor(xs.value.repeat(n // block + 1, 1)[:n], xs.meta)
    assert long.value.numel() > 1 << 32
    got = Gemm.fp8_gemm_fused(ws, long, Dtypes.kbfloat16, activation='silu')
    z = x.double() @ w.double().t() * 2.0**-10
    y = oact.value(z, 'silu')
    assert_within(got[:block], y, allowed(torch.bfloat16, y, epilogue_error(z, None, y, None)), 'first block')
    assert same_blocks(got, block)
    del long, got

    m = 4104
    x, xs = whole_codes(block, 64, 113)
    w, ws = whole_codes(m, 64, 114)
    gate = torch.randn(block, m, generator=gen(115)).bfloat16()
    many = gate.cuda().repeat(n // block + 1, 1)[:n]
    long = ScalingTensor(xs.value.repeat(n // block + 1, 1)[:n], xs.meta)
    got, z8, g8 = Gemm.fp8_gemm_fused(ws, long, Dtypes.kbfloat16, activation='silu', gate=many, residual=many, checkpoint=True)
    z = x.double() @ w.double().t() * 2.0**-10
    y = oact.value(z, 'silu') * gate.double() + gate.double()
    assert_within(got[:block], y, allowed(torch.bfloat16, y, epilogue_error(z, gate, y, gate)), 'first block')
    assert same_blocks(got, block)
    for packed, of in ((z8, z.float()), (g8, gate), (BlockTensor.pack(many), gate)):
        codes, exponents = oact.pack(of)
        assert packed.value.numel() > 1 << 32
        assert torch.equal(packed.value[:block].cpu(), codes) and torch.equal(packed.exponent[:block].cpu(), exponents)
        assert same_blocks(packed.value, block) and same_blocks(packed.exponent, block)
    assert same_blocks(g8.to(torch.bfloat16), block)
    want_dz, want_dg, _ = oact.gradients(gate, oact.unpack(*oact.pack(z.float()), m), 'silu', oact.unpack(*oact.pack(gate), m))
    zq, gq = oact.unpack(*oact.pack(z.float()), m), oact.unpack(*oact.pack(gate), m)
    error = gate.double().abs() * gq.abs() * slope_error(zq) + 2.0**-22 * want_dz.abs()
    error_dg = gate.double().abs() * zq.abs() * 1e-6 + 2.0**-23 * want_dg.abs()
    for bias_dtype in (None, torch.float32):
        dz, dg, _ = Activation.backward(many, z8, 'silu', gate=g8, bias_dtype=bias_dtype)
        assert_within(dz[:block], want_dz, allowed(torch.bfloat16, want_dz, error), ('dz', bias_dtype))
        assert_within(dg[:block], want_dg, allowed(torch.bfloat16, want_dg, error_dg), ('dgate', bias_dtype))
        assert same_blocks(dz, block) and same_blocks(dg, block)
        del dz, dg
    meta = ScalingMeta(Dtypes.kfloat8_e5m2, window_size=4)
    dz, _, _ = Activation.backward_cast(many, z8, 'silu', meta, gate=g8, bias_dtype=torch.float32)
    assert abs(float(meta.amax[0]) - float(want_dz.abs().max())) <= 1e-5 * float(want_dz.abs().max())
    assert same_blocks(dz.value, block)


# (few rows in 16-byte accesses and not; paired, small and large tiles; tiles of two sizes; rows that begin anywhere in tiles)
@pytest.mark.parametrize('n,m,k', [(5, 96, 256), (48, 65, 1040), (130, 512, 512), (2048, 1024, 1024), (1024, 1032, 2064), (2304, 8192, 256), (4289, 4096, 4096),
                                   (300, 72, 1040), (2500, 4101, 384), (150, 513, 1040)])
@pytest.mark.parametrize('dtype', DTYPES)
def test_fused_product_in_place_of_its_residual(n, m, k, dtype):
    """The output may be the residual, in every kernel: the same bits as beside it."""
    x, xs = whole_codes(n, k, 121)
    w, ws = whole_codes(m, k, 122)
    gate, residual = torch.randn(n, m, device='cuda').to(dtype), torch.randn(n, m, device='cuda').to(dtype)
    bias, code = torch.randn(m, device='cuda').to(dtype), _backend.activation_code('gelu')
    for g, checkpoint in ((None, False), (gate, True)):
        outs = []
        for in_place in (False, True):
            old = residual.clone()
            z8 = BlockTensor._empty((n, m), old.device) if checkpoint else None
            g8 = BlockTensor._empty((n, m), old.device) if checkpoint else None
            out = _backend.fp8_gemm_fused(ws.value, ws.meta.scale_inv, xs.value, xs.meta.scale_inv, old if in_place else torch.empty_like(old), bias, code, g, old,
                                          (0, 0) if z8 is None else z8._pointers(), (0, 0) if g8 is None else g8._pointers())
            assert (out.data_ptr() == old.data_ptr()) == in_place
            outs.append([out] + ([z8.value, z8.exponent, g8.value, g8.exponent] if checkpoint else []))
        for a, b in zip(*outs):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), (n, m, k, dtype, checkpoint)


def test_operands_on_the_host_are_refused():
    """All of them, before anything is launched: scales, exponents and parts of a meta as well as tensors."""
    x, xs = whole_codes(4, 64, 131)
    w, ws = whole_codes(8, 64, 132)
    host = ScalingTensor(xs.value, ScalingMeta(Dtypes.kfloat8_e4m3, device='cpu'))
    host_codes = ScalingTensor(xs.value.cpu(), xs.meta)
    for a, b in ((ws, host), (host, ws), (ws, host_codes), (host_codes, ws)):
        with pytest.raises(ValueError):
            Gemm.fp8_gemm_fused(a, b, Dtypes.kbfloat16)
    out = Gemm.fp8_gemm_fused(ws, xs, Dtypes.kbfloat16)
    for beside in (dict(bias=out[0].cpu()), dict(gate=out.cpu()), dict(residual=out.cpu())):
        with pytest.raises(ValueError):
            Gemm.fp8_gemm_fused(ws, xs, Dtypes.kbfloat16, **beside)
    z8, z = held(4, 64, 133)
    dy = torch.randn(4, 64, device='cuda')
    with pytest.raises(ValueError):
        BlockTensor(z8.value, z8.exponent.cpu(), (4, 64))
    on_host = BlockTensor(z8.value.cpu(), z8.exponent.cpu(), (4, 64))
    for of, gate in ((on_host, None), (z8, on_host)):
        with pytest.raises(ValueError):
            Activation.backward(dy, of, 'gelu', gate=gate)
    for name in ('scale', 'scale_inv', 'amax', 'amax_counter'):
        meta = ScalingMeta(Dtypes.kfloat8_e5m2, window_size=16)
        setattr(meta, name, getattr(meta, name).cpu())
        with pytest.raises(ValueError):
            Activation.backward_cast(dy, z8, 'gelu', meta)


@pytest.mark.parametrize('name', oact.NAMES)
@pytest.mark.parametrize('gated', [False, True])
def test_gradients_of_values_whose_square_leaves_float32(name, gated):
    """Exponents up to the largest: a slope there is 0 or 1 (the oracle's, in 64 bits, as well), with a bias gradient and without."""
    exponents = [139, 180, 187, 190, 191, 192, 200, 230, 239]
    rows, cols = len(exponents), 256
    codes = (torch.arange(256) & 0xfe).to(torch.uint8)    # (without the two NaN codes)
    value, exponent = codes.repeat(rows, 1).cuda(), torch.tensor(exponents, dtype=torch.uint8)[:, None].expand(rows, cols // 32).contiguous().cuda()
    z8 = BlockTensor(value, exponent, (rows, cols))
    z = oact.unpack(value.cpu(), exponent.cpu(), cols)
    assert bool(torch.isfinite(z).all()) and float(z.abs().max()) < 2.0**121 * 448
    g8, g = held(rows, cols, 141) if gated else (None, None)
    dy = torch.randn(rows, cols, generator=gen(142))
    want_dz, want_dg, _ = oact.gradients(dy, z, name, g)
    error = dy.double().abs() * (1.0 if g is None else g.abs()) * torch.where(z.abs() > 16.0, 1e-6, slope_error(z.clamp(-16.0, 16.0)))
    for bias_dtype in (None, torch.float32):
        dz, dg, db = Activation.backward(dy.cuda(), z8, name, gate=g8, bias_dtype=bias_dtype)
        assert_within(dz, want_dz, allowed(torch.float32, want_dz, error + 2.0**-22 * want_dz.abs()), (name, gated, bias_dtype))
        if gated:
            assert_within(dg, want_dg, allowed(torch.float32, want_dg, dy.double().abs() * z.abs() * 1e-6 + 2.0**-23 * want_dg.abs()), (name, 'dgate'))
        assert db is None or bool(torch.isfinite(db).all())


def test_more_rows_than_a_grid_has():
    """Operands that begin anywhere, past 65535 workgroups of 64 rows: stretches, with their part of every operand."""
    n, m, block = 65535 * 64 + 70, 3, 4096
    x, xs = whole_codes(block, 1, 151)
    w, ws = whole_codes(m, 1, 152)
    codes = xs.value.repeat(n // block + 1, 1)[:n].contiguous()
    gate = torch.randn(block, m, generator=gen(153)).bfloat16()
    many = gate.cuda().repeat(n // block + 1, 1)[:n]
    out, z8, g8 = torch.empty_like(many), BlockTensor._empty((n, m), many.device), BlockTensor._empty((n, m), many.device)
    _backend.fp8_gemm_fused(ws.value, ws.meta.scale_inv, codes, xs.meta.scale_inv, out, None, _backend.activation_code('silu'), many, many, z8._pointers(),
                            g8._pointers())
    z = 0.0 + x.double() @ w.double().t() * 2.0**-10    # (a sum that begins at zero is no negative zero)
    y = oact.value(z, 'silu') * gate.double() + gate.double()
    assert_within(out[:block], y, allowed(torch.bfloat16, y, epilogue_error(z, gate, y, gate)), 'first block')
    for packed, of in ((z8, z.float()), (g8, gate)):
        want, exponents = oact.pack(of)
        assert torch.equal(packed.value[:block].cpu(), want) and torch.equal(packed.exponent[:block].cpu(), exponents)
        assert same_blocks(packed.value, block) and same_blocks(packed.exponent, block)
    assert same_blocks(out, block)


# (few rows in 16-byte accesses and not; paired, small and large tiles, whole and ragged slices of K; tiles of two sizes; rows that begin anywhere in tiles)
@pytest.mark.parametrize('n,m,k', [(1, 1000, 1040), (48, 300, 200), (130, 512, 512), (2048, 1024, 1024), (1024, 1032, 2064), (2304, 8192, 400), (4289, 4096, 2048),
                                   (2500, 4101, 384)])
@pytest.mark.parametrize('dtype', DTYPES)
def test_fused_product_of_sums_that_round(n, m, k, dtype):
    """Codes of every size.  The FP8 matrix instruction itself sums to some 16 bits: 1.5e-5 of a product's norm (measured on random
    operands, whatever K).  Of normal values an error is that of the product's spread, |x| |w| / sqrt(K) of its row and its column, and
    32 times it is allowed to a single output (2^-11), 6 times it to the norm."""
    xs, ws = (ScalingTensor((torch.randn(rows, k, generator=gen(s)) * 60.0).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).cuda(),
                            ScalingMeta(Dtypes.kfloat8_e4m3, scale_inv=torch.tensor(inv, device='cuda')))
              for rows, s, inv in ((n, 161, 0.013), (m, 162, 0.0007)))
    x, w = (t.value.view(torch.float8_e4m3fn).double() * t.meta.scale_inv.double() for t in (xs, ws))
    product = (x @ w.t()).cpu()
    off = 2.0**-11 * (x.norm(dim=1)[:, None] * w.norm(dim=1)[None, :]).cpu() / math.sqrt(k)
    plain = Gemm.fp8_gemm_fused(ws, xs, Dtypes.kfloat32).double().cpu()
    assert float((plain - product).norm()) <= 6 * 1.5e-5 * float(product.norm())
    bias, gate, residual = (torch.randn(shape, generator=gen(s)).to(dtype) for shape, s in (((m, ), 163), ((n, m), 164), ((n, m), 165)))
    z = product + bias.double()
    out, z8, g8 = Gemm.fp8_gemm_fused(ws, xs, Dtypes.dtype_to_qtype[dtype], bias=bias.cuda(), activation='gelu', gate=gate.cuda(), residual=residual.cuda(),
                                      checkpoint=True)
    y = oact.value(z, 'gelu') * gate.double() + residual.double()
    off = off + 2.0**-23 * z.abs()
    # (GELU's slope is at most 1.13)
    assert_within(out, y, allowed(dtype, y, epilogue_error(z, gate, y, residual) + 1.13 * off * gate.double().abs()), (n, m, k, dtype))
    assert_packed(g8, gate)
    block = oact.blocks(z).abs().amax(2).repeat_interleave(32, 1)[:, :m]
    bound = torch.maximum(z.abs() / 16, block / 448 * 2.0**-9) + 2 * off
    assert_within(z8.float(), z, bound, 'checkpoint')


def test_lazily_negated_values_are_read_as_what_they_are():
    """The imaginary part of a conjugate is a view of the original's with a mark that its sign is turned; of a single column nothing
    else tells it from rows that lie apart."""
    for cols in (1, 96):
        c = torch.randn(64, cols, device='cuda', dtype=torch.complex64)
        view, side = c.conj().imag, -torch.view_as_real(c)[..., 1].contiguous()
        assert view.is_neg() and torch.equal(view, side)
        assert_packed(BlockTensor.pack(view), side.cpu())
        z8, z = held(64, cols, 171)
        assert torch.equal(Activation.backward(view, z8, 'silu')[0], Activation.backward(side, z8, 'silu')[0])
        x, xs = whole_codes(64, 256, 172)
        w, ws = whole_codes(cols, 256, 173)
        assert torch.equal(Gemm.fp8_gemm_fused(ws, xs, Dtypes.kfloat32, gate=view, residual=view), Gemm.fp8_gemm_fused(ws, xs, Dtypes.kfloat32, gate=side, residual=side))
