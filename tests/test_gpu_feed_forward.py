"""GPU tests of FP8Linear with an epilogue, of the feed-forward block built from it, and of activations saved in 8 bits."""

import contextlib
import copy

import pytest
import torch
import torch.utils.checkpoint
from torch.nn.attention import SDPBackend, sdpa_kernel

import msamp
from msamp.common.dtype import Dtypes
from msamp.common.tensor import ScalingMeta, TypeCast
from msamp.nn import FeedForward, FP8Linear, LinearReplacer, model_state, saved_in_8_bits
from msamp.nn.functional import linear_fused
from msamp.optim import LBAdamW
from oracle import activation as oact
from tests.gpu_util import rel_fro

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _fresh_state():
    model_state.clear()
    ScalingMeta.in_time_scaling = True
    yield
    model_state.clear()


def fp8_layer(d_in, d_out, dtype, bias=True, seed=0):
    torch.manual_seed(seed)
    linear = torch.nn.Linear(d_in, d_out, bias=bias, device='cuda', dtype=dtype)
    return LinearReplacer.replace(linear)


def codes64(codes, meta_scale_inv, fmt=torch.float8_e4m3fn):
    return codes.cpu().view(fmt).double() * float(meta_scale_inv)


# E4M3 rounds to 2^-4 of a value at most (3.6e-2 / sqrt(3) of it on average), E5M2 to 2^-3 (7.2e-2 / sqrt(3)): a product of two
# rounded operands is within the root of the sum of their squares of the exact one, twice that is allowed for outliers.
E4M3_RMS, E5M2_RMS = 0.036 / 3**0.5 * 1.5, 0.072 / 3**0.5 * 1.5


@pytest.mark.parametrize('tokens,d_in,d_out', [(64, 128, 256), (300, 256, 512), (1, 256, 192), (33, 200, 99), (512, 64, 1040)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
def test_layer_with_an_epilogue_is_the_layer_and_the_operators_behind_it(tokens, d_in, d_out, dtype):
    """Forward and all gradients against 64 bits of the unquantized layer, within what FP8 rounds."""
    for name, gated, residual, bias in (('gelu', False, False, True), ('silu', True, True, False), (None, True, False, True), (None, False, True, True),
                                        ('relu', False, True, True)):
        model_state.clear()
        layer = fp8_layer(d_in, d_out, dtype, bias, seed=tokens)
        x = torch.randn(tokens, d_in, device='cuda', dtype=dtype, requires_grad=True)
        # (a gate that is half of a wider tensor)
        wide = torch.randn(tokens, 2 * d_out, device='cuda', dtype=dtype, requires_grad=True) if gated else None
        r = torch.randn(tokens, d_out, device='cuda', dtype=dtype, requires_grad=True) if residual else None
        dy = torch.randn(tokens, d_out, device='cuda', dtype=dtype) * 1e-2
        y = layer(x, activation=name, gate=wide[:, d_out:] if gated else None, residual=r)
        y.backward(dy)

        x64, w64 = x.detach().double().cpu().requires_grad_(True), (layer.weight.value.double().cpu() * float(layer.weight.meta.scale_inv)).requires_grad_(True)
        b64 = layer.bias.detach().double().cpu().requires_grad_(True) if bias else None
        g64 = wide.detach().double().cpu().requires_grad_(True) if gated else None
        z = x64 @ w64.t() + (b64 if bias else 0.0)
        want = {None: lambda t: t, 'relu': torch.relu, 'gelu': torch.nn.functional.gelu, 'silu': torch.nn.functional.silu}[name](z)
        want = (want * g64[:, d_out:] if gated else want) + (r.detach().double().cpu() if residual else 0.0)
        want.backward(dy.double().cpu())
        what = (tokens, d_in, d_out, dtype, name)
        product = 2 * (2 * E4M3_RMS**2)**0.5
        assert y.dtype == dtype and rel_fro(y, want) < product + 1e-2, what
        # dz: the checkpoints' rounding of z (through act') and of the gate, then E5M2 and the other operand's E4M3.  A sign of z that
        # the product's rounding turns moves ReLU's gradient by all of itself: the share of such z is that rounding over the spread of z.
        grads = 2 * (E5M2_RMS**2 + 3 * E4M3_RMS**2)**0.5 + (product**0.5 if name == 'relu' else product)
        assert x.grad.dtype == dtype and rel_fro(x.grad, x64.grad) < grads, what
        assert rel_fro(layer.weight.grad.float(), w64.grad) < grads + E4M3_RMS, what
        if bias:
            assert layer.bias.grad.dtype == layer.bias.dtype and rel_fro(layer.bias.grad, b64.grad) < grads, what
        if gated:
            assert rel_fro(wide.grad, g64.grad) < grads, what
        if residual:
            assert torch.equal(r.grad, dy)


def test_layer_with_an_epilogue_takes_the_same_casts_as_the_layer():
    """The metas' windows and scales move as those of the plain layer, and the outputs are the plain layer's behind torch's operators
    up to the roundings in between."""
    runs = []
    for fused in (True, False):
        model_state.clear()    # (a program has one model)
        layer = fp8_layer(256, 512, torch.bfloat16, seed=3)
        optimizer = LBAdamW(layer.parameters(), lr=0.0)
        steps = []
        for step in range(20):
            torch.manual_seed(100 + step)
            x = torch.randn(192, 256, device='cuda', dtype=torch.bfloat16)
            dy = torch.randn(192, 512, device='cuda', dtype=torch.bfloat16) * 1e-3
            y = layer(x, activation='silu') if fused else torch.nn.functional.silu(layer(x))
            y.backward(dy)
            metas = layer.scaling_metas
            steps.append([t.detach().clone() for t in (y, metas['input'].amax, metas['input'].scale, metas['ograd'].amax_counter, metas['ograd'].amax)])
            optimizer.step()
            optimizer.zero_grad()
        runs.append(steps)
    for (y, amax, scale, counter, ograd), (y2, amax2, scale2, counter2, ograd2) in zip(*runs):
        # one rounding to bfloat16 (2^-8) against two, and silu's slope of at most 1.1 on the first
        assert float((y.double() - y2.double()).abs().max()) <= 3.2 * 2.0**-8 * float(y2.double().abs().max())
        assert torch.equal(amax, amax2) and torch.equal(scale, scale2) and int(counter) == int(counter2)
        # (the output gradient's maximum: of dy * silu'(z), here with z from 8 bits)
        assert torch.allclose(ograd, ograd2, rtol=0.15)
    assert int(counter) >= 16


def test_layer_with_an_epilogue_accumulates_and_goes_without_gradients():
    layer = fp8_layer(128, 256, torch.bfloat16, seed=5)
    x = torch.randn(4, 40, 128, device='cuda', dtype=torch.bfloat16)
    gate = torch.randn(4, 40, 256, device='cuda', dtype=torch.bfloat16)
    with torch.no_grad():
        a = layer(x, activation='gelu_tanh', gate=gate)
    b = layer(x, activation='gelu_tanh', gate=gate)
    assert a.shape == (4, 40, 256) and torch.equal(a, b) and not a.requires_grad
    b.float().square().mean().backward()
    first = layer.weight.grad.float().clone()
    layer(x, activation='gelu_tanh', gate=gate).float().square().mean().backward()
    assert rel_fro(layer.weight.grad.float(), 2 * first) < 3 * E4M3_RMS
    # autocast: the output takes its type, gate and residual are converted
    with torch.autocast('cuda', dtype=torch.bfloat16):
        y = layer(x.float(), activation='silu', gate=gate.float(), residual=gate.float())
    assert y.dtype == torch.bfloat16
    for bad in (dict(activation='swish'), dict(activation='silu', gate=gate[:1]), dict(residual=gate[..., :8])):
        with pytest.raises(ValueError):
            layer(x, **bad)
    with pytest.raises(TypeError):
        linear_fused(x, torch.randn(256, 128, device='cuda'), activation='silu')


@pytest.mark.parametrize('gated', [False, True])
def test_feed_forward_block_trains_as_its_plain_form_does(gated):
    torch.manual_seed(7)

    def block():
        return FeedForward(torch.nn.Linear(64, 256), torch.nn.Linear(256, 64), gate=torch.nn.Linear(64, 256) if gated else None,
                           activation='silu' if gated else 'gelu')

    plain = block().cuda()
    x = torch.randn(512, 64, device='cuda')
    target = torch.tanh(x @ torch.randn(64, 64, device='cuda') / 4)
    model, optimizer = msamp.initialize(copy.deepcopy(plain), None, opt_level='O2')
    reference = torch.optim.AdamW(plain.parameters(), lr=1e-3, weight_decay=0.01)
    assert isinstance(model.up, FP8Linear) and isinstance(model.down, FP8Linear)
    for group in optimizer.param_groups:
        group['lr'] = 1e-3
    losses = []
    for _ in range(60):
        pair = []
        for m, o in ((model, optimizer), (plain, reference)):
            o.zero_grad()
            loss = (m(x, residual=x) - target).square().mean()
            loss.backward()
            o.step()
            pair.append(float(loss.detach()))
        losses.append(pair)
    # the same course, to the 10 % by which FP8 gradients (5e-2 each, averaged by Adam) may move it
    assert losses[-1][0] < 0.5 * losses[0][0]
    assert abs(losses[0][0] - losses[0][1]) < 0.05 * losses[0][1] and abs(losses[-1][0] - losses[-1][1]) < 0.1 * losses[0][1]


def test_feed_forward_block_replays_from_a_graph():
    torch.manual_seed(9)
    block = LinearReplacer.replace(FeedForward(torch.nn.Linear(128, 512), torch.nn.Linear(512, 128), gate=torch.nn.Linear(128, 512), activation='silu').bfloat16().cuda())
    x = torch.randn(256, 128, device='cuda', dtype=torch.bfloat16)
    dy = torch.randn(256, 128, device='cuda', dtype=torch.bfloat16) * 1e-2

    def step():
        for p in block.parameters():
            p.grad = None
        xx = x.detach().requires_grad_(True)
        y = block(xx, residual=x)
        y.backward(dy)
        return y, xx.grad, block.up.weight.grad.value, block.gate.bias.grad

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step()
    for seed in range(4):
        torch.manual_seed(seed)
        x.copy_(torch.randn(256, 128, device='cuda'))
        with torch.cuda.stream(side):
            eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, eager):
            assert torch.equal(got, want), seed


def test_saved_in_8_bits():
    torch.manual_seed(11)
    norm = torch.nn.LayerNorm(512).cuda()
    linear = torch.nn.Linear(512, 1024).cuda()
    x = torch.randn(4096, 512, device='cuda')

    def loss():
        return torch.nn.functional.gelu(linear(norm(x))).square().mean()

    def grads(packed):
        norm.zero_grad()
        linear.zero_grad()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        if packed:
            with saved_in_8_bits():
                value = loss()
        else:
            value = loss()
        held = torch.cuda.memory_allocated() - before
        value.backward()
        return held, float(value.detach()), [p.grad.clone() for p in (*norm.parameters(), *linear.parameters())]

    held, value, want = grads(False)
    held8, value8, got = grads(True)
    assert value8 == value
    # norm's output and GELU's input and output in 4 bytes against 1.03; norm's input, a leaf without a gradient, is packed as well
    assert held8 < 0.5 * held
    for a, b in zip(got, want):
        assert rel_fro(a, b) < 3 * E4M3_RMS
    # parameters, small tensors and short rows are left alone
    w = torch.nn.Parameter(torch.randn(512, 512, device='cuda'))
    small, short = torch.randn(16, 512, device='cuda'), torch.randn(65536, 8, device='cuda', requires_grad=True)
    with saved_in_8_bits():
        y = small @ w.t()
        z = (short * short).sum()
    y.sum().backward()
    z.backward()
    assert torch.equal(short.grad, 2 * short)
    assert torch.allclose(w.grad, small.sum(0).expand(512, 512), rtol=1e-4, atol=1e-4)


def saved_gradients(f, inputs, packed, autocast=False):
    """(gradients of f, with and without 8 bits, bytes held between forward and backward pass)."""
    for t in inputs:
        t.grad = None
    before = torch.cuda.memory_allocated()
    with saved_in_8_bits() if packed else contextlib.nullcontext():
        with torch.autocast('cuda', dtype=torch.bfloat16) if autocast else contextlib.nullcontext():
            out = f(*inputs)
    held = torch.cuda.memory_allocated() - before
    torch.manual_seed(17)
    (out.float() * torch.randn(out.shape, device='cuda')).sum().backward()
    return [t.grad for t in inputs if t.requires_grad], held


@pytest.mark.parametrize('dtype', [
    torch.bfloat16,
    pytest.param(torch.float32, marks=pytest.mark.skip(reason="torch's fused attention in float32 ended in an illegal memory access here; its cause is not known"))
])
def test_saved_in_8_bits_leaves_attention_alone(dtype):
    """Its logsumexp has the sequence as its last dimension and an error of it lies in an exponent; its other inputs are compared with it."""
    # (never the path of plain products, whose transposed operands are not for the GPU in 16 bits)
    backends = [SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION]
    torch.manual_seed(13)
    q, k, v = (torch.randn(4, 16, 1024, 64, device='cuda', dtype=dtype, requires_grad=True) for _ in range(3))
    attention = lambda q, k, v: torch.nn.functional.scaled_dot_product_attention(q * 1.0, k * 1.0, v * 1.0, is_causal=True)    # noqa: E731
    with sdpa_kernel(backends):
        want, _ = saved_gradients(attention, (q, k, v), False)
        got, _ = saved_gradients(attention, (q, k, v), True)
    for a, b in zip(got, want):    # (the order of its sums may change from run to run: a rounding of the result)
        assert rel_fro(a, b) < 2 * torch.finfo(dtype).eps


def test_saved_in_8_bits_leaves_logarithms_alone():
    """The loss of a classifier: its backward pass exponentiates the logarithms that it saves."""
    torch.manual_seed(14)
    x = torch.randn(512, 32000, device='cuda', requires_grad=True)
    target = torch.randint(0, 32000, (512, ), device='cuda')
    for f in (lambda x: torch.nn.functional.cross_entropy(x * 0.5, target, reduction='none'), lambda x: torch.log_softmax(x * 0.5, -1),
              lambda x: torch.logsumexp(x * 0.5, -1)):
        want, _ = saved_gradients(f, (x, ), False)
        got, _ = saved_gradients(f, (x, ), True)
        assert torch.equal(got[0], want[0])


@pytest.mark.parametrize('frozen', [False, True])
def test_saved_in_8_bits_leaves_weights_alone_under_autocast(frozen):
    torch.manual_seed(15)
    linear, norm = torch.nn.Linear(512, 512).cuda(), torch.nn.LayerNorm(512).cuda()
    linear.weight.requires_grad_(not frozen)
    x = torch.randn(512, 512, device='cuda', requires_grad=True)
    want, held = saved_gradients(lambda x: linear(x * 2.0), (x, ), False, autocast=True)
    whole = None if frozen else linear.weight.grad.clone()
    linear.weight.grad = None
    got, held8 = saved_gradients(lambda x: linear(x * 2.0), (x, ), True, autocast=True)
    assert torch.equal(got[0], want[0])
    if not frozen:    # (and the input is packed)
        assert rel_fro(linear.weight.grad, whole) < 3 * E4M3_RMS and not torch.equal(linear.weight.grad, whole) and held8 < held
    # the rest of what autocast casts: values and types stay as they are
    for f in (lambda x: norm(x.bfloat16() * 2), lambda x: (x.bfloat16() * 2).square(), lambda x: (x.bfloat16() * 2)**2, lambda x: (x * 2) @ linear.weight,
              lambda x: torch.nn.functional.gelu(linear(norm(x * 2))), lambda x: torch.nn.functional.group_norm((x.bfloat16() * 2).view(4, 128, 512), 8)):
        with torch.autocast('cuda', dtype=torch.bfloat16):
            want = f(x)
            with saved_in_8_bits():
                got = f(x)
        assert got.dtype == want.dtype and torch.equal(got, want)


def test_saved_in_8_bits_around_fp8_layers():
    """A block of FP8 layers inside: what they keep themselves does not pass through, what stands beside them does."""
    torch.manual_seed(16)
    block = LinearReplacer.replace(FeedForward(torch.nn.Linear(256, 512), torch.nn.Linear(512, 256)).bfloat16().cuda())
    norm = torch.nn.RMSNorm(256).bfloat16().cuda()
    x = torch.randn(1024, 256, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    want, held = saved_gradients(lambda x: block(norm(x * 2.0), residual=x), (x, ), False)
    got, held8 = saved_gradients(lambda x: block(norm(x * 2.0), residual=x), (x, ), True)
    assert held8 < held and rel_fro(got[0], want[0]) < 3 * E4M3_RMS


@pytest.mark.parametrize('d_in,d_out', [(1024, 4096), (1000, 4000)])
def test_backward_frees_what_the_forward_pass_kept(d_in, d_out):
    """While the output is still referenced, as a training loop's last loss is through the next forward pass."""
    def requested():    # (what is allocated counts the rest of a block that the allocator does not split, up to 1 MiB a tensor)
        return torch.cuda.memory_stats()['requested_bytes.all.current']

    tokens = 2048
    layer = fp8_layer(d_in, d_out, torch.bfloat16)
    x = torch.randn(tokens, d_in, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    gate = torch.randn(tokens, d_out, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn(tokens, d_out, device='cuda', dtype=torch.bfloat16)
    kept = []
    for _ in range(3):    # (the first time brings the gradients and workspaces)
        before = requested()
        y = layer(x, activation='silu', gate=gate)
        after = requested()
        y.backward(dy, retain_graph=True)
        first = x.grad.clone()
        x.grad = None
        y.backward(dy)
        assert torch.equal(x.grad, first)    # (the checkpoints are there for as long as the graph is)
        first = None
        kept.append((after - before, requested() - before))
        with pytest.raises(RuntimeError):
            y.backward(dy)
        x.grad = gate.grad = None
        layer.weight.grad = layer.bias.grad = None
        y_bytes, y = y.numel() * y.element_size(), None
        torch.cuda.synchronize()
    grads = x.numel() * 2 + gate.numel() * 2 + layer.weight.numel() + d_out * 4
    codes = tokens * d_out * 2 * 33 // 32
    held, left = kept[-1]
    assert held > codes and left < y_bytes + grads + (1 << 20)


@pytest.mark.parametrize('tokens,d_in,d_out', [(64, 128, 256), (33, 200, 99), (300, 100, 60), (512, 64, 1040)])
@pytest.mark.parametrize('form', ['no window', 'no window, frozen weight', 'fp8 ddp', 'fp8 ddp, no window'])
def test_backward_of_the_layer_by_its_other_ways(tokens, d_in, d_out, form, monkeypatch):
    """Metas without a window (casts apart from the gradients), operands that the products want transposed, gradients that a data-parallel
    reducer casts: against 64 bits of the unquantized layer, one backward pass behind another."""
    layer = fp8_layer(d_in, d_out, torch.bfloat16, seed=tokens)
    if 'no window' in form:
        for name in ('input', 'ograd'):
            layer.scaling_metas[name].window_size = 1
    if 'frozen' in form:
        layer.weight.requires_grad = False
    model_state.use_fp8_ddp = 'ddp' in form
    taken = []
    take = TypeCast.takes_column_sums
    monkeypatch.setattr(TypeCast, 'takes_column_sums', staticmethod(lambda *args: taken.append(1) or take(*args)))
    x = torch.randn(tokens, d_in, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    gate = torch.randn(tokens, d_out, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn(tokens, d_out, device='cuda', dtype=torch.bfloat16)
    for _ in range(2):
        layer(x, activation='silu', gate=gate).backward(dy)
    assert not taken    # (the bias' gradient is there before)

    x64, g64, b64 = (t.detach().double().cpu().requires_grad_(True) for t in (x, gate, layer.bias))
    w64 = (layer.weight.value.double().cpu() * float(layer.weight.meta.scale_inv)).requires_grad_(True)
    (torch.nn.functional.silu(x64 @ w64.t() + b64) * g64).backward(2 * dy.double().cpu())
    product = 2 * (2 * E4M3_RMS**2)**0.5
    grads = 2 * (E5M2_RMS**2 + 3 * E4M3_RMS**2)**0.5 + product
    assert rel_fro(x.grad, x64.grad) < grads and rel_fro(gate.grad, g64.grad) < grads and rel_fro(layer.bias.grad, b64.grad) < grads
    if 'frozen' in form:
        assert layer.weight.grad is None
    else:
        assert isinstance(layer.weight.grad, torch.Tensor) == ('ddp' in form)
        assert rel_fro(layer.weight.grad.float(), w64.grad) < grads + 2 * E4M3_RMS    # (two casts of it)


@pytest.mark.parametrize('d_in,d_out', [(256, 512), (200, 99)])
def test_layer_with_an_epilogue_under_hooks_of_autograd(d_in, d_out):
    """Activation checkpointing, which runs the forward pass again, and saved tensors that go to the host and back: the same gradients."""
    tokens = 160
    grads = []
    for how in ('plain', 'again', 'host', '8 bits'):
        model_state.clear()
        layer = fp8_layer(d_in, d_out, torch.bfloat16, seed=2)
        torch.manual_seed(3)
        x = torch.randn(tokens, d_in, device='cuda', dtype=torch.bfloat16, requires_grad=True)
        gate = torch.randn(tokens, d_out, device='cuda', dtype=torch.bfloat16, requires_grad=True)
        dy = torch.randn(tokens, d_out, device='cuda', dtype=torch.bfloat16)
        call = lambda x, gate: layer(x, activation='gelu', gate=gate)    # noqa: E731
        if how == 'again':
            y = torch.utils.checkpoint.checkpoint(call, x, gate, use_reentrant=False)
        else:
            with {'plain': contextlib.nullcontext, 'host': torch.autograd.graph.save_on_cpu, '8 bits': lambda: saved_in_8_bits(min_numel=1)}[how]():
                y = call(x, gate)
        y.backward(dy)
        grads.append([y.detach(), x.grad, gate.grad, layer.bias.grad, layer.weight.grad.value])
    for other in grads[1:]:
        for a, b in zip(other, grads[0]):
            assert torch.equal(a, b)
