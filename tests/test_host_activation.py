"""Host side of the operators between two linear layers, without a GPU: argument blocks, constants, checks of arguments, and the
oracle against what torch computes."""

import ctypes
import os
import re

import pytest
import torch

from msamp import _backend
from msamp.common.tensor import BlockTensor
from msamp.operators.activation import Activation
from oracle import activation as oact

HEADER = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include', 'msamp_hip.h')).read()


@pytest.mark.parametrize('name,packer', [('gemm_fused', _backend._GEMM_FUSED), ('activation_backward', _backend._ACTIVATION_BACKWARD)])
def test_argument_blocks_have_the_fields_of_the_header(name, packer):
    body = re.search(r'typedef struct msamp_%s_args \{(.*?)\}' % name, HEADER, re.S).group(1)
    members = [m.strip() for m in re.sub(r'/\*.*?\*/', '', body, flags=re.S).split(';') if m.strip()]
    assert all('*' in m or m.startswith('int64_t ') for m in members)
    assert packer.size == 8 * sum(len(m.split(',')) for m in members)


def test_constants_are_those_of_the_header():
    for name, code in _backend.ACTIVATIONS.items():
        assert int(re.search(r'MSAMP_ACT_%s = (\d+)' % (name or 'none').upper(), HEADER).group(1)) == code
    assert int(re.search(r'#define MSAMP_CKPT_BLOCK (\d+)', HEADER).group(1)) == _backend.CKPT_BLOCK
    assert int(re.search(r'#define MSAMP_FUSED_ROWS (\d+)', HEADER).group(1)) == _backend.FUSED_ROWS
    assert int(re.search(r'#define MSAMP_ACT_CAST_COLS (\d+)', HEADER).group(1)) == _backend.ACT_CAST_COLS
    assert Activation.NAMES == ('relu', 'gelu', 'gelu_tanh', 'silu')


def test_tensors_outside_the_gpu_are_refused():
    with pytest.raises(ValueError):
        BlockTensor.pack(torch.zeros(4, 32))
    packed = BlockTensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), (4, 33))
    assert packed.size() == (4, 33) and packed.size(1) == 33 and packed.numel() == 132 and packed.nbytes == 264 and not packed.is_cuda
    with pytest.raises(ValueError):
        packed.float()
    with pytest.raises(ValueError):
        Activation.backward(torch.zeros(4, 33), packed, 'gelu')
    for bad in ('tanh', 7, ['gelu']):
        with pytest.raises(ValueError):
            _backend.activation_code(bad)
    for shape in ((4, 65), (5, 33), (4, 32, 33)):
        with pytest.raises(ValueError):
            BlockTensor(packed.value, packed.exponent, shape)


@pytest.mark.parametrize('name', oact.NAMES[1:])
def test_oracle_activations_are_torchs(name):
    z = torch.linspace(-9, 9, 1801, dtype=torch.float64, requires_grad=True)
    torch_act = {'relu': torch.relu, 'gelu': torch.nn.functional.gelu, 'silu': torch.nn.functional.silu,
                 'gelu_tanh': lambda t: torch.nn.functional.gelu(t, approximate='tanh')}[name]
    want = torch_act(z)
    want.sum().backward()
    # 1 + tanh and 1 - tanh^2 lose up to 2^-53 and 2^-52, in both formulas, times |z| / 2 <= 4.5 and the inner derivative <= 9.5
    assert torch.allclose(oact.value(z.detach(), name), want.detach(), rtol=1e-12, atol=2 * 4.5 * 2.0**-53)
    assert torch.allclose(oact.slope(z.detach(), name), z.grad, rtol=1e-12, atol=2 * 4.5 * 9.5 * 2.0**-52)


def test_oracle_checkpoint_is_the_nearest_value_of_its_block():
    """Every code is the nearest of all that its block's exponent allows, and no smaller exponent would do."""
    x = torch.randn(40, 100, generator=torch.Generator().manual_seed(7)).double() * torch.logspace(-30, 30, 40, dtype=torch.float64).unsqueeze(1)
    codes, exponents = oact.pack(x.float())
    held = oact.unpack(codes, exponents, 100)
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    table = table[torch.isfinite(table)]
    unit = torch.exp2(exponents.double() - 127).repeat_interleave(32, 1)[:, :100]
    x = x.float().double()
    nearest = (x.unsqueeze(2) - unit.unsqueeze(2) * table).abs().amin(2)
    assert torch.equal((held - x).abs(), nearest)
    top = oact.blocks(x).abs().amax(2)
    assert bool((top <= 448 * torch.exp2(exponents.double() - 127)).all()) and bool((top > 448 * torch.exp2(exponents.double() - 128)).all())


def test_feed_forward_of_plain_layers_is_the_formula():
    from msamp.nn import FeedForward
    torch.manual_seed(0)
    up, gate, down = torch.nn.Linear(8, 24), torch.nn.Linear(8, 24), torch.nn.Linear(24, 8)
    x = torch.randn(5, 8)
    for name, act in (('relu', torch.relu), ('gelu', torch.nn.functional.gelu), ('silu', torch.nn.functional.silu)):
        assert torch.allclose(FeedForward(up, down, activation=name)(x), down(act(up(x))))
        assert torch.allclose(FeedForward(up, down, gate=gate, activation=name)(x, residual=x), down(act(gate(x)) * up(x)) + x)
    assert 'activation=silu' in repr(FeedForward(up, down, activation='silu'))
    with pytest.raises(ValueError):
        FeedForward(up, down, activation='swish')


def test_saved_in_8_bits_leaves_tensors_outside_the_gpu_alone():
    from msamp.nn import saved_in_8_bits
    x = torch.randn(64, 64, requires_grad=True)
    with saved_in_8_bits(min_numel=1):
        y = (x * 2).exp().sum()
    y.backward()
    assert torch.allclose(x.grad, 2 * (2 * x).exp().detach())


ERR_SHAPE = int(re.search(r'MSAMP_ERR_SHAPE = (-?\d+)', HEADER).group(1))


def test_sizes_beyond_the_kernels_are_refused_and_not_cut():
    """Sizes past 31 and 32 bits (the library refuses them before it looks at a pointer), in every call that takes one by value."""
    assert int(re.search(r'#define MSAMP_CKPT_COLS (\w+)', HEADER).group(1), 16) == _backend.CKPT_COLS
    lib, p, size = _backend.load(), 64, ctypes.c_size_t()
    for cols in (_backend.CKPT_COLS + 1, 2**31, 2**32 + 64, 2**40):
        assert lib.msamp_checkpoint_pack(p, _backend.DT_BF16, 1, cols, cols, p, p, None) == ERR_SHAPE
        assert lib.msamp_checkpoint_unpack(p, p, 1, cols, p, _backend.DT_BF16, None) == ERR_SHAPE
        assert lib.msamp_activation_backward_scratch(4, cols, 1, 0, ctypes.addressof(size)) == ERR_SHAPE
        assert lib.msamp_activation_backward_scratch(cols + 2**31, 64, 1, 0, ctypes.addressof(size)) == ERR_SHAPE
        assert lib.msamp_pad_codes(p, 1, p, p, 1, p, cols, None) == ERR_SHAPE
        with pytest.raises(ValueError):
            _backend.checkpoint_empty(1, cols, 'cpu')
        with pytest.raises(ValueError):
            BlockTensor(torch.zeros(1, 32, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.uint8), (1, cols))
        with pytest.raises(ValueError):
            BlockTensor._empty((cols, ), 'cpu')


def test_codes_and_exponents_lie_on_one_device():
    """(The codes alone used to be asked where they are, and kernels were given the address of exponents on the host.)"""
    with pytest.raises(ValueError):
        BlockTensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8, device='meta'), (4, 33))
    with pytest.raises(ValueError):
        BlockTensor(torch.zeros(4, 64, dtype=torch.uint8, device='meta'), torch.zeros(4, 2, dtype=torch.uint8), (4, 33))
