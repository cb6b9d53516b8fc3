"""What saved_in_8_bits packs and what it leaves alone, without a GPU: with the oracle's rounding in the place of the kernels."""

import contextlib
import math

import pytest
import torch
import torch.nn.functional as F

from msamp.nn import saved, saved_in_8_bits
from oracle import activation as oact


class Rounded:
    """A BlockTensor's part here; `taken` lists what was packed."""
    taken = []

    def __init__(self, x):
        self.x = oact.unpack(*oact.pack(x.detach().reshape(-1, x.shape[-1]).float()), x.shape[-1]).reshape(x.shape)

    @classmethod
    def pack(cls, x):
        cls.taken.append((tuple(x.shape), x.dtype))
        return cls(x)

    def to(self, dtype):
        return self.x.to(dtype)


@pytest.fixture(autouse=True)
def _without_a_gpu(monkeypatch):
    monkeypatch.setattr(saved, '_on_gpu', lambda tensor: True)
    monkeypatch.setattr(saved, 'BlockTensor', Rounded)
    Rounded.taken = []


def rand(*shape, seed=0, dtype=torch.float32, grad=True):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).requires_grad_(grad)


def gradients(f, *inputs, hooks=True, autocast=None):
    """The gradients of sum(f) with respect to `inputs`, which f gets as results of an operator, as a model's activations are."""
    with saved_in_8_bits(min_numel=1) if hooks else contextlib.nullcontext():
        with torch.autocast('cpu', dtype=autocast) if autocast else contextlib.nullcontext():
            out = f(*(x.clone().div(1.0) if not isinstance(x, torch.nn.Parameter) else x for x in inputs))
    weights = rand(*out.shape, seed=99, grad=False)
    return torch.autograd.grad((out.float() * weights).sum(), [x for x in inputs if x.requires_grad])


LEFT_ALONE = {
    'log_softmax': lambda x: F.log_softmax(x, -1),
    'cross_entropy': lambda x: F.cross_entropy(x, torch.arange(x.shape[0]), reduction='none'),
    'softmax': lambda x: torch.softmax(x, -1),
    'logsumexp': lambda x: torch.logsumexp(x, -1),
    'exp': lambda x: torch.exp(x),
    'tanh': lambda x: torch.tanh(x),
    'mse_loss': lambda x: F.mse_loss(x, torch.ones_like(x), reduction='none'),
    'cube': lambda x: x**3,
    'masked': lambda x: x * torch.full_like(x, 1.3),
    'attention': lambda x: F.scaled_dot_product_attention(x[None], x[None], x[None], is_causal=True),
    'std': lambda x: (x - x.mean(-1, keepdim=True)) / x.std(-1, keepdim=True),
}


@pytest.mark.parametrize('name', LEFT_ALONE)
def test_what_must_not_be_rounded_is_left_alone(name):
    x = rand(24, 96, seed=1)
    got, want = gradients(LEFT_ALONE[name], x), gradients(LEFT_ALONE[name], x, hooks=False)
    assert Rounded.taken == [] and torch.equal(got[0], want[0])


PACKED = {
    'linear': lambda x, w: F.linear(x, w),
    'linear_3d': lambda x, w: F.linear(x.view(4, 6, 96), w),
    'matmul': lambda x, w: x @ w.t(),
    'addmm': lambda x, w: torch.addmm(torch.zeros(96), x, w),
    'square': lambda x: x.square(),
    'power': lambda x: x**2,
    'pow': lambda x: torch.pow(x, 2),
    'gelu': lambda x: F.gelu(x),
    'gelu_tanh': lambda x: F.gelu(x, approximate='tanh'),
    'silu': lambda x: F.silu(x),
    'mish': lambda x: F.mish(x),
    'leaky_relu': lambda x: F.leaky_relu(x),
    'relu': lambda x: F.relu(x),
    'relu_method': lambda x: x.relu(),
    'layer_norm': lambda x: F.layer_norm(x, (96, )),
    'rms_norm': lambda x: F.rms_norm(x, (96, )),
    'group_norm': lambda x: F.group_norm(x.view(4, 6, 96), 3),
    'conv': lambda x: F.conv1d(x.view(4, 6, 96), torch.nn.Parameter(rand(8, 6, 3, grad=False))),
    'glu': lambda x: F.glu(x),
}


@pytest.mark.parametrize('name', PACKED)
def test_activations_are_packed(name):
    x, w = rand(24, 96, seed=2), torch.nn.Parameter(rand(96, 96, seed=3, grad=False))
    args = (x, w) if name in ('linear', 'linear_3d', 'matmul', 'addmm') else (x, )
    got, want = gradients(PACKED[name], *args), gradients(PACKED[name], *args, hooks=False)
    assert len(Rounded.taken) == (2 if name == 'rms_norm' else 1)    # (two operators here, one on the GPU)
    assert all(shape[-1] == 96 and math.prod(shape) == x.numel() for shape, _ in Rounded.taken)
    for a, b in zip(got, want):    # four significant bits: 2^-4 of a factor at most; the slopes and the norms bend by as much
        assert float((a - b).norm()) <= 2.0**-4 * 2 * float(b.norm())
    if len(args) == 2:
        assert torch.equal(got[0], want[0])    # the weight came back whole


@pytest.mark.parametrize('frozen', [False, True])
def test_copies_of_weights_that_autocast_makes_are_left_alone(frozen):
    """Of shapes in which a weight, its transpose and an activation cannot be told apart."""
    x = rand(96, 96, seed=4)
    w, b = torch.nn.Parameter(rand(96, 96, seed=5, grad=False), requires_grad=not frozen), torch.nn.Parameter(rand(96, seed=6, grad=False))
    for f in (lambda x: F.linear(x, w, b), lambda x: F.linear(x, w), lambda x: x @ w, lambda x: x @ w.t(), lambda x: torch.mm(x, w)):
        Rounded.taken = []
        got, want = gradients(f, x, autocast=torch.bfloat16), gradients(f, x, hooks=False, autocast=torch.bfloat16)
        assert torch.equal(got[0], want[0])
        assert Rounded.taken == ([] if frozen else [((96, 96), torch.bfloat16)])


def test_copies_of_parameters_are_left_alone():
    x, gamma = rand(96, 96, seed=7, dtype=torch.bfloat16), torch.nn.Parameter(rand(96, 96, seed=8, grad=False))
    for copy in (lambda: gamma.bfloat16(), lambda: gamma.t().bfloat16(), lambda: gamma.bfloat16().view(96, 96).t(), lambda: gamma.detach().bfloat16(),
                 lambda: gamma[:, :]):
        Rounded.taken = []
        got, want = gradients(lambda x: x * copy(), x), gradients(lambda x: x * copy(), x, hooks=False)
        assert torch.equal(got[0], want[0])
        assert len(Rounded.taken) == (1 if copy().requires_grad else 0)    # (x, for the parameter's gradient)


def test_small_tensors_and_short_rows_are_left_alone():
    for shape, taken in (((1024, 64), 1), ((1023, 64), 0), ((4096, 31), 0), ((65536, ), 1)):
        Rounded.taken = []
        with saved_in_8_bits():
            y = F.gelu(rand(*shape) * 2)
        assert len(Rounded.taken) == taken, shape
        y.sum().backward()


def test_contexts_nest_and_end():
    x = rand(96, 96)
    with saved_in_8_bits(min_numel=1):
        with saved_in_8_bits(min_numel=1 << 20):
            F.gelu(x * 2)
        assert Rounded.taken == []
        F.gelu(x * 2)
        assert len(Rounded.taken) == 1
        with torch.no_grad():
            F.gelu(x * 2)
    F.gelu(x * 2)
    assert len(Rounded.taken) == 1


def test_results_that_are_left_alone_are_freed_with_their_graph():
    class Sentinel:
        freed = 0

        def __del__(self):
            Sentinel.freed += 1

    x = rand(96, 96)
    for hooks in (contextlib.nullcontext(), saved_in_8_bits(), saved_in_8_bits(min_numel=1)):
        before = Sentinel.freed
        with hooks:
            y = torch.exp(x * 1.0)    # (saves its result)
        y.grad_fn.metadata['sentinel'] = Sentinel()
        del y
        assert Sentinel.freed == before + 1


def test_gradients_of_gradients_pass_through_what_is_left_alone():
    x, w = rand(8, 16, seed=21), torch.nn.Parameter(rand(16, 16, seed=22, grad=False))

    def second():
        first, = torch.autograd.grad((torch.exp(x @ w) * x).sum(), x, create_graph=True)
        return torch.autograd.grad(first.square().sum(), (x, w))

    want = second()
    with saved_in_8_bits():
        got = second()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_changes_in_place_are_noticed():
    """Of what is left alone, as without the context; what was packed is what it was when it was saved."""
    for hooks in (contextlib.nullcontext(), saved_in_8_bits(), saved_in_8_bits(min_numel=1)):
        x, mask = rand(96, 96), torch.ones(96, 96)
        with hooks:
            y = x * 1.0 * mask
        mask.add_(1.0)
        with pytest.raises(RuntimeError, match='in-?place'):
            y.sum().backward()
        w = torch.nn.Parameter(rand(96, 96, grad=False))
        with hooks:
            y = F.linear(x * 1.0, w)
        with torch.no_grad():
            w.add_(1.0)    # (an optimizer's step between the forward and the backward pass)
        with pytest.raises(RuntimeError, match='in-?place'):
            y.sum().backward()
    x = rand(96, 96)
    with saved_in_8_bits(min_numel=1):
        h = x * 2.0
        y = F.gelu(h)
    want, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    h.detach().zero_()
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], want)


class Other(torch.Tensor):
    """A subclass, whose memory need not be what it shows."""


def test_other_kinds_of_tensors_are_left_alone():
    x, w = rand(96, 96, seed=31, grad=False).relu(), rand(96, 96, seed=32)
    sparse = x.to_sparse().requires_grad_(True)
    for f in (lambda: torch.mm(sparse * 1.0, w * 1.0).sum(), lambda: (torch.sparse.mm(sparse, w * 1.0) * 2.0).sum(),
              lambda: torch.relu(torch.nested.nested_tensor([w[:3], w[3:7]], requires_grad=True)).to_padded_tensor(0.0).sum(),
              lambda: F.gelu((w * 1.0).as_subclass(Other)).sum()):
        w.grad = None
        f().backward()
        want, w.grad = w.grad, None
        Rounded.taken = []
        with saved_in_8_bits(min_numel=1):
            loss = f()
        loss.backward()
        assert all(shape == (96, 96) for shape, _ in Rounded.taken)
        assert (w.grad is None) == (want is None) and (want is None or bool(Rounded.taken) or torch.equal(w.grad, want))
