"""saved_in_8_bits: activations that autograd saves for the backward pass, held as BlockTensors (not in the reference)."""

import numbers

import torch
import torch.nn.functional as F
from torch.overrides import TorchFunctionMode

from msamp import _backend
from msamp.common.tensor import BlockTensor

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_ALL = object()    # whatever the operator saves

# The operators whose backward pass has an activation as a factor or takes a bounded slope at it, so that what 8 bits round of it is as
# small in the gradient; which of their arguments (place, name) that is, and the type that autocast gives those ('low': its own,
# 'full': float32).  Everything else that an operator saves is left alone, of these operators and of all others: logarithms and what
# is compared with them (the loss of a classifier, attention's statistics), results that are subtracted from one or from each other, weights.
_FIRST, _BOTH = ((0, 'input'), ), ((0, 'input'), (1, 'other'))
_PRODUCT_OF = {torch.mm: 'mat2', torch.bmm: 'mat2', torch.matmul: 'other'}
_OPERATORS = {
    torch._C._nn.linear: (_FIRST, 'low'),
    torch.conv1d: (_FIRST, 'low'), torch.conv2d: (_FIRST, 'low'), torch.conv3d: (_FIRST, 'low'),
    F.layer_norm: (_FIRST, 'full'), torch.layer_norm: (_FIRST, 'full'), F.group_norm: (_FIRST, 'full'), F.rms_norm: (_FIRST, None),
    torch.rms_norm: (_FIRST, None),
    F.gelu: (_FIRST, None), F.silu: (_FIRST, None), F.mish: (_FIRST, None), F.leaky_relu: (_FIRST, None), F.glu: (_FIRST, None),
    F.relu: (_ALL, None), torch.relu: (_ALL, None), torch.Tensor.relu: (_ALL, None),    # (their result)
    torch.square: (_FIRST, 'full'), torch.Tensor.square: (_FIRST, 'full'),
    torch.pow: (_FIRST, 'full'), torch.Tensor.pow: (_FIRST, 'full'), torch.Tensor.__pow__: (_FIRST, 'full'),    # (to the power of two)
    torch.mul: (_BOTH, None), torch.Tensor.mul: (_BOTH, None), torch.Tensor.__mul__: (_BOTH, None), torch.Tensor.__rmul__: (_BOTH, None),
    torch.addmm: (((1, 'mat1'), (2, 'mat2')), 'low'),
    torch.Tensor.mm: (((0, 'input'), (1, 'mat2')), 'low'), torch.Tensor.bmm: (((0, 'input'), (1, 'mat2')), 'low'),
    torch.Tensor.matmul: (_BOTH, 'low'), torch.Tensor.__matmul__: (_BOTH, 'low'),
    **{f: (((0, 'input'), (1, name)), 'low') for f, name in _PRODUCT_OF.items()},
}
_POWERS = (torch.pow, torch.Tensor.pow, torch.Tensor.__pow__)
# nodes through which a tensor is still the leaf that it came from, in another type or shape
_SAME = tuple(name + 'Backward0' for name in ('ToCopy', 'T', 'Transpose', 'Permute', 'View', 'UnsafeView', 'ReshapeAlias', 'Expand', 'Unsqueeze',
                                              'Squeeze', 'Slice', 'Select', 'AsStrided', 'Clone', 'Alias'))


def _on_gpu(tensor):
    return tensor.is_cuda


def _dense(tensor):
    """A tensor whose values lie in memory of its own: not a sparse or nested one, and no subclass, whose memory need not be what it shows."""
    return type(tensor) in (torch.Tensor, torch.nn.Parameter) and tensor.layout == torch.strided and not tensor.is_nested


def _of_leaf(tensor):
    """A parameter, another leaf that wants a gradient, or either in another type or shape."""
    if isinstance(tensor, torch.nn.Parameter) or isinstance(tensor._base, torch.nn.Parameter):
        return True
    if not tensor.requires_grad or tensor.is_leaf:
        return tensor.requires_grad
    node = tensor.grad_fn
    while node is not None and node.name() in _SAME:
        node = node.next_functions[0][0]
    return node is not None and node.name() == 'torch::autograd::AccumulateGrad'


class _Operators(TorchFunctionMode):
    """Knows, while one of _OPERATORS runs, the memory of the activations among its arguments."""

    def __init__(self):
        super().__init__()
        self.packs = ()    # addresses of storages, or _ALL

    def __torch_function__(self, func, types, args=(), kwargs=None):
        kwargs = kwargs or {}
        rule = _OPERATORS.get(func)
        if rule is None or not torch.is_grad_enabled():
            return func(*args, **kwargs)
        places, autocast = rule
        if func in _POWERS:
            exponent = args[1] if len(args) > 1 else kwargs.get('exponent')
            if not isinstance(exponent, numbers.Number) or exponent != 2:
                return func(*args, **kwargs)
        packs = set()
        if places is _ALL:
            packs = _ALL
        else:
            args, several = list(args), len(places) > 1
            for at, name in places:
                held, key = (args, at) if at < len(args) else (kwargs, name)
                x = args[at] if held is args else kwargs.get(name)
                # (of several factors one without a gradient is a mask, a table or a frozen weight)
                if not isinstance(x, torch.Tensor) or not _dense(x) or not _on_gpu(x) or several and not x.requires_grad or _of_leaf(x):
                    continue
                # Autocast would make a copy of its own, which could not be told from one of a weight.
                if autocast is not None and x.dtype in _FLOATS and torch.is_autocast_enabled(x.device.type):
                    held[key] = x = x.to(torch.float32 if autocast == 'full' else torch.get_autocast_dtype(x.device.type))
                packs.add(x.untyped_storage().data_ptr())
        self.packs = packs
        try:
            return func(*args, **kwargs)
        finally:
            self.packs = ()


class saved_in_8_bits(torch.autograd.graph.saved_tensors_hooks):
    """Context manager under which operators of torch save the activations for their backward pass in 8 bits:

        with msamp.nn.saved_in_8_bits():
            loss = model(x)
        loss.backward()

    An activation is rounded to 8 bits when it is saved and comes back in its own type, so gradients are those of an activation with four
    significant bits.  That is done for the inputs of linear layers, convolutions, matrix products, products, squares, layer, group and
    RMS norms, GELU, SiLU, Mish, GLU and leaky ReLU, and for ReLU's result, where a program calls them on activations.  Left as they are:
    whatever other operators save (attention's inputs and statistics, logarithms, probabilities, a custom autograd function's own), the
    statistics of norms, parameters, views of them and copies in another type (autocast's among them), other leaves that want a gradient,
    factors that want none, sparse and nested tensors and subclasses, and tensors that are not float32, float16 or bfloat16 on the GPU, of
    fewer than min_numel values, or whose last dimension is shorter than a block of 32.  A tensor that several operators save is held
    once for each of them.  What FP8Linear layers keep is in 8 bits already.  (A weight that is computed from others is an activation
    like any other, unless it is a linear layer's or a convolution's.)"""

    def __init__(self, min_numel=1 << 16):
        self._operators = operators = _Operators()

        def pack(tensor):
            packs = operators.packs
            if not packs or not _dense(tensor) or packs is not _ALL and tensor.untyped_storage().data_ptr() not in packs or not _on_gpu(tensor) or \
                    tensor.dtype not in _FLOATS or tensor.numel() < min_numel or tensor.dim() == 0 or not 32 <= tensor.shape[-1] <= _backend.CKPT_COLS:
                # (detached: an operator's result would hold the operator, and so itself.  Autograd takes no note of versions behind hooks.)
                return tensor.detach(), tensor._version
            return BlockTensor.pack(tensor), tensor.dtype

        def unpack(saved):
            held, what = saved
            if not isinstance(held, torch.Tensor):
                return held.to(what)
            if held._version != what:
                raise RuntimeError('a tensor that the backward pass needs has been modified by an in-place operation: its shape is '
                                   f'{tuple(held.shape)}, it is at version {held._version}, expected version {what}.')
            return held

        super().__init__(pack, unpack)

    def __enter__(self):
        super().__enter__()
        self._operators.__enter__()
        return self

    def __exit__(self, *args):
        self._operators.__exit__(*args)
        super().__exit__(*args)
