"""Activation.backward: the gradients of act(z) * gate from 8-bit checkpoints of z and of the gate (not in the reference,
which leaves activations to torch and keeps their inputs in 16 or 32 bits)."""

import torch

from msamp import _backend
from msamp.common.dtype import Dtypes
from msamp.common.tensor import BlockTensor, ScalingTensor

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


class Activation:
    """Gradients of y = act(z) * gate, the activations being those of Gemm.fp8_gemm_fused."""
    NAMES = tuple(name for name in _backend.ACTIVATIONS if name is not None)

    @staticmethod
    def _checked(output_grad, z, gate, bias_dtype):
        if not isinstance(z, BlockTensor) or not (gate is None or isinstance(gate, BlockTensor)):
            raise TypeError('z and the gate should be BlockTensors.')
        gpu = output_grad.get_device()    # (-1 in host memory)
        if gpu < 0 or z._codes.get_device() != gpu or gate is not None and gate._codes.get_device() != gpu:
            raise ValueError('The output gradient and the checkpoints are not all on one GPU.')
        if output_grad.dtype not in _FLOATS or bias_dtype not in _FLOATS + (None, ):
            raise TypeError(f'unsupported types: output gradient {output_grad.dtype}, bias gradient {bias_dtype}.')
        if output_grad.shape != z.shape or gate is not None and gate.shape != z.shape:
            raise ValueError(f'shape mismatch: output gradient {tuple(output_grad.shape)}, z {tuple(z.shape)}' +
                             ('.' if gate is None else f', gate {tuple(gate.shape)}.'))
        if output_grad.dim() == 0:
            raise ValueError('The output gradient has no dimension.')
        dy = output_grad
        cols = dy.shape[-1]
        if dy.numel() and dy.dim() != 2:
            dy = dy.detach().reshape(-1, cols)
        if dy.numel() and (cols > 1 and dy.stride(1) != 1 or dy.shape[0] > 1 and dy.stride(0) < cols or dy.is_neg()):
            dy = dy.detach().resolve_neg().contiguous()
        return dy

    @classmethod
    def backward(cls, output_grad, z, activation, gate=None, bias_dtype=None):
        """(dz, dgate, dbias): dz = output_grad * gate * act'(z) and dgate = output_grad * act(z) in output_grad's type, dgate
        None without a gate; dbias the sum of dz over all but the last dimension, in float32 and rounded to bias_dtype, None if
        that is None.

        z, gate: the BlockTensors of the forward pass, gate None where there was none.  activation: as in
        Gemm.fp8_gemm_fused.  output_grad: float32 / float16 / bfloat16 of z's shape; rows may lie apart."""
        code = _backend.activation_code(activation)
        dy = cls._checked(output_grad, z, gate, bias_dtype)
        if dy.numel() == 0:
            return torch.empty_like(dy), None if gate is None else torch.empty_like(dy), \
                None if bias_dtype is None else dy.new_zeros(dy.shape[-1], dtype=bias_dtype)
        dz, dgate, sums = _backend.activation_backward(
            dy, z._pointers(), None if gate is None else gate._pointers(), code, bias_dtype
        )
        if output_grad.dim() != 2:
            dz, dgate = dz.view(output_grad.shape), None if dgate is None else dgate.view(output_grad.shape)
        return dz, dgate, sums

    @staticmethod
    def takes_cast(meta, cols):
        """True if backward_cast takes an output gradient of `cols` columns with this meta."""
        return Dtypes.is_fp8_qtype(meta.qtype) and meta.scaling_mode() == 'gated' and 0 < cols <= _backend.ACT_CAST_COLS and \
            meta.scale.is_cuda and meta.scale_inv.is_cuda and meta.amax.is_cuda

    @classmethod
    def backward_cast(cls, output_grad, z, activation, meta, gate=None, bias_dtype=None):
        """backward with dz cast on to FP8 with `meta` as TypeCast.cast_to_fp8 casts with it (the warm-up test is taken on the
        device), from float32 and without dz in between: returns (ScalingTensor, dgate, dbias).  For metas with a window, on the GPU
        (takes_cast); output_grad is 2-D and not empty."""
        payload, dgate, sums = cls._backward_codes(output_grad, z, activation, meta, gate, bias_dtype)
        return ScalingTensor(payload, meta), dgate, sums

    @classmethod
    def _backward_codes(cls, output_grad, z, activation, meta, gate, bias_dtype, pitch=None):
        """backward_cast's payload, in rows of `pitch`, and the rest."""
        code = _backend.activation_code(activation)
        dy = cls._checked(output_grad, z, gate, bias_dtype)
        if output_grad.dim() != 2 or dy.numel() == 0:
            raise ValueError(f'The output gradient should be 2-D and not empty, not {tuple(output_grad.shape)}.')
        if not cls.takes_cast(meta, dy.shape[1]):
            raise ValueError('The meta should be of an FP8 type, with a window and on the GPU, and the gradient not too wide.')
        return _backend.activation_backward(
            dy, z._pointers(), None if gate is None else gate._pointers(), code, bias_dtype, meta, pitch
        )
