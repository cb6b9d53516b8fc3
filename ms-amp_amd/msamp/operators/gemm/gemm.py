"""Gemm.fp8_gemm (msamp/operators/gemm/gemm.py:58-179) on the gfx950 FP8 MFMA kernel."""

import torch
import torch.nn.functional as F

from msamp import _backend
from msamp.common.dtype import Dtypes
from msamp.common.tensor import BlockTensor, ScalingTensor


class Gemm:
    """FP8 GEMM entry point."""
    _te_base = 16
    _FLOATS = {int(qtype): dtype for dtype, qtype in Dtypes.dtype_to_qtype.items() if dtype.is_floating_point}

    @staticmethod
    def _round2times(value, base):
        """Smallest multiple of base that is >= value."""
        return (value + base - 1) // base * base

    @staticmethod
    def _aligned(payload):
        """The kernels fetch operands 16 bytes at a time.  A payload that starts elsewhere (a view into a flat buffer
        at an odd offset) is copied to a fresh allocation first, as the reference pads and copies what its library
        cannot take (msamp/operators/gemm/gemm.py:107-121)."""
        return payload if payload.data_ptr() % 16 == 0 else payload.clone()

    @classmethod
    def kmajor_supported(cls, m, n, k, a_kmajor=True, b_kmajor=False):
        """True if fp8_gemm reads K-major operands of this problem in place (else it transposes them first)."""
        return _backend.gemm_kmajor_supported(m, n, k, a_kmajor, b_kmajor)

    @classmethod
    @torch.no_grad()
    def fp8_gemm_cast(cls, mat_a, mat_b, out_qtype, meta, sync=False, a_kmajor=False, b_kmajor=False, accumulate=False,
                      out=None):
        """fp8_gemm(mat_a, mat_b, out_qtype, accumulate=accumulate, out=out).cast(meta.qtype, meta=meta, sync=sync) for a
        meta with in-time scaling, without reading the product back (not in the reference, which takes the two steps:
        nn/functional.py:100-123).  Small products take one launch and are never stored; larger ones are stored in
        `out` (a scratch tensor if not given) next to the codes for the scale the meta holds, and are read again only
        when the scale rule moves the scale.  Returns the FP8 ScalingTensor, or None if the kernel does not take this
        problem -- the caller then takes the two steps itself; the result is the same bit for bit."""
        assert isinstance(mat_a, ScalingTensor) and isinstance(mat_b, ScalingTensor)
        assert mat_a.is_cuda and mat_a.is_contiguous() and mat_b.is_cuda and mat_b.is_contiguous()
        assert Dtypes.is_fp8_qtype(mat_a.qtype) and Dtypes.is_fp8_qtype(mat_b.qtype) and Dtypes.is_fp8_qtype(meta.qtype)
        if meta.scaling_mode() != 'in_time' or (a_kmajor != b_kmajor):
            return None
        out_dtype = Dtypes.get_dtype_from_qtype(out_qtype)
        if out is not None:
            assert out.is_cuda and out.is_contiguous() and out.dtype == out_dtype
        else:
            assert not accumulate, 'accumulate needs an output tensor'
        payload = _backend.fp8_gemm_cast(
            cls._aligned(mat_a.value), int(mat_a.qtype), mat_a.meta.scale_inv, cls._aligned(mat_b.value), int(mat_b.qtype),
            mat_b.meta.scale_inv, out_dtype, int(meta.qtype), meta.scale, meta.amax[0:1], meta.scale_inv,
            nan_to_inf=sync, a_kmajor=a_kmajor, b_kmajor=b_kmajor, hp_out=out, accumulate=accumulate
        )
        return None if payload is None else ScalingTensor(payload, meta)

    @classmethod
    @torch.no_grad()
    def fp8_gemm(
        cls, mat_a, mat_b, out_qtype, bias=None, accumulate=False, out=None, use_split_accumulator=False, a_kmajor=False,
        b_kmajor=False
    ):
        """out[N, M] = (mat_b[N, K] @ mat_a[M, K].T) * a.scale_inv * b.scale_inv.

        mat_a, mat_b: contiguous FP8 ScalingTensors on the GPU.  The kernel accumulates in fp32
        over the full K (use_split_accumulator has nothing to switch) and writes out_qtype; with
        `accumulate` it adds into `out`.  Only K needs padding (to a multiple of 16 bytes, with
        FP8 zeros); ragged M and N are handled inside the kernel.

        a_kmajor / b_kmajor (not in the reference): the tensor passed is the transpose of the operand,
        [K, M] / [K, N], as the backward pass of a linear layer has them; the kernel reads it in place
        when the shape allows, otherwise it is transposed first.  Same result either way, except that with both
        K-major and an output of a few tiles the float32 sum may be taken in parts of K (msamp_fp8_gemm_ksplit):
        another order of the same sum, which depends on the sizes and the device only.
        """
        assert isinstance(mat_a, ScalingTensor)
        assert isinstance(mat_b, ScalingTensor)
        assert mat_a.is_cuda and mat_a.is_contiguous()
        assert mat_b.is_cuda and mat_b.is_contiguous()
        assert Dtypes.is_fp8_qtype(mat_a.qtype) and Dtypes.is_fp8_qtype(mat_b.qtype)

        if a_kmajor or b_kmajor:
            K, M = mat_a.shape if a_kmajor else mat_a.shape[::-1]
            N = mat_b.shape[1] if b_kmajor else mat_b.shape[0]
            if cls.kmajor_supported(M, N, K, a_kmajor, b_kmajor):
                out_dtype = Dtypes.get_dtype_from_qtype(out_qtype)
                if out is None:
                    assert not accumulate, 'accumulate needs an output tensor'
                    out = torch.empty(N, M, dtype=out_dtype, device=mat_a.device)
                else:
                    assert out.is_cuda and out.is_contiguous() and out.dtype == out_dtype
                operands = (
                    cls._aligned(mat_a.value), int(mat_a.qtype), mat_a.meta.scale_inv, cls._aligned(mat_b.value),
                    int(mat_b.qtype), mat_b.meta.scale_inv, out, accumulate
                )
                if not (a_kmajor and b_kmajor and bias is None and _backend.fp8_gemm_ksplit(*operands)):
                    _backend.fp8_gemm(*operands, bias, a_kmajor=a_kmajor, b_kmajor=b_kmajor)
                return out
            if a_kmajor:
                mat_a = mat_a.fp8_transpose()
            if b_kmajor:
                mat_b = mat_b.fp8_transpose()

        M, K = mat_a.shape
        N = len(mat_b)
        a, b = cls._aligned(mat_a.value), cls._aligned(mat_b.value)
        pK = cls._round2times(K, cls._te_base) - K
        if pK > 0:
            a = F.pad(a, (0, pK))
            b = F.pad(b, (0, pK))
        out_dtype = Dtypes.get_dtype_from_qtype(out_qtype)
        if out is None:
            assert not accumulate, 'accumulate needs an output tensor'
            out = torch.empty(N, M, dtype=out_dtype, device=a.device)
        else:
            assert out.is_cuda and out.is_contiguous() and out.dtype == out_dtype
        _backend.fp8_gemm(
            a, int(mat_a.qtype), mat_a.meta.scale_inv, b, int(mat_b.qtype), mat_b.meta.scale_inv, out, accumulate, bias
        )
        return out

    @staticmethod
    def _beside_output(tensor, what, n, m, dtype, gpu):
        """A gate or residual as the kernel takes it: [N, M] in the output's type, its rows contiguous, any distance apart."""
        if tensor.shape != (n, m):
            raise ValueError(f'the {what} has shape {tuple(tensor.shape)}, the output ({n}, {m}).')
        if tensor.dtype != dtype:
            raise TypeError(f'the {what} is {tensor.dtype}, the output {dtype}.')
        if tensor.get_device() != gpu:
            raise ValueError(f'The {what} is on {tensor.device}, the operands on cuda:{gpu}.')
        return tensor if tensor.stride(1) == 1 and (n == 1 or tensor.stride(0) >= m) else tensor.contiguous()

    @classmethod
    def fp8_gemm_fused(cls, mat_a, mat_b, out_qtype, bias=None, activation=None, gate=None, residual=None, checkpoint=False):
        """out[N, M] = act(z) * gate + residual with z = (mat_b[N, K] @ mat_a[M, K].T) * a.scale_inv * b.scale_inv + bias (not in
        the reference, whose layers return z and leave the rest to element-wise operators).

        mat_a, mat_b: contiguous E4M3 ScalingTensors on the GPU, a weight and its input.  All of it is float32 from the product on
        and rounded once, to out_qtype (kfloat32, kfloat16 or kbfloat16).
        bias: [M], any of these types.  activation: None, 'relu', 'gelu', 'gelu_tanh' or 'silu'.  gate, residual: [N, M] in the
        output's type; their rows may lie apart (a half of a wider tensor).
        Of what a float32 output shows: the FP8 matrix instruction sums its products to some 16 bits (1.5e-5 of a product's norm, whatever
        K), and GELU is held to an absolute 4e-7, so its far negative side has no relative accuracy.
        With `checkpoint` the call returns (out, z8, gate8): BlockTensors with the 8-bit checkpoints of z and of the gate (None
        without one), written on the way, from which Activation.backward takes the gradients.  Not recorded by autograd."""
        if not (isinstance(mat_a, ScalingTensor) and isinstance(mat_b, ScalingTensor)):
            raise TypeError('the operands should be ScalingTensors.')
        a, b, a_meta, b_meta = mat_a.value, mat_b.value, mat_a.meta, mat_b.meta
        if int(a_meta.qtype) != _backend.DT_E4M3 or int(b_meta.qtype) != _backend.DT_E4M3:
            raise TypeError('the operands should be in e4m3 format.')
        if a.dim() != 2 or b.dim() != 2:
            raise ValueError(f'the operands should be 2-D, not {tuple(a.shape)} and {tuple(b.shape)}.')
        (m, k), (n, b_k), device = a.shape, b.shape, a.device
        if k != b_k or k == 0:
            raise ValueError(f'shape mismatch: mat_a {tuple(a.shape)}, mat_b {tuple(b.shape)}.')
        gpu = a.get_device()    # (-1 in host memory; a number is compared in half the time of a device)
        if gpu < 0 or not (a.is_contiguous() and b.is_contiguous()):
            raise ValueError('The operands are not in cuda memory or contiguous.')
        if b.get_device() != gpu or a_meta.scale_inv.get_device() != gpu or b_meta.scale_inv.get_device() != gpu:
            raise ValueError('The operands and their reciprocal scales are not all on one device.')
        code = _backend.activation_code(activation)
        dtype = cls._FLOATS.get(int(out_qtype))
        if dtype is None:
            raise TypeError(f'the output should be float32, float16 or bfloat16, not {out_qtype}.')
        if bias is not None and not (bias.get_device() == gpu and bias.is_contiguous() and bias.numel() == m):
            raise ValueError(f'The bias is not on cuda:{gpu}, not contiguous or not of {m} values.')
        if gate is not None:
            gate = cls._beside_output(gate, 'gate', n, m, dtype, gpu)
        if residual is not None:
            residual = cls._beside_output(residual, 'residual', n, m, dtype, gpu)
        out = torch.empty((n, m), dtype=dtype, device=device)
        z = g = None
        if checkpoint:
            z = BlockTensor._empty((n, m), device)
            g = None if gate is None else BlockTensor._empty((n, m), device)
        if n > 0 and m > 0:
            if n > _backend.FUSED_ROWS:
                if k % cls._te_base == 0:
                    a, b = cls._aligned(a), cls._aligned(b)
                elif (pitch := _backend.fp8_gemm_fused_pitch(m, n, k, device.index)) != k:
                    a, b = _backend.pad_codes(a, b, pitch)
            _backend.fp8_gemm_fused(a, a_meta.scale_inv, b, b_meta.scale_inv, out, bias, code, gate, residual,
                                    (0, 0) if z is None else z._pointers(), (0, 0) if g is None else g._pointers())
        return (out, z, g) if checkpoint else out
