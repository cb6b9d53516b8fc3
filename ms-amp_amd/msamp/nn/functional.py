"""F.linear with ScalingTensor weights: FP8 forward, dgrad and wgrad (msamp/nn/functional.py:16-194)."""

import torch
import torch.nn.functional as F

from msamp import _backend
from msamp.common.dtype import Dtypes
from msamp.common.tensor import BlockTensor, ScalingMeta, ScalingTensor, TypeCast
from msamp.operators.activation import Activation
from msamp.operators.gemm import Gemm
from msamp.nn.state import model_state


# What the library's calls for a whole direction take; everything else goes through the same entry points one by one, with
# their own checks.  (A problem whose tile walks are yet to be timed is one of those.)
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _walk_settled(d_in, d_out, *problem):
    # Only the calls for a direction read codes in padded rows, and they time no walks: a gradient product of a ragged width
    # that waited to be timed waited for ever, and its layer went over transposed copies (forward and backward, bfloat16, us:
    # 8192 x 4096 -> 50257 5911, 4596 so; 8192 x 4100 -> 4096 with a bias 629, 536).  Any walk gives the same bits.
    return d_in % 16 != 0 or d_out % 16 != 0 or _backend.gemm_walk_settled(*problem)


def _casts_in_one_call(x, meta, weight, output_dtype, bias):
    w, w_meta = weight.value, weight.meta
    if not (meta.scaling_mode() == 'gated' and meta.qtype == Dtypes.kfloat8_e4m3 and x.dim() == 2 and x.numel() > 0 and x.is_cuda and
            x.dtype in _FLOATS and output_dtype in _FLOATS and meta.scale.is_cuda):
        return False
    (tokens, d_in), device = x.shape, x.device
    return w.dim() == 2 and w.numel() > 0 and w.shape[1] == d_in and w.dtype in _FLOATS and w.device == device and \
        w.is_contiguous() and w_meta.amax.device == device and 1 <= w_meta.window_size <= w_meta.amax.numel() and \
        (bias is None or (bias.device == device and bias.dtype in _FLOATS and bias.numel() == w.shape[0])) and \
        (d_in % 16 == 0 and w.shape[0] % 16 == 0 or _backend.linear_fits(tokens, d_in, w.shape[0]))


def _forward_in_one_call(x, meta, weight, output_dtype, bias):
    return _casts_in_one_call(x, meta, weight, output_dtype, bias) and \
        _backend.gemm_walk_settled(weight.shape[0], x.shape[0], _backend.linear_pitch(x.shape[1]), False, False)


def _backward_in_one_call(ctx, dy, d_in, need_dgrad):
    meta = ctx.metas['ograd']
    (tokens, d_out), device = dy.shape, dy.device
    # (under create_graph the casts themselves may have to be recorded)
    return not torch.is_grad_enabled() and meta.scaling_mode() == 'gated' and meta.qtype == Dtypes.kfloat8_e5m2 and \
        meta.scale.is_cuda and dy.numel() > 0 and dy.dtype in _FLOATS and ctx.output_dtype in _FLOATS and \
        ctx.input_codes.device == device and (not need_dgrad or _walk_settled(d_in, d_out, d_in, tokens, d_out, True, False))


def _wgrad_in_one_call(ctx, tokens, d_in, d_out):
    meta, old = ctx.metas['wgrad'], ctx.weight.grad
    if model_state.use_fp8_ddp or _backend._shared_device() or meta.scaling_mode() != 'in_time' or \
            meta.qtype != Dtypes.kfloat8_e4m3 or not _backend.gemm_cast_declines(d_in, d_out, tokens):
        return False
    if old is None:
        return _walk_settled(d_in, d_out, d_in, d_out, tokens, True, True)
    # (a product that is added to something is not timed)
    return type(old) is ScalingTensor and old.meta.qtype == Dtypes.kfloat8_e4m3 and old.value.shape == (d_out, d_in) and \
        old.value.device == ctx.input_codes.device and old.value.is_contiguous()


class _FP8GemmFunction(torch.autograd.Function):
    """y = x W^T (+ bias) with x, W in E4M3; dx = dy W and dW = dy^T x with dy in E5M2; fp32 accumulation.

    The reference adds the bias in a separate elementwise pass after the function (nn/functional.py:184-185); here it
    rides in the epilogue of the forward GEMM (fma(acc, scale, bias), one rounding to the output type instead of
    two) and its gradient, the column sums of dy in the output type, is returned from backward as autograd would
    have formed it."""
    @staticmethod
    def forward(ctx, input, weight, metas, dtype_holder, bias=None, differentiable=True):
        ctx.metas = metas
        model_state.check_metas_in_flat(metas)
        output_dtype = dtype_holder.dtype
        ctx.need_input_grad = input.requires_grad
        ctx.weight, ctx.d_in = weight, input.shape[1]
        ctx.output_dtype = output_dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.need_bias_grad = bias is not None and bias.requires_grad
        if bias is not None and not (bias.dtype == output_dtype and bias.is_contiguous()):
            bias = bias.detach().to(output_dtype).contiguous()
        src = input.contiguous()
        meta = metas['input']
        if _forward_in_one_call(src, meta, weight, output_dtype, bias):
            out, ctx.input_codes, ctx.weight_codes, ctx.weight_words = _backend.linear_forward(
                src, meta, weight.value, weight.meta, output_dtype, bias, differentiable
            )
            return out
        input_fp8 = src.cast(Dtypes.kfloat8_e4m3, meta=meta)
        weight_fp8 = weight.cast(Dtypes.kfloat8_e4m3)
        ctx.input_codes, ctx.weight_codes = input_fp8.value, weight_fp8.value
        ctx.weight_words = weight_fp8.meta
        return Gemm.fp8_gemm(weight_fp8, input_fp8, Dtypes.dtype_to_qtype[output_dtype], bias=bias, use_split_accumulator=False)

    @staticmethod
    def _products(ctx, ograd_fp8, ograd_fp8_t, in_place, input_codes, weight_codes, need_dgrad, need_wgrad):
        """The products of the backward pass from the codes of the output gradient: returns the input's gradient (None unless
        need_dgrad) and stores the weight's."""
        metas, words = ctx.metas, ctx.weight_words
        output_qtype = Dtypes.dtype_to_qtype[ctx.output_dtype]
        input_grad = None
        input_fp8 = ScalingTensor(input_codes, metas['input'])
        weight_fp8 = ScalingTensor(weight_codes, words if isinstance(words, ScalingMeta) else
                                   ScalingMeta._of_words(Dtypes.kfloat8_e4m3, words))
        if need_dgrad:
            if in_place:
                input_grad = Gemm.fp8_gemm(weight_fp8, ograd_fp8, output_qtype, use_split_accumulator=True, a_kmajor=True)
            else:
                weight_fp8_t = weight_fp8.fp8_transpose()
                input_grad = Gemm.fp8_gemm(weight_fp8_t, ograd_fp8, output_qtype, use_split_accumulator=True)

        if need_wgrad:
            if in_place:
                mat_a, mat_b, layout = input_fp8, ograd_fp8, dict(a_kmajor=True, b_kmajor=True)
            else:
                mat_a, mat_b, layout = input_fp8.fp8_transpose(), ograd_fp8_t, {}
            wgrad = None
            old_wgrad = None
            if ctx.weight.grad is not None:
                # gradient accumulation: add into the dequantized previous gradient
                old_wgrad = ctx.weight.grad.to(ctx.output_dtype)
            if not model_state.use_fp8_ddp:
                # GEMM and cast without reading the product back, where the kernel takes the problem (same bits as the
                # two steps below)
                wgrad = Gemm.fp8_gemm_cast(
                    mat_a, mat_b, output_qtype, metas['wgrad'], sync=True, accumulate=old_wgrad is not None, out=old_wgrad,
                    **layout
                )
            if wgrad is None:
                if old_wgrad is None:
                    wgrad = Gemm.fp8_gemm(mat_a, mat_b, output_qtype, use_split_accumulator=True, **layout)
                else:
                    wgrad = Gemm.fp8_gemm(
                        mat_a, mat_b, output_qtype, accumulate=True, out=old_wgrad, use_split_accumulator=True, **layout
                    )
                if model_state.use_fp8_ddp:
                    wgrad.meta = metas['wgrad']
                else:
                    wgrad = wgrad.cast(Dtypes.kfloat8_e4m3, meta=metas['wgrad'], sync=True)
            del old_wgrad
            ctx.weight.backward_grad_update(wgrad)
        return input_grad

    @staticmethod
    def backward(ctx, output_grad):
        return _FP8GemmFunction._gradients(ctx, output_grad, ctx.need_bias_grad)

    @staticmethod
    def _gradients(ctx, output_grad, need_bias_grad):
        output_grad = output_grad.contiguous()
        metas = ctx.metas
        tokens, d_out = output_grad.shape
        d_in = ctx.d_in
        input_codes, weight_codes = ctx.input_codes, ctx.weight_codes
        need_dgrad, need_wgrad = ctx.need_input_grad, ctx.weight.requires_grad
        # The reference materializes dy^T, W^T and x^T (fused cast-transpose + two FP8 transposes) because its
        # GEMM reads K-contiguous operands only.  This kernel also reads [K, rows] operands in place, so when
        # the shapes allow, dy is only cast and W, x, dy go to the GEMMs as they are (same results, up to the order of
        # the float32 sum where the weight gradient is taken in parts of K).
        # Codes of widths that are no multiples of 16 come from the forward call in padded rows, which linear_backward reads.
        pitched = input_codes.shape[1] != d_in or weight_codes.shape[0] != d_out
        if pitched and not ((not need_wgrad or _wgrad_in_one_call(ctx, tokens, d_in, d_out)) and
                            _backward_in_one_call(ctx, output_grad, d_in, need_dgrad)):
            pitched = False
            input_codes, weight_codes = input_codes[:, :d_in].contiguous(), weight_codes[:d_out, :d_in].contiguous()
        in_place = pitched or (not need_dgrad or Gemm.kmajor_supported(d_in, tokens, d_out, True, False)) and \
            (not need_wgrad or Gemm.kmajor_supported(d_in, d_out, tokens, True, True))
        if not in_place and (not need_wgrad or _wgrad_in_one_call(ctx, tokens, d_in, d_out)):
            in_place = _backend.linear_takes_short_k(tokens, d_in, d_out) and _backward_in_one_call(ctx, output_grad, d_in, need_dgrad)
        words = ctx.weight_words
        input_grad = bias_grad = None
        column_sums = in_place and need_bias_grad and TypeCast.takes_column_sums(output_grad, metas['ograd'], ctx.bias_dtype)
        if in_place and _backward_in_one_call(ctx, output_grad, d_in, need_dgrad):
            # (a weight gradient that is cast inside its product keeps a call of its own)
            with_wgrad = need_wgrad and _wgrad_in_one_call(ctx, tokens, d_in, d_out)
            payload, input_grad, wgrad, bias_grad = _backend.linear_backward(
                output_grad, d_in, metas['ograd'], input_codes, metas['input'].scale_inv, weight_codes,
                words.scale_inv.data_ptr() if isinstance(words, ScalingMeta) else words.data_ptr() + 4, ctx.output_dtype, need_dgrad,
                metas['wgrad'] if with_wgrad else None, ctx.weight.grad, ctx.bias_dtype if column_sums else None
            )
            if with_wgrad:
                ctx.weight.backward_grad_update(ScalingTensor(wgrad, metas['wgrad']))
                need_wgrad = False
            need_dgrad = False
            ograd_fp8, ograd_fp8_t = ScalingTensor(payload, metas['ograd']), None
        elif column_sums:
            payload, bias_grad = TypeCast.cast_to_fp8_with_column_sums(output_grad, metas['ograd'], ctx.bias_dtype)
            ograd_fp8, ograd_fp8_t = ScalingTensor(payload, metas['ograd']), None
        elif in_place:
            ograd_fp8 = output_grad.cast(Dtypes.kfloat8_e5m2, meta=metas['ograd'])
            ograd_fp8_t = None
        else:
            ograd_fp8, ograd_fp8_t = output_grad.fused_cast_transpose(Dtypes.kfloat8_e5m2, meta=metas['ograd'])

        if need_dgrad or need_wgrad:
            grad = _FP8GemmFunction._products(ctx, ograd_fp8, ograd_fp8_t, in_place, input_codes, weight_codes, need_dgrad, need_wgrad)
            if need_dgrad:
                input_grad = grad

        if need_bias_grad and bias_grad is None:
            bias_grad = output_grad.sum(0).to(ctx.bias_dtype)
        return input_grad, None, None, None, bias_grad, None


class _FP8FusedLinearFunction(torch.autograd.Function):
    """y = act(x W^T + bias) * gate + residual in one product, with the pre-activation and the gate kept in 8 bits for the
    backward pass, which takes the gradients of activation and gate from them on the way to the two products of
    _FP8GemmFunction (not in the reference, whose layers hand 16-bit tensors to element-wise operators that save them)."""
    @staticmethod
    def forward(ctx, input, weight, metas, dtype_holder, bias, activation, gate, residual, differentiable):
        ctx.metas = metas
        model_state.check_metas_in_flat(metas)
        output_dtype = dtype_holder.dtype
        ctx.need_input_grad = input.requires_grad
        ctx.weight, ctx.d_in = weight, input.shape[1]
        ctx.output_dtype = output_dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.need_bias_grad = bias is not None and bias.requires_grad
        ctx.activation = activation
        if bias is not None and not (bias.dtype == output_dtype and bias.is_contiguous()):
            bias = bias.detach().to(output_dtype).contiguous()
        src, meta = input.contiguous(), metas['input']
        z = g = None
        keeps = differentiable and (activation is not None or gate is not None)
        if _casts_in_one_call(src, meta, weight, output_dtype, bias):
            (n, m), device = (src.shape[0], weight.shape[0]), src.device
            gate = None if gate is None else Gemm._beside_output(gate, 'gate', n, m, output_dtype, device.index)
            residual = None if residual is None else Gemm._beside_output(residual, 'residual', n, m, output_dtype, device.index)
            if keeps:
                z = BlockTensor._empty((n, m), device)
                g = None if gate is None else BlockTensor._empty((n, m), device)
            out, input_codes, weight_codes, words = _backend.linear_forward_fused(
                src, meta, weight.value, weight.meta, output_dtype, bias, _backend.activation_code(activation), gate, residual,
                (0, 0) if z is None else z._pointers(), (0, 0) if g is None else g._pointers()
            )
            ctx.weight_meta = None
        else:
            input_fp8, weight_fp8 = src.cast(Dtypes.kfloat8_e4m3, meta=meta), weight.cast(Dtypes.kfloat8_e4m3)
            input_codes, weight_codes, words, ctx.weight_meta = input_fp8.value, weight_fp8.value, None, weight_fp8.meta
            out = Gemm.fp8_gemm_fused(weight_fp8, input_fp8, Dtypes.dtype_to_qtype[output_dtype], bias=bias, activation=activation, gate=gate,
                                      residual=residual, checkpoint=keeps)
            if keeps:
                out, z, g = out
        # (what autograd saves is freed behind the backward pass, attributes live as long as the output does)
        ctx.save_for_backward(input_codes, weight_codes, words, None if z is None else z._buffer, None if g is None else g._buffer)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, output_grad):
        ctx.input_codes, ctx.weight_codes, words, z, gate = ctx.saved_tensors
        ctx.weight_words = ctx.weight_meta if words is None else words
        shape = output_grad.shape
        ctx.z = None if z is None else BlockTensor._empty(shape, None, shape[0], z)
        ctx.gate = None if gate is None else BlockTensor._empty(shape, None, shape[0], gate)
        try:
            return _FP8FusedLinearFunction._gradients(ctx, output_grad)
        finally:
            del ctx.input_codes, ctx.weight_codes, ctx.weight_words, ctx.z, ctx.gate

    @staticmethod
    def _gradients(ctx, output_grad):
        need_gate_grad, need_residual_grad = ctx.needs_input_grad[6], ctx.needs_input_grad[7]
        gate_grad = bias_grad = input_grad = None
        (tokens, d_out), d_in, meta = output_grad.shape, ctx.d_in, ctx.metas['ograd']
        need_dgrad, need_wgrad = ctx.need_input_grad, ctx.weight.requires_grad
        bias_dtype = ctx.bias_dtype if ctx.need_bias_grad else None
        # (codes of widths that are no multiples of 16 lie in padded rows, which linear_backward reads)
        pitched = ctx.input_codes.shape[1] != d_in or ctx.weight_codes.shape[0] != d_out
        casts = ctx.z is not None and output_grad.numel() > 0 and Activation.takes_cast(meta, d_out) and meta.qtype == Dtypes.kfloat8_e5m2
        with_wgrad = casts and need_wgrad and _wgrad_in_one_call(ctx, tokens, d_in, d_out)
        if casts and isinstance(ctx.weight_words, torch.Tensor) and (with_wgrad or not need_wgrad or not pitched) and \
                _backend.linear_fits(tokens, d_in, d_out) and (not need_dgrad or _walk_settled(d_in, d_out, d_in, tokens, d_out, True, False)):
            payload, gate_grad, bias_grad = Activation._backward_codes(
                output_grad, ctx.z, ctx.activation, meta, ctx.gate, bias_dtype, _backend.linear_pitch(d_out)
            )
            _, input_grad, wgrad, _ = _backend.linear_backward(
                output_grad, d_in, meta, ctx.input_codes, ctx.metas['input'].scale_inv, ctx.weight_codes, ctx.weight_words.data_ptr() + 4,
                ctx.output_dtype, need_dgrad, ctx.metas['wgrad'] if with_wgrad else None, ctx.weight.grad, None, codes=payload
            )
            if with_wgrad:
                ctx.weight.backward_grad_update(ScalingTensor(wgrad, ctx.metas['wgrad']))
            elif need_wgrad:    # (one that is cast inside its product keeps a call of its own)
                _FP8GemmFunction._products(ctx, ScalingTensor(payload, meta), None, True, ctx.input_codes, ctx.weight_codes, False, True)
        elif ctx.z is None:
            input_grad, _, _, _, bias_grad, _ = _FP8GemmFunction.backward(ctx, output_grad)
        elif casts and not pitched and (not need_dgrad or Gemm.kmajor_supported(d_in, tokens, d_out, True, False)) and \
                (not need_wgrad or Gemm.kmajor_supported(d_in, d_out, tokens, True, True)):
            ograd_fp8, gate_grad, bias_grad = Activation.backward_cast(output_grad, ctx.z, ctx.activation, meta, gate=ctx.gate, bias_dtype=bias_dtype)
            input_grad = _FP8GemmFunction._products(ctx, ograd_fp8, None, True, ctx.input_codes, ctx.weight_codes, need_dgrad, need_wgrad)
        else:    # a shape whose products want transposed copies, or a meta without a window
            preact_grad, gate_grad, bias_grad = Activation.backward(output_grad, ctx.z, ctx.activation, gate=ctx.gate, bias_dtype=bias_dtype)
            input_grad = _FP8GemmFunction._gradients(ctx, preact_grad, False)[0]
        return input_grad, None, None, None, bias_grad, None, gate_grad if need_gate_grad else None, \
            output_grad if need_residual_grad else None, None


def _output_dtype(input):
    return torch.get_autocast_dtype('cuda') if torch.is_autocast_enabled() else input.dtype


def linear_fused(input, weight, bias=None, activation=None, gate=None, residual=None):
    """act(linear(input, weight, bias)) * gate + residual for a ScalingTensor weight that carries `_scaling_metas`: one FP8 product
    with all of it in its epilogue, rounded once.

    activation: None, 'relu', 'gelu', 'gelu_tanh' or 'silu'.  gate, residual: tensors of the output's shape (converted to its
    type if they are not); a 2-D view whose rows lie apart, such as a half of a wider tensor, is read in place.  Where a gradient is
    recorded and there is an activation or a gate, the pre-activation and the gate are kept in 8 bits (BlockTensor) and nothing in 16.
    The weight is cast on every call; of up to 64 tokens without a gradient the plain layer does not need its codes, and with
    torch's operators behind it takes less (4096 -> 12288, SiLU and a gate, us, here | so: 1 token 46 | 38, 64 52 | 47; 256 57 | 65)."""
    if not isinstance(input, torch.Tensor):
        raise TypeError(f'input should be a torch.Tensor. current type: {type(input)}')
    if not isinstance(weight, ScalingTensor) or not hasattr(weight, '_scaling_metas'):
        raise TypeError(f'weight should be a ScalingTensor with _scaling_metas. current type: {type(weight)}')
    _backend.activation_code(activation)
    output_dtype = _output_dtype(input)
    shape = input.shape[:-1] + (weight.shape[0], )
    beside = []
    for what, tensor in (('gate', gate), ('residual', residual)):
        if tensor is not None:
            if tensor.shape != shape:
                raise ValueError(f'the {what} has shape {tuple(tensor.shape)}, the output {tuple(shape)}.')
            tensor = tensor.to(output_dtype).reshape(-1, shape[-1]) if tensor.dim() != 2 else tensor.to(output_dtype)
        beside.append(tensor)
    model_state.ready_to_scale_tensor = True
    if input.dim() != 2:
        input = input.reshape(-1, input.shape[-1])
    out = _FP8FusedLinearFunction.apply(input, weight, weight._scaling_metas, FunctionalOverider.EMPTY_GRAD_TENSOR.type(output_dtype), bias,
                                        activation, *beside, torch.is_grad_enabled())
    return out if len(shape) == 2 else out.view(shape)


class FunctionalOverider:
    """Replaces torch.nn.functional.linear with a version that routes ScalingTensor weights to FP8."""
    EMPTY_GRAD_TENSOR = torch.nn.Parameter(torch.tensor([]))
    _installed = False

    @classmethod
    def override(cls):
        if cls._installed:
            return
        cls._installed = True
        F.linear = cls._get_wrapper_for_linear(F.linear)

    @classmethod
    def _get_wrapper_for_linear(cls, old_fn):
        def new_fn(input, weight, bias=None):
            """linear(input, weight, bias=None): y = x A^T + b; `weight` may be a ScalingTensor carrying
            `_scaling_metas`, in which case the three GEMMs run in FP8 and the bias, rounded to the output dtype
            (the autocast dtype if autocast is on, else the input's), is added in the forward GEMM's epilogue."""
            if not isinstance(input, torch.Tensor):
                raise TypeError(f'input should be a torch.Tensor. current type: {type(input)}')
            if not isinstance(weight, (torch.Tensor, ScalingTensor)):
                raise TypeError(f'weight should be a torch.Tensor or ScalingTensor. current type: {type(weight)}')
            if bias is not None and not isinstance(bias, torch.Tensor):
                raise TypeError(f'bias should be a torch.Tensor. current type: {type(bias)}')
            if isinstance(weight, torch.Tensor):
                return old_fn(input, weight, bias=bias)
            if not hasattr(weight, '_scaling_metas'):
                raise ValueError('weight (ScalingTensor) should have _scaling_metas attribute.')

            model_state.ready_to_scale_tensor = True
            shape = input.shape
            if len(shape) != 2:
                input = input.reshape(-1, shape[-1])
            output_dtype = _output_dtype(input)
            out = _FP8GemmFunction.apply(input, weight, weight._scaling_metas, cls.EMPTY_GRAD_TENSOR.type(output_dtype), bias,
                                         torch.is_grad_enabled())
            if len(shape) != 2:
                out = out.view(shape[:-1] + (-1, ))
            return out

        return new_fn


FunctionalOverider.override()
