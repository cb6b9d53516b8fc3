"""BlockTensor: an activation held in 8 bits, with a power of two for every 32 neighbouring values of a row (not in the
reference, which keeps activations in the type they were computed in)."""

import torch

from msamp import _backend


class BlockTensor:
    """`value`: uint8 E4M3 codes in rows of the last dimension rounded up to 32; `exponent`: a byte E + 127 for every 32 of them.
    A code stands for its value times 2^E.  E is the smallest exponent with which no finite value of the block is beyond the
    format's 448, so values near the block's largest keep four significant bits and those more than 2^15 below it vanish; NaN and
    the infinities come back as NaN.  1.03 bytes a value, for tensors that a backward pass needs again and that no scale of a
    whole tensor fits.  `shape` is the shape of the tensor that was packed."""

    def __init__(self, value, exponent, shape):
        shape = torch.Size(shape)
        rows, cols = (shape[:-1].numel(), shape[-1]) if shape else (1, 1)
        blocks = (cols + _backend.CKPT_BLOCK - 1) // _backend.CKPT_BLOCK
        if value.dtype != torch.uint8 or exponent.dtype != torch.uint8:
            raise TypeError(f'codes and exponents should be torch.uint8, not {value.dtype} and {exponent.dtype}.')
        if cols > _backend.CKPT_COLS:
            raise ValueError(f'a checkpoint has at most {_backend.CKPT_COLS} columns, not {cols}.')
        if tuple(value.shape) != (rows, blocks * _backend.CKPT_BLOCK) or tuple(exponent.shape) != (rows, blocks):
            raise ValueError(f'codes {tuple(value.shape)} and exponents {tuple(exponent.shape)} do not hold a tensor of shape {tuple(shape)}.')
        if not (value.is_contiguous() and exponent.is_contiguous()):
            raise ValueError('The codes or the exponents are not contiguous.')
        if value.device != exponent.device:
            raise ValueError(f'The codes are on {value.device}, the exponents on {exponent.device}.')
        self._value, self._exponent, self._buffer = value, exponent, None
        self.shape, self._rows, self._cols = shape, rows, cols

    @classmethod
    def _empty(cls, shape, device, rows=None, buffer=None):
        """A BlockTensor whose codes and exponents hold nothing yet, in one allocation."""
        self = cls.__new__(cls)
        self.shape = torch.Size(shape)
        self._cols = self.shape[-1] if self.shape else 1
        self._rows = rows if rows is not None else self.shape[0] if len(self.shape) == 2 else self.shape[:-1].numel()
        self._buffer = buffer if buffer is not None else _backend.checkpoint_empty(self._rows, self._cols, device)
        self._value = self._exponent = None
        return self

    @classmethod
    def pack(cls, tensor):
        """Round a float32 / float16 / bfloat16 tensor on the GPU to 8 bits.  Rows may lie apart; any other order of the
        values in memory is copied first."""
        if not isinstance(tensor, torch.Tensor):
            raise TypeError(f'input should be a torch.Tensor. current type: {type(tensor)}')
        rows, shape = tensor, tensor.shape
        if len(shape) != 2:
            cols = shape[-1] if shape else 1
            rows = tensor.detach()
            rows = rows.reshape(-1, cols) if tensor.numel() else rows.new_empty(shape[:-1].numel(), cols)
        n, cols = rows.shape
        if cols > 1 and rows.stride(1) != 1 or n > 1 and rows.stride(0) < cols or rows.is_neg():
            rows = rows.detach().resolve_neg().contiguous()
        return cls._empty(shape, rows.device, n, _backend.checkpoint_pack(rows))

    def _pointers(self):
        """Addresses of the codes and of the exponents."""
        if self._buffer is not None:
            return _backend.checkpoint_pointers(self._buffer, self._rows, self._cols)
        return self._value.data_ptr(), self._exponent.data_ptr()

    @property
    def value(self):
        if self._value is None:
            pitch = _backend.checkpoint_pitch(self._cols)
            self._value = self._buffer[:self._rows * pitch].view(self._rows, pitch)
        return self._value

    @property
    def exponent(self):
        if self._exponent is None:
            pitch = _backend.checkpoint_pitch(self._cols)
            self._exponent = self._buffer[self._rows * pitch:].view(self._rows, pitch // _backend.CKPT_BLOCK)
        return self._exponent

    def to(self, dtype):
        """The values in a float type, rounded once."""
        if not self.is_cuda:
            raise ValueError('The codes are not in GPU memory; the FP8 kernels only run on the HIP device.')
        return _backend.checkpoint_unpack(*self._pointers(), self._rows, self._cols, self.shape, dtype, self.device)

    def float(self):
        return self.to(torch.float32)

    def half(self):
        return self.to(torch.float16)

    def bfloat16(self):
        return self.to(torch.bfloat16)

    def size(self, dim=None):
        return self.shape if dim is None else self.shape[dim]

    def numel(self):
        return self.shape.numel()

    @property
    def _codes(self):
        return self._value if self._buffer is None else self._buffer

    @property
    def device(self):
        return self._codes.device

    @property
    def is_cuda(self):
        return self._codes.is_cuda

    @property
    def nbytes(self):
        """Bytes of the codes and the exponents."""
        return self._value.numel() + self._exponent.numel() if self._buffer is None else self._buffer.numel()

    def __repr__(self):
        return f'BlockTensor(shape={tuple(self.shape)}, device={self.device})'
