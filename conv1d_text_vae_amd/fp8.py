"""8-bit operands with a scale for each block of 128, and the products over them (c1v_fp8_* of include/c1dvae.h).

    w = fp8.quantize_cols(kernel)              # once per weight update; kernel [in, out] as Keras keeps it
    y = fp8.dense(x, w, bias)                  # serving: x is quantised on the way (one launch for few rows)
    y = fp8.linear(x, kernel, bias)            # training: forward and both gradients in 8 bits
    c = fp8.product(fp8.quantize_rows(a), fp8.quantize_rows(b))      # a @ b.T

Values are e4m3, a scale is a power of two (one exponent byte), sums are fp32.  float32 and bfloat16 tensors on the GPU only;
like the rest of the package there is no CPU fallback.  The reference has no counterpart (its dense layers are fp32 Keras ones).
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
from typing import Optional, Tuple

import torch

from . import _lib as L

BLOCK = L.FP8_BLOCK
_CODE = {torch.float32: L.F32, torch.bfloat16: L.BF16}


# The argument structs as packed bytes: building them field by field costs more than the launch.  (Layouts of the ctypes mirrors
# in _lib.py.)
_GEMM = 'PPPPqqqPiiPqPq'
_QUANT = struct.Struct('@PiqqqPPPPPP').pack
_PRODUCT = struct.Struct('@' + _GEMM).pack
_DENSE = struct.Struct('@Piqq' + _GEMM).pack
_LINEAR = struct.Struct('@qqqiiiiiPqPqPPPqPPPPP').pack
# torch's own accessors of the current stream and device: the public ones build objects
_stream, _current = (getattr(torch._C, n, None) for n in ('_cuda_getCurrentRawStream', '_cuda_getDevice'))
_entry = {}


def _bind(name: str):
    f = L.load()[name]                                             # a function object of its own: takes the struct's bytes
    f.argtypes, f.restype = [C.c_char_p, C.c_void_p], C.c_int
    _entry[name] = f
    return f


@functools.lru_cache(maxsize=4096)
def _work_bytes(m: int, n: int, kp: int) -> int:
    return L.load().c1v_fp8_gemm_work(m, n, kp)


@functools.lru_cache(maxsize=4096)
def _direct(m: int, n: int, kp: int) -> bool:
    return bool(L.load().c1v_fp8_dense_direct(m, n, kp))


@functools.lru_cache(maxsize=4096)
def _linear_sizes(*shape_types_needs) -> Tuple[int, int, int]:
    sizes = [C.c_int64() for _ in range(3)]
    L.check(L.load().c1v_fp8_linear_sizes(C.byref(L.Fp8LinearArgs(*shape_types_needs)), *(C.byref(v) for v in sizes)),
            'c1v_fp8_linear_sizes')
    return tuple(v.value for v in sizes)


class Fp8Rows:
    """A matrix [rows, cols] in 8 bits, its blocks of 128 along the columns: `data` float8_e4m3fn [rows, cols rounded up to
    128] (zeros behind the last column), `scale` uint8 [blocks, rows rounded up to 16]; value = data * 2^(scale - 127).
    Tensors at other strides (a transposition, a slice) are laid out once, here."""

    __slots__ = ('data', 'scale', 'cols')

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, cols: int):
        rows, kp = data.shape
        if data.dtype != torch.float8_e4m3fn or scale.dtype != torch.uint8:
            raise ValueError('data must be float8_e4m3fn and scale uint8, got {0} and {1}'.format(data.dtype, scale.dtype))
        if kp != -(-cols // BLOCK) * BLOCK or tuple(scale.shape) != (kp // BLOCK, (rows + 15) // 16 * 16):
            raise ValueError('{0} columns need data [rows, {1}] and scale [{2}, {3}], got {4} and {5}'.format(
                cols, -(-cols // BLOCK) * BLOCK, -(-cols // BLOCK), (rows + 15) // 16 * 16, tuple(data.shape), tuple(scale.shape)))
        if data.device != scale.device:
            raise ValueError('data and scale are on {0} and {1}'.format(data.device, scale.device))
        self.data, self.scale, self.cols = data.contiguous(), scale.contiguous(), int(cols)

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    def dequantize(self) -> torch.Tensor:
        """float32 [rows, cols]"""
        s = (self.scale[:, :self.rows].to(torch.int32) << 23).view(torch.float32).t()
        kp = self.data.shape[1]
        return (self.data.float().view(self.rows, kp // BLOCK, BLOCK) * s.unsqueeze(-1)).view(self.rows, kp)[:, :self.cols]


def _empty(rows: int, cols: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    kb = -(-cols // BLOCK)
    return (torch.empty((rows, kb * BLOCK), dtype=torch.float8_e4m3fn, device=device),
            torch.empty((kb, (rows + 15) // 16 * 16), dtype=torch.uint8, device=device))


def _wrap(pair, cols: int) -> Fp8Rows:
    q = Fp8Rows.__new__(Fp8Rows)
    q.data, q.scale, q.cols = pair[0], pair[1], cols
    return q


def _matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    """x as a matrix whose rows are runs of memory (a copy only where they are not)."""
    if x.dtype not in _CODE:
        raise ValueError('{0} must be float32 or bfloat16, got {1}'.format(what, x.dtype))
    shape = x.shape
    if len(shape) != 2:
        raise ValueError('{0} must be a matrix, got shape {1}'.format(what, tuple(shape)))
    rows, cols = shape
    if cols < 1:
        raise ValueError('{0} has no columns'.format(what))
    if not x.is_cuda:
        raise L.C1VError('{0} is on {1}: the HIP kernels are the only implementation of this operator.'.format(what, x.device))
    step, unit = x.stride()
    if (cols > 1 and unit != 1) or (rows > 1 and step < cols):
        return x.contiguous()
    return x


def _call(name: str, args: bytes, i: int):
    """On the current stream of GPU `i`, whichever one is current."""
    f = _entry.get(name) or _bind(name)
    if _current() == i:
        rc = f(args, _stream(i))
    else:
        with torch.cuda.device(i):
            rc = f(args, _stream(i))
    if rc:
        L.check(rc, name)


def _quantize(x: torch.Tensor, rows: bool, cols: bool):
    x = _matrix(x, 'x')
    R, K = x.shape
    dev = x.device
    q = _empty(R, K, dev) if rows else None
    qt = _empty(K, R, dev) if cols else None
    if R:
        _call('c1v_fp8_quantize', _QUANT(
            x.data_ptr(), _CODE[x.dtype], R, K, x.stride(0) if R > 1 else K, q[0].data_ptr() if rows else 0,
            q[1].data_ptr() if rows else 0, qt[0].data_ptr() if cols else 0, qt[1].data_ptr() if cols else 0, 0, 0), x.get_device())
    return _wrap(q, K) if rows else None, _wrap(qt, R) if cols else None


def quantize_rows(x: torch.Tensor) -> Fp8Rows:
    """x [R, K] in 8 bits, blocks along K (the contraction of x @ w.T)."""
    return _quantize(x, True, False)[0]


def quantize_cols(x: torch.Tensor) -> Fp8Rows:
    """x.T [K, R] in 8 bits, blocks along R: the weight operand of a kernel [in, out], or the operand of x.T @ dy."""
    return _quantize(x, False, True)[1]


def quantize_both(x: torch.Tensor) -> Tuple[Fp8Rows, Fp8Rows]:
    """(quantize_rows(x), quantize_cols(x)) from one read of x."""
    return _quantize(x, True, True)


def _check_bias(bias, n: int, device):
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (n,) or bias.device != device or
                             not bias.is_contiguous()):
        raise ValueError('bias must be a contiguous float32 vector of {0} values on {1}'.format(n, device))


def _no_gradient(what: str):
    """A product that has no gradient does not drop out of a graph unnoticed."""
    if torch.is_grad_enabled():
        raise ValueError('{0} has no gradient, and one of its inputs requires one: use linear, detach() or torch.no_grad()'.format(what))


def product(a: Fp8Rows, b: Fp8Rows, bias: Optional[torch.Tensor] = None, relu: bool = False,
            out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[a.rows, b.rows] = relu(a @ b.T + bias).  No gradient: a bias that requires one is refused while gradients are enabled."""
    if bias is not None and bias.requires_grad:
        _no_gradient('product')
    dev = a.data.device
    if a.cols != b.cols:
        raise ValueError('the operands have {0} and {1} columns'.format(a.cols, b.cols))
    if b.data.device != dev:
        raise ValueError('the operands are on {0} and {1}'.format(dev, b.data.device))
    if out_dtype not in _CODE:
        raise ValueError('out_dtype must be float32 or bfloat16, got {0}'.format(out_dtype))
    if not a.data.is_cuda:
        raise L.C1VError('operands on {0}: the HIP kernels are the only implementation of this operator.'.format(dev))
    m, n, kp = a.data.shape[0], b.data.shape[0], a.data.shape[1]
    _check_bias(bias, n, dev)
    if not (m and n and kp):
        out = torch.zeros((m, n), dtype=out_dtype, device=dev)
        if bias is not None:
            out += bias
        return out.relu_() if relu else out
    out = torch.empty((m, n), dtype=out_dtype, device=dev)
    need = _work_bytes(m, n, kp)
    work = torch.empty(need // 4, dtype=torch.float32, device=dev) if need else None
    _call('c1v_fp8_gemm', _PRODUCT(a.data.data_ptr(), a.scale.data_ptr(), b.data.data_ptr(), b.scale.data_ptr(), m, n, kp,
                                   0 if bias is None else bias.data_ptr(), relu, _CODE[out_dtype], out.data_ptr(), n,
                                   work.data_ptr() if need else 0, need), dev.index)
    return out


def dense(x: torch.Tensor, w: Fp8Rows, bias: Optional[torch.Tensor] = None, relu: bool = False,
          out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """relu(x @ w.T + bias) for x [..., w.cols] in float32 or bfloat16, quantised on the way; out_dtype: x's by default.
    No gradient (`linear` has one): an x or a bias that requires one is refused while gradients are enabled."""
    if x.requires_grad or (bias is not None and bias.requires_grad):
        _no_gradient('dense')
    shape = x.shape
    if len(shape) != 2:
        x = x.reshape(-1, shape[-1])
    x = _matrix(x, 'x')
    m, k = x.shape
    q, sc = w.data, w.scale
    n, kp = q.shape
    if k != w.cols:
        raise ValueError('x has {0} columns, the weights {1}'.format(k, w.cols))
    i = x.get_device()
    if q.get_device() != i:
        raise ValueError('x is on {0}, the weights on {1}'.format(x.device, q.device))
    kind = x.dtype if out_dtype is None else out_dtype
    code = _CODE.get(kind)
    if code is None:
        raise ValueError('out_dtype must be float32 or bfloat16, got {0}'.format(kind))
    if bias is not None:
        _check_bias(bias, n, q.device)
    out = x.new_empty((m, n), dtype=kind)
    if m and n:
        qa = sa = work = need = 0
        if m > L.FP8_ROWS and not _direct(m, n, kp):               # x's values, its scales and the product's workspace in one piece
            at, need = m * kp, _work_bytes(m, n, kp)
            end = at + kp // BLOCK * ((m + 15) // 16 * 16)
            room = torch.empty(end + need, dtype=torch.uint8, device=x.device)
            qa = room.data_ptr()
            sa, work = qa + at, qa + end
        _call('c1v_fp8_dense', _DENSE(
            x.data_ptr(), _CODE[x.dtype], x.stride(0) if m > 1 else k, k, qa, sa, q.data_ptr(), sc.data_ptr(), m, n, kp,
            0 if bias is None else bias.data_ptr(), relu, code, out.data_ptr(), n, work, need), i)
    return out if len(shape) == 2 else out.view(*shape[:-1], n)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel, bias):
        need_x, need_k, need_b = ctx.needs_input_grad
        x, kernel = _matrix(x, 'x'), _matrix(kernel, 'kernel')
        rows, k = x.shape
        n = kernel.shape[1]
        dev, x_type, ctx.k_type = x.device, x.dtype, kernel.dtype
        if not rows:
            ctx.args = None
            ctx.empty = (x_type, k, n)
            return torch.empty((0, n), dtype=x_type, device=dev)
        y = torch.empty((rows, n), dtype=x_type, device=dev)
        what = (rows, k, n, _CODE[x_type], _CODE[ctx.k_type], need_x, need_k, need_b)
        keep_bytes, temp_bytes, ctx.temp_bytes = _linear_sizes(*what)
        keep = torch.empty(keep_bytes, dtype=torch.uint8, device=dev) if keep_bytes else None
        temp = torch.empty(temp_bytes, dtype=torch.uint8, device=dev)
        _call('c1v_fp8_linear_fwd', _LINEAR(
            *what, x.data_ptr(), x.stride(0) if rows > 1 else k, kernel.data_ptr(), kernel.stride(0) if k > 1 else n,
            0 if bias is None else bias.data_ptr(), y.data_ptr(), 0, 0, 0, 0, 0, keep.data_ptr() if keep_bytes else 0, temp.data_ptr()),
            dev.index)
        ctx.args = what
        ctx.save_for_backward(keep)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need_x, need_k, need_b = ctx.needs_input_grad
        dev = dy.device
        if ctx.args is None:
            x_type, k, n = ctx.empty
            return (torch.empty((0, k), dtype=x_type, device=dev) if need_x else None,
                    torch.zeros((k, n), dtype=ctx.k_type, device=dev) if need_k else None,
                    torch.zeros(n, dtype=torch.float32, device=dev) if need_b else None)
        keep, = ctx.saved_tensors
        dy = _matrix(dy, 'the gradient')
        rows, k, n = ctx.args[:3]
        dx = torch.empty((rows, k), dtype=dy.dtype, device=dev) if need_x else None
        dk = torch.empty((k, n), dtype=ctx.k_type, device=dev) if need_k else None
        db = torch.empty(n, dtype=torch.float32, device=dev) if need_b else None
        temp = torch.empty(ctx.temp_bytes, dtype=torch.uint8, device=dev)
        _call('c1v_fp8_linear_bwd', _LINEAR(
            *ctx.args, 0, 0, 0, 0, 0, 0, dy.data_ptr(), dy.stride(0) if rows > 1 else n, dx.data_ptr() if need_x else 0,
            dk.data_ptr() if need_k else 0, db.data_ptr() if need_b else 0, 0 if keep is None else keep.data_ptr(), temp.data_ptr()),
            dev.index)
        return dx, dk, db


def linear(x: torch.Tensor, kernel: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [..., in] @ kernel [in, out] + bias with every product in 8 bits; differentiable once.

    y = Q(x) Q(kernel), blocks along `in`;  dx = Q(dy) Q(kernel)^T, blocks along `out`;  dkernel = Q(x)^T Q(dy), blocks along
    the rows;  dbias = the fp32 sum of dy.  The gradients are those of the quantised operands with the quantiser taken as the
    identity.  What is kept for the backward pass is x and the kernel in 8 bits, not x itself.

    A forward and backward pass can be captured into a HIP graph; as for every torch operator, no eager graph over the same
    leaves may be alive while a backward pass is captured (its gradient accumulators belong to another stream)."""
    shape = x.shape
    if kernel.dim() != 2 or x.dim() < 1 or shape[-1] != kernel.shape[0]:
        raise ValueError('x [..., in] and kernel [in, out] expected, got {0} and {1}'.format(tuple(shape), tuple(kernel.shape)))
    if kernel.device != x.device:
        raise ValueError('x is on {0}, the kernel on {1}'.format(x.device, kernel.device))
    _check_bias(bias, kernel.shape[1], x.device)
    y = _Linear.apply(x if x.dim() == 2 else x.reshape(-1, shape[-1]), kernel, bias)
    return y if x.dim() == 2 else y.view(*shape[:-1], kernel.shape[1])
