"""Projections with 4-bit weights on the gfx950 kernels (csrc/w4_linear.hip): quantised
at load, or packed from given codes, multiplied at decode batch sizes, read back as
values for prefill.  They stand beside the fp8 weights (_sm70_ops.sm70_attn_fp8_gemv,
sm70_attn_fp8_dequant, ops.attn_fp8_quantize) at half the bytes.

A weight of row n and column k is (code - zero point) * scale, codes and zero points
0..15, scale and zero point those of the row and of its group of 32, 64 or 128 columns.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib, ops
from .ops import _check, _contig, _launch, _no_grad, _rows16, _traced

MAX_ROWS = 64  # of x in w4_linear
_DTYPE_CODE = {torch.float16: 0, torch.bfloat16: 1}


@dataclass(frozen=True)
class W4Weight:
    """Weights [n, k] as the kernels read them: q int32 [ceil(n / 16), ceil(k / 128), 64, 4],
    sz int32 [ceil(n / 16), ceil(k / 128) * 128 / group, 16] (mi355_dsa.h has the layout)."""
    q: torch.Tensor
    sz: torch.Tensor
    n: int
    k: int
    group: int
    dtype: torch.dtype

    def __post_init__(self):
        _check_weights(self.q, self.sz, self.n, self.k, self.group, self.dtype)


def _check_weights(q, sz, n: int, k: int, group: int, dtype: torch.dtype) -> None:
    _check(dtype in _DTYPE_CODE, "w4: fp16 or bf16 weights")
    _check(group in (32, 64, 128), "w4: group must be 32, 64 or 128")
    _check(k % 8 == 0, "w4: K must be a multiple of 8")
    t, b = -(-n // 16), -(-k // 128)
    _check(q.shape == (t, b, 64, 4) and sz.shape == (t, b * (128 // group), 16)
           and q.dtype == torch.int32 and sz.dtype == torch.int32 and q.is_contiguous()
           and sz.is_contiguous() and sz.device == q.device,
           "w4: q and sz are not of weights [n, k]")


def _empty(n: int, k: int, group: int, dtype: torch.dtype, dev) -> W4Weight:
    _check(group in (32, 64, 128), "w4: group must be 32, 64 or 128")
    t, b = -(-n // 16), -(-k // 128)
    return W4Weight(torch.empty(t, b, 64, 4, dtype=torch.int32, device=dev),
                    torch.empty(t, b * (128 // group), 16, dtype=torch.int32, device=dev),
                    n, k, group, dtype)


def w4_quantize(weight: torch.Tensor, group: int = 128, symmetric: bool = False) -> W4Weight:
    """Quantises weight [N, K] (fp16 or bf16, K a multiple of 8) group by group: with lo and
    hi the least and largest value of a group and 0, scale = (hi - lo) / 15 and zero point
    RN(-lo / scale), or (symmetric) max(hi / 7, -lo / 8) and 8; codes are
    clamp(RN(w / scale) + zero point, 0, 15).  Scales are of the weights' type.  A group
    that holds an infinity has no finite scale; NaN does not count and has some code."""
    _no_grad(weight)
    _check(weight.dim() == 2, "weight must be 2-D [N, K]")
    w = _empty(weight.size(0), weight.size(1), group, weight.dtype, weight.device)
    run = ops.op("w4_quantize") if _traced(weight) else _quantize
    run(w.q, w.sz, weight, group, symmetric)
    return w


def _quantize(q, sz, weight, group, symmetric):
    _check(weight.is_cuda, "weight must be on the GPU")
    x = weight if weight.is_contiguous() and weight.data_ptr() % 16 == 0 else \
        weight.clone(memory_format=torch.contiguous_format)
    _launch("mi355_dsa_w4_quantize", x.device, q.data_ptr(), sz.data_ptr(), x.data_ptr(),
            _DTYPE_CODE[x.dtype], x.size(0), x.size(1), group, symmetric)


def w4_pack(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
            group: int = 128) -> W4Weight:
    """Weights quantised elsewhere: codes uint8 [N, K] (their low four bits), scales fp16
    or bf16 [N, ceil(K / group)], zeros uint8 of that shape, or None for 8."""
    _check(codes.dim() == 2 and codes.dtype == torch.uint8, "codes must be uint8 [N, K]")
    w = _empty(codes.size(0), codes.size(1), group, scales.dtype, codes.device)
    _check_scales(codes, scales, zeros, group)
    _no_grad(scales)
    run = ops.op("w4_pack") if _traced(codes) else _pack
    run(w.q, w.sz, codes, scales, zeros, group)
    return w


def _check_scales(codes, scales, zeros, group) -> None:
    n, k = codes.shape
    _check(scales.shape == (n, -(-k // group)), "scales must be [N, ceil(K / group)]")
    _check(zeros is None or (zeros.shape == scales.shape and zeros.dtype == torch.uint8),
           "zeros must be uint8 [N, ceil(K / group)]")


def _pack(q, sz, codes, scales, zeros, group):
    _check(codes.is_cuda and scales.device == codes.device
           and (zeros is None or zeros.device == codes.device), "all tensors must be on one GPU")
    c = codes if codes.is_contiguous() and codes.data_ptr() % 8 == 0 else \
        codes.clone(memory_format=torch.contiguous_format)
    s, z = _contig(scales), None if zeros is None else _contig(zeros)
    _launch("mi355_dsa_w4_pack", c.device, q.data_ptr(), sz.data_ptr(), c.data_ptr(), s.data_ptr(),
            None if z is None else z.data_ptr(), _DTYPE_CODE[s.dtype], c.size(0), c.size(1), group)


def w4_linear(x: torch.Tensor, w: W4Weight, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [M, K] times the transposed weights: [M, N] in x's type (the weights'), M at most
    64 rows.  Weights enter unrounded, sums are fp32.  In bf16 two sums are subtracted, so
    that fp32's error is in units of 31 * scale * sum |x| of a group whatever its codes
    (fp16: of |x (code - zero point)|), and an infinity of x makes its row of y NaN, also
    where the formula gives an infinity.  Prefill-sized products: w4_dequant and a matrix
    product."""
    _no_grad(x)
    _check(x.dim() == 2 and x.size(1) == w.k, "x must be [M, K]")
    _check(x.dtype == w.dtype, "x must have the weights' type")
    _check(x.size(0) <= MAX_ROWS, f"w4_linear: at most {MAX_ROWS} rows, got {x.size(0)}")
    if out is None:
        out = torch.empty(x.size(0), w.n, dtype=x.dtype, device=x.device)
    else:
        _check_out(out, x, w.n)
    run = ops.op("w4_linear") if _traced(x) else _linear
    run(out, x, w.q, w.sz, w.group)
    return out


def _check_out(out, x, n: int) -> None:
    _check(out.shape == (x.size(0), n) and out.dtype == x.dtype and out.is_contiguous()
           and out.device == x.device, "out must be contiguous [M, N] of x's type")


def _linear(y, x, q, sz, group):
    _check(x.is_cuda and q.device == x.device and sz.device == x.device,
           "all tensors must be on one GPU")
    M, K = x.shape
    if M:
        x = _rows16(x)
        if M * x.stride(0) >= 1 << 29:  # the kernel's offsets are 32-bit
            x = x.contiguous()
    N = y.size(1)
    need = _lib.lib().mi355_dsa_w4_linear_workspace_size(M, N, K)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _launch("mi355_dsa_w4_linear", x.device, y.data_ptr(), x.data_ptr(), x.stride(0), q.data_ptr(),
            sz.data_ptr(), _DTYPE_CODE[x.dtype], M, N, K, group, ops._ptr(ws), need)


def w4_dequant(w: W4Weight) -> torch.Tensor:
    """The weights as values [N, K] of their type, RN((code - zero point) * scale)."""
    out = torch.empty(w.n, w.k, dtype=w.dtype, device=w.q.device)
    run = ops.op("w4_dequant") if _traced(w.q) else _dequant
    run(out, w.q, w.sz, w.group)
    return out


def _dequant(out, q, sz, group):
    _check(q.is_cuda, "the weights must be on the GPU")
    _launch("mi355_dsa_w4_dequant", q.device, out.data_ptr(), q.data_ptr(), sz.data_ptr(),
            _DTYPE_CODE[out.dtype], out.size(0), out.size(1), group)


# The ops may be called with any tensors: what the functions above have checked, or made.
def _op_quantize(q, sz, weight, group, symmetric):
    _check(weight.dim() == 2 and q.device == weight.device, "weight must be 2-D [N, K]")
    _check_weights(q, sz, *weight.shape, group, weight.dtype)
    _quantize(q, sz, weight, group, symmetric)


def _op_pack(q, sz, codes, scales, zeros, group):
    _check(codes.dim() == 2 and codes.dtype == torch.uint8 and q.device == codes.device,
           "codes must be uint8 [N, K]")
    _check_weights(q, sz, *codes.shape, group, scales.dtype)
    _check_scales(codes, scales, zeros, group)
    _pack(q, sz, codes, scales, zeros, group)


def _op_linear(y, x, q, sz, group):
    _check(x.dim() == 2 and y.dim() == 2, "x must be [M, K], y [M, N]")
    _check_out(y, x, y.size(1))
    _check_weights(q, sz, y.size(1), x.size(1), group, x.dtype)
    _linear(y, x, q, sz, group)


def _op_dequant(out, q, sz, group):
    _check(out.dim() == 2 and out.is_contiguous() and out.device == q.device,
           "out must be contiguous [N, K]")
    _check_weights(q, sz, *out.shape, group, out.dtype)
    _dequant(out, q, sz, group)


ops.define("w4_quantize(Tensor(a!) q, Tensor(b!) sz, Tensor weight, int group, bool symmetric) -> ()",
           _op_quantize)
ops.define("w4_pack(Tensor(a!) q, Tensor(b!) sz, Tensor codes, Tensor scales, Tensor? zeros, "
           "int group) -> ()", _op_pack)
ops.define("w4_linear(Tensor(a!) y, Tensor x, Tensor q, Tensor sz, int group) -> ()", _op_linear)
ops.define("w4_dequant(Tensor(a!) out, Tensor q, Tensor sz, int group) -> ()", _op_dequant)
