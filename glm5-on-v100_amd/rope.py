"""Rotary positions on the gfx950 kernel (csrc/rope.hip, C ABI mi355_dsa_rotary):
the step in front of the layer's attention, which takes q, k_pe and the indexer's
q and k rotated.

A table row holds the cosines of a position's rot_dim / 2 pairs and then the
sines, in fp32 (`rotary_table`, built in fp64).  In the interleaved layout pair i
of the rotated part is (2 i, 2 i + 1), as MLA's rope dims are kept; in the half
layout (i, i + rot_dim / 2), as the indexer's are.
"""
from __future__ import annotations

import math

import torch

from . import _lib, ops
from .ops import _check, _launch, _no_grad, _traced

_DTYPE_CODE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
MAX_TENSORS = 4  # of one launch


def rotary_table(rot_dim: int, max_positions: int, base: float = 10000.0,
                 scaling: dict | None = None, device="cuda") -> torch.Tensor:
    """cos | sin fp32 [max_positions, rot_dim] of position * base^(-2 i / rot_dim).

    scaling, for contexts longer than the model was trained on:
      {"type": "linear", "factor": f}: positions divided by f;
      {"type": "ntk", "factor": f}: base times f^(rot_dim / (rot_dim - 2));
      {"type": "yarn", "factor": f, "original_max_positions": n, and optionally
       "beta_fast" (32), "beta_slow" (1), "mscale" (1), "mscale_all_dim" (0)}: the
      method of Peng et al. 2023 -- frequencies of more than beta_fast turns over
      the n positions stay, those below beta_slow are divided by f, a linear ramp
      over the dims between; cos and sin times m(mscale) / m(mscale_all_dim) with
      m(s) = 0.1 s ln f + 1."""
    _check(rot_dim > 0 and rot_dim % 2 == 0, "rotary_table: rot_dim must be even and > 0")
    _check(max_positions >= 0, "rotary_table: max_positions must be >= 0")
    _check(base > 0, "rotary_table: base must be > 0")
    half = rot_dim // 2
    exponent = torch.arange(half, dtype=torch.float64) * 2 / rot_dim
    freq, mag = float(base) ** -exponent, 1.0
    if scaling is not None:
        kind, f = scaling.get("type"), float(scaling.get("factor", 1.0))
        _check(kind in ("linear", "ntk", "yarn"), f"rotary_table: unknown scaling {kind!r}")
        _check(f >= 1.0, "rotary_table: factor must be >= 1")
        if kind == "linear":
            freq = freq / f
        elif kind == "ntk":
            _check(rot_dim > 2, "rotary_table: ntk scaling needs rot_dim > 2")
            freq = (base * f ** (rot_dim / (rot_dim - 2))) ** -exponent
        else:
            n = scaling.get("original_max_positions", 0)
            _check(n > 0, "rotary_table: yarn needs original_max_positions")
            _check(base > 1, "rotary_table: yarn needs base > 1")

            def dim_of(turns):
                return rot_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

            lo = max(math.floor(dim_of(scaling.get("beta_fast", 32.0))), 0)
            hi = min(math.ceil(dim_of(scaling.get("beta_slow", 1.0))), rot_dim - 1)
            ramp = ((torch.arange(half, dtype=torch.float64) - lo)
                    / (hi - lo if hi > lo else 0.001)).clamp(0, 1)
            freq = freq / f * ramp + freq * (1 - ramp)

            def m(s):
                return 0.1 * s * math.log(f) + 1.0

            mag = m(scaling.get("mscale", 1.0)) / m(scaling.get("mscale_all_dim", 0.0))
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] \
        * freq.to(device)
    return (torch.cat([angle.cos(), angle.sin()], dim=1) * mag).float()


def _part(x: torch.Tensor, out: torch.Tensor | None, offset: int, interleaved: bool, n_tok: int,
          dev: torch.device):
    """(packed mi355_dsa_rotary_part, out) of x [T, H, D] or [T, D]; out allocated if None.
    Nothing is packed of a tensor of no head."""
    shape, code = x.shape, _DTYPE_CODE.get(x.dtype)
    _check(len(shape) in (2, 3) and shape[0] == n_tok,
           "apply_rotary: tensors are [tokens, heads, dim] or [tokens, dim]")
    _check(code is not None, "apply_rotary: fp16, bf16 or fp32 tensors")
    _check(x.device == dev, "all tensors must be on one GPU")
    xs = x.stride()
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out is not x:
        _check(out.shape == shape and out.dtype == x.dtype and out.device == dev,
               "apply_rotary: out must have x's shape, type and device")
    os = out.stride()
    _check((xs[-1] == 1 and os[-1] == 1) or shape[-1] <= 1,
           "apply_rotary: the last dim must be contiguous")
    heads = shape[1] if len(xs) == 3 else 1
    if heads == 0:
        return b"", out
    return _lib.ROTARY_PART.pack(out.data_ptr(), x.data_ptr(), os[0], os[-2], xs[0], xs[-2], heads,
                                 shape[-1], offset, code, interleaved), out


def _table_args(positions: torch.Tensor, table: torch.Tensor):
    _check(table.is_cuda and positions.device == table.device,
           "positions and table must be on the GPU")
    _check(positions.dim() == 1 and positions.dtype in (torch.int32, torch.int64),
           "positions must be int32 or int64 [tokens]")
    _check(table.dtype == torch.float32 and table.dim() == 2 and table.is_contiguous(),
           "table must be contiguous fp32 [positions, rot_dim]")
    return positions if positions.is_contiguous() else positions.contiguous()


def apply_rotary(xs, positions: torch.Tensor, table: torch.Tensor, offsets=0, interleaved=True,
                 outs=None):
    """Rotates dims [offset, offset + rot_dim) of every head of x [T, H, D] or
    [T, D] (fp16, bf16 or fp32, last dim contiguous) by the table row of the
    token's position; other dims are copied.  xs is a tensor, or a list of up to
    4 (a step's q, k_pe and the indexer's q and k) with one offset and layout
    each, rotated in one launch.  outs: tensors to write, xs themselves for in
    place (only the rotated part moves then); otherwise they must not overlap
    xs, and no two of them may hold the same elements (of two places in one tensor,
    both in place, the rotated parts).  A token whose position is outside the table (a padded one, -1) is not
    rotated.  Returns what was written, a tensor or a list as xs."""
    single = isinstance(xs, torch.Tensor)
    xl = [xs] if single else xs
    n = len(xl)
    if not 1 <= n <= MAX_TENSORS:
        raise RuntimeError(f"apply_rotary: 1 to {MAX_TENSORS} tensors")
    offs = [offsets] * n if isinstance(offsets, int) else offsets
    inter = [interleaved] * n if isinstance(interleaved, bool) else interleaved
    ol = [None] * n if outs is None else [outs] if isinstance(outs, torch.Tensor) else outs
    _check(len(offs) == n and len(inter) == n and len(ol) == n,
           "apply_rotary: one offset, layout and out for each tensor")
    _no_grad(*xl)
    if _traced(positions):
        ol = [torch.empty_like(x, memory_format=torch.contiguous_format) if o is None else o
              for x, o in zip(xl, ol)]
        ops.op("apply_rotary")(ol, xl, positions, table, offs, inter)
    else:
        ol = _rotary(ol, xl, positions, table, offs, inter)
    return ol[0] if single else ol


def _rotary(ol, xl, positions, table, offs, inter) -> list[torch.Tensor]:
    positions = _table_args(positions, table)
    T, dev = positions.shape[0], table.device
    parts = [_part(x, o, a, i, T, dev) for x, o, a, i in zip(xl, ol, offs, inter)]
    packed = b"".join([p[0] for p in parts])
    _launch("mi355_dsa_rotary", dev, packed, len(packed) // _lib.ROTARY_PART.size,
            positions.data_ptr(), positions.dtype == torch.int64, T, table.data_ptr(),
            table.shape[0], table.shape[1])
    return [p[1] for p in parts]


def _op_rotary(*args):
    _rotary(*args)


ops.define("apply_rotary(Tensor(a!)[] outs, Tensor[] xs, Tensor positions, Tensor table, "
           "int[] offsets, bool[] interleaved) -> ()", _op_rotary)
