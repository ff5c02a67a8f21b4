"""Drop-in for vLLM's MLA cache writer (vllm/_custom_ops.py
concat_and_cache_mla), the producer of the latent cache the sparse MLA
kernels read: same name, argument order and semantics for kv_cache_dtype
"auto" and "fp8_ds_mla".  It dispatches to the torch op registered by
ops.py, which runs the gfx950 HIP kernel.

Beside it, for servers that rotate and re-read by themselves:
rope_concat_and_cache_mla rotates k_pe (and q) and writes the row in one launch,
gather_latent_cache reads rows back as values.
"""
from __future__ import annotations

import torch

from . import ops, rope
from ._sm70_ops import _op
from .ops import DSMLA_ROW_BYTES, _check, _contig, _launch, _no_grad, _rows16, _traced


def concat_and_cache_mla(kv_c: torch.Tensor, k_pe: torch.Tensor, kv_cache: torch.Tensor,
                         slot_mapping: torch.Tensor, kv_cache_dtype: str,
                         scale: torch.Tensor) -> None:
    """Writes token t of kv_c [T, 512] and k_pe [T, 64] into the latent cache
    row slot_mapping[t] (T = slot_mapping.numel(); negative slots skipped).

    "auto": kv_cache fp16 [n_blocks, page, 576] = [kv_c | k_pe].
    "fp8_ds_mla": kv_cache uint8 [n_blocks, page, 656]: 512 e4m3 bytes with a
    max(amax/448, FLT_MIN) scale per 128-dim tile, the 4 fp32 scales, then the
    64 16-bit RoPE values in k_pe's type (sparse attention reads fp16).
    `scale` is unused by both (vLLM reads it only for per-tensor fp8 caches)."""
    _op("concat_and_cache_mla")(kv_c, k_pe, kv_cache, slot_mapping, kv_cache_dtype, scale)


def _latent_rows(kv_cache: torch.Tensor) -> tuple[bool, int]:
    """(fp8 rows, number of rows) of a latent cache [n_blocks, page, 656 | 576]."""
    fp8 = kv_cache.dtype == torch.uint8
    _check(fp8 or kv_cache.dtype == torch.float16,
           "kv_cache must be fp16 or uint8 (fp8_ds_mla)")
    _check(kv_cache.dim() >= 2 and kv_cache.size(-1) == (DSMLA_ROW_BYTES if fp8 else 576),
           "kv_cache last dim must be 656 (fp8_ds_mla) or 576 (fp16)")
    _check(kv_cache.is_contiguous(), "kv_cache must be contiguous")
    return fp8, kv_cache.numel() // kv_cache.size(-1)


def rope_concat_and_cache_mla(positions: torch.Tensor, table: torch.Tensor, kv_c: torch.Tensor,
                              k_pe: torch.Tensor, kv_cache: torch.Tensor,
                              slot_mapping: torch.Tensor, kv_cache_dtype: str,
                              interleaved: bool = True, q: torch.Tensor | None = None,
                              q_offset: int = 0, q_out: torch.Tensor | None = None):
    """concat_and_cache_mla of a step whose k_pe is not rotated yet, and
    rope.apply_rotary of its q, in one launch; equal, bit for bit, to the two.

    table [positions, 64] (rope.rotary_table); T = slot_mapping.numel() tokens,
    positions [T]; q [T, H, D] of kv_c's type, its dims [q_offset, q_offset + 64)
    rotated into q_out (q itself for in place; allocated if not given).  k_pe is
    not changed.  The 64 rope values of an fp8_ds_mla row are stored in k_pe's type, as
    the writer alone does: gather_latent_cache and mla_tree.tree_attention take that type
    (pe_dtype), sparse and dense attention read fp16 (DsaLayer stores fp16 for them).
    A token with a negative slot writes no row, its q is rotated all the same; one with a
    position outside the table is not rotated.  Valid slots must be distinct.  Returns
    q_out, or None without q."""
    _no_grad(kv_c, k_pe, q)
    if not _traced(kv_c):
        return _rope_write(positions, table, kv_c, k_pe, kv_cache, slot_mapping, kv_cache_dtype,
                           interleaved, q, q_offset, q_out)
    if q is not None and q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    ops.op("rope_concat_and_cache_mla")(positions, table, kv_c, k_pe, kv_cache, slot_mapping,
                                        kv_cache_dtype, interleaved, q, q_offset, q_out)
    return q_out


def _rope_write(positions, table, kv_c, k_pe, kv_cache, slot_mapping, kv_cache_dtype, interleaved,
                q, q_offset, q_out):
    if kv_cache_dtype not in ("auto", "fp8_ds_mla"):
        raise RuntimeError(f"rope_concat_and_cache_mla: unsupported kv_cache_dtype {kv_cache_dtype!r}")
    fp8, n_rows = _latent_rows(kv_cache)
    _check(fp8 == (kv_cache_dtype == "fp8_ds_mla"),
           "kv_cache's type is not that of kv_cache_dtype")
    _check(kv_c.is_cuda and k_pe.device == kv_c.device and kv_cache.device == kv_c.device
           and slot_mapping.device == kv_c.device and table.device == kv_c.device,
           "all tensors must be on one GPU")
    _check(kv_c.dim() == 2 and k_pe.dim() == 2 and kv_c.size(1) == 512 and k_pe.size(1) == 64,
           "kv_lora_rank must be 512 and the rope dim 64")
    _check(kv_c.dtype in ((torch.float16, torch.bfloat16) if fp8 else (torch.float16,))
           and k_pe.dtype == kv_c.dtype,
           "kv_c and k_pe must be of one type: fp16, or bf16 into fp8_ds_mla")
    _check(slot_mapping.dim() == 1 and slot_mapping.dtype in (torch.int64, torch.int32),
           "slot_mapping must be int64 or int32 [tokens]")
    positions = rope._table_args(positions, table)
    _check(table.shape[1] == 64, "table must be [positions, 64]")
    T = slot_mapping.size(0)
    _check(positions.size(0) == T, "one position for each slot")
    _check(kv_c.size(0) >= T and k_pe.size(0) >= T, "fewer kv_c / k_pe rows than slots")
    part = None
    if q is not None:
        _check(q.dtype == kv_c.dtype, "q must have kv_c's type")
        part, q_out = rope._part(q, q_out, q_offset, interleaved, T, kv_c.device)
        part = part or None  # no head
    else:
        _check(q_out is None, "q_out without q")

    kv_c, k_pe, slot_mapping = _rows16(kv_c), _rows16(k_pe), _contig(slot_mapping)
    _launch("mi355_dsa_rope_concat_and_cache_mla", kv_c.device, kv_cache.data_ptr(), fp8, n_rows,
            kv_c.data_ptr(), kv_c.stride(0), k_pe.data_ptr(), k_pe.stride(0),
            kv_c.dtype == torch.bfloat16, T, slot_mapping.data_ptr(),
            slot_mapping.dtype == torch.int64, positions.data_ptr(),
            positions.dtype == torch.int64, table.data_ptr(), table.shape[0], interleaved, part)
    return q_out


def gather_latent_cache(kv_cache: torch.Tensor, block_table: torch.Tensor,
                        cu_seqlens: torch.Tensor, total: int,
                        starts: torch.Tensor | None = None, dtype: torch.dtype = torch.float16,
                        pe_dtype: torch.dtype = torch.float16,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """Latent rows of paged requests as values: out [total, 576] (kv_c | k_pe), the
    gathered context of SM70MLAPrefill.run_prefill_context_chunk before its
    projections.

    Row cu_seqlens[r] + i of out is position starts[r] + i (starts None: i) of
    request r, through block_table [requests, blocks] int32; cu_seqlens int32
    [requests + 1], total its last entry (or more: rows of no request are not
    written, they stay as they were in a given out).  dtype fp16, bf16 or fp32;
    pe_dtype: the type that the 64 rope values of fp8_ds_mla rows were written in.
    A position whose row does not resolve reads as zeros."""
    if _traced(kv_cache):
        if out is None:
            out = torch.empty(total, 576, dtype=dtype, device=kv_cache.device)
        ops.op("gather_latent_cache")(out, kv_cache, block_table, cu_seqlens, starts, dtype, pe_dtype)
        return out
    return _gather(out, kv_cache, block_table, cu_seqlens, total, starts, dtype, pe_dtype)


def _gather(out, kv_cache, block_table, cu_seqlens, total, starts, dtype, pe_dtype):
    fp8, n_rows = _latent_rows(kv_cache)
    _check(kv_cache.is_cuda and block_table.device == kv_cache.device
           and cu_seqlens.device == kv_cache.device
           and (starts is None or starts.device == kv_cache.device),
           "all tensors must be on one GPU")
    _check(block_table.dim() == 2 and block_table.dtype == torch.int32,
           "block_table must be int32 [requests, blocks]")
    R = block_table.size(0)
    _check(cu_seqlens.dim() == 1 and cu_seqlens.dtype == torch.int32
           and cu_seqlens.size(0) == R + 1, "cu_seqlens must be int32 [requests + 1]")
    _check(starts is None or (starts.dim() == 1 and starts.dtype == torch.int32
                              and starts.size(0) == R), "starts must be int32 [requests]")
    _check(dtype in rope._DTYPE_CODE, "gather_latent_cache: fp16, bf16 or fp32 values")
    _check(pe_dtype in ((torch.float16, torch.bfloat16) if fp8 else (torch.float16,)),
           "pe_dtype must be fp16, or bf16 for fp8_ds_mla rows")
    _check(total >= 0, "total must be >= 0")
    if out is None:
        out = torch.empty(total, 576, dtype=dtype, device=kv_cache.device)
    else:
        _check(out.dim() == 2 and out.shape == (total, 576) and out.dtype == dtype
               and out.device == kv_cache.device, "out must be [total, 576] of dtype")
        _check(out.stride(1) == 1 and out.stride(0) >= 576
               and out.stride(0) * out.element_size() % 16 == 0 and out.data_ptr() % 16 == 0,
               "out rows must be contiguous and 16-byte aligned")
    block_table, cu_seqlens = _contig(block_table), _contig(cu_seqlens)
    starts = _contig(starts) if starts is not None else None
    _launch("mi355_dsa_gather_latent_cache", kv_cache.device, out.data_ptr(), out.stride(0),
            rope._DTYPE_CODE[dtype], total, kv_cache.data_ptr(), fp8, pe_dtype == torch.bfloat16,
            n_rows, kv_cache.size(-2), block_table.data_ptr(), block_table.size(1),
            cu_seqlens.data_ptr(), starts.data_ptr() if starts is not None else None, R)
    return out


def _op_rope_write(*args):
    _rope_write(*args)


def _op_gather(out, kv_cache, block_table, cu_seqlens, starts, dtype, pe_dtype):
    _gather(out, kv_cache, block_table, cu_seqlens, out.size(0), starts, dtype, pe_dtype)


ops.define("rope_concat_and_cache_mla(Tensor positions, Tensor table, Tensor kv_c, Tensor k_pe, "
           "Tensor(a!) kv_cache, Tensor slot_mapping, str kv_cache_dtype, bool interleaved, "
           "Tensor? q, int q_offset, Tensor(b!)? q_out) -> ()", _op_rope_write)
ops.define("gather_latent_cache(Tensor(a!) out, Tensor kv_cache, Tensor block_table, "
           "Tensor cu_seqlens, Tensor? starts, ScalarType dtype, ScalarType pe_dtype) -> ()",
           _op_gather)
