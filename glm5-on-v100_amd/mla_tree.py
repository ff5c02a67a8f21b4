"""Attention of drafted token trees over the paged latent cache on the gfx950
kernel (csrc/mla_tree.hip, C ABI mi355_dsa_mla_tree_attention): the verification
step of speculative decoding where the drafts of a request form a tree.

It stands beside the dense decode (_sm70_ops.sm70_mla_decode), which takes one
token per row and no mask: all drafted tokens of a request and all heads share
every key tile here, the cache may hold fp16 or fp8_ds_mla rows, and any head
count goes.
"""
from __future__ import annotations

import torch

from . import _lib, ops
from ._cache_ops import _latent_rows
from .ops import _check, _contig, _launch, _no_grad, _traced

MAX_DRAFT = 64  # drafted tokens of a request that a mask can name


def tree_masks(parents) -> tuple[list[int], list[int]]:
    """(mask, depth) of the nodes of one tree from their parents (an earlier node's
    index, or -1 for a child of the context): bit i of mask[j] is set for j itself
    and its ancestors i, as int64 values; the position of node j is the context's
    length + depth[j]."""
    mask, depth = [], []
    for j, p in enumerate(parents):
        _check(-1 <= p < j, "tree_masks: a parent must be an earlier node, or -1")
        _check(j < MAX_DRAFT, f"tree_masks: at most {MAX_DRAFT} nodes")
        m = (mask[p] & (2 ** 64 - 1) if p >= 0 else 0) | 1 << j
        mask.append(m - 2 ** 64 if m >> 63 else m)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return mask, depth


def _check_trees(n_tok: int, block_table: torch.Tensor, seq_lens: torch.Tensor,
                 cu_seqlens_q: torch.Tensor, tree_mask: torch.Tensor, dev: torch.device) -> None:
    _check(block_table.dim() == 2 and block_table.dtype == torch.int32,
           "block_table must be int32 [requests, max_blocks]")
    R = block_table.size(0)
    _check(seq_lens.dim() == 1 and seq_lens.dtype == torch.int32 and seq_lens.size(0) == R,
           "seq_lens must be int32 [requests]")
    _check(cu_seqlens_q.dim() == 1 and cu_seqlens_q.dtype == torch.int32
           and cu_seqlens_q.size(0) == R + 1, "cu_seqlens_q must be int32 [requests + 1]")
    _check(tree_mask.dim() == 1 and tree_mask.dtype == torch.int64 and tree_mask.size(0) == n_tok,
           "tree_mask must be int64 [tokens]")
    _check(block_table.device == dev and seq_lens.device == dev and cu_seqlens_q.device == dev
           and tree_mask.device == dev, "all tensors must be on one GPU")


def tree_attention(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor,
                   seq_lens: torch.Tensor, cu_seqlens_q: torch.Tensor, tree_mask: torch.Tensor,
                   scale: float, out: torch.Tensor | None = None,
                   lse: torch.Tensor | None = None, pe_dtype: torch.dtype = torch.float16):
    """q [T, H, 576] fp16 (q_latent form); request r's drafted tokens are the rows
    cu_seqlens_q[r] .. cu_seqlens_q[r + 1] - 1 (int32 [R + 1]), n of them, already
    written to the cache at positions seq_lens[r] - n .. seq_lens[r] - 1.  Token j
    of them sees every position below seq_lens[r] - n and drafted token i where bit
    i of its tree_mask (int64 [T]) is set, its own bit included; at most 64 drafted
    tokens of a request can be seen.  kv_cache [n_blocks, page, 576] fp16 or
    [n_blocks, page, 656] uint8 (fp8_ds_mla, read as the fp16 values that
    gather_latent_cache gives; the 64 rope values must have been written as fp16); block_table int32 [R, max_blocks], seq_lens int32 [R].

    Returns o [T, H, 512] fp16 and lse [T, H] fp32; a row that sees nothing has
    o = 0 and lse = -inf.  Rows of no request (behind the last one) are not
    written: they stay as they were in a given out / lse."""
    _no_grad(q, kv_cache)
    _check(q.dim() == 3, "q must be [tokens, heads, 576]")
    T, H = q.shape[:2]
    if out is None:
        out = torch.empty(T, H, 512, dtype=torch.float16, device=q.device)
    if lse is None:
        lse = torch.empty(T, H, dtype=torch.float32, device=q.device)
    run = ops.op("mla_tree_attention") if _traced(q) else _attention
    run(out, lse, q, kv_cache, block_table, seq_lens, cu_seqlens_q, tree_mask, scale, pe_dtype)
    return out, lse


def _attention(out, lse, q, kv_cache, block_table, seq_lens, cu_seqlens_q, tree_mask, scale,
               pe_dtype):
    _check(q.is_cuda and kv_cache.device == q.device, "q and kv_cache must be on the GPU")
    _check(q.dtype == torch.float16, "q must be fp16")
    _check(q.dim() == 3 and q.size(2) == 576, "q must be [tokens, heads, 576]")
    fp8, n_rows = _latent_rows(kv_cache)
    _check(pe_dtype in ((torch.float16, torch.bfloat16) if fp8 else (torch.float16,)),
           "pe_dtype must be fp16, or bf16 for fp8_ds_mla rows")
    T, H = q.size(0), q.size(1)
    _check(H > 0, "n_head must be > 0")
    _check_trees(T, block_table, seq_lens, cu_seqlens_q, tree_mask, q.device)
    R = block_table.size(0)
    _check(out.dtype == torch.float16 and out.shape == (T, H, 512) and out.is_contiguous()
           and out.device == q.device, "out must be contiguous fp16 [tokens, heads, 512]")
    _check(lse.dtype == torch.float32 and lse.shape == (T, H) and lse.is_contiguous()
           and lse.device == q.device, "lse must be contiguous fp32 [tokens, heads]")
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    block_table, seq_lens = _contig(block_table), _contig(seq_lens)
    cu_seqlens_q, tree_mask = _contig(cu_seqlens_q), _contig(tree_mask)
    need = _lib.lib().mi355_dsa_mla_tree_workspace_size(T, H)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    _launch("mi355_dsa_mla_tree_attention", q.device, out.data_ptr(), lse.data_ptr(), q.data_ptr(),
            T, H, kv_cache.data_ptr(), 2 if pe_dtype == torch.bfloat16 else fp8, n_rows,
            kv_cache.size(-2), block_table.data_ptr(), block_table.size(1), seq_lens.data_ptr(),
            cu_seqlens_q.data_ptr(), R, tree_mask.data_ptr(), scale, ws.data_ptr(), need)


ops.define("mla_tree_attention(Tensor(a!) o, Tensor(b!) lse, Tensor q, Tensor kv_cache, "
           "Tensor block_table, Tensor seq_lens, Tensor cu_seqlens_q, Tensor tree_mask, "
           "float scale, ScalarType pe_dtype) -> ()", _attention)
