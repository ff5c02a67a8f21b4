"""Attention of requests that share a long prefix over the paged latent cache, on the
gfx950 kernel (csrc/mla_prefix.hip, C ABI mi355_dsa_mla_prefix_attention): many answers
to one prompt, or many users behind one system prompt.

It stands beside the dense decode (_sm70_ops.sm70_mla_decode) and tree attention
(mla_tree), which read a prefix once for every request: here the rows of all requests
that share meet every shared key tile together, and then each request its own keys.
"""
from __future__ import annotations

import torch

from . import _lib, ops
from ._cache_ops import _latent_rows
from .mla_tree import _check_trees
from .ops import _check, _contig, _launch, _no_grad, _traced


def pays(n_tok: int, n_head: int, n_req: int, n_group: int, positions: int) -> bool:
    """Whether drafted trees of requests that share most of `positions` are expected to be
    attended to faster here than by tree_attention, from what the host knows.

    Row groups of 128 (token, head) rows meet each 32 keys as one tile: tree attention needs
    ceil(n_head * tokens / 128) of them for each request, here the requests' rows fill them
    together.  A tile spared saves 3 to 5 ns, and the division of the work, a launch of its own,
    costs 8 to 12 us.  us here / by tree attention, 16 heads, one token a request, 2048
    positions of fp16 rows: 16 requests 40 / 36, 64 (3520 tiles spared) 51 / 52, 128 56 / 82; 64
    heads: 64 (1984) 66 / 56, 128 (4032) 81 / 88.  Tree attention's workgroups each sum over
    all requests: with two drafted tokens of 64 heads, where no tile is spared, 128 requests
    117 / 114, 160 137 / 148, 256 170 / 190; but 160 groups of one request 171 / 159, 130 of
    two (16 heads, 1024 positions) 100 / 140."""
    alone = n_req * -(-n_tok * n_head // (128 * max(n_req, 1)))
    spared = (alone - n_tok * n_head // 128 - n_group) * (positions // 32)
    return (n_req > 128 and 2 * n_group <= n_req) or spared >= 3500


def shared_prefix_attention(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor,
                            seq_lens: torch.Tensor, cu_shared: torch.Tensor,
                            shared_lens: torch.Tensor, scale: float,
                            cu_seqlens_q: torch.Tensor | None = None,
                            tree_mask: torch.Tensor | None = None,
                            out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                            pe_dtype: torch.dtype = torch.float16):
    """The requests cu_shared[g] .. cu_shared[g + 1] - 1 (int32 [groups + 1]) hold their first
    shared_lens[g] positions (int32 [groups]; paging.shared_lengths finds them) in the
    same cache rows, which are read through the block-table row of the first one that has a
    token.  A group may be one request, and share nothing; positions that a drafted token
    takes, or that the shortest request of a group lacks, do not count as shared (requests
    without a token, which cu_seqlens_q may have, are not looked at).  So an ended request of
    length 0 that stays in its group with a token ends the sharing, though not the results: 32
    answers over 32768 positions 166 us, with one ended 235, or 171 where cu_shared puts it
    into a group of its own.

    q [T, H, 576] fp16 (q_latent form).  Without cu_seqlens_q: one token a request, T of them,
    token r at position seq_lens[r] - 1, which sees everything up to itself.  With
    cu_seqlens_q and tree_mask: each request's drafted tokens, as in
    mla_tree.tree_attention.  kv_cache, block_table, seq_lens, scale and pe_dtype are as there;
    the block table holds less than 2^23 positions.

    Returns o [T, H, 512] fp16 and lse [T, H] fp32; a row that sees nothing has o = 0
    and lse = -inf.  Rows of no request, and of requests of no group, stay as they were in
    a given out / lse.  An own cache row (not shared) that holds an infinity or NaN does not touch
    the rows that do not see it."""
    _no_grad(q, kv_cache)
    _check(q.dim() == 3, "q must be [tokens, heads, 576]")
    T, H = q.shape[:2]
    if out is None:
        out = torch.empty(T, H, 512, dtype=torch.float16, device=q.device)
    if lse is None:
        lse = torch.empty(T, H, dtype=torch.float32, device=q.device)
    run = ops.op("mla_prefix_attention") if _traced(q) else _attention
    run(out, lse, q, kv_cache, block_table, seq_lens, cu_shared, shared_lens, scale, cu_seqlens_q,
        tree_mask, pe_dtype)
    return out, lse


def _check_shared(cu_shared: torch.Tensor, shared_lens: torch.Tensor, dev: torch.device) -> None:
    _check(cu_shared.dim() == 1 and cu_shared.dtype == torch.int32 and cu_shared.size(0) >= 1,
           "cu_shared must be int32 [groups + 1]")
    _check(shared_lens.dim() == 1 and shared_lens.dtype == torch.int32
           and shared_lens.size(0) == cu_shared.size(0) - 1, "shared_lens must be int32 [groups]")
    _check(cu_shared.device == dev and shared_lens.device == dev, "all tensors must be on one GPU")


def _attention(out, lse, q, kv_cache, block_table, seq_lens, cu_shared, shared_lens, scale,
               cu_seqlens_q, tree_mask, pe_dtype):
    _check(q.is_cuda and kv_cache.device == q.device, "q and kv_cache must be on the GPU")
    _check(q.dtype == torch.float16, "q must be fp16")
    _check(q.dim() == 3 and q.size(2) == 576, "q must be [tokens, heads, 576]")
    fp8, n_rows = _latent_rows(kv_cache)
    _check(pe_dtype in ((torch.float16, torch.bfloat16) if fp8 else (torch.float16,)),
           "pe_dtype must be fp16, or bf16 for fp8_ds_mla rows")
    T, H = q.size(0), q.size(1)
    _check(H > 0, "n_head must be > 0")
    _check((cu_seqlens_q is None) == (tree_mask is None),
           "cu_seqlens_q and tree_mask go together")
    if cu_seqlens_q is not None:
        _check_trees(T, block_table, seq_lens, cu_seqlens_q, tree_mask, q.device)
        cu_seqlens_q, tree_mask = _contig(cu_seqlens_q), _contig(tree_mask)
    else:
        _check(block_table.dim() == 2 and block_table.dtype == torch.int32
               and block_table.size(0) == T, "block_table must be int32 [requests, max_blocks], "
               "one request for each token without cu_seqlens_q")
        _check(seq_lens.dim() == 1 and seq_lens.dtype == torch.int32 and seq_lens.size(0) == T,
               "seq_lens must be int32 [requests]")
        _check(block_table.device == q.device and seq_lens.device == q.device,
               "all tensors must be on one GPU")
    _check_shared(cu_shared, shared_lens, q.device)
    R, S = block_table.size(0), shared_lens.size(0)
    _check(out.dtype == torch.float16 and out.shape == (T, H, 512) and out.is_contiguous()
           and out.device == q.device, "out must be contiguous fp16 [tokens, heads, 512]")
    _check(lse.dtype == torch.float32 and lse.shape == (T, H) and lse.is_contiguous()
           and lse.device == q.device, "lse must be contiguous fp32 [tokens, heads]")
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    block_table, seq_lens = _contig(block_table), _contig(seq_lens)
    cu_shared, shared_lens = _contig(cu_shared), _contig(shared_lens)
    need = _lib.lib().mi355_dsa_mla_prefix_workspace_size(T, H, R, S)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    _launch("mi355_dsa_mla_prefix_attention", q.device, out.data_ptr(), lse.data_ptr(),
            q.data_ptr(), T, H, kv_cache.data_ptr(), 2 if pe_dtype == torch.bfloat16 else fp8,
            n_rows, kv_cache.size(-2), block_table.data_ptr(), block_table.size(1),
            seq_lens.data_ptr(), None if cu_seqlens_q is None else cu_seqlens_q.data_ptr(), R,
            None if tree_mask is None else tree_mask.data_ptr(), cu_shared.data_ptr(),
            shared_lens.data_ptr(), S, scale, ws.data_ptr(), need)


ops.define("mla_prefix_attention(Tensor(a!) o, Tensor(b!) lse, Tensor q, Tensor kv_cache, "
           "Tensor block_table, Tensor seq_lens, Tensor cu_shared, Tensor shared_lens, float scale, "
           "Tensor? cu_seqlens_q, Tensor? tree_mask, ScalarType pe_dtype) -> ()", _attention)
