"""Block tables and slot maps of a step, built on the GPU (csrc/paging.hip): what the
cache writers and attentions of this package take (block_table, seq_lens, slot_mapping,
positions, cu_seqlens_q), from the requests' lengths, without a read back to the host.

A program keeps block_table int32 [requests, max_blocks], seq_lens int32 [requests] and
a stack of free pages: free_pages int32 [pages of the pool], of which the first
free_count[0] (int32 [1]) are free, the last of them taken first.  All calls are
capture-safe, and no call synchronises.
"""
from __future__ import annotations

import torch

from . import _lib, ops
from .ops import _check, _contig, _launch, _traced


def _tables(block_table: torch.Tensor, seq_lens: torch.Tensor, kept: bool) -> tuple[int, int]:
    """Checks the two and returns (requests, max_blocks); kept: they are written."""
    _check(block_table.is_cuda and seq_lens.device == block_table.device,
           "all tensors must be on one GPU")
    _check(block_table.dim() == 2 and block_table.dtype == torch.int32,
           "block_table must be int32 [requests, max_blocks]")
    R = block_table.size(0)
    _check(seq_lens.dim() == 1 and seq_lens.dtype == torch.int32 and seq_lens.size(0) == R,
           "seq_lens must be int32 [requests]")
    _check(not kept or (block_table.is_contiguous() and seq_lens.is_contiguous()),
           "block_table and seq_lens are written: they must be contiguous")
    return R, block_table.size(1)


def _stack(free_pages: torch.Tensor, free_count: torch.Tensor, page_size: int,
           dev: torch.device) -> None:
    _check(free_pages.dim() == 1 and free_pages.dtype == torch.int32 and free_pages.is_contiguous()
           and free_pages.device == dev, "free_pages must be contiguous int32 [pages] on the GPU")
    _check(free_count.numel() == 1 and free_count.dtype == torch.int32 and free_count.device == dev,
           "free_count must be int32 [1] on the GPU")
    _check(page_size > 0, "page size must be > 0")


def _per_request(x: torch.Tensor, name: str, R: int, dev: torch.device) -> torch.Tensor:
    _check(x.dim() == 1 and x.dtype == torch.int32 and x.size(0) == R and x.device == dev,
           f"{name} must be int32 [requests] on the GPU")
    return _contig(x)


def extend_tables(block_table: torch.Tensor, seq_lens: torch.Tensor, new_tokens: torch.Tensor,
                  free_pages: torch.Tensor, free_count: torch.Tensor, page_size: int,
                  max_tokens: int):
    """Room for new_tokens[r] (int32 [R]; 0: idle) further tokens of every request, in
    place: pages from the free stack into block_table, seq_lens and free_count moved on.

    Returns slot_mapping and positions int32 [max_tokens], cu_seqlens_q int32 [R + 1] and
    granted bool [R].  The step's tokens stand request by request, as new_tokens has them;
    token cu_seqlens_q[r] + i is position seq_lens[r] (the old one) + i.  Rows behind the
    last token (a padded batch) have slot and position -1, which the cache writers skip
    and the rotation leaves alone.

    A request is refused (granted false; its tokens keep their rows, with slot and position
    -1; its table and length stay) if its table or max_tokens is too short for it, or if the
    pages left do not suffice: pages go to the requests in order, and from the first
    that they do not suffice for on, only requests that need none are granted."""
    if not _traced(block_table):
        return _extend(None, block_table, seq_lens, new_tokens, free_pages, free_count, page_size,
                       max_tokens)
    outs = _extend_outs(block_table, max_tokens)
    ops.op("extend_tables")(*outs, block_table, seq_lens, new_tokens, free_pages, free_count,
                            page_size)
    return outs


def _extend_outs(block_table, max_tokens):
    _check(max_tokens >= 0, "max_tokens must be >= 0")
    R, dev = block_table.size(0), block_table.device
    return (torch.empty(max_tokens, dtype=torch.int32, device=dev),
            torch.empty(max_tokens, dtype=torch.int32, device=dev),
            torch.empty(R + 1, dtype=torch.int32, device=dev),
            torch.empty(R, dtype=torch.bool, device=dev))


def _extend(outs, block_table, seq_lens, new_tokens, free_pages, free_count, page_size, max_tokens):
    R, W = _tables(block_table, seq_lens, True)
    dev = block_table.device
    _stack(free_pages, free_count, page_size, dev)
    new_tokens = _per_request(new_tokens, "new_tokens", R, dev)
    outs = _extend_outs(block_table, max_tokens) if outs is None else outs
    slots, pos, cu, granted = outs
    _launch("mi355_dsa_extend_tables", dev, block_table.data_ptr(), seq_lens.data_ptr(),
            new_tokens.data_ptr(), R, W, free_pages.data_ptr(), free_count.data_ptr(),
            free_pages.size(0), page_size, slots.data_ptr(), pos.data_ptr(), slots.size(0),
            cu.data_ptr(), granted.data_ptr())
    return outs


def truncate_tables(block_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor,
                    free_pages: torch.Tensor, free_count: torch.Tensor, page_size: int) -> None:
    """Requests cut back to new_lens (int32 [R]; at or above seq_lens[r]: as they are), in
    place: rejected drafts, ended requests (0), answers to a shared prompt (its length, a
    whole number of pages: those stay).  Pages that no position needs any more go back to
    the free stack, their entries become -1.  Pages that others hold too must not be cut
    off.  Entries that are already negative give nothing back; free_pages must have room
    for every page of the pool (what does not fit is dropped).  extend_tables followed by
    a cut to the old lengths leaves the stack as it was."""
    run = ops.op("truncate_tables") if _traced(block_table) else _truncate
    run(block_table, seq_lens, new_lens, free_pages, free_count, page_size)


def _truncate(block_table, seq_lens, new_lens, free_pages, free_count, page_size):
    R, W = _tables(block_table, seq_lens, True)
    dev = block_table.device
    _stack(free_pages, free_count, page_size, dev)
    new_lens = _per_request(new_lens, "new_lens", R, dev)
    ws = torch.empty(R + 1, dtype=torch.int32, device=dev)
    _launch("mi355_dsa_truncate_tables", dev, block_table.data_ptr(), seq_lens.data_ptr(),
            new_lens.data_ptr(), R, W, free_pages.data_ptr(), free_count.data_ptr(),
            free_pages.size(0), page_size, ws.data_ptr(), 4 * (R + 1))


def token_tables(block_table: torch.Tensor, seq_lens: torch.Tensor, cu_seqlens_q: torch.Tensor,
                 n_tok: int, cols: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(rows [n_tok, cols], lens [n_tok]) int32, one for each token, as sparse and dense
    decode take them: the block-table row of the token's request (its first cols columns),
    and the positions up to and with the token, seq_lens[r] - n + j + 1 for token j of
    the n of request r (rows cu_seqlens_q[r] .. cu_seqlens_q[r + 1] - 1).  A row of no
    request is -1 with length 0.  block_table rows may be strided."""
    cols = block_table.size(-1) if cols is None else cols
    _check(0 <= cols <= block_table.size(-1) and n_tok >= 0,
           "token_tables: cols must be 0 .. max_blocks, n_tok >= 0")
    dev = block_table.device
    out = torch.empty(n_tok, cols, dtype=torch.int32, device=dev)
    lens = torch.empty(n_tok, dtype=torch.int32, device=dev)
    run = ops.op("token_tables") if _traced(block_table) else _token_tables
    run(out, lens, block_table, seq_lens, cu_seqlens_q)
    return out, lens


def _token_tables(out, lens, block_table, seq_lens, cu_seqlens_q):
    R, W = _tables(block_table, seq_lens, False)
    dev = block_table.device
    _check(cu_seqlens_q.dim() == 1 and cu_seqlens_q.dtype == torch.int32
           and cu_seqlens_q.size(0) == R + 1 and cu_seqlens_q.device == dev,
           "cu_seqlens_q must be int32 [requests + 1] on the GPU")
    if W > 1 and block_table.stride(1) != 1 or block_table.stride(0) < W:
        block_table = block_table.contiguous()
    seq_lens, cu = _contig(seq_lens), _contig(cu_seqlens_q)
    _launch("mi355_dsa_token_tables", dev, out.data_ptr(), lens.data_ptr(), out.size(0),
            out.size(1), block_table.data_ptr(), block_table.stride(0), seq_lens.data_ptr(),
            cu.data_ptr(), R)


def shared_lengths(block_table: torch.Tensor, seq_lens: torch.Tensor, cu_shared: torch.Tensor,
                   page_size: int) -> torch.Tensor:
    """int32 [groups]: the leading positions that the requests of each group hold in the
    same pages (group g: requests cu_shared[g] .. cu_shared[g + 1] - 1, int32
    [groups + 1]) -- whole pages, at most the shortest of their lengths.  0 for a group
    of no request, or with one of length 0 (an ended answer, a padded row: to be given a
    group of its own); the length of one that is alone."""
    _check(cu_shared.dim() == 1 and cu_shared.size(0) >= 1, "cu_shared must be int32 [groups + 1]")
    out = torch.empty(cu_shared.size(0) - 1, dtype=torch.int32, device=block_table.device)
    run = ops.op("shared_lengths") if _traced(block_table) else _shared_lengths
    run(out, block_table, seq_lens, cu_shared, page_size)
    return out


def _shared_lengths(out, block_table, seq_lens, cu_shared, page_size):
    R, W = _tables(block_table, seq_lens, False)
    dev = block_table.device
    _check(cu_shared.dtype == torch.int32 and cu_shared.device == dev,
           "cu_shared must be int32 [groups + 1] on the GPU")
    _check(page_size > 0, "page size must be > 0")
    block_table, seq_lens, cu = _contig(block_table), _contig(seq_lens), _contig(cu_shared)
    ws = torch.empty(R, dtype=torch.int32, device=dev)
    _launch("mi355_dsa_shared_lengths", dev, out.data_ptr(), cu.data_ptr(), out.size(0),
            block_table.data_ptr(), seq_lens.data_ptr(), R, W, page_size, ws.data_ptr(), 4 * R)


# The ops may be called with any tensors: what the functions above make.
def _written(x, shape, dtype, dev, name: str) -> None:
    _check(x.shape == shape and x.dtype == dtype and x.is_contiguous() and x.device == dev,
           f"{name} must be contiguous {dtype} {list(shape)} on the GPU")


def _op_extend(slots, pos, cu, granted, block_table, seq_lens, new_tokens, free_pages, free_count,
               page_size):
    R, dev, T = seq_lens.numel(), block_table.device, slots.numel()
    _written(slots, (T,), torch.int32, dev, "slot_mapping")
    _written(pos, (T,), torch.int32, dev, "positions")
    _written(cu, (R + 1,), torch.int32, dev, "cu_seqlens_q")
    _written(granted, (R,), torch.bool, dev, "granted")
    _extend((slots, pos, cu, granted), block_table, seq_lens, new_tokens, free_pages, free_count,
            page_size, T)


def _op_token_tables(out, lens, block_table, seq_lens, cu_seqlens_q):
    _check(out.dim() == 2 and block_table.dim() == 2 and out.size(1) <= block_table.size(1),
           "out must be [tokens, cols] of a block table's first columns")
    _written(out, tuple(out.shape), torch.int32, block_table.device, "out")
    _written(lens, (out.size(0),), torch.int32, block_table.device, "lens")
    _token_tables(out, lens, block_table, seq_lens, cu_seqlens_q)


def _op_shared_lengths(out, block_table, seq_lens, cu_shared, page_size):
    _check(cu_shared.dim() == 1 and cu_shared.size(0) >= 1, "cu_shared must be int32 [groups + 1]")
    _written(out, (cu_shared.size(0) - 1,), torch.int32, block_table.device, "out")
    _shared_lengths(out, block_table, seq_lens, cu_shared, page_size)


ops.define("extend_tables(Tensor(a!) slot_mapping, Tensor(b!) positions, Tensor(c!) cu_seqlens_q, "
           "Tensor(d!) granted, Tensor(e!) block_table, Tensor(f!) seq_lens, Tensor new_tokens, "
           "Tensor free_pages, Tensor(g!) free_count, int page_size) -> ()", _op_extend)
ops.define("truncate_tables(Tensor(a!) block_table, Tensor(b!) seq_lens, Tensor new_lens, "
           "Tensor(c!) free_pages, Tensor(d!) free_count, int page_size) -> ()", _truncate)
ops.define("token_tables(Tensor(a!) out, Tensor(b!) lens, Tensor block_table, Tensor seq_lens, "
           "Tensor cu_seqlens_q) -> ()", _op_token_tables)
ops.define("shared_lengths(Tensor(a!) out, Tensor block_table, Tensor seq_lens, Tensor cu_shared, "
           "int page_size) -> ()", _op_shared_lengths)
