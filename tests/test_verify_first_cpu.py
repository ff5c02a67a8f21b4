"""DsaLayer.verify_tree refuses bad metadata and indexer tensors before it writes a cache:
on CPU tensors, whose own refusal comes from the first launch."""
import pytest
import torch

from test_verify_tree_cpu import args

I32 = dict(dtype=torch.int32)


@pytest.mark.parametrize("kw,msg", [
    (dict(block_table=torch.zeros(1, 1, dtype=torch.int64)), "block_table must be int32"),
    (dict(block_table=torch.zeros(1, **I32)), "block_table must be int32"),
    (dict(seq_lens=torch.ones(1, dtype=torch.int64)), "seq_lens must be int32"),
    (dict(seq_lens=torch.ones(2, **I32)), "seq_lens must be int32"),
    (dict(cu_seqlens_q=torch.zeros(1, **I32)), "cu_seqlens_q must be int32"),
    (dict(tree_mask=torch.zeros(3, dtype=torch.int64)), "tree_mask must be int64"),
    (dict(tree_mask=torch.zeros(2, **I32)), "tree_mask must be int64"),
    (dict(tree_mask=torch.zeros(2, dtype=torch.int64, device="meta")), "one GPU"),
    (dict(idx_k=torch.zeros(2, 64).half()), "idx_k must be"),
    (dict(idx_k=torch.zeros(2, 128, dtype=torch.float64)), "idx_k and idx_q must be"),
    (dict(idx_k=torch.zeros(2, 256).half()[:, ::2]), "idx_k and idx_q must be"),
    (dict(idx_k=torch.zeros(2, 128).half().requires_grad_()), "no backward pass"),
    (dict(idx_k=torch.zeros(2, 128).half()), "GPU")])
def test_refuses(pkg, kw, msg):
    m = pkg.dsa_layer
    w = m.DsaLayerWeights(torch.zeros(3, 128, 512).half(), torch.zeros(3, 512, 128).half(), 0.1)
    L = m.DsaLayer(w, torch.zeros(2, 16, 576).half(), torch.zeros(2, 16, 128).half())
    with pytest.raises(RuntimeError, match=msg):
        L.verify_tree(**{**args(pkg), **kw})
