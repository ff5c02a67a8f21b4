"""DsaLayer.verify_tree refuses tables of more than topk positions without the indexer's
tensors, before anything is launched."""
import pytest
import torch

from test_verify_tree_cpu import args


@pytest.mark.parametrize("kw,msg", [
    ({}, "more than topk = 16 positions"),
    (dict(idx_q=torch.zeros(2, 32, 128).half()), "more than topk = 16 positions"),
    (dict(idx_q=torch.zeros(2, 32, 64).half(), idx_w=torch.zeros(2, 32).half()), "idx_q must be"),
    (dict(idx_q=torch.zeros(2, 32, 128).half(), idx_w=torch.zeros(1, 32).half()), "idx_q must be"),
    (dict(block_table=torch.zeros(1, 1, dtype=torch.int32)), "GPU"),  # 16 positions: none needed
])
def test_refuses(pkg, kw, msg):
    m = pkg.dsa_layer
    w = m.DsaLayerWeights(torch.zeros(3, 128, 512).half(), torch.zeros(3, 512, 128).half(), 0.1)
    L = m.DsaLayer(w, torch.zeros(4, 16, 576).half(), torch.zeros(4, 16, 128).half(), topk=16)
    with pytest.raises(RuntimeError, match=msg):
        L.verify_tree(**{**args(pkg), "block_table": torch.zeros(1, 2, dtype=torch.int32), **kw})


def test_page_of_the_indexer_cache(pkg):
    m = pkg.dsa_layer
    w = m.DsaLayerWeights(torch.zeros(3, 128, 512).half(), torch.zeros(3, 512, 128).half(), 0.1)
    L = m.DsaLayer(w, torch.zeros(4, 24, 576).half(), torch.zeros(4, 24, 128).half(), topk=16)
    kw = dict(idx_q=torch.zeros(2, 32, 128).half(), idx_w=torch.zeros(2, 32).half())
    with pytest.raises(RuntimeError, match="power of two"):
        L.verify_tree(**{**args(pkg), **kw})
