"""What DsaLayer.verify_tree refuses, on CPU tensors."""
import pytest
import torch


def args(pkg, T=2, H=3):
    return dict(q=torch.zeros(T, H, 192, dtype=torch.float16), kv_c=torch.zeros(T, 512).half(),
                k_pe=torch.zeros(T, 64).half(), positions=torch.zeros(T, dtype=torch.int64),
                table=torch.zeros(8, 64), slot_mapping=torch.zeros(T, dtype=torch.int64),
                block_table=torch.zeros(1, 1, dtype=torch.int32),
                seq_lens=torch.ones(1, dtype=torch.int32),
                cu_seqlens_q=torch.tensor([0, T], dtype=torch.int32),
                tree_mask=torch.zeros(T, dtype=torch.int64))


@pytest.mark.parametrize("kw,msg", [
    (dict(q=torch.zeros(2, 4, 192).half()), "q must be"),
    (dict(q=torch.zeros(2, 3, 128).half()), "q must be"),
    (dict(q=torch.zeros(3, 3, 192).half()), "a slot for each token"),
    (dict(q=torch.zeros(2, 3, 192)), "fp16"),
    (dict(positions=torch.zeros(1, dtype=torch.int64)), "positions"),
    ({}, "GPU"),
])
def test_refuses(pkg, kw, msg):
    m = pkg.dsa_layer
    w = m.DsaLayerWeights(torch.zeros(3, 128, 512).half(), torch.zeros(3, 512, 128).half(), 0.1)
    L = m.DsaLayer(w, torch.zeros(2, 16, 576).half(), torch.zeros(2, 16, 128).half())
    with pytest.raises(RuntimeError, match=msg):
        L.verify_tree(**{**args(pkg), **kw})
