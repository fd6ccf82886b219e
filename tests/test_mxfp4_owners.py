"""MXFP4 keys at the expert owners of a parallel layer: what is refused before any exchange (no GPU), and the owners'
steps on source-major segments against each source by itself."""

import pytest
import torch

from mirai_b200 import expert_parallel as ep
from mirai_b200 import ops


def keys_of_shape(E, H, I):
    """Three MXFP4 keys without buffers: enough for what a call looks at before it launches anything."""
    keys = []
    for out, inp in ((I, H), (I, H), (H, I)):
        w = ops.Mxfp4Tensor.__new__(ops.Mxfp4Tensor)
        w.shape, w.device = (E, out, inp), torch.device("cpu")
        keys.append(w)
    return tuple(keys)


@pytest.mark.parametrize("H,I", [(96, 64), (64, 160)])
def test_training_widths_are_refused_before_any_exchange(H, I, monkeypatch):
    """Every rank refuses alike: none is left waiting for a peer that stopped at its owner's GEMMs, or in the backward."""
    def exchange(*a, **k):
        raise AssertionError("an exchange began")
    monkeypatch.setattr(ep.dist, "all_to_all_single", exchange)
    monkeypatch.setattr(ep.dist, "all_gather_into_tensor", exchange)
    E, T, k = 4, 6, 2
    shard = ep.ExpertShard(E, 2, 0)
    x, logits = torch.zeros(T, H, dtype=torch.bfloat16), torch.zeros(T, E)
    with pytest.raises(ValueError, match="steps of 64"):
        ep.ep_moe_forward(x, logits, keys_of_shape(2, H, I), shard=shard, top_k=k, inter=I, train=True)
    layer = ep.ExpertParallelMoE.__new__(ep.ExpertParallelMoE)
    layer.ops, layer.shard, layer.top_k, layer.inter, layer._gen = ep.CudaStepOps(), shard, k, I, 0
    with pytest.raises(ValueError, match="steps of 64"):
        layer.forward(x, logits, keys_of_shape(2, H, I), train=True)
    assert layer._gen == 0
    with pytest.raises(ValueError, match="steps of 64"):
        ep.CudaStepOps().experts_train(x, None, keys_of_shape(E, H, I), I)
