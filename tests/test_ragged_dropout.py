"""HipRaggedAttention does not drop attention weights, and says so in place of training without."""
import pytest
import torch

from hipkittens_b200.attention import HipRaggedAttention


def test_a_rate_is_refused_in_training(native_built):
    q, kv = torch.zeros(10, 4, 64, dtype=torch.bfloat16), torch.zeros(10, 2, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 10], dtype=torch.int32)
    module = HipRaggedAttention(attention_dropout=0.1)
    with pytest.raises(RuntimeError, match="no dropout"):
        module(q, kv, cu)
    # without it, and where none would be applied, the call goes on to what else it asks for
    for other in (module.eval(), HipRaggedAttention(), HipRaggedAttention(attention_dropout=0.0).train()):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            other(q, kv, cu)
