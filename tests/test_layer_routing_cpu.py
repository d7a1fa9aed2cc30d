"""The one-GPU layers refuse routing arguments whose shapes do not belong together, before anything is launched: transposed
weights have as many entries as the pairs and used to give an output of the wrong shape."""

import pytest
import torch

from triton_grouped_gemm_b200.ep.autograd import moe_ffn
from triton_grouped_gemm_b200.ep.w4_layer import W4MoELayer

BF = torch.bfloat16
X, IDX, WEIGHT = torch.zeros(6, 32, dtype=BF), torch.zeros(6, 2, dtype=torch.int64), torch.zeros(6, 2)
W13, W2 = torch.zeros(2, 64, 32, dtype=BF), torch.zeros(2, 32, 32, dtype=BF)


def _w4(x, idx, weight):
    layer = W4MoELayer.__new__(W4MoELayer)     # without the quantiser, which needs a GPU
    layer.num_experts, layer.activation = 2, "silu"
    layer.w13 = layer.w2 = None
    return layer(x, idx, weight)


@pytest.mark.parametrize("layer", [lambda *a: moe_ffn(*a, W13, W2), _w4])
def test_shapes(layer):
    for idx, weight in ((IDX, WEIGHT.t()), (IDX, WEIGHT[:, :1]), (IDX, WEIGHT[:5]), (IDX, WEIGHT.reshape(-1))):
        with pytest.raises(AssertionError, match="topk_weight must have topk_idx's shape"):
            layer(X, idx, weight)
    for idx in (IDX.t(), IDX[:5], IDX.reshape(-1)):
        with pytest.raises(AssertionError, match="topk_idx 2D"):
            layer(X, idx, WEIGHT)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        layer(X, IDX, WEIGHT)
