"""What the training modules and the 4-bit experts refuse before anything runs (no GPU)."""
import pytest
import torch

from light_moe_b200.fp4 import FP4Experts, FP4MoELayer
from light_moe_b200.grouped import GroupedExperts, GroupedLinear, grouped_linear

OFF = torch.tensor([0, 2, 4])


@pytest.mark.parametrize("x,w,off", [
    (torch.zeros(4, 8), torch.zeros(2, 6, 7), OFF), (torch.zeros(4, 8), torch.zeros(6, 8), OFF),
    (torch.zeros(4, 2, 8), torch.zeros(2, 6, 8), OFF), (torch.zeros(4, 8), torch.zeros(2, 6, 8).half(), OFF),
    (torch.zeros(4, 8).double(), torch.zeros(2, 6, 8).double(), OFF), (torch.zeros(4, 8), torch.zeros(2, 6, 8), OFF[:2]),
])
def test_grouped_linear_refusals(x, w, off):
    with pytest.raises(ValueError):
        grouped_linear(x, w, off)


def test_experts_refusals_and_parameters():
    m = GroupedExperts(2, 8, 6)
    assert [tuple(p.shape) for p in m.parameters()] == [(2, 6, 8), (2, 6, 8), (2, 8, 6)]
    bound = 8 ** -0.5
    assert m.gate_proj.weight.abs().max() <= bound and "num_experts=2" in repr(GroupedLinear(2, 8, 6))
    x, ids, w = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    for bad in ((x, ids, w[:, :1]), (x[:2], ids, w), (x, ids[:, :0], w[:, :0]), (x, ids[0], w[0]), (x[None], ids, w)):
        with pytest.raises(ValueError):
            m(*bad)


def test_fp4_layer_refusals():
    z = torch.zeros
    for w1, w3, w2 in ((z(2, 64, 48), z(2, 64, 48), z(2, 48, 64)), (z(2, 64, 32), z(2, 32, 32), z(2, 32, 64)),
                       (z(2, 64, 32), z(2, 64, 32), z(2, 64, 32))):
        with pytest.raises(ValueError):
            FP4Experts.from_dense(w1, w3, w2)
    ex = FP4Experts("mxfp4", (None, None), (None, None), (None, None), None, None, None, 2, 0, 32, 64)
    with pytest.raises(ValueError):
        FP4MoELayer(z(3, 32), ex, 1)
    with pytest.raises(ValueError):
        FP4MoELayer(z(2, 32), ex, 1, input_scale=torch.ones(1))


def test_fp4_layer_refuses_hidden_sizes_that_its_router_does_not_take():
    z = torch.zeros
    for d in (32, 96):
        ex = FP4Experts("mxfp4", (None, None), (None, None), (None, None), None, None, None, 2, 0, d, 64)
        with pytest.raises(ValueError, match="64"):
            FP4MoELayer(z(2, d), ex, 1)
    ex = FP4Experts("mxfp4", (None, None), (None, None), (None, None), None, None, None, 2, 0, 192, 32)
    FP4MoELayer(z(2, 192), ex, 1)
