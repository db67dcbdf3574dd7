"""A training step of the relation head for a clip without pairs."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_relation_logits_of_no_pairs():
    from trace_amd.config import TraceConfig
    from trace_amd.model_builder_rel import Generalized_RCNN
    m = Generalized_RCNN(TraceConfig(RESIZE_HIDDEN_DIM=4), conv_bodies=False)
    m.relation_infer_sem.to(DEV)
    m.relation_infer_spa.to(DEV)
    m.train()
    K = m.relation_infer_sem[2].in_features
    a, b = (torch.zeros((0, K), dtype=torch.bfloat16, device=DEV, requires_grad=True) for _ in range(2))
    out = m.relation_logits_train(a, b, 11, 3)
    assert out.shape == (0, m.cfg.NUM_PRD_CLASSES)
    out.sum().backward()
    assert a.grad.shape == a.shape
    assert not m.relation_infer_sem[2].weight.grad.any() and not m.relation_infer_sem[2].bias.grad.any()


@pytest.mark.parametrize("relu", [False, True])
def test_gemm_nt_gradients_of_no_rows(relu):
    from trace_amd import autograd as tag
    x = torch.zeros((0, 64), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    w, b = torch.randn((40, 64), device=DEV, requires_grad=True), torch.randn(40, device=DEV, requires_grad=True)
    y = tag.gemm_nt(x, w, b, relu)
    assert y.shape == (0, 40)
    y.float().sum().backward()
    for t in (x, w, b):
        assert t.grad.shape == t.shape and t.grad.dtype == t.dtype and not t.grad.any()
