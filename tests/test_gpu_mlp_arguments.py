"""Calls of the adaptation MLP whose tensors do not fit one another are refused before a kernel reads behind one of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _module(k, o):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(k, 128), torch.nn.ReLU(), torch.nn.Linear(128, o, bias=False)).cuda()


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("checkpoint", [True, False])
@pytest.mark.parametrize("engine", ["tcgen05", "mma.sync"])
def test_rows_of_another_width(engine, checkpoint, grad, monkeypatch):
    from npa_b200 import mlp
    monkeypatch.setattr(mlp, "TENSOR_ENGINE", engine)
    module = _module(66, 18)
    for p in module.parameters():
        p.requires_grad_(grad)
    for shape in ((40, 200), (40, 65), (40, 0), ()):
        with pytest.raises((RuntimeError, ValueError)):
            mlp.apply_mlp(module, torch.ones(shape, device="cuda"), checkpoint=checkpoint)


@pytest.mark.parametrize("grad", [True, False])
def test_the_operators_themselves(grad):
    from npa_b200 import _native as n
    module = _module(66, 18)
    w1, b1, w2 = (p.detach().requires_grad_(grad) for p in module.parameters())
    z = torch.randn(40, 66, device="cuda")
    for call in (n.ops.mlp, n.ops.mlp_checkpoint):
        for wrong in (z[:, :65].contiguous(), torch.randn(40, 200, device="cuda"), z[:, :0], z[0, 0]):
            with pytest.raises(RuntimeError, match="66 columns"):
                call(wrong, w1, b1, w2)
        with pytest.raises(TypeError, match="expected float32 tensors on"):
            call(z, w1, b1.detach().cpu(), w2)
        with pytest.raises(TypeError, match="expected float32 tensors on"):
            call(z, w1, b1, w2.detach().cpu())
        with pytest.raises(TypeError, match="expected float32 tensors on"):
            call(z, w1, b1.detach().half(), w2)
        with pytest.raises(RuntimeError, match="at least one input"):
            call(z[:, :0], w1[:, :0], b1, w2)
        gap = torch.zeros(256, device="cuda")[::2]
        gap.copy_(b1)
        assert torch.equal(call(z, w1, gap, w2), call(z, w1, b1, w2))
