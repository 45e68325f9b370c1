"""An Int8MLP keeps its layout, and with it the kernel for both layers, wherever its buffers come from."""
import copy
import io

import pytest
import torch

pytestmark = pytest.mark.gpu


def _quick(k=66, n=18):
    from npa_b200.int8 import Int8MLP
    torch.manual_seed(0)
    return Int8MLP(torch.nn.Sequential(torch.nn.Linear(k, 128), torch.nn.ReLU(), torch.nn.Linear(128, n, bias=False)).cuda())


def _moved(quick):
    """The module after everything that gives its buffers other memory."""
    from npa_b200.int8 import Int8MLP
    saved = io.BytesIO()
    torch.save(quick, saved)
    saved.seek(0)
    k, n = quick.in_features, quick.out_features
    fresh = lambda: Int8MLP(torch.nn.Sequential(torch.nn.Linear(k, 128), torch.nn.ReLU(), torch.nn.Linear(128, n, bias=False)).cuda())
    dense = {name: value.detach().clone(memory_format=torch.contiguous_format) for name, value in quick.state_dict().items()}
    loaded, assigned = fresh(), fresh()
    loaded.load_state_dict(dense)
    assigned.load_state_dict(dense, assign=True)
    return {"cpu and back": copy.deepcopy(quick).cpu().cuda(), "copied": copy.deepcopy(quick), "saved": torch.load(saved, weights_only=False),
            "loaded": loaded, "assigned": assigned, "empty": copy.deepcopy(quick).to_empty(device="cuda"), "to": copy.deepcopy(quick).to("cpu").to("cuda:0")}


def _kernels(call):
    call()
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    return [e.name for e in p.events() if e.device_type == torch.autograd.DeviceType.CUDA]


@pytest.mark.parametrize("k,n", [(66, 18), (163, 35), (64, 16)])
def test_buffers_that_were_moved(k, n):
    quick = _quick(k, n)
    z = torch.randn(500, k, device="cuda")
    want = quick(z)
    before = {name: (value.shape, value.dtype) for name, value in quick.state_dict().items()}
    for how, module in _moved(quick).items():
        assert {name: (value.shape, value.dtype) for name, value in module.state_dict().items()} == before, how
        for w in (module.w1, module.w2):
            assert w.stride(0) % 16 == 0 and w.stride(1) == 1 and w.data_ptr() % 16 == 0, (how, w.stride())
        if how != "empty":  # its values are anything
            assert torch.equal(module(z), want), how


def test_one_launch_after_a_move():
    quick = _quick()
    z = torch.randn(500, 66, device="cuda")
    for how, module in _moved(quick).items():
        names = _kernels(lambda: module(z))
        assert len(names) == 1 and "mlp_int8_kernel" in names[0], (how, names)
