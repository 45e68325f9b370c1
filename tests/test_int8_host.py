"""CPU-only checks of the 8-bit operators: refusals of tensors that are not on a GPU, and of the C ABI before any launch."""
import ctypes

import pytest
import torch


def test_host_tensors_are_refused():
    from npa_b200.int8 import dequantize_rows, linear_int8, mlp_int8, quantize_rows
    from npa_b200.rows8 import Rows8, compress_rows
    x, w, t = torch.randn(3, 8), torch.zeros(4, 8, dtype=torch.int8), torch.ones(4)
    for call in (lambda: quantize_rows(x), lambda: dequantize_rows(w, t), lambda: linear_int8(x, w, t), lambda: mlp_int8(x, w, t, t, w, t), lambda: compress_rows(x),
                 lambda: Rows8(w, torch.zeros(4, 1, dtype=torch.uint8), torch.float32).restore()):
        with pytest.raises(TypeError, match="CUDA tensor"):
            call()


def test_bad_arguments_of_the_c_abi():
    """Addresses here are never dereferenced: the checks come first."""
    from npa_b200 import _native as n
    lib, ok, odd = n.lib, ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 1)
    F32, F16, I8 = 0, 1, 3
    inv, uns, small = n.NPA_ERR_INVALID_ARGUMENT, n.NPA_ERR_UNSUPPORTED, n.NPA_ERR_SCRATCH_TOO_SMALL
    calls = [
        (inv, "positive", lib.npa_quantize_rows(ok, F32, 8, 0, 8, ok, I8, 16, ok, None)),
        (inv, "floating", lib.npa_quantize_rows(ok, I8, 8, 1, 8, ok, I8, 16, ok, None)),
        (inv, "8-bit", lib.npa_quantize_rows(ok, F32, 8, 1, 8, ok, F32, 16, ok, None)),
        (inv, "non-NULL", lib.npa_quantize_rows(ok, F32, 8, 1, 8, None, I8, 16, ok, None)),
        (inv, "aligned", lib.npa_quantize_rows(odd, F16, 8, 1, 8, ok, I8, 16, ok, None)),
        (inv, "overlap", lib.npa_quantize_rows(ok, F32, 8, 1, 8, ok, I8, 4, ok, None)),
        (inv, "floating", lib.npa_dequantize_rows(ok, I8, 16, ok, 1, 8, ok, I8, None)),
        (inv, "positive", lib.npa_linear_int8(ok, F32, 8, None, ok, 8, ok, None, 0, 0, ok, F32, 1, 8, 0, ok, 1 << 20, None)),
        (uns, "65536", lib.npa_linear_int8(ok, F32, 8, None, ok, 8, ok, None, 0, 0, ok, F32, 1, 65537, 8, ok, 1 << 20, None)),
        (inv, "scales", lib.npa_linear_int8(ok, I8, 8, None, ok, 8, ok, None, 0, 0, ok, F32, 1, 8, 8, None, 0, None)),
        (inv, "scratch", lib.npa_linear_int8(ok, F32, 8, None, ok, 16, ok, None, 0, 0, ok, F32, 100, 8, 8, None, 0, None)),
        (small, "needed", lib.npa_linear_int8(ok, F32, 8, None, ok, 16, ok, None, 0, 0, ok, F32, 100, 8, 8, ok, 8, None)),
        (inv, "unknown type", lib.npa_linear_int8(ok, 9, 8, None, ok, 8, ok, None, 0, 0, ok, F32, 1, 8, 8, ok, 1 << 20, None)),
        (inv, "must be there", lib.npa_mlp_int8(ok, 8, ok, 16, ok, None, ok, 128, ok, ok, 1, 8, 128, 4, ok, 1 << 20, None)),
        (uns, "2^30 columns", lib.npa_quantize_rows(ok, F32, 0, 1, (1 << 31) - 8, ok, I8, 1 << 31, ok, None)),
        (uns, "2^30 columns", lib.npa_dequantize_rows(ok, I8, 0, ok, 1, (1 << 30) + 1, ok, F32, None)),
        (uns, "2^30 columns", lib.npa_rows8_compress(ok, F32, 0, 1, (1 << 31) - 1, ok, 1 << 31, ok, None)),
        (uns, "2^30 columns", lib.npa_rows8_restore(ok, 1 << 31, ok, 1, (1 << 30) + 1, ok, F32, None)),
        (inv, "positive", lib.npa_rows8_compress(ok, F32, 8, 1, 0, ok, 16, ok, None)),
        (inv, "overlap", lib.npa_rows8_compress(ok, F32, 8, 1, 8, ok, 7, ok, None)),
        (inv, "unknown type", lib.npa_rows8_restore(ok, 16, ok, 1, 8, ok, I8, None)),
        (uns, "out <= 48", lib.npa_mlp_checkpoint_forward(ok, ok, ok, ok, ok, 1, 8, 49, 8, 1, 128, 1, ok, ok, ok, ok, 1 << 24, None)),
        (small, "needed", lib.npa_mlp_checkpoint_forward(ok, ok, ok, ok, ok, 1, 8, 4, 8, 1, 128, 1, ok, ok, ok, ok, 16, None)),
        (inv, "aligned", lib.npa_mlp_checkpoint_forward(ok, ok, ok, ok, ok, 1, 8, 4, 8, 1, 128, 1, odd, ok, ok, ok, 1 << 24, None)),
        (inv, "non-NULL", lib.npa_mlp_checkpoint_backward(ok, ok, None, ok, 1 << 24, ok, ok, ok, ok, ok, ok, 1, 8, 4, ok, 1 << 24, None)),
        (inv, "together", lib.npa_mlp_checkpoint_backward(ok, ok, ok, ok, 1 << 24, ok, ok, ok, None, ok, ok, 1, 8, 4, ok, 1 << 24, None)),
        (small, "needed", lib.npa_mlp_checkpoint_backward(ok, ok, ok, ok, 1 << 24, ok, ok, ok, ok, ok, ok, 1, 8, 4, ok, 64, None)),
        (small, "needed", lib.npa_mlp_checkpoint_backward(ok, ok, ok, ok, 64, ok, ok, ok, ok, ok, ok, 1, 8, 4, ok, 1 << 24, None)),
    ]
    # (each message is the last error of its own call only when read at once)
    assert [rc for _, _, rc in calls] == [want for want, _, _ in calls]
    rc = lib.npa_mlp_checkpoint_backward(ok, ok, ok, ok, 1 << 24, ok, ok, ok, None, ok, ok, 1, 8, 4, ok, 1 << 24, None)
    assert rc == inv and "together" in n.last_error()
    room = lib.npa_linear_int8_scratch_bytes
    assert room(ok, I8, 16, ok, 16, 100, 8, 4) == 0 and room(ok, F32, 8, ok, 16, 100, 8, 4) >= 100 * 16 + 400  # codes and scales of the rows
    assert room(odd, I8, 16, ok, 16, 100, 8, 4) >= 100 * 16 and room(ok, I8, 8, ok, 16, 100, 8, 4) >= 100 * 16 and room(ok, I8, 16, odd, 16, 100, 8, 4) >= 4 * 16
    assert room(ok, F32, 8, ok, 16, 1, 8, 4) == 0  # few rows: inside the kernel


def test_int8_module_checks_its_shape_first():
    from npa_b200.int8 import Int8MLP
    for module in (torch.nn.Linear(3, 4), torch.nn.Sequential(torch.nn.Linear(3, 4)), torch.nn.Sequential(torch.nn.Linear(3, 4), torch.nn.ReLU(), torch.nn.Linear(4, 2))):
        with pytest.raises(ValueError, match="Sequential"):
            Int8MLP(module)


def test_checkpoints_of_an_unsupported_module_are_refused():
    from npa_b200.mlp import apply_mlp
    module = torch.nn.Sequential(torch.nn.Linear(8, 128), torch.nn.ReLU(), torch.nn.Linear(128, 4, bias=False))
    with pytest.raises(ValueError, match="checkpoint=True"):
        apply_mlp(module, torch.zeros(3, 8), checkpoint=True)
    with torch.no_grad():
        assert apply_mlp(module, torch.zeros(3, 8), checkpoint=True).shape == (3, 4)
