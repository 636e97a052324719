"""What the microscaled rows refuse before they reach the library: runs without a GPU."""
import importlib

import pytest
import torch

bts = importlib.import_module("bot-sort-onnx-tensorrt_amd")


@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_rows_live_on_a_gpu(device):
    """room for rows in host memory would hand its address to a kernel"""
    with pytest.raises(bts.BtsError):
        bts.MxRows.empty(4, 64, "e2m1", device=device)
    with pytest.raises(bts.BtsError):
        bts.MxRows(torch.zeros((4, 64), dtype=torch.uint8, device=device), torch.zeros((4, 4), dtype=torch.uint8, device=device), 64, "e2m1")


def test_host_tensors_are_refused():
    for call in (lambda: bts.mx_quantize(torch.ones(4, 64)), lambda: bts.rms_norm_mx(torch.ones(4, 64))):
        with pytest.raises(bts.BtsError):
            call()


def test_forward_mode_tangents_are_refused(monkeypatch):
    from torch.autograd import forward_ad
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    x, w = torch.ones(2, 64), torch.ones(64)
    with forward_ad.dual_level():
        dx, dw = forward_ad.make_dual(x, x), forward_ad.make_dual(w, w)
        for call in (lambda: bts.mx_quantize(dx), lambda: bts.rms_norm_mx(dx), lambda: bts.rms_norm_mx(x, residual=dx), lambda: bts.rms_norm_mx(x, weight=dw)):
            with pytest.raises(bts.BtsError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(bts.BtsError, match="tangent"):       # (forward mode goes on there)
                call()
