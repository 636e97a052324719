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


def test_what_is_not_a_tensor_is_refused_by_name(monkeypatch):
    """lists, arrays and rows of another kind: the package's error, saying which argument"""
    import numpy as np
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    x, rows, a = torch.ones(2, 64), bts.MxRows.empty(2, 64, "e4m3", device="cpu"), np.ones((2, 64), np.float32)
    for name, call in (("x", lambda: bts.mx_quantize([[1.0] * 64])), ("x", lambda: bts.mx_quantize(a)), ("x", lambda: bts.rms_norm_mx(a)), ("x", lambda: bts.mx_quantize(None)),
                       ("out", lambda: bts.mx_quantize(x, "e4m3", out=x)), ("out", lambda: bts.rms_norm_mx(x, out=torch.ones(2, 64))),
                       ("residual", lambda: bts.rms_norm_mx(x, residual=a)), ("weight", lambda: bts.rms_norm_mx(x, weight=a[0])),
                       ("weight", lambda: bts.rms_norm_mx(x, weight=[1.0] * 64)), ("sum_out", lambda: bts.rms_norm_mx(x, sum_out=a)),
                       ("y_out", lambda: bts.rms_norm_mx(x, y_out=rows)), ("out", lambda: bts.mx_product(rows, rows, out=a)),
                       ("out", lambda: bts.mx_product(rows, rows, out=rows)), ("MxRows", lambda: bts.mx_product(rows, x)),
                       ("codes", lambda: bts.MxRows(np.zeros((2, 128), np.uint8), rows.scales, 64, "e4m3")), ("scales", lambda: bts.MxRows(rows.codes, None, 64, "e4m3"))):
        with pytest.raises(bts.BtsError, match=name):
            call()


def test_views_that_hold_the_negative_are_refused(monkeypatch):
    """the imaginary part of a conjugate is a view whose memory holds the other sign: one column of it has rows like any matrix's"""
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    z = torch.complex(torch.ones(4, 1), torch.ones(4, 1)).conj().imag
    assert z.is_neg() and (z == -1).all()
    for call in (lambda: bts.mx_quantize(z), lambda: bts.rms_norm_mx(z), lambda: bts.rms_norm_mx(torch.ones(4, 1), weight=z[0])):
        with pytest.raises(bts.BtsError, match="conjugate"):
            call()
