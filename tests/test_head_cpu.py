"""The C entry points of the head and of the distillation loss refuse what their declarations exclude, before a device is
touched; the Python calls refuse CPU tensors."""
import ctypes

import pytest
import torch

FAKE = 4096  # non-NULL, 16-byte aligned, never dereferenced on these paths


@pytest.fixture(scope="module")
def L():
    from ddfnet_b200.csrc import build
    build.build()
    from ddfnet_b200 import _lib
    return _lib.load()


def test_top_logits(L):
    call = lambda rows=2, classes=100, stride=100, k=5, t=1.0, dtype=0, p=FAKE: L.ddf_b200_top_logits(
        p, FAKE, FAKE, FAKE, rows, classes, stride, k, t, dtype, None)
    assert call(p=None) == -1
    for bad in ({"rows": 0}, {"classes": 0}, {"k": 0}, {"k": 101}, {"stride": 99}, {"t": 0.0}, {"t": float("nan")},
                {"t": float("inf")}, {"t": -1.0}, {"classes": 1000, "stride": 1000, "k": 257}):
        assert call(**bad) == -12, bad
    assert call(classes=1 << 31, stride=1 << 31) == -9
    assert L.ddf_b200_strerror(-12).startswith(b"ddf_b200:")


def test_distill(L):
    from ddfnet_b200 import _lib

    def args(**kw):
        a = {"logits": FAKE, "values": FAKE, "indices": FAKE, "rest": None, "rows": 2, "classes": 100, "row_stride": 100, "k": 5,
             "dtype": 0, "values_dtype": 0, "wide_indices": 1, "reduction": _lib.MEAN, "temperature": 1.0, **kw}
        return ctypes.byref(_lib.DistillArgs(**a))
    forward = lambda a: L.ddf_b200_distill_forward(a, FAKE, FAKE, FAKE, FAKE, None)
    both = lambda a: L.ddf_b200_distill_loss_grad(a, FAKE, FAKE, FAKE, 1.0, FAKE, None)
    backward = lambda a: L.ddf_b200_distill_backward(a, FAKE, FAKE, FAKE, 0, FAKE, None)
    for call in (forward, both, backward):
        assert call(None) == -1
        for bad, status in (({"logits": None}, -1), ({"indices": None}, -1), ({"rows": 0}, -12), ({"k": 0}, -12), ({"k": 257}, -12),
                            ({"row_stride": 99}, -12), ({"temperature": 0.0}, -12), ({"reduction": 3}, -12), ({"dtype": 3}, -5),
                            ({"values_dtype": 9}, -5), ({"classes": (1 << 23) + 1, "row_stride": 1 << 24}, -9)):
            assert call(args(**bad)) == status, bad


def test_linear(L):
    from ddfnet_b200 import _lib

    def args(**kw):
        a = {"x": FAKE, "weight": FAKE, "bias": None, "residual": None, "rows": 4, "inputs": 32, "outputs": 16, "x_stride": 32,
             "weight_stride": 32, "residual_stride": 16, "activation": 0, "after": 0, "dtype": 1, **kw}
        return ctypes.byref(_lib.LinearArgs(**a))
    forward = lambda a: L.ddf_b200_linear_forward(a, FAKE, None, None, 0, None)
    backward = lambda a: L.ddf_b200_linear_backward(a, FAKE, 16, None, FAKE, FAKE, None, None, None, 0, None)
    for call in (forward, backward):
        assert call(None) == -1
        for bad, status in (({"x": None}, -1), ({"weight": None}, -1), ({"rows": 0}, -12), ({"inputs": 0}, -12), ({"x_stride": 31}, -12),
                            ({"weight_stride": 8}, -12), ({"activation": 4}, -12), ({"activation": -1}, -12), ({"dtype": 0}, -5),
                            ({"dtype": 3}, -5), ({"residual": FAKE, "residual_stride": 8}, -12), ({"rows": (1 << 30) + 1}, -9)):
            assert call(args(**bad)) == status, bad
    assert L.ddf_b200_linear_forward(args(), None, None, None, 0, None) == -1
    assert L.ddf_b200_linear_backward(args(activation=2), FAKE, 16, None, FAKE, None, None, None, None, 0, None) == -1
    assert L.ddf_b200_linear_backward(args(), FAKE, 8, None, FAKE, None, None, None, None, 0, None) == -12
    assert L.ddf_b200_linear_waitlimit(args(), FAKE, None, 0, 0, 0, None) == -12
    assert L.ddf_b200_linear_workspace(args(rows=0)) == 0


def test_cpu_tensors_are_refused():
    from ddfnet_b200 import distill_loss, distill_loss_grad, linear_act, top_logits
    x, i = torch.zeros(3, 10), torch.zeros(3, 2, dtype=torch.int64)
    for call in (lambda: top_logits(x, 2), lambda: distill_loss(x, x[:, :2], i), lambda: distill_loss_grad(x, x[:, :2], i),
                 lambda: linear_act(x.half(), x.half())):
        with pytest.raises(ValueError, match="CUDA"):
            call()
