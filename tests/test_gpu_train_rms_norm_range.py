"""Rows of very large and very small values: the norm behind a fold and its backward hold while a row's squares add up inside the
32-bit range, without eps down to a root mean square of 2^-55, each row for itself."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_train_rms_norm as base  # noqa: E402
from test_gpu_train_rms_norm import AR, DEV, RS, Case  # noqa: E402

WIDTHS = [5, 100, 200, 500, 1000, 9000, 20000]  # a width of each variant


def sizes(cols):
    """Factors for values of order one: up to a sum of squares of 4 * 2^124, down to a mean of 4 * 2^-112."""
    return torch.tensor([2.0 ** 62 * cols ** -0.5, 1e15, 1.0, 1e-14, 2.0 ** -56], device=DEV)[:, None]


@pytest.fixture(autouse=True)
def no_eps(monkeypatch):
    monkeypatch.setattr(base, "EPS", 0.0)


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("kind,stream,out", [("bf16", "bf16", None), ("fp32", "fp32", None), ("bf16", "fp32", "e4m3"), ("fp32", "fp32", "int8")])
def test_forward(kind, stream, out, cols):
    for collective, n in ((AR, 2), (RS, 3)):
        c = Case(collective, n, 5, cols, kind, stream, out=out, seed=cols)
        for v in c.send.views:
            for part in v.view(-1, 5, cols):
                part.copy_(part.float() * sizes(cols))
        for v in c.residual.views:
            v.copy_(v.float() * sizes(cols))
        c.outputs()
        c.run_forward()
        c.check_forward()


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("kind,stream", [("bf16", "bf16"), ("fp32", "fp32"), ("bf16", "fp32")])
def test_backward(kind, stream, cols):
    """The hidden state's rows are large and small, the gradients of order one: the projection that is taken off, h * r^3 * mean(g * weight * h),
    is as large as what it is taken from in every row."""
    for collective, n in ((AR, 2), (RS, 3)):
        c = Case(collective, n, 5, cols, kind, stream, seed=cols)
        c.gradients(arriving=False, both=True)
        for v in c.h.views:
            v.copy_(v.float() * sizes(cols))
        for v in c.send.views:
            v.add_(1.0)  # with a mean, and so a projection
        for v in c.h.views:
            v.copy_(v.float().abs())
        c.run_backward()
        c.check_backward()
