"""The norm behind a fold and its backward where every row begins on a cache line and the last vector of a row does not
lie on the vectors' grid: such a vector is moved back to end with the row, to any element boundary.  Rows that end on a 4-byte
boundary leave by buffer stores, others through the caches; both against 64 bits, with the bytes around the rows watched."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_train_rms_norm as base  # noqa: E402
from test_gpu_train_rms_norm import AR, DEV, RS, Case  # noqa: E402

LINE = 128  # elements: whole lines of every type


class OnLines:
    """`count` matrices, each in an allocation of its own and its rows cols + gap elements apart, with a known fill around the rows."""

    def __init__(self, count, rows, cols, dtype, offset=0, gap=0):
        self.rows, self.cols, self.stride = rows, cols, cols + gap
        size = (rows * self.stride + LINE) * dtype.itemsize
        self.raw = [torch.full((size,), 0xA5, dtype=torch.uint8, device=DEV) for _ in range(count)]
        self.views = [b.view(dtype)[:rows * self.stride].view(rows, self.stride)[:, :cols] for b in self.raw]
        assert all(v.data_ptr() % 128 == 0 for v in self.views)

    def all(self):
        return torch.stack([v.clone() for v in self.views])

    def fill(self, values):
        for v, x in zip(self.views, values):
            v.copy_(x)
        return self

    def intact(self):
        for b, v in zip(self.raw, self.views):
            around = torch.ones(b.numel(), dtype=torch.bool, device=DEV)
            size = v.element_size()
            around[:self.rows * self.stride * size].view(self.rows, self.stride * size)[:, :self.cols * size] = False
            if not bool((b[around] == 0xA5).all()):
                return False
        return True


# each variant's widths, one to three elements off a multiple of four, and even ones off a multiple of eight
WIDTHS = [131, 257, 509, 510, 511, 513, 1001, 1002, 4099, 4100, 5001, 8191, 8193, 8201, 8206, 12292, 16383]


@pytest.fixture(autouse=True)
def on_lines(monkeypatch):
    monkeypatch.setattr(base, "Strided", OnLines)


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("kind,stream,out", [("bf16", "bf16", None), ("fp16", "fp32", None), ("bf16", "bf16", "e4m3"), ("fp16", "fp16", "int8"),
                                             ("fp32", "fp32", "e4m3")])
def test_forward(kind, stream, out, rows, cols):
    for collective, n in ((AR, 3), (RS, 2), (AR, 1)):
        c = Case(collective, n, rows, cols, kind, stream, out=out, gap=-cols % LINE, seed=cols)
        c.outputs()
        c.run_forward()
        c.check_forward()
        assert c.hidden.intact() and c.y.intact() and (c.scales is None or c.scales.intact())


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("kind,stream", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp32"), ("fp32", "fp32")])
def test_backward(kind, stream, rows, cols):
    for collective, n, both in ((AR, 3, True), (RS, 2, True), (AR, 1, False)):
        c = Case(collective, n, rows, cols, kind, stream, gap=-cols % LINE, seed=cols)
        c.gradients(both=both)
        c.run_backward()
        c.check_backward()
        assert c.dh.intact() and c.dw.intact() and (c.dsend is None or c.dsend.intact())


@pytest.mark.parametrize("cols", [509, 4099, 8201])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_in_place(cols, kind):
    """The outputs in the inputs' places: the bits of the call beside them."""
    for collective in (AR, RS):
        n, rows, gap = 2, 3, -cols % LINE
        c = Case(collective, n, rows, cols, kind, gap=gap, seed=cols)
        c.outputs()
        c.run_forward()
        want = c.y.all(), c.hidden.all()
        own = [v if c.gathered else v[r * rows:(r + 1) * rows] for r, v in enumerate(c.send.views)]
        hidden = [c.residual.views[0]] + c.hidden.views[1:] if c.gathered else c.residual.views
        args, more = c.forward_args()
        more["residual_outs"] = hidden
        call = base.mr.all_reduce_rms_norm if c.gathered else base.mr.reduce_scatter_rms_norm
        call(args[0], own, *args[2:], **more)
        torch.cuda.synchronize()
        assert torch.equal(torch.stack(own), want[0]) and torch.equal(torch.stack(hidden), want[1])
        assert c.send.intact() and c.residual.intact()
