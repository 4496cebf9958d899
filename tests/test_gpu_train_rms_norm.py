"""The norm behind a fold and its backward against their formulas in 64 bits, on the GPU.

Tolerances are counted from the arithmetic the calls promise (32-bit sums, one rounding of the result):
U = 2^-24 is half a step of a 32-bit value.  A sum of N ranks and a residual is off by at most N * U times the sum of its terms'
magnitudes.  A row's sums pass fewer than 64 additions one behind the other (at most 16 in a lane, 6 across a
wavefront, 16 across a workgroup, for rows up to 16384), so 1 / rms is off by 64 * U relative, plus what the sums' own terms are
off; TAIL = 80 * U covers it with its square root, quotient and products.  A result rounded to type t adds eps(t) / 2."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import megray_amd as mr  # noqa: E402

DEV = "cuda:0"
U = 2.0 ** -24
TAIL = 80 * U
AR, RS = mr.Collective.ALL_REDUCE, mr.Collective.REDUCE_SCATTER
TYPES = {"fp16": (torch.float16, mr.DType.FLOAT16), "bf16": (torch.bfloat16, mr.DType.BFLOAT16), "fp32": (torch.float32, mr.DType.FLOAT32),
         "e4m3": (torch.float8_e4m3fn, mr.DType.FLOAT8_E4M3), "int8": (torch.int8, mr.DType.INT8)}
EPS = 1e-5


def half_step(t):
    return torch.finfo(t).eps / 2


def smallest(t):
    """Half the distance of the type's smallest values: what a rounding among its subnormal values is off."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


class Strided:
    """`count` matrices of rows x cols inside one allocation: an element offset and a row stride of their own, a known
    fill around them.  intact() tells whether anything but the matrices was written."""

    def __init__(self, count, rows, cols, dtype, offset=0, gap=0):
        self.rows, self.cols, self.stride = rows, cols, cols + gap
        size = offset + rows * self.stride + 64
        self.raw = torch.full((count, size * dtype.itemsize), 0xA5, dtype=torch.uint8, device=DEV)
        self.base = self.raw.view(dtype)
        self.views = [b[offset:offset + rows * self.stride].view(rows, self.stride)[:, :cols] for b in self.base]

    def all(self):
        return torch.stack([v.clone() for v in self.views])

    def fill(self, values):
        for v, x in zip(self.views, values):
            v.copy_(x)
        return self

    def intact(self):
        raw = self.raw.clone().view(self.base.dtype)
        offset = self.views[0].storage_offset()
        for b in raw:
            b[offset:offset + self.rows * self.stride].view(self.rows, self.stride)[:, :self.cols].view(torch.uint8 if b.dtype.itemsize == 1 else b.dtype).zero_()
        want = torch.full_like(self.raw, 0xA5).view(self.base.dtype)
        for b in want:
            b[offset:offset + self.rows * self.stride].view(self.rows, self.stride)[:, :self.cols].view(torch.uint8 if b.dtype.itemsize == 1 else b.dtype).zero_()
        return bool(torch.equal(raw.view(torch.uint8), want.view(torch.uint8)))


def rand(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


class Case:
    def __init__(self, collective, n, rows, cols, kind="bf16", stream=None, weight=None, out=None, offset=0, gap=0, seed=0, residual=True):
        self.collective, self.n, self.rows, self.cols = collective, n, rows, cols
        self.kind, self.stream, self.weight_kind, self.out = kind, stream or kind, weight or kind, out or kind
        self.gathered = collective == AR
        self.folded = rows if self.gathered else rows * n
        self.copies = 1 if self.gathered else n
        g = torch.Generator(device=DEV).manual_seed(seed)
        t, r = TYPES[kind][0], TYPES[self.stream][0]
        self.send = Strided(n, self.folded, cols, t, offset, gap).fill([rand((self.folded, cols), t, g, 0.5) for _ in range(n)])
        self.residual = Strided(self.copies, rows, cols, r, offset, gap).fill([rand((rows, cols), r, g, 2.0) for _ in range(self.copies)]) if residual else None
        self.weight = (1 + 0.3 * torch.randn(cols, generator=g, device=DEV)).to(TYPES[self.weight_kind][0])
        self.offset, self.gap, self.g = offset, gap, g

    def fold(self):
        """The sum over ranks in 64 bits and the sum of the terms' magnitudes, [copies, rows, cols]."""
        x = self.send.all().double()
        return x.sum(0).view(self.copies, self.rows, self.cols), x.abs().sum(0).view(self.copies, self.rows, self.cols)

    def types(self):
        return dict(residual_dtype=TYPES[self.stream][1], weight_dtype=TYPES[self.weight_kind][1])

    # forward

    def outputs(self):
        r, o = TYPES[self.stream][0], TYPES[self.out][0]
        self.hidden = Strided(self.n, self.rows, self.cols, r, self.offset, self.gap)
        self.y = Strided(self.n, self.rows, self.cols, o, self.offset, self.gap)
        self.scales = Strided(self.n, 1, self.rows, torch.float32, self.offset) if self.out in ("e4m3", "int8") else None

    def forward_args(self):
        args = dict(residuals=self.residual.views if self.residual else None, residual_outs=self.hidden.views,
                    scales=self.scales.views if self.scales else None, out_dtype=TYPES[self.out][1], **self.types())
        stride = self.cols + self.gap
        args.update(send_stride=stride, residual_stride=stride, residual_out_stride=stride, out_stride=stride)
        return (self.send.views, self.y.views, self.weight, self.rows, self.cols, TYPES[self.kind][1], EPS), args

    def run_forward(self, stream=None):
        args, more = self.forward_args()
        call = mr.all_reduce_rms_norm if self.gathered else mr.reduce_scatter_rms_norm
        call(*args, stream=stream, **more)
        torch.cuda.synchronize()

    def want_forward(self):
        s, terms = self.fold()
        if self.residual:
            res = self.residual.all().double()
            s, terms = s + res, terms + res.abs()
        dh = self.n * U * terms
        w = self.weight.double()
        r = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + EPS)
        y = s * r * w
        lost = dh.norm(dim=-1, keepdim=True) / (s.norm(dim=-1, keepdim=True) + 1e-300)
        dy = dh * r * w.abs() + y.abs() * (lost + TAIL)
        return s, dh, y, dy

    def check_forward(self, hidden=None, outs=None):
        h, dh, y, dy = self.want_forward()
        r = TYPES[self.stream][0]
        for k in range(self.n):
            c = 0 if self.gathered else k
            got = (hidden or self.hidden.views)[k].double()
            off = (got - h[c]).abs() - (dh[c] + half_step(r) * (h[c].abs() + dh[c]) + smallest(r))
            assert float(off.max()) <= 0, f"hidden of rank {k}: {float(off.max())} over its tolerance"
            got = (outs or self.y.views)[k]
            if self.scales is None:
                t = TYPES[self.kind][0]
                off = (got.double() - y[c]).abs() - (dy[c] + half_step(t) * (y[c].abs() + dy[c]) + smallest(t))
                assert float(off.max()) <= 0, f"output of rank {k}: {float(off.max())} over its tolerance"
                continue
            q_max = 448.0 if self.out == "e4m3" else 127.0
            scale = self.scales.views[k][0].double()
            top = y[c].abs().amax(-1).clamp(min=2.0 ** -100)
            assert bool(((scale - top / q_max).abs() <= (dy[c].amax(-1) / q_max + 4 * U * top / q_max)).all())
            q = y[c] / scale[:, None]
            half = torch.clamp(2.0 ** -4 * q.abs(), min=2.0 ** -10) if self.out == "e4m3" else 0.5
            off = (got.float().double() - q).abs() - (half + dy[c] / scale[:, None] + 4 * U * q.abs())
            assert float(off.max()) <= 1e-9, f"codes of rank {k}: {float(off.max())} over their tolerance"
        if self.gathered:  # every rank gets the same bits
            for k in range(1, self.n):
                assert torch.equal(self.hidden.views[0], self.hidden.views[k])
                assert torch.equal(self.y.views[0].view(torch.uint8 if self.scales else self.y.views[0].dtype), self.y.views[k].view(torch.uint8 if self.scales else self.y.views[0].dtype))

    # backward

    def gradients(self, arriving=True, both=False):
        t, r = TYPES[self.kind][0], TYPES[self.stream][0]
        self.h = Strided(self.copies, self.rows, self.cols, r, self.offset, self.gap).fill([rand((self.rows, self.cols), r, self.g, 2.0) for _ in range(self.copies)])
        self.arriving = Strided(self.copies, self.rows, self.cols, r, self.offset, self.gap).fill([rand((self.rows, self.cols), r, self.g) for _ in range(self.copies)]) if arriving else None
        self.dh = Strided(self.n, self.rows, self.cols, r, self.offset, self.gap)
        self.dsend = Strided(self.n, self.rows, self.cols, t, self.offset, self.gap) if both else None
        self.dw = Strided(self.n, 1, self.cols, torch.float32, self.offset)
        size = mr.rms_norm_backward_workspace(self.collective, self.n, self.rows, self.cols)
        self.workspace = torch.full((size // 4 + 64,), float("nan"), device=DEV)
        self.workspace_bytes = size

    def backward_args(self):
        stride = self.cols + self.gap
        args = dict(residual_grads=self.arriving.views if self.arriving else None, send_grads=self.dsend.views if self.dsend else None,
                    weight_grads=[v[0] for v in self.dw.views], workspace=self.workspace, workspace_bytes=self.workspace_bytes,
                    send_stride=stride, hidden_stride=stride, residual_grad_stride=stride, residual_out_grad_stride=stride,
                    send_grad_stride=stride, **self.types())
        return (self.send.views, self.h.views, self.weight, self.dh.views, self.rows, self.cols, TYPES[self.kind][1], EPS), args

    def run_backward(self, stream=None):
        args, more = self.backward_args()
        call = mr.all_reduce_rms_norm_backward if self.gathered else mr.reduce_scatter_rms_norm_backward
        call(*args, stream=stream, **more)
        torch.cuda.synchronize()

    def want_backward(self):
        g, terms = self.fold()
        dg = self.n * U * terms
        h, w = self.h.all().double(), self.weight.double()
        r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
        gw = g * w
        c = (gw * h).mean(-1, keepdim=True)
        dc = (w.abs() * h.abs() * dg).mean(-1, keepdim=True) + TAIL * (gw * h).abs().mean(-1, keepdim=True)
        a = self.arriving.all().double() if self.arriving else torch.zeros_like(h)
        want = r * gw - h * r ** 3 * c + a
        off = r * w.abs() * dg + h.abs() * r ** 3 * dc + 3 * TAIL * ((r * gw).abs() + (h * r ** 3 * c).abs()) + 4 * U * a.abs()
        dw = (g * h * r).sum(1)
        # the additions of a column: its group's rows one by one, then the groups
        dw_off = ((h * r).abs() * dg).sum(1) + (TAIL + (self.rows + 16) * U) * (g * h * r).abs().sum(1)
        return want, off, dw, dw_off

    def check_backward(self, dh=None, dsend=None):
        want, off, dw, dw_off = self.want_backward()
        t, r = TYPES[self.kind][0], TYPES[self.stream][0]
        for k in range(self.n):
            c = 0 if self.gathered else k
            got = (dh or self.dh.views)[k].double()
            over = (got - want[c]).abs() - (off[c] + half_step(r) * (want[c].abs() + off[c]) + smallest(r))
            assert float(over.max()) <= 0, f"gradient of rank {k}: {float(over.max())} over its tolerance"
            if self.dsend:
                got = (dsend or self.dsend.views)[k].double()
                over = (got - want[c]).abs() - (off[c] + half_step(t) * (want[c].abs() + off[c]) + smallest(t))
                assert float(over.max()) <= 0, f"send gradient of rank {k}: {float(over.max())} over its tolerance"
            over = (self.dw.views[k][0].double() - dw[c]).abs() - dw_off[c] - 1e-30
            assert float(over.max()) <= 0, f"weight gradient of rank {k}: {float(over.max())} over its tolerance"


# every variant's first and last width, odd ones, a head and a tail that share a vector
WIDTHS = [1, 3, 7, 8, 9, 15, 64, 100, 511, 512, 513, 1000, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 5000, 8191, 8192, 8193, 12001, 16384]


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("collective,n,rows", [(AR, 2, 5), (RS, 3, 2)])
def test_forward_widths(cols, collective, n, rows):
    c = Case(collective, n, rows, cols, seed=cols)
    c.outputs()
    c.run_forward()
    c.check_forward()
    assert c.hidden.intact() and c.y.intact()


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("collective,n,rows", [(AR, 2, 5), (RS, 3, 2)])
def test_backward_widths(cols, collective, n, rows):
    c = Case(collective, n, rows, cols, seed=cols)
    c.gradients()
    c.run_backward()
    c.check_backward()
    assert c.dh.intact() and c.dw.intact() and bool(torch.isnan(c.workspace[c.workspace_bytes // 4:]).all())


@pytest.mark.parametrize("cols", [16385, 24576 + 3, 40000])
@pytest.mark.parametrize("collective,n,rows,out", [(AR, 2, 2, "bf16"), (RS, 2, 1, "e4m3"), (AR, 3, 1, "int8")])
def test_rows_no_variant_holds(cols, collective, n, rows, out):
    c = Case(collective, n, rows, cols, out=out, seed=cols)
    c.outputs()
    c.run_forward()
    c.check_forward()
    assert c.hidden.intact() and c.y.intact()
    c = Case(collective, n, 3 * rows, cols, seed=cols)
    c.gradients()
    c.run_backward()
    c.check_backward()
    assert c.dh.intact() and c.dw.intact()


@pytest.mark.parametrize("kind,stream,weight", [("bf16", "bf16", "fp32"), ("bf16", "fp32", "bf16"), ("fp16", "fp16", "fp16"),
                                                ("fp16", "fp32", "fp32"), ("fp32", "fp32", "fp32")])
@pytest.mark.parametrize("out", [None, "e4m3", "int8"])
@pytest.mark.parametrize("cols", [5, 200, 1000, 2001, 4096, 7777, 10000])
def test_forward_types(kind, stream, weight, out, cols):
    c = Case(AR if cols % 2 else RS, 3, 6, cols, kind, stream, weight, out, seed=cols)
    c.outputs()
    c.run_forward()
    c.check_forward()
    assert c.hidden.intact() and c.y.intact() and (c.scales is None or c.scales.intact())


@pytest.mark.parametrize("kind,stream,weight", [("bf16", "bf16", "fp32"), ("bf16", "fp32", "bf16"), ("fp16", "fp16", "fp16"),
                                                ("fp16", "fp32", "fp32"), ("fp32", "fp32", "fp32")])
@pytest.mark.parametrize("cols", [5, 200, 1000, 2001, 4096, 7777, 10000])
def test_backward_types(kind, stream, weight, cols):
    c = Case(AR if cols % 2 else RS, 3, 6, cols, kind, stream, weight, seed=cols)
    c.gradients(arriving=cols % 3 != 0, both=True)
    c.run_backward()
    c.check_backward()
    assert c.dh.intact() and c.dsend.intact()


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 12, 16, 31, 32])
@pytest.mark.parametrize("cols,kind", [(512, "bf16"), (2100, "fp32"), (9000, "fp16")])
def test_rank_counts(n, cols, kind):
    for collective in (AR, RS):
        c = Case(collective, n, 3, cols, kind, seed=n)
        c.outputs()
        c.run_forward()
        c.check_forward()
        c = Case(collective, n, 3, cols, kind, seed=n)
        c.gradients()
        c.run_backward()
        c.check_backward()


@pytest.mark.parametrize("offset,gap", [(1, 0), (3, 5), (0, 8), (7, 1)])
@pytest.mark.parametrize("cols", [3, 640, 1500, 4099, 8200])
@pytest.mark.parametrize("kind,out", [("bf16", None), ("fp32", "e4m3"), ("fp16", "int8")])
def test_rows_off_every_boundary(offset, gap, cols, kind, out):
    c = Case(AR, 2, 4, cols, kind, out=out, offset=offset, gap=gap, seed=cols)
    c.outputs()
    c.run_forward()
    c.check_forward()
    assert c.hidden.intact() and c.y.intact()
    c = Case(RS, 2, 4, cols, kind, offset=offset, gap=gap, seed=cols)
    c.gradients(both=True)
    c.run_backward()
    c.check_backward()
    assert c.dh.intact() and c.dsend.intact() and c.dw.intact()


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 255, 256, 257, 1000, 5000])
@pytest.mark.parametrize("cols", [72, 1536])
def test_row_counts(rows, cols):
    for collective, n in ((AR, 2), (RS, 2)):
        c = Case(collective, n, rows, cols, seed=rows)
        c.outputs()
        c.run_forward()
        c.check_forward()
        assert c.hidden.intact() and c.y.intact()
        c = Case(collective, n, rows, cols, seed=rows)
        c.gradients()
        c.run_backward()
        c.check_backward()
        assert c.dh.intact()


@pytest.mark.parametrize("cols", [6, 500, 1003, 4096, 8185, 20001])
def test_in_place(cols):
    n, rows = 3, 4
    for collective in (AR, RS):
        c = Case(collective, n, rows, cols, seed=cols)
        c.outputs()
        want = c.want_forward  # of the inputs as they are now
        h, dh, y, dy = want()
        own = [v if c.gathered else v[r * rows:(r + 1) * rows] for r, v in enumerate(c.send.views)]
        hidden = [c.residual.views[0]] + c.hidden.views[1:] if c.gathered else c.residual.views
        args, more = c.forward_args()
        more["residual_outs"] = hidden
        call = mr.all_reduce_rms_norm if c.gathered else mr.reduce_scatter_rms_norm
        call(args[0], own, *args[2:], **more)
        torch.cuda.synchronize()
        c.want_forward = lambda: (h, dh, y, dy)
        c.scales = None
        c.gathered, keep = False, c.gathered  # compare rank by rank
        if keep:
            h, dh, y, dy = (x.expand(n, rows, cols) for x in (h, dh, y, dy))
        c.check_forward(hidden=hidden, outs=own)

        c = Case(collective, n, rows, cols, seed=cols)
        c.gradients(both=True)
        wanted = c.want_backward()
        own = [v if c.gathered else v[r * rows:(r + 1) * rows] for r, v in enumerate(c.send.views)]
        source = c.h if cols % 2 else c.arriving
        out = [source.views[0]] + c.dh.views[1:] if c.gathered else source.views
        args, more = c.backward_args()
        more["send_grads"] = own
        call = mr.all_reduce_rms_norm_backward if c.gathered else mr.reduce_scatter_rms_norm_backward
        call(args[0], args[1], args[2], out, *args[4:], **more)
        torch.cuda.synchronize()
        c.want_backward = lambda: wanted
        c.check_backward(dh=out, dsend=own)


def test_optional_parts():
    c = Case(AR, 2, 5, 300, residual=False)
    c.outputs()
    c.run_forward()
    c.check_forward()
    args, more = c.forward_args()
    first = c.y.all()
    more["residual_outs"] = None
    mr.all_reduce_rms_norm(*args, **more)
    torch.cuda.synchronize()
    assert torch.equal(first, c.y.all())
    c = Case(RS, 2, 5, 300)
    c.gradients()
    c.run_backward()
    dh, dw = c.dh.all(), c.dw.all()
    args, more = c.backward_args()
    more.update(weight_grads=None, workspace=None, workspace_bytes=0)
    for v in c.dh.views:
        v.zero_()
    mr.reduce_scatter_rms_norm_backward(*args, **more)
    torch.cuda.synchronize()
    assert torch.equal(dh, c.dh.all())
    args, more = c.backward_args()
    for v in c.dw.views:
        v.zero_()
    mr.reduce_scatter_rms_norm_backward(*args[:3], None, *args[4:], **more)
    torch.cuda.synchronize()
    assert torch.equal(dw, c.dw.all())


def test_no_rows():
    for collective in (AR, RS):
        c = Case(collective, 2, 0, 100)
        c.outputs()
        c.run_forward()
        c.gradients()
        c.run_backward()
        assert c.y.intact() and c.dh.intact()
        assert all(bool((v == 0).all()) for v in c.dw.views)


@pytest.mark.parametrize("cols", [4, 100, 3000, 17000])
def test_rows_that_are_not_finite_stay_among_themselves(cols):
    for out in ("bf16", "e4m3", "int8"):
        c = Case(AR, 2, 6, cols, out=out)
        c.send.views[0][1, cols // 2] = float("nan")
        c.send.views[1][3, 0] = float("inf")
        c.residual.views[0][4, cols - 1] = float("-inf")
        c.send.views[0][5] = 0
        c.send.views[1][5] = 0
        c.residual.views[0][5] = 0
        c.outputs()
        c.run_forward()
        y = c.y.views[1].float()
        assert bool(torch.isnan(c.hidden.views[0][1, cols // 2])) and float(c.hidden.views[0][3, 0]) == float("inf")
        if c.scales is None:
            assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[3, 0])) and bool(torch.isnan(y[4, cols - 1]))
        else:
            scale = c.scales.views[1][0]
            assert bool(torch.isnan(scale[[1, 3, 4]]).all())
            bad = y[[1, 3, 4]]
            assert bool(torch.isnan(bad).all()) if out == "e4m3" else bool((bad == 0).all())
            assert 0 < float(scale[5]) < 1e-30
        assert bool((y[5] == 0).all())
        for row in (0, 2):
            assert bool(torch.isfinite(y[row]).all())


def test_the_same_bits_every_time():
    c = Case(AR, 8, 700, 1111)
    c.outputs()
    c.run_forward()
    first = c.y.all(), c.hidden.all()
    c.gradients()
    c.run_backward()
    grads = c.dh.all(), c.dw.all()
    for _ in range(3):
        for s in (c.y, c.hidden, c.dh, c.dw):
            for v in s.views:
                v.zero_()
        c.workspace.fill_(7.0)
        c.run_forward()
        c.run_backward()
        assert torch.equal(first[0], c.y.all()) and torch.equal(first[1], c.hidden.all())
        assert torch.equal(grads[0], c.dh.all()) and torch.equal(grads[1], c.dw.all())


def test_plans_and_streams_and_graphs():
    """A plan launches what the call does; both may sit in a graph that is replayed on new data between eager work."""
    c = Case(AR, 4, 33, 2222, "fp16", "fp32")
    c.outputs()
    args, more = c.forward_args()
    forward = mr.RmsNormPlan(AR, *args, **more)
    c.gradients(both=True)
    bargs, bmore = c.backward_args()
    backward = mr.RmsNormBackwardPlan(AR, *bargs, **bmore)
    assert forward.launch_count == 1 and backward.launch_count == 2
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    forward.launch(stream=side)
    backward.launch(stream=side)
    side.synchronize()
    c.check_forward()
    c.check_backward()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        forward.launch(stream=torch.cuda.current_stream())
        backward.launch(stream=torch.cuda.current_stream())
    for replay in range(3):
        g = torch.Generator(device=DEV).manual_seed(100 + replay)
        for v in c.send.views + c.residual.views + c.h.views:
            v.copy_(rand(v.shape, torch.float32, g))
        for s in (c.y, c.hidden, c.dh, c.dw, c.dsend):
            for v in s.views:
                v.fill_(replay + 3)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.check_forward()
        c.check_backward()


@pytest.mark.parametrize("collective", [AR, RS])
def test_gradients_against_differences(collective):
    """With L = sum of y * a + h * b in 64 bits, (L(x + t d) - L(x - t d)) / 2t is the gradient along d up to t^2 times the third
    derivative.  Inputs are 32-bit; h and y are off by about 2^-23 of themselves, independently, which moves the quotient by
    about 2^-23 * |a . y| / t, and t = 2^-6 with 1 / rms about 1/2 leaves a third-order term of t^2 / 4 of |d| |a|:
    6e-5, so 5e-4 of the norms' product is tight enough to tell a wrong term and wide enough for both."""
    n, rows, cols = 2, 4, 96
    c = Case(collective, n, rows, cols, "fp32")
    c.outputs()
    g = torch.Generator(device=DEV).manual_seed(5)
    a = [rand((rows, cols), torch.float32, g) for _ in range(1 if c.gathered else n)]
    b = [rand((rows, cols), torch.float32, g) for _ in range(1 if c.gathered else n)]

    def loss():
        c.run_forward()
        return sum(float((c.y.views[k].double() * a[k].double() + c.hidden.views[k].double() * b[k].double()).sum()) for k in range(len(a)))

    loss()
    # the gradient of y arrives as the ranks' partial gradients, that of h as the residual's
    grad = Case(collective, n, rows, cols, "fp32")
    grad.gradients()
    grad.weight.copy_(c.weight)
    for v in grad.send.views[1:]:
        v.copy_(0.25 * grad.send.views[0])
    whole = torch.cat(a) if not c.gathered else a[0]
    grad.send.views[0].copy_(whole - sum(v for v in grad.send.views[1:]))
    for k in range(len(a)):
        grad.h.views[k].copy_(c.hidden.views[k])
        grad.arriving.views[k].copy_(b[k])
    grad.run_backward()
    t = 2.0 ** -6
    for what in ("send", "residual", "weight"):
        for k in range(3):
            if what == "weight":
                d = rand((cols,), torch.float32, g)
                want = sum(float((grad.dw.views[r][0].double() * d.double()).sum()) for r in range(1 if c.gathered else n))
                target, size = c.weight, float(d.norm()) * float(torch.stack(a).norm())
            else:
                d = rand((c.folded if what == "send" else rows, cols), torch.float32, g)
                target = c.send.views[k % n] if what == "send" else c.residual.views[k % c.copies]
                if what == "send":
                    dh = grad.dh.views[0] if c.gathered else torch.cat(grad.dh.views)
                else:
                    dh = grad.dh.views[k % c.copies]
                want = float((dh.double() * d.double()).sum())
                size = float(d.norm()) * float((torch.stack(a).norm() + torch.stack(b).norm()))
            keep = target.clone()
            target.copy_(keep + t * d)
            up = loss()
            target.copy_(keep - t * d)
            down = loss()
            target.copy_(keep)
            assert abs((up - down) / (2 * t) - want) <= 5e-4 * size, what
