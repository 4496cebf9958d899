"""The norm behind a fold, its backward, the gradients' norm and the AdamW step, run together as a model runs them: a tensor- and
data-parallel training step, the same chain from a graph, a decoding step, launches long enough for every store policy.

U = 2^-24 is half a step of a 32-bit value."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import megray_amd as mr  # noqa: E402

DEV = "cuda:0"
U = 2.0 ** -24
AR, RS = mr.Collective.ALL_REDUCE, mr.Collective.REDUCE_SCATTER
FP32, FP16, BF16, E4M3 = mr.DType.FLOAT32, mr.DType.FLOAT16, mr.DType.BFLOAT16, mr.DType.FLOAT8_E4M3
EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS = 1e-2, 0.9, 0.95, 1e-8


def randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def norm64(h, w):
    return h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * w


class Block:
    """h1 = x + sum over tensor ranks of x[k] @ first[k];  h2 = h1 + sum of norm(h1)[k] @ second[k];  y = norm(h2): the products'
    inputs are split over the ranks, so each rank has a part of every sum."""

    def __init__(self, ranks, cols, g):
        self.ranks, self.cols = ranks, cols
        part = cols // ranks
        make = lambda: [randn(g, part, cols, scale=cols ** -0.5) for _ in range(ranks)]  # noqa: E731
        self.first, self.second = make(), make()
        self.w1, self.w2 = 1 + randn(g, cols, scale=0.2), 1 + randn(g, cols, scale=0.2)

    def tensors(self):
        return self.first + self.second + [self.w1, self.w2]

    def split(self, x):
        return [p.contiguous() for p in x.split(self.cols // self.ranks, -1)]

    def step(self, x, targets, grads):
        """Forward, the loss sum over ranks of (y * targets[k]).sum(), backward; `grads` get the tensors' gradients."""
        n, rows, cols = self.ranks, x.shape[0], self.cols
        new = lambda count: [torch.full((rows, cols), float("nan"), device=DEV) for _ in range(count)]  # noqa: E731
        h1, y1, h2, y2 = new(n), new(n), new(n), new(n)
        mr.all_reduce_rms_norm([a @ b for a, b in zip(self.split(x), self.first)], y1, self.w1, rows, cols, FP32, EPS, residuals=[x], residual_outs=h1)
        halves = [self.split(y1[k])[k] for k in range(n)]
        mr.all_reduce_rms_norm([a @ b for a, b in zip(halves, self.second)], y2, self.w2, rows, cols, FP32, EPS, residuals=[h1[0]], residual_outs=h2)
        loss = sum((y2[k] * targets[k]).double().sum() for k in range(n))
        space = torch.empty(mr.rms_norm_backward_workspace(AR, n, rows, cols), dtype=torch.uint8, device=DEV)
        dh2, dh1 = new(n), new(n)
        dw1, dw2 = ([torch.full((cols,), float("nan"), device=DEV) for _ in range(n)] for _ in range(2))
        mr.all_reduce_rms_norm_backward(targets, [h2[0]], self.w2, dh2, rows, cols, FP32, EPS, weight_grads=dw2, workspace=space)
        # a rank knows its own columns' gradient of y1: zeros elsewhere make it a part of the sum
        part = cols // n
        dy1 = [torch.zeros(rows, cols, device=DEV) for _ in range(n)]
        for k in range(n):
            dy1[k][:, k * part:(k + 1) * part] = dh2[k] @ self.second[k].T
            grads[n + k].copy_(halves[k].T @ dh2[k])
        mr.all_reduce_rms_norm_backward(dy1, [h1[0]], self.w1, dh1, rows, cols, FP32, EPS, residual_grads=[dh2[0]], weight_grads=dw1, workspace=space)
        for k in range(n):
            grads[k].copy_(self.split(x)[k].T @ dh1[k])
        grads[2 * n].copy_(dw1[n - 1])
        grads[2 * n + 1].copy_(dw2[0])
        return float(loss)

    def reference(self, x, targets):
        leaves = [t.double().cpu().requires_grad_() for t in self.tensors()]
        n = self.ranks
        x = x.double().cpu()
        h1 = x + sum(a @ b for a, b in zip(x.split(self.cols // n, -1), leaves[:n]))
        h2 = h1 + sum(a @ b for a, b in zip(norm64(h1, leaves[2 * n]).split(self.cols // n, -1), leaves[n:2 * n]))
        loss = (norm64(h2, leaves[2 * n + 1]) * sum(t.double().cpu() for t in targets)).sum()
        loss.backward()
        return float(loss.detach()), [t.grad for t in leaves]


@pytest.mark.parametrize("ranks,replicas,rows,cols", [(4, 2, 24, 256), (2, 3, 1, 96), (1, 1, 7, 40)])
def test_a_training_step(ranks, replicas, rows, cols):
    """Gradients: five products with at most 256 terms and four norms lie one behind the other; each loses at most 256 * U of its terms'
    norms, which are at most 16 times its result's (the root of 256, for terms without a common direction): 9 * 2^8 * 2^4 * 2^-24 < 2^-8
    of a tensor's norm.  A rank's share, a residual's or a replica's left out is several percent and more.

    The step is compared from the gradients themselves: clip and update are off by a few U of lr."""
    g = torch.Generator(device=DEV).manual_seed(ranks)
    block = Block(ranks, cols, g)
    params = block.tensors()
    copies = [params] + [[t.clone() for t in params] for _ in range(replicas - 1)]  # every replica's parameters
    lengths = [t.numel() for t in params]
    grads = [[torch.full_like(t, float("nan")) for t in params] for _ in range(replicas)]
    m, v = [torch.zeros_like(t) for t in params], [torch.zeros_like(t) for t in params]
    decays = [0.1] * (2 * ranks) + [0.0, 0.0]
    plan = mr.AdamWPlan(grads, lengths, FP32, copies, FP32, None, m, v, weight_decays=decays)
    out = torch.empty(plan.norm_floats, device=DEV)
    m64, v64 = [t.double() for t in m], [t.double() for t in v]
    for step in (1, 2, 3):
        for k in range(replicas):
            x = randn(g, rows, cols)
            targets = [randn(g, rows, cols) for _ in range(ranks)]
            loss = block.step(x, targets, grads[k])
            want_loss, want = block.reference(x, targets)
            scale = sum(float(t.norm()) for t in targets) * (rows * cols) ** 0.5
            assert abs(loss - want_loss) < 2.0 ** -8 * scale
            for got, exact in zip(grads[k], want):
                assert float((got.double().cpu() - exact).norm()) < 2.0 ** -8 * float(exact.norm())
        before = [t.double() for t in params]
        plan.grad_norm(out, grad_scale=1.0 / replicas, max_norm=0.5)
        plan.step(LR, step, BETA1, BETA2, ADAM_EPS, grad_scale=1.0 / replicas, clip=out[1:])
        torch.cuda.synchronize()
        mean = [sum(grads[k][t].double() for k in range(replicas)) / replicas for t in range(len(params))]
        total = sum(float((t * t).sum()) for t in mean) ** 0.5
        clip = min(1.0, 0.5 / (total + 1e-6))
        assert abs(float(out[0]) - total) < 16 * U * total and abs(float(out[1]) - clip) < 16 * U * clip
        for t, decay in enumerate(decays):
            x = mean[t] * clip
            m64[t] = BETA1 * m64[t] + (1 - BETA1) * x
            v64[t] = BETA2 * v64[t] + (1 - BETA2) * x * x
            # |m| <= 4 sqrt(v) in the first three steps, so an update is at most 8 LR; a mean that nearly cancels is off by U of its
            # terms, not of itself: 64 U of the largest update
            move = LR * (m64[t] / (1 - BETA1 ** step)) / ((v64[t] / (1 - BETA2 ** step)).sqrt() + ADAM_EPS)
            want = before[t] * (1 - LR * decay) - move
            # where the gradients' sum itself nearly cancels its rounding is no small part of it
            terms = sum(grads[k][t].double().abs() for k in range(replicas)) / replicas
            firm = mean[t].abs() > 2.0 ** -6 * terms
            off = (params[t].double() - want).abs() - (4 * U * before[t].abs() + 64 * U * 8 * LR * 2 ** 6)
            assert bool((off <= 0)[firm].all())
            m64[t], v64[t] = m[t].double(), v[t].double()
        for other in copies[1:]:
            for a, b in zip(params, other):
                assert torch.equal(a.view(torch.int32), b.view(torch.int32))


def test_the_chain_from_a_graph():
    """Norm, its backward, the gradients' norm and a clipped step on the weight's gradients, captured once and replayed on new data,
    with eager work between: the same bits as the calls."""
    n, rows, cols = 4, 37, 1000
    g = torch.Generator(device=DEV).manual_seed(3)
    new = lambda dtype, count=n: [torch.zeros(rows, cols, dtype=dtype, device=DEV) for _ in range(count)]  # noqa: E731
    sends, partials, residual = new(torch.bfloat16), new(torch.bfloat16), new(torch.float32, 1)
    h, y, dh, dsend = new(torch.float32), new(torch.bfloat16), new(torch.float32), new(torch.bfloat16)
    weight = torch.ones(cols, device=DEV)
    weights = [weight] + [weight.clone() for _ in range(n - 1)]
    dw = [torch.zeros(cols, device=DEV) for _ in range(n)]
    space = torch.empty(mr.rms_norm_backward_workspace(RS, n, rows, cols) + mr.rms_norm_backward_workspace(AR, n, rows, cols), dtype=torch.uint8, device=DEV)
    more = dict(residual_dtype=FP32, weight_dtype=FP32)
    forward = mr.RmsNormPlan(AR, sends, y, weight, rows, cols, BF16, EPS, residuals=residual, residual_outs=h, **more)
    backward = mr.RmsNormBackwardPlan(AR, partials, [h[0]], weight, dh, rows, cols, BF16, EPS, send_grads=dsend, weight_grads=dw, workspace=space, **more)
    m, v = torch.zeros(cols, device=DEV), torch.zeros(cols, device=DEV)
    adam = mr.AdamWPlan([[dw[0]]], [cols], FP32, [[t] for t in weights], FP32, None, [m], [v], weight_decays=[0.01])
    out = torch.empty(adam.norm_floats, device=DEV)

    def chain(stream):
        forward.launch(stream=stream)
        backward.launch(stream=stream)
        adam.grad_norm(out, max_norm=1.0, stream=stream)
        adam.step(LR, 5, BETA1, BETA2, ADAM_EPS, clip=out[1:], stream=stream)

    results = h + y + dh + dsend + dw + weights + [m, v]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    chain(side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        chain(torch.cuda.current_stream())
    for _ in range(3):
        for t in sends + partials + residual:
            t.copy_(randn(g, rows, cols))
        state = [t.clone() for t in (*weights, m, v)]
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in results]
        for t, old in zip((*weights, m, v), state):
            t.copy_(old)
        chain(torch.cuda.current_stream())
        torch.cuda.synchronize()
        for a, b in zip(got, results):
            assert torch.equal(a, b)


@pytest.mark.parametrize("tokens", [1, 2, 5])
@pytest.mark.parametrize("cols", [64, 520, 4096])
def test_decoding_carries_the_stream_in_place(tokens, cols):
    """Layer after layer of one token (or a few) to 8 bits, the residual stream in one buffer that the calls replace: as a chain of 64-bit
    norms, each from the stream as it is stored."""
    n = 8
    g = torch.Generator(device=DEV).manual_seed(cols)
    stream = randn(g, tokens, cols).bfloat16()
    spare = [stream] + [torch.empty_like(stream) for _ in range(n - 1)]
    codes = [torch.empty(tokens, cols, dtype=torch.float8_e4m3fn, device=DEV) for _ in range(n)]
    scales = [torch.empty(tokens, device=DEV) for _ in range(n)]
    for _ in range(4):
        sends = [randn(g, tokens, cols, scale=0.3).bfloat16() for _ in range(n)]
        weight = (1 + randn(g, cols, scale=0.2)).bfloat16()
        h = stream.double() + sum(s.double() for s in sends)
        mr.all_reduce_rms_norm(sends, codes, weight, tokens, cols, BF16, EPS, residuals=[stream], residual_outs=spare, scales=scales, out_dtype=E4M3)
        torch.cuda.synchronize()
        # terms of at most 8 + 1 ranks' sums: 9 U of their magnitudes, and the rounding
        terms = stream.double().abs() + h.abs() + sum(s.double().abs() for s in sends)
        assert bool(((stream.double() - h).abs() <= 2.0 ** -8 * h.abs() + 10 * U * terms + 1e-38).all())
        y = norm64(h, weight.double())
        for k in range(n):
            assert torch.equal(spare[k], stream) and torch.equal(codes[k].view(torch.uint8), codes[0].view(torch.uint8)) and torch.equal(scales[k], scales[0])
        got = codes[0].double() * scales[0].double()[:, None]
        # half a step of the code, 2^-10 of the scale among the smallest codes; a hundred U for sums, root, quotient
        room = 2.0 ** -4 * y.abs() + 2.0 ** -10 * scales[0].double()[:, None] + 100 * U * y.abs().amax(-1, keepdim=True)
        assert bool(((got - y).abs() <= room).all())
        assert bool(((scales[0].double() * 448 / y.abs().amax(-1) - 1).abs() < 100 * U).all())


@pytest.mark.parametrize("n", [3, 5, 8])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_few_rows_out_of_place_and_in_place_agree(n, rows):
    """Few rows are shared among workgroups by destination, but not where an output takes an input's place."""
    cols = 2056
    g = torch.Generator(device=DEV).manual_seed(n)
    sends = [randn(g, rows, cols).half() for _ in range(n)]
    residual, weight = randn(g, rows, cols).half(), randn(g, cols).half()
    out, h = [torch.empty_like(s) for s in sends], [torch.empty_like(s) for s in sends]
    mr.all_reduce_rms_norm(sends, out, weight, rows, cols, FP16, EPS, residuals=[residual], residual_outs=h)
    torch.cuda.synchronize()
    total = residual.double() + sum(s.double() for s in sends)
    terms = residual.double().abs() + sum(s.double().abs() for s in sends)
    per = torch.rsqrt((total * total).mean(-1, keepdim=True) + EPS) * weight.double()  # y / total, also where the total is zero
    y = total * per
    # h is off by at most (n + 1) U of its terms, y by that times |per|, and by fewer than 90 U of itself through the row's sum
    room = 2.0 ** -11 * y.abs() + 100 * U * terms * per.abs() + 2.0 ** -25
    for k in range(n):
        assert bool(((out[k].double() - y).abs() <= room).all())
    moved, spare = [s.clone() for s in sends], [residual.clone()] + [torch.empty_like(residual) for _ in range(n - 1)]
    mr.all_reduce_rms_norm(moved, moved, weight, rows, cols, FP16, EPS, residuals=[spare[0]], residual_outs=spare)
    torch.cuda.synchronize()
    for k in range(n):
        assert torch.equal(moved[k], out[k]) and torch.equal(spare[k], h[k])


@pytest.mark.parametrize("n,rows,cols", [(3, 11500, 4096), (5, 6500, 4096), (5, 6500, 4101), (2, 17000, 4096), (5, 3400, 8200)])
def test_long_launches(n, rows, cols):
    """More than 256 MiB written: streamed stores, one at a time, rows walked (up to four destinations) or a workgroup each.  Rows from
    every part are compared with 64 bits, all ranks with the first, and the backward's weight gradient with the rows' sum."""
    assert n * rows * cols * 4 >= 256 << 20
    g = torch.Generator(device=DEV).manual_seed(n)
    sends = [randn(g, rows, cols).bfloat16() for _ in range(n)]
    residual, weight = randn(g, rows, cols).bfloat16(), (1 + randn(g, cols, scale=0.2)).bfloat16()
    out, h = [torch.empty_like(s) for s in sends], [torch.empty_like(s) for s in sends]
    mr.all_reduce_rms_norm(sends, out, weight, rows, cols, BF16, EPS, residuals=[residual], residual_outs=h)
    torch.cuda.synchronize()
    pick = torch.cat([torch.arange(0, 70), torch.arange(rows // 2, rows // 2 + 70), torch.arange(rows - 70, rows)]).to(DEV)
    total = residual[pick].double() + sum(s[pick].double() for s in sends)
    terms = residual[pick].double().abs() + sum(s[pick].double().abs() for s in sends)
    r = torch.rsqrt((total * total).mean(-1, keepdim=True) + EPS)
    y = total * r * weight.double()
    assert bool(((h[0][pick].double() - total).abs() <= 2.0 ** -8 * total.abs() + 8 * U * terms).all())
    assert bool(((out[0][pick].double() - y).abs() <= 2.0 ** -8 * y.abs() + 100 * U * terms * r * weight.double().abs()).all())
    # every row of every rank: the mean of squares of y / weight is 1 but for eps, and each y is off by half a step at most
    for k in range(n):
        assert torch.equal(out[k], out[0]) and torch.equal(h[k], h[0])
    for i in range(0, rows, 2048):
        z = out[0][i:i + 2048].float() / weight.float()
        assert bool((((z * z).mean(-1)) - 1).abs().max() < 2.0 ** -6)
    del out
    dh, dsend = [torch.empty_like(s) for s in sends], [torch.empty_like(s) for s in sends]
    dw = [torch.empty(cols, device=DEV) for _ in range(n)]
    space = torch.empty(mr.rms_norm_backward_workspace(AR, n, rows, cols), dtype=torch.uint8, device=DEV)
    mr.all_reduce_rms_norm_backward(sends, [h[0]], weight, dh, rows, cols, BF16, EPS, send_grads=dsend, weight_grads=dw, workspace=space)
    torch.cuda.synchronize()
    grad, hidden, w = sum(s[pick].double() for s in sends), h[0][pick].double(), weight.double()
    r = torch.rsqrt((hidden * hidden).mean(-1, keepdim=True) + EPS)
    want = r * grad * w - hidden * r ** 3 * (grad * w * hidden).mean(-1, keepdim=True)
    terms = sum(s[pick].double().abs() for s in sends)
    near = 100 * U * r * (terms * w.abs() + hidden.abs() * r * (terms * w.abs() * hidden.abs() * r).mean(-1, keepdim=True))
    assert bool(((dh[0][pick].double() - want).abs() <= 2.0 ** -8 * want.abs() + near).all())
    for k in range(n):
        assert torch.equal(dh[k], dh[0]) and torch.equal(dsend[k], dsend[0]) and torch.equal(dw[k], dw[0])
    exact, size = torch.zeros(cols, dtype=torch.float64, device=DEV), torch.zeros(cols, dtype=torch.float64, device=DEV)
    for i in range(0, rows, 1024):
        rows_ = slice(i, i + 1024)
        hidden = h[0][rows_].double()
        unit = hidden * torch.rsqrt((hidden * hidden).mean(-1, keepdim=True) + EPS)
        exact += (sum(s[rows_].double() for s in sends) * unit).sum(0)
        size += (sum(s[rows_].double().abs() for s in sends) * unit.abs()).sum(0)
    # at most 64 rows of a group, 64 groups of a wavefront and 16 wavefronts are added one behind the other, the rows' values are off by 80 U
    assert bool(((dw[0].double() - exact).abs() <= 256 * U * size).all())


@pytest.mark.parametrize("cols", [8192 + 1, 8192 + 5, 8200, 9221, 12293, 16383])
@pytest.mark.parametrize("stream", [FP16, FP32])
def test_wide_rows_in_place_of_the_arriving_gradient(cols, stream):
    """Rows of two vectors per lane whose last vector overlaps another wavefront's (8193: the first lane of the eighth wavefront ends the row):
    the gradient in the arriving one's place is, bit for bit or within the sums' order, the one beside it."""
    n, rows = 2, 700
    g = torch.Generator(device=DEV).manual_seed(cols)
    t = torch.float32 if stream == FP32 else torch.float16
    sends, weight = [randn(g, rows, cols).half() for _ in range(n)], randn(g, cols).half()
    hidden, arriving = randn(g, rows, cols).to(t), randn(g, rows, cols).to(t)
    space = torch.empty(mr.rms_norm_backward_workspace(AR, n, rows, cols), dtype=torch.uint8, device=DEV)
    results = []
    for place in (torch.empty_like(arriving), arriving.clone()):
        source = place if results else arriving
        dh, dw = [place, torch.empty_like(place)], [torch.empty(cols, device=DEV) for _ in range(n)]
        mr.all_reduce_rms_norm_backward(sends, [hidden], weight, dh, rows, cols, FP16, EPS, residual_dtype=stream, residual_grads=[source],
                                        weight_grads=dw, workspace=space)
        torch.cuda.synchronize()
        assert torch.equal(dh[0], dh[1])
        results.append((dh[0].double(), dw[0].double()))
    (beside, dw_beside), (over, dw_over) = results
    # the two kernels add a row's terms in another order: their sums differ by fewer than 2 * 80 U of the terms' magnitudes
    r = torch.rsqrt((hidden.double() ** 2).mean(-1, keepdim=True) + EPS)
    size = sum(s.double().abs() for s in sends) * weight.double().abs()
    near = 160 * U * (r * size + (hidden.double().abs() * r) * r * (size * hidden.double().abs() * r).mean(-1, keepdim=True) + arriving.double().abs())
    step = 2 * torch.finfo(t).eps / 2
    assert bool(((over - beside).abs() <= step * torch.maximum(over.abs(), beside.abs()) + near + torch.finfo(t).smallest_normal * step).all())
    total = (sum(s.double().abs() for s in sends) * hidden.double().abs() * r).sum(0)
    assert bool(((dw_over - dw_beside).abs() <= 512 * U * total).all())


@pytest.mark.parametrize("cols", [8, 17, 88, 127, 128, 129, 136, 250, 255, 256, 257])
@pytest.mark.parametrize("collective", [AR, RS])
@pytest.mark.parametrize("rows", [1, 15, 33, 3000])
def test_short_rows(cols, collective, rows):
    """Rows that share a wavefront, and row groups whose shares of the weight's gradient meet before they are stored: against 64 bits, and
    in place bit for bit."""
    n = 3
    g = torch.Generator(device=DEV).manual_seed(cols + rows)
    total = rows if collective == AR else rows * n
    copies = 1 if collective == AR else n
    sends = [randn(g, total, cols).bfloat16() for _ in range(n)]
    hidden, arriving = [[randn(g, rows, cols) for _ in range(copies)] for _ in range(2)]
    weight = randn(g, cols)
    space = torch.empty(mr.rms_norm_backward_workspace(collective, n, rows, cols), dtype=torch.uint8, device=DEV)
    call = mr.all_reduce_rms_norm_backward if collective == AR else mr.reduce_scatter_rms_norm_backward
    results = []
    for in_place in (False, True):
        h = [t.clone() for t in hidden]
        dh = (h + [torch.empty_like(h[0]) for _ in range(n - copies)]) if in_place else [torch.empty(rows, cols, device=DEV) for _ in range(n)]
        dw = [torch.empty(cols, device=DEV) for _ in range(n)]
        call(sends, h, weight, dh, rows, cols, BF16, EPS, residual_dtype=FP32, weight_dtype=FP32, residual_grads=arriving, weight_grads=dw, workspace=space)
        torch.cuda.synchronize()
        results.append((dh, dw))
    for a, b in zip(results[0][0] + results[0][1], results[1][0] + results[1][1]):
        assert torch.equal(a, b)
    grads, sizes = sum(s.double() for s in sends).view(copies, rows, cols), sum(s.double().abs() for s in sends).view(copies, rows, cols)
    for c in range(copies):
        h, w, grad, size = hidden[c].double(), weight.double(), grads[c], sizes[c] * weight.double().abs()
        r = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
        want = r * grad * w - h * r ** 3 * (grad * w * h).mean(-1, keepdim=True) + arriving[c].double()
        near = 100 * U * (r * size + h.abs() * r ** 3 * (size * h.abs()).mean(-1, keepdim=True) + arriving[c].double().abs())
        assert bool(((results[0][0][c].double() - want).abs() <= near).all())
        dw, per = (grad * h * r).sum(0), (sizes[c] * (h * r).abs()).sum(0)
        # a group's rows (3000 / 94 at most, 2 a turn), its sixteen slots and 94 groups in turn: fewer than 200 additions, the rows' values off by 80 U
        assert bool(((results[0][1][c].double() - dw).abs() <= 300 * U * per).all())


@pytest.mark.parametrize("cols", [5, 100, 200, 500, 1000, 9000, 20000])
def test_rows_four_gigabytes_apart(cols):
    """Offsets past 32 bits: the third row begins 2^32 bytes and more behind the first, in every buffer; the results are those of rows beside each
    other, bit for bit where the same kernel takes them."""
    rows, stride = 3, (1 << 30) + 64
    g = torch.Generator(device=DEV).manual_seed(cols)
    far = [torch.empty(2 * stride + cols, dtype=torch.float16, device=DEV) for _ in range(4)]
    rows_of = lambda t: [t[r * stride:r * stride + cols] for r in range(rows)]  # noqa: E731
    near = [randn(g, rows, cols).half() for _ in range(2)]
    weight = randn(g, cols).half()
    for t, x in zip(far, near):
        for r, v in enumerate(rows_of(t)):
            v.copy_(x[r])
    out, h = torch.empty_like(near[0]), torch.empty_like(near[0])
    mr.all_reduce_rms_norm([near[0]], [out], weight, rows, cols, FP16, EPS, residuals=[near[1]], residual_outs=[h])
    mr.all_reduce_rms_norm([far[0]], [far[2]], weight, rows, cols, FP16, EPS, residuals=[far[1]], residual_outs=[far[3]], send_stride=stride,
                           residual_stride=stride, residual_out_stride=stride, out_stride=stride)
    torch.cuda.synchronize()
    assert torch.equal(torch.stack(rows_of(far[3])), h)
    got = torch.stack(rows_of(far[2])).double()
    assert bool(((got - out.double()).abs() <= 2.0 ** -10 * out.double().abs() + 2.0 ** -24).all())  # a step, if a sum took another order
    dh, dsend, dw = torch.empty_like(h), torch.empty_like(h), [torch.empty(cols, device=DEV) for _ in range(2)]
    space = torch.empty(mr.rms_norm_backward_workspace(AR, 1, rows, cols), dtype=torch.uint8, device=DEV)
    mr.all_reduce_rms_norm_backward([near[0]], [h], weight, [dh], rows, cols, FP16, EPS, send_grads=[dsend], weight_grads=dw[:1], workspace=space)
    mr.all_reduce_rms_norm_backward([far[0]], [far[3]], weight, [far[1]], rows, cols, FP16, EPS, send_grads=[far[2]], weight_grads=dw[1:], workspace=space,
                                    send_stride=stride, hidden_stride=stride, residual_out_grad_stride=stride, send_grad_stride=stride)
    torch.cuda.synchronize()
    size = dh.double().abs().amax()
    for t, want in ((far[1], dh), (far[2], dsend)):
        assert bool(((torch.stack(rows_of(t)).double() - want.double()).abs() <= 2.0 ** -10 * want.double().abs() + 200 * U * size + 2.0 ** -24).all())
    # three rows' terms |g| * |h * r|, the second at most 20 (a normal value beside its row's root mean square), each off by at most 2 * 100 U
    assert bool(((dw[0] - dw[1]).abs() <= 200 * U * 3 * near[0].float().abs().amax() * 20).all())


def test_two_plans_at_once():
    """Two backwards with a workspace each and two optimizers with an `out` each, on two streams at the same time."""
    n, rows, cols = 2, 900, 1024
    g = torch.Generator(device=DEV).manual_seed(1)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    made, results = [], []
    for _ in side:
        sends, hidden = [randn(g, rows, cols).half() for _ in range(n)], randn(g, rows, cols).half()
        dh, dw = [torch.empty_like(s) for s in sends], [torch.empty(cols, device=DEV) for _ in range(n)]
        space = torch.empty(mr.rms_norm_backward_workspace(AR, n, rows, cols), dtype=torch.uint8, device=DEV)
        weight = randn(g, cols).half()
        back = mr.RmsNormBackwardPlan(AR, sends, [hidden], weight, dh, rows, cols, FP16, EPS, weight_grads=dw, workspace=space)
        adam = mr.AdamWPlan([[s] for s in sends], [rows * cols], FP16)
        made.append((back, adam, torch.empty(adam.norm_floats, device=DEV)))
        results.append(dh + dw + [made[-1][2][:2]])
    torch.cuda.synchronize()
    alone = []
    for (back, adam, out), mine in zip(made, results):
        back.launch()
        adam.grad_norm(out, max_norm=1.0)
        torch.cuda.synchronize()
        alone.append([t.clone() for t in mine])
        for t in mine:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(8):
        for (back, adam, out), s in zip(made, side):
            back.launch(stream=s)
            adam.grad_norm(out, max_norm=1.0, stream=s)
    torch.cuda.synchronize()
    for mine, want in zip(results, alone):
        for a, b in zip(mine, want):
            assert torch.equal(a, b)


def test_one_buffer_as_several_ranks():
    """Inputs may be the same buffer: the sum counts it as often as it is named.  Outputs may not."""
    rows, cols = 3, 333
    g = torch.Generator(device=DEV).manual_seed(9)
    x, weight = randn(g, rows, cols), randn(g, cols)
    out = [torch.empty_like(x) for _ in range(4)]
    mr.all_reduce_rms_norm([x] * 4, out, weight, rows, cols, FP32, EPS)
    other = [torch.empty_like(x)]
    mr.all_reduce_rms_norm([4 * x], other, weight, rows, cols, FP32, EPS)
    torch.cuda.synchronize()
    assert torch.equal(out[3], other[0])  # powers of two: the same bits
    with pytest.raises(mr.MegRayError, match="two outputs overlap"):
        mr.all_reduce_rms_norm([x] * 2, [out[0]] * 2, weight, rows, cols, FP32, EPS)
    flat = x.view(-1)
    plan, twice = mr.AdamWPlan([[flat], [flat]], [flat.numel()], FP32), mr.AdamWPlan([[flat]], [flat.numel()], FP32)
    a, b = torch.empty(plan.norm_floats, device=DEV), torch.empty(twice.norm_floats, device=DEV)
    plan.grad_norm(a)
    twice.grad_norm(b, grad_scale=2.0)
    torch.cuda.synchronize()
    assert float(a[0]) == float(b[0]) and float(a[1]) == 1.0


def test_what_an_adamw_plan_refuses_to_write_or_read():
    values = torch.randn(5000, device=DEV)
    params, m, v = torch.zeros(5000, device=DEV), torch.zeros(5000, device=DEV), torch.zeros(5000, device=DEV)
    plan = mr.AdamWPlan([[values]], [5000], FP32, [[params]], FP32, None, [m], [v])
    with pytest.raises(mr.MegRayError, match="floats"):
        plan.grad_norm(torch.empty(plan.norm_floats - 1, device=DEV))
    before = values.clone()
    for t in (values, params, m, v):
        with pytest.raises(mr.MegRayError, match="overlaps a tensor"):
            plan.grad_norm(t)
        with pytest.raises(mr.MegRayError, match="overlaps a tensor"):
            plan.grad_norm(t.data_ptr() + 4 * 5000 - 8)
    for t in (params, m, v):
        with pytest.raises(mr.MegRayError, match="clip"):
            plan.step(LR, 1, clip=t[7:])
    torch.cuda.synchronize()
    assert torch.equal(values, before) and not bool(params.any())
