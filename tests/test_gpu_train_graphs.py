"""Captured calls of the folds with an epilogue, and how long their handles have to live: a norm's plan may go once its launches are
captured; an AdamW plan stays, since its launches read its table."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import megray_amd as mr  # noqa: E402

DEV = "cuda:0"
AR, BF16, FP32 = mr.Collective.ALL_REDUCE, mr.DType.BFLOAT16, mr.DType.FLOAT32


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


@pytest.mark.parametrize("rows,cols", [(3, 1000), (65, 256), (2, 20000)])
def test_a_captured_norm_outlives_its_plans(rows, cols):
    n = 3
    g = torch.Generator(device=DEV).manual_seed(cols)
    new = lambda count=n: [torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV) for _ in range(count)]  # noqa: E731
    sends, partials, residual, y, h, dh = new(), new(), new(1), new(), new(), new()
    weight = randn(g, cols).bfloat16()
    dw = [torch.zeros(cols, device=DEV) for _ in range(n)]
    space = torch.empty(mr.rms_norm_backward_workspace(AR, n, rows, cols), dtype=torch.uint8, device=DEV)

    def plans():
        return (mr.RmsNormPlan(AR, sends, y, weight, rows, cols, BF16, 1e-5, residuals=residual, residual_outs=h),
                mr.RmsNormBackwardPlan(AR, partials, [h[0]], weight, dh, rows, cols, BF16, 1e-5, weight_grads=dw, workspace=space))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    captured = plans()
    for p in captured:
        p.launch(stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for p in captured:
            p.launch(stream=torch.cuda.current_stream())
    for p in captured:
        p.close()
    del captured
    results = y + h + dh + dw
    for _ in range(3):
        for t in sends + partials + residual:
            t.copy_(randn(g, rows, cols))
        for t in results:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in results]
        for t in results:
            t.zero_()
        for p in plans():
            p.launch()
        torch.cuda.synchronize()
        for a, b in zip(got, results):
            assert torch.equal(a, b)


def test_captured_steps_of_two_plans_share_nothing():
    """Two plans, a graph each, replayed in turn with eager steps of a third on the same values between: the same bits everywhere."""
    n = 5000
    g = torch.Generator(device=DEV).manual_seed(2)
    grads = [randn(g, n) for _ in range(2)]
    start = randn(g, n)
    made, graphs = [], []
    for k in range(3):
        p, m, v = start.clone(), torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
        plan = mr.AdamWPlan([[t] for t in grads], [n], FP32, [[p]], FP32, None, [m], [v])
        made.append((plan, torch.zeros(plan.norm_floats, device=DEV), p, m, v))

    def both(plan, out, stream):
        plan.grad_norm(out, max_norm=1.0, stream=stream)
        plan.step(1e-2, 4, clip=out[1:], stream=stream)

    side = torch.cuda.Stream()
    for plan, out, *_ in made[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            both(plan, out, torch.cuda.current_stream())
        graphs.append(graph)
    for _ in range(3):
        for t in grads:
            t.copy_(randn(g, n))
        graphs[0].replay()
        both(made[2][0], made[2][1], None)
        graphs[1].replay()
        torch.cuda.synchronize()
        for other in made[1:]:
            for a, b in zip(made[0][2:], other[2:]):
                assert torch.equal(a, b)
            assert made[0][1][:2].tolist() == other[1][:2].tolist()
