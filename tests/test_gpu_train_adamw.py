"""AdamW over many tensors and the gradients' norm against their formulas in 64 bits, on the GPU.

Tolerances: U = 2^-24 is half a step of a 32-bit value.  A sum of N gradients is off by at most N * U of its terms' magnitudes; each
product, quotient or root after it adds one U of its result."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import megray_amd as mr  # noqa: E402

DEV = "cuda:0"
U = 2.0 ** -24
BLOCK = 256
TYPES = {"fp16": (torch.float16, mr.DType.FLOAT16), "bf16": (torch.bfloat16, mr.DType.BFLOAT16), "fp32": (torch.float32, mr.DType.FLOAT32),
         "e4m3": (torch.float8_e4m3fn, mr.DType.FLOAT8_E4M3)}
GUARD = 64
HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)


def blocks(n):
    return -(-n // BLOCK)


class Flat:
    """Tensors of `lengths` elements inside one allocation, `offset` elements off its start and with a guard around each."""

    def __init__(self, lengths, dtype, offset=0, fill=0.0):
        self.at, size = [], offset
        for n in lengths:
            size += GUARD
            self.at.append(size)
            size += n
        self.lengths = lengths
        self.data = torch.zeros(size + GUARD, dtype=torch.float32, device=DEV).fill_(fill).to(dtype)
        self.views = [self.data[a:a + n] for a, n in zip(self.at, lengths)]
        self.before = self.data.clone()

    def intact(self):
        now, then = self.data.clone().view(torch.uint8), self.before.view(torch.uint8)
        size = self.data.element_size()
        for a, n in zip(self.at, self.lengths):
            now[a * size:(a + n) * size] = then[a * size:(a + n) * size]
        return bool(torch.equal(now, then))


def encode(x, keep=False):
    """Codes and scales of one tensor in 64 bits' arithmetic, rounded by torch."""
    pad = torch.zeros(blocks(x.numel()) * BLOCK, dtype=torch.float64, device=DEV)
    pad[:x.numel()] = x
    pad = pad.view(-1, BLOCK)
    scale = (pad.abs().amax(1).clamp(min=2.0 ** -100) / 448).float()
    q = pad / scale.double()[:, None]
    q = q.clamp(-448, 448)
    if keep:
        q = torch.where(pad > 0, q.clamp(min=2.0 ** -9), q)
    return q.float().to(torch.float8_e4m3fn).view(-1)[:x.numel()], scale


def decode(codes, scale):
    return codes.double() * scale.double().repeat_interleave(BLOCK)[:codes.numel()]


class Model:
    def __init__(self, lengths, grad_ranks, param_ranks, grad="bf16", param="bf16", states="fp32", offset=0, masters=True, seed=0,
                 step=10, scale=1e-2):
        self.lengths, self.grad_ranks, self.param_ranks = list(lengths), grad_ranks, param_ranks
        self.grad, self.param, self.states = grad, param, states
        g = torch.Generator(device=DEV).manual_seed(seed)
        normal = lambda n: torch.randn(n, generator=g, device=DEV)  # noqa: E731
        self.grads = [Flat(lengths, TYPES[grad][0], offset) for _ in range(grad_ranks)]
        for f in self.grads:
            for v in f.views:
                v.copy_(normal(v.numel()) * scale)
        self.params = [Flat(lengths, TYPES[param][0], offset) for _ in range(param_ranks)]
        self.master = Flat(lengths, torch.float32, offset) if masters else self.params[0]
        for v in self.master.views:
            v.copy_(normal(v.numel()) * 0.1)
        self.m, self.v = Flat(lengths, TYPES[states][0], offset), Flat(lengths, TYPES[states][0], offset)
        self.m_scale = self.v_scale = None
        if states == "e4m3":
            self.m_scale, self.v_scale = Flat([blocks(n) for n in lengths], torch.float32, offset), Flat([blocks(n) for n in lengths], torch.float32, offset)
        for k, n in enumerate(lengths):
            m, v = normal(n) * scale * 0.3, (torch.rand(n, generator=g, device=DEV) + 0.2) * scale * scale
            if states == "e4m3":
                if n:
                    q, s = encode(m.double())
                    self.m.views[k].view(torch.uint8).copy_(q.view(torch.uint8)), self.m_scale.views[k].copy_(s)
                    q, s = encode(v.double().sqrt(), True)
                    self.v.views[k].view(torch.uint8).copy_(q.view(torch.uint8)), self.v_scale.views[k].copy_(s)
            else:
                self.m.views[k].copy_(m), self.v.views[k].copy_(v)
        self.decays = [0.1 if k % 2 else 0.0 for k in range(len(lengths))]
        self.masters = masters
        self.number = step

    def flats(self):
        return self.grads + self.params + [self.master, self.m, self.v] + ([self.m_scale, self.v_scale] if self.m_scale else [])

    def plan(self, **changed):
        args = dict(params=[f.views for f in self.params], param_dtype=TYPES[self.param][1], masters=self.master.views if self.masters else None,
                    exp_avgs=self.m.views, exp_avg_sqs=self.v.views, state_dtype=TYPES[self.states][1], weight_decays=self.decays,
                    exp_avg_scales=self.m_scale.views if self.m_scale else None, exp_avg_sq_scales=self.v_scale.views if self.v_scale else None)
        args.update(changed)
        return mr.AdamWPlan([f.views for f in self.grads], self.lengths, TYPES[self.grad][1], **args)

    def fold(self, k):
        x = torch.stack([f.views[k].double() for f in self.grads])
        return x.sum(0), x.abs().sum(0)

    def want(self, factor=1.0, hyper=HYPER):
        """Per tensor: m, v, sqrt(v) and p in 64 bits, each with what 32 bits may be off."""
        b1, b2, lr = hyper["beta1"], hyper["beta2"], hyper["lr"]
        got = []
        for k, n in enumerate(self.lengths):
            s, terms = self.fold(k)
            x, dx = s * factor, (self.grad_ranks + 3) * U * terms * abs(factor)
            if self.states == "e4m3":
                m, v = decode(self.m.views[k], self.m_scale.views[k]), decode(self.v.views[k], self.v_scale.views[k]).square()
            else:
                m, v = self.m.views[k].double(), self.v.views[k].double()
            size_m = b1 * m.abs() + (1 - b1) * x.abs()
            m2, v2 = b1 * m + (1 - b1) * x, b2 * v + (1 - b2) * x * x
            dm = 5 * U * size_m + (1 - b1) * dx
            dv = 6 * U * v2 + 2 * (1 - b2) * x.abs() * dx + 2.0 ** -148
            root = v2.sqrt()
            droot = dv / (2 * root.clamp(min=2.0 ** -70)) + U * root
            rate, c2 = lr / (1 - b1 ** self.number), 1 / math.sqrt(1 - b2 ** self.number)
            den = root * c2 + hyper["eps"]
            update = rate * m2 / den
            dupdate = rate * dm / den + update.abs() * (droot * c2 / den + 6 * U)
            p = self.master.views[k].double()
            shrink = lr * self.decays[k]
            p2 = p * (1 - shrink) - update
            dp = dupdate + 2 * U * shrink * p.abs() + 2 * U * p.abs() + U * p2.abs()
            got.append((m2, dm, v2, dv, root, droot, p2, dp))
        return got

    def check(self, want):
        t = TYPES[self.param][0]
        half = torch.finfo(t).eps / 2
        for k, (m, dm, v, dv, root, droot, p, dp) in enumerate(want):
            n = self.lengths[k]
            if not n:
                continue

            def near(got, value, off, what):
                over = float(((got.double() - value).abs() - off).max())
                assert over <= 0, f"{what} of tensor {k} ({n} elements): {over} over its tolerance"

            near(self.master.views[k], p, dp, "master")
            for r, f in enumerate(self.params):
                near(f.views[k], p, dp + half * (p.abs() + dp) + torch.finfo(t).smallest_normal * half, f"rank {r}'s parameter")
            if self.states == "fp32":
                near(self.m.views[k], m, dm, "m")
                near(self.v.views[k], v, dv, "v")
                continue
            for name, x, dx, codes, scales, alive in (("m", m, dm, self.m, self.m_scale, False), ("sqrt(v)", root, droot, self.v, self.v_scale, True)):
                pad = torch.zeros(blocks(n) * BLOCK, dtype=torch.float64, device=DEV)
                pad[:n] = x.abs()
                off = torch.zeros_like(pad)
                off[:n] = dx
                top, most = pad.view(-1, BLOCK).amax(1).clamp(min=2.0 ** -100), off.view(-1, BLOCK).amax(1)
                scale = scales.views[k]
                near(scale, top / 448, most / 448 + 4 * U * top / 448, name + "'s scale")
                each = scale.double().repeat_interleave(BLOCK)[:n]
                q = x / each
                if alive:
                    q = torch.where(x > 0, q.clamp(min=2.0 ** -9), q)
                near(codes.views[k], q, torch.clamp(2.0 ** -4 * q.abs(), min=2.0 ** -10) + dx / each + 4 * U * q.abs(), name + "'s codes")
                if alive:
                    assert bool((codes.views[k].float()[x > 1e-30] > 0).all())
        for f in self.flats():
            assert f.intact()


LENGTHS = [1, 2, 7, 8, 9, 255, 256, 257, 300, 0, 2047, 2048, 2049, 5000, 20001]


@pytest.mark.parametrize("grad,param", [("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32"), ("fp32", "bf16"), ("bf16", "fp32"), ("fp16", "bf16"),
                                        ("bf16", "fp16"), ("fp16", "fp32"), ("fp32", "fp16")])
@pytest.mark.parametrize("states", ["fp32", "e4m3"])
@pytest.mark.parametrize("offset", [0, 3])
def test_types_and_lengths(grad, param, states, offset):
    m = Model(LENGTHS, 3, 2, grad, param, states, offset)
    plan = m.plan()
    want = m.want(0.25)
    plan.step(step=m.number, grad_scale=0.25, **HYPER)
    torch.cuda.synchronize()
    m.check(want)


@pytest.mark.parametrize("grad_ranks,param_ranks", [(1, 1), (1, 8), (2, 2), (4, 4), (5, 3), (8, 8), (9, 1), (16, 16), (32, 32)])
def test_rank_counts(grad_ranks, param_ranks):
    for grad, states in (("bf16", "e4m3"), ("fp32", "fp32")):
        m = Model([2500, 33], grad_ranks, param_ranks, grad, "bf16", states)
        plan = m.plan()
        want = m.want(1.0 / grad_ranks)
        plan.step(step=m.number, grad_scale=1.0 / grad_ranks, **HYPER)
        out = torch.zeros(plan.norm_floats + 2, device=DEV)
        plan.grad_norm(out, grad_scale=0.5, max_norm=0.01)
        torch.cuda.synchronize()
        m.check(want)
        squares = sum(float((m.fold(k)[0] * 0.5).square().sum()) for k in range(2))
        off = sum(float((m.fold(k)[1] * 0.5).square().sum()) for k in range(2))
        norm = math.sqrt(squares)
        assert abs(float(out[0]) - norm) <= (grad_ranks + 3) * U * math.sqrt(off) + 2 * U * norm
        assert abs(float(out[1]) - min(1.0, 0.01 / (norm + 1e-6))) <= 4 * U + (grad_ranks + 3) * U * math.sqrt(off) / norm
        assert out[plan.norm_floats:].tolist() == [0.0, 0.0]


def test_parameters_that_are_their_own_masters():
    m = Model([4097, 12], 2, 3, "fp32", "fp32", "fp32", masters=False)
    plan = m.plan()
    want = m.want()
    plan.step(step=m.number, **HYPER)
    torch.cuda.synchronize()
    m.check(want)
    same = Model([4097, 12], 2, 3, "fp32", "fp32", "fp32", masters=False)
    same.plan(masters=same.params[0].views).step(step=same.number, **HYPER)
    torch.cuda.synchronize()
    for a, b in zip(m.params[2].views, same.params[2].views):
        assert torch.equal(a, b)


@pytest.mark.parametrize("states", ["fp32", "e4m3"])
def test_states_begin_at_zero(states):
    """Step 1 on zeroed states: m / c1 = g, sqrt(v / c2) = |g|: a parameter moves by lr against its gradient's sign, and one without
    a gradient stays."""
    m = Model([3000], 2, 1, "fp32", "fp32", states, step=1)
    for f in [m.m, m.v] + ([m.m_scale, m.v_scale] if m.m_scale else []):
        for v in f.views:
            v.view(torch.uint8).zero_()
    for f in m.grads:
        f.views[0][100:600] = 0
    p = m.master.views[0].clone()
    want = m.want()
    m.plan().step(step=1, **HYPER)
    torch.cuda.synchronize()
    m.check(want)
    assert torch.equal(p[100:600], m.master.views[0][100:600])
    moved = (p - m.master.views[0]).double()
    g = m.fold(0)[0]
    strong = g.abs() > 1e-4  # eps is 1e-4 of these; both signs and 1 % of lr
    assert bool(((moved[strong] - HYPER["lr"] * g[strong].sign()).abs() < 0.01 * HYPER["lr"]).all())


def test_small_roots_keep_a_code():
    """One element of a block 10^6 times the others: their roots are below half the smallest code and still do not vanish."""
    m = Model([512], 1, 1, "fp32", "fp32", "e4m3", scale=1e-3)
    m.grads[0].views[0].fill_(1e-6)
    m.grads[0].views[0][7] = 10.0
    for f in (m.m, m.v, m.m_scale, m.v_scale):
        f.views[0].view(torch.uint8).zero_()
    want = m.want()
    plan = m.plan()
    plan.step(step=m.number, **HYPER)
    torch.cuda.synchronize()
    m.check(want)
    assert bool((m.v.views[0].float() > 0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_step_whose_clip_is_not_finite_changes_nothing(bad):
    m = Model([700, 3000], 2, 2, states="e4m3")
    before = [f.data.clone().view(torch.uint8) for f in m.flats()]
    plan = m.plan()
    plan.step(step=3, clip=torch.tensor([bad], device=DEV), **HYPER)
    torch.cuda.synchronize()
    for f, b in zip(m.flats(), before):
        assert torch.equal(f.data.view(torch.uint8), b)
    want = m.want(0.5)
    m.number = 10
    plan.step(step=10, clip=torch.tensor([0.5], device=DEV), **HYPER)
    torch.cuda.synchronize()
    m.check(want)


def test_the_norm_of_gradients_that_are_not_finite_and_of_large_ones():
    m = Model([5000, 9], 2, 1, "fp32", "fp32", "fp32")
    plan = m.plan()
    out = torch.zeros(plan.norm_floats, device=DEV)
    m.grads[0].views[0].fill_(1e30)  # squares past 32 bits
    m.grads[1].views[0].fill_(1e30)
    plan.grad_norm(out, max_norm=1.0)
    torch.cuda.synchronize()
    assert abs(float(out[0]) / (2e30 * math.sqrt(5000)) - 1) < 4 * U and abs(float(out[1]) * float(out[0]) - 1) < 4 * U
    for bad in (float("inf"), float("nan")):
        m.grads[1].views[1][3] = bad
        plan.grad_norm(out, max_norm=1.0)
        torch.cuda.synchronize()
        assert not math.isfinite(float(out[0])) and math.isnan(float(out[1]))
    before = m.master.data.clone()
    plan.step(step=1, clip=out[1:], **HYPER)
    torch.cuda.synchronize()
    assert torch.equal(before, m.master.data)


def test_no_gradients_at_all():
    for lengths in ([], [0, 0]):
        m = Model(lengths, 2, 2)
        plan = m.plan()
        out = torch.full((plan.norm_floats,), 7.0, device=DEV)
        plan.grad_norm(out, max_norm=2.0)
        plan.step(step=1, **HYPER)
        torch.cuda.synchronize()
        assert out.tolist() == [0.0, 1.0]


def test_what_a_made_plan_refuses():
    m = Model([100], 1, 1)
    plan = m.plan()
    out = torch.zeros(plan.norm_floats + 1, device=DEV)
    for call, text in ((lambda: plan.step(step=0, **HYPER), "counts from 1"), (lambda: plan.step(step=-1, **HYPER), "counts from 1"),
                       (lambda: plan.step(step=1, **dict(HYPER, beta1=1.0)), "beta"), (lambda: plan.step(step=1, **dict(HYPER, eps=-1.0)), "eps"),
                       (lambda: plan.step(step=1, **dict(HYPER, lr=float("nan"))), "lr"), (lambda: plan.step(step=1, clip=out.data_ptr() + 2, **HYPER), "clip"),
                       (lambda: plan.grad_norm(out[1:]), "multiple of 8"), (lambda: plan.grad_norm(None), "out is null"),
                       (lambda: plan.grad_norm(out, max_norm=-1.0), "max_norm"), (lambda: plan.grad_norm(out, grad_scale=float("inf")), "grad_scale"),
                       (lambda: m.plan(params=None).step(step=1, **HYPER), "without parameters")):
        with pytest.raises(mr.MegRayError, match=text):
            call()
    torch.cuda.synchronize()


def test_the_same_bits_every_time_and_from_a_graph():
    """A captured norm and clipped step, replayed on new gradients between the program's own work, give the bits of eager ones."""
    lengths = [30000, 5, 4096]
    captured, eager = (Model(lengths, 4, 4, "bf16", "bf16", "e4m3", seed=3) for _ in range(2))
    plans = [m.plan() for m in (captured, eager)]
    outs = [torch.zeros(p.norm_floats, device=DEV) for p in plans]
    side = torch.cuda.Stream()

    def both(plan, out, stream):
        plan.grad_norm(out, grad_scale=0.25, max_norm=0.1, stream=stream)
        plan.step(step=5, grad_scale=0.25, clip=out[1:], stream=stream, **HYPER)

    side.wait_stream(torch.cuda.current_stream())
    both(plans[0], outs[0], side)
    both(plans[1], outs[1], None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        both(plans[0], outs[0], torch.cuda.current_stream())
    for replay in range(4):
        g = torch.Generator(device=DEV).manual_seed(replay)
        for a, b in zip(captured.grads, eager.grads):
            for x, y in zip(a.views, b.views):
                x.copy_(torch.randn(x.numel(), generator=g, device=DEV) * 0.01)
                y.copy_(x)
        torch.cuda.synchronize()
        graph.replay()
        both(plans[1], outs[1], None)
        torch.cuda.synchronize()
        for a, b in zip(captured.flats(), eager.flats()):
            assert torch.equal(a.data.view(torch.uint8), b.data.view(torch.uint8)), replay
        assert outs[0][:2].tolist() == outs[1][:2].tolist()


def test_a_long_tensor():
    """Enough elements for every workgroup of the norm to walk several tiles, and for the step's grid to be a large one."""
    n = 12_000_001
    m = Model([n], 2, 1, "bf16", "bf16", "fp32", offset=1)
    plan = m.plan()
    want = m.want()
    out = torch.zeros(plan.norm_floats, device=DEV)
    plan.grad_norm(out)
    plan.step(step=m.number, clip=out[1:], **HYPER)
    torch.cuda.synchronize()
    m.check(want)
    norm = math.sqrt(float(m.fold(0)[0].square().sum()))
    assert abs(float(out[0]) / norm - 1) <= 8 * U and float(out[1]) == 1.0
