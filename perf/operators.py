"""What follows a reduction in a tensor- and data-parallel model, measured: the fold of the ranks' partial activations
with the residual's addition and a root-mean-square norm (forward and backward), the norm of the folded gradients, and
the AdamW step that takes them and writes the new parameters to every rank.

`run` computes a case in elementary torch operations, or, where `own` is true, through megray_amd's entry points.
All ranks' buffers lie in one GPU's memory, as everywhere in this library: axis 0 of a tensor here is the rank.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5
BLOCK = 256           # elements that share a scale in an 8-bit optimizer state
Q_MAX = 448.0         # largest finite float8_e4m3fn
AMAX_MIN = 2.0 ** -100  # the smallest row or block maximum a scale is made from
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
SIZES = {"fp16": 2, "bf16": 2, "fp32": 4, "e4m3": 1}
LARGEST = 3.4e9       # bytes of the largest listed activations case

STEP = dict(lr=5e-5, step=1000, beta1=0.9, beta2=0.95, eps=1e-8)
DECAY = 0.1
GRAD_SCALE = 1.0 / 8
CLIP = 0.7
MAX_NORM = 1.0


def listed():
    return [
        # decoding one token: one row behind a layer's output projection, eight tensor-parallel ranks; latency
        {"name": "norm one token", "op": "norm", "way": "all_reduce", "ranks": 8, "rows": 1, "cols": 8192,
         "type": "bf16", "stream": "bf16", "out": "bf16", "gap": 0},
        # decoding a batch whose next product runs in 8 bits: a code per value, a scale per row
        {"name": "norm batch to 8 bits", "op": "norm", "way": "all_reduce", "ranks": 8, "rows": 128, "cols": 5120,
         "type": "bf16", "stream": "bf16", "out": "e4m3", "gap": 0},
        # prompts / a training batch: the layer boundary at its full size
        {"name": "norm prompt", "op": "norm", "way": "all_reduce", "ranks": 8, "rows": 8192, "cols": 8192,
         "type": "bf16", "stream": "bf16", "out": "bf16", "gap": 0},
        # sequence parallel: each rank keeps its own rows of a 32-bit residual stream; odd sizes, padded rows
        {"name": "norm ragged shards", "op": "norm", "way": "reduce_scatter", "ranks": 4, "rows": 1023, "cols": 4099,
         "type": "fp16", "stream": "fp32", "out": "fp16", "gap": 3},
        # backward of a small fine-tuning batch
        {"name": "norm gradient small", "op": "norm_grad", "way": "all_reduce", "ranks": 2, "rows": 64, "cols": 2048,
         "type": "fp16", "stream": "fp16", "out": "fp16", "gap": 0},
        # backward of a training batch at its full size
        {"name": "norm gradient batch", "op": "norm_grad", "way": "all_reduce", "ranks": 8, "rows": 8192, "cols": 8192,
         "type": "bf16", "stream": "bf16", "out": "bf16", "gap": 0},
        # backward of the sequence-parallel form, three ranks, odd width, 32-bit residual stream
        {"name": "norm gradient ragged shards", "op": "norm_grad", "way": "reduce_scatter", "ranks": 3, "rows": 1365,
         "cols": 5001, "type": "bf16", "stream": "fp32", "out": "bf16", "gap": 0},
        # a small model's step: dozens of tensors, most of them a few KiB; launches
        {"name": "adamw small tensors", "op": "adamw", "ranks": 2, "width": 96, "layers": 6, "type": "fp16",
         "params": "fp16", "states": "fp32", "skew": 0},
        # a shard of a large model's step: eight data-parallel ranks, 32-bit states
        {"name": "adamw large", "op": "adamw", "ranks": 8, "width": 1280, "layers": 5, "type": "bf16",
         "params": "bf16", "states": "fp32", "skew": 0},
        # the same step with 8-bit states, odd widths, buffers off every boundary
        {"name": "adamw 8-bit states", "op": "adamw", "ranks": 4, "width": 1025, "layers": 4, "type": "bf16",
         "params": "bf16", "states": "e4m3", "skew": 1},
        # the gradients' norm of a small model, on which the step waits
        {"name": "gradient norm small", "op": "grad_norm", "ranks": 4, "width": 128, "layers": 4, "type": "fp32",
         "skew": 0},
        # the gradients' norm of a large model's shard
        {"name": "gradient norm large", "op": "grad_norm", "ranks": 8, "width": 1280, "layers": 5, "type": "bf16",
         "skew": 0},
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng: random.Random):
    op = rng.choice(["norm", "norm", "norm_grad", "norm_grad", "adamw", "grad_norm"])
    ranks = rng.choice([1, 2, 3, 4, 5, 6, 8, 8, 16])
    kind = rng.choice(["fp16", "bf16", "bf16", "fp32"])
    if op in ("norm", "norm_grad"):
        case = {"op": op, "way": rng.choice(["all_reduce", "all_reduce", "reduce_scatter"]), "ranks": ranks}
        case["rows"], case["cols"] = _spread(rng, 1, 8192), _spread(rng, 64, 16384)
        case["type"], case["stream"] = kind, rng.choice([kind, kind, "fp32"])
        case["out"] = rng.choice([kind, "e4m3"]) if op == "norm" else kind
        case["gap"] = rng.choice([0, 0, 0, 8, 3])
        while work(case)["bytes"] > LARGEST:
            case["rows"] = max(1, case["rows"] // 2)
        return case
    case = {"op": op, "ranks": ranks, "width": _spread(rng, 32, 1280), "layers": _spread(rng, 1, 8), "type": kind}
    if op == "adamw":
        case["params"] = rng.choice([kind, kind, "bf16"])
        case["states"] = rng.choice(["fp32", "e4m3"])
    case["skew"] = rng.choice([0, 0, 1, 5])
    while work(case)["bytes"] > LARGEST and case["layers"] > 1:
        case["layers"] -= 1
    while work(case)["bytes"] > LARGEST:
        case["width"] = case["width"] * 3 // 4
    return case


def _lengths(case):
    """The tensors of `layers` transformer layers: four square matrices, two of a four times wider hidden layer, and the
    vectors of norms and biases."""
    w = case["width"]
    return ([w * w] * 4 + [4 * w * w] * 2 + [w] * 4 + [4 * w]) * case["layers"]


def _places(case):
    """(offset of each tensor in a rank's flat buffer, the buffer's length): tensors start a multiple of BLOCK apart."""
    offsets, at = [], 0
    for n in _lengths(case):
        offsets.append(at)
        at += -(-n // BLOCK) * BLOCK
    return offsets, at


def work(case):
    n = case["ranks"]
    t = SIZES[case["type"]]
    if case["op"] in ("norm", "norm_grad"):
        rows, cols, r = case["rows"], case["cols"], SIZES[case["stream"]]
        copies = n if case["way"] == "all_reduce" else 1
        folded = rows * cols * (1 if case["way"] == "all_reduce" else n)  # elements behind the fold
        if case["op"] == "norm":
            moved = folded * (n * t + r + copies * (r + SIZES[case["out"]])) + cols * t
            moved += folded // cols * copies * 4 * (case["out"] == "e4m3")
            return {"bytes": moved, "flops": folded * (n + 6)}
        both = copies * t if case["stream"] != case["type"] else 0
        return {"bytes": folded * (n * t + 2 * r + copies * r + both) + cols * t + n * cols * 4, "flops": folded * (n + 12)}
    total = sum(_lengths(case))
    if case["op"] == "grad_norm":
        return {"bytes": total * n * t + 8, "flops": total * (n + 2)}
    state = 24 if case["states"] == "fp32" else 12
    scales = 0 if case["states"] == "fp32" else 4 * 4 * _places(case)[1] // BLOCK
    return {"bytes": total * (n * t + state + n * SIZES[case["params"]]) + scales, "flops": total * (n + 16)}


def _normal(shape, kind, g, scale=1.0):
    return torch.randn(shape, device=DEV, generator=g, dtype=torch.float32).mul_(scale).to(TYPES[kind])


def _inputs(case, seed):
    """The tensors a case works on, from the seed alone."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    n, kind = case["ranks"], case["type"]
    if case["op"] in ("norm", "norm_grad"):
        rows, cols = case["rows"], case["cols"]
        folded = rows if case["way"] == "all_reduce" else rows * n
        shards = (rows, cols) if case["way"] == "all_reduce" else (n, rows, cols)
        s = {"send": torch.empty(n, folded, cols + case["gap"], device=DEV, dtype=TYPES[kind])}
        for r in range(n):
            s["send"][r] = _normal((folded, cols + case["gap"]), kind, g, 0.5)
        s["weight"] = (1 + 0.2 * torch.randn(cols, device=DEV, generator=g)).to(TYPES[kind])
        if case["op"] == "norm":
            s["residual"] = _normal(shards, case["stream"], g, 2.0)
            s["hidden"] = torch.empty(n, rows, cols, device=DEV, dtype=TYPES[case["stream"]])
            s["out"] = torch.empty(n, rows, cols, device=DEV, dtype=TYPES[case["out"]])
            if case["out"] == "e4m3":
                s["scales"] = torch.empty(n, rows, device=DEV)
            return s
        s["hidden"] = _normal(shards, case["stream"], g, 2.0)
        s["arriving"] = _normal(shards, case["stream"], g, 0.5)
        s["dhidden"] = torch.empty(n, rows, cols, device=DEV, dtype=TYPES[case["stream"]])
        if case["stream"] != kind:
            s["dsend"] = torch.empty(n, rows, cols, device=DEV, dtype=TYPES[kind])
        s["dweight"] = torch.empty(n, cols, device=DEV)
        return s
    offsets, total = _places(case)
    lengths, skew = _lengths(case), case["skew"]
    used = torch.zeros(total, device=DEV)
    for at, m in zip(offsets, lengths):
        used[at:at + m] = 1
    s = {"grads": torch.zeros(n, total + 8, device=DEV, dtype=TYPES[kind])[:, skew:skew + total]}
    for r in range(n):
        s["grads"][r] = torch.randn(total, device=DEV, generator=g).mul_(1e-2).mul_(used).to(TYPES[kind])
    if case["op"] == "grad_norm":
        return s
    s["master"] = torch.zeros(total + 8, device=DEV)[skew:skew + total]
    s["master"].copy_(torch.randn(total, device=DEV, generator=g).mul_(0.05).mul_(used))
    s["params"] = torch.zeros(n, total + 8, device=DEV, dtype=TYPES[case["params"]])[:, skew:skew + total]
    s["params"].copy_(s["master"])
    m = torch.randn(total, device=DEV, generator=g).mul_(1e-3).mul_(used)
    v = torch.rand(total, device=DEV, generator=g).add_(0.5).mul_(4e-6).mul_(used)
    if case["states"] == "fp32":
        s["m"], s["v"] = m, v
    else:
        s["m"], s["m_scale"] = _to_8_bits(m)
        s["v"], s["v_scale"] = _to_8_bits(v.sqrt(), keep=True)
    s["decay"] = torch.tensor([DECAY if k > case["width"] * 4 else 0.0 for k in lengths], device=DEV)
    s["tensor_of"] = torch.repeat_interleave(torch.arange(len(lengths), device=DEV),
                                             torch.tensor([-(-k // BLOCK) for k in lengths], device=DEV))
    s["clip"] = torch.tensor([CLIP], device=DEV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        s["plan"] = _plan(case, s)
    return s


def _plan(case, s):
    """What a program that makes the same call on the same buffers again and again keeps of it."""
    import megray_amd as mr
    types = {"fp16": mr.DType.FLOAT16, "bf16": mr.DType.BFLOAT16, "fp32": mr.DType.FLOAT32, "e4m3": mr.DType.FLOAT8_E4M3}
    if case["op"] in ("norm", "norm_grad"):
        gathered = case["way"] == "all_reduce"
        way = mr.Collective.ALL_REDUCE if gathered else mr.Collective.REDUCE_SCATTER
        each = (lambda t: [t]) if gathered else list
        if case["op"] == "norm":
            return mr.RmsNormPlan(way, list(s["send"]), list(s["out"]), s["weight"], case["rows"], case["cols"],
                                  types[case["type"]], EPS, residuals=each(s["residual"]), residual_outs=list(s["hidden"]),
                                  scales=list(s["scales"]) if "scales" in s else None, residual_dtype=types[case["stream"]],
                                  out_dtype=types[case["out"]], send_stride=case["cols"] + case["gap"])
        size = mr.rms_norm_backward_workspace(way, case["ranks"], case["rows"], case["cols"])
        s["workspace"] = torch.empty(size, device=DEV, dtype=torch.uint8)
        return mr.RmsNormBackwardPlan(way, list(s["send"]), each(s["hidden"]), s["weight"], list(s["dhidden"]), case["rows"],
                                      case["cols"], types[case["type"]], EPS, residual_grads=each(s["arriving"]),
                                      send_grads=list(s["dsend"]) if "dsend" in s else None,
                                      weight_grads=list(s["dweight"]), workspace=s["workspace"],
                                      residual_dtype=types[case["stream"]], send_stride=case["cols"] + case["gap"])
    offsets, _ = _places(case)
    lengths = _lengths(case)
    views = lambda t: [t[at:at + k] for at, k in zip(offsets, lengths)]  # noqa: E731
    ranks = lambda t: [views(x) for x in t]  # noqa: E731
    if case["op"] == "grad_norm":
        plan = mr.AdamWPlan(ranks(s["grads"]), lengths, types[case["type"]])
        s["norm"] = torch.empty(plan.norm_floats, device=DEV)
        return plan
    blocks = lambda t: [t[at // BLOCK:] for at in offsets]  # noqa: E731
    return mr.AdamWPlan(ranks(s["grads"]), lengths, types[case["type"]], params=ranks(s["params"]), param_dtype=types[case["params"]],
                        masters=views(s["master"]), exp_avgs=views(s["m"]), exp_avg_sqs=views(s["v"]),
                        state_dtype=types[case["states"]],
                        exp_avg_scales=blocks(s["m_scale"]) if "m_scale" in s else None,
                        exp_avg_sq_scales=blocks(s["v_scale"]) if "v_scale" in s else None,
                        weight_decays=[DECAY if k > case["width"] * 4 else 0.0 for k in lengths])


def run(s):
    case = s["case"]
    if case["op"] == "norm":
        if own:
            s["plan"].launch()
        else:
            _norm(case, s)
        return {k: s[k] for k in ("out", "hidden", "scales") if k in s}
    if case["op"] == "norm_grad":
        if own:
            s["plan"].launch()
        else:
            _norm_grad(case, s)
        return {k: s[k] for k in ("dhidden", "dsend", "dweight") if k in s}
    if case["op"] == "grad_norm":
        if own:
            s["plan"].grad_norm(s["norm"], grad_scale=GRAD_SCALE, max_norm=MAX_NORM)
            return s["norm"][:2]
        g = s["grads"].sum(0, dtype=torch.float32) * GRAD_SCALE
        norm = (g * g).sum(dtype=torch.float64).sqrt()
        return torch.stack([norm, torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)]).float()
    if own:
        s["plan"].step(grad_scale=GRAD_SCALE, clip=s["clip"], **STEP)
    else:
        _adamw(case, s)
    return {k: s[k] for k in ("params", "master", "m", "v", "m_scale", "v_scale") if k in s}


# the plain forms: elementary operations in 32 bits, rounded once at the end

def _fold(case, s):
    """The ranks' rows summed in 32 bits: [rows, cols] for an all_reduce, [ranks, rows, cols] for a reduce_scatter."""
    x = s["send"][:, :, :case["cols"]].sum(0, dtype=torch.float32)
    return x if case["way"] == "all_reduce" else x.view(case["ranks"], case["rows"], case["cols"])


def _norm(case, s):
    h = s["residual"].float() + _fold(case, s)
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    s["hidden"].copy_(h.to(s["hidden"].dtype))  # one row set for every rank of an all_reduce
    if case["out"] == "e4m3":
        scale = torch.clamp(y.abs().amax(-1, keepdim=True), min=AMAX_MIN) / Q_MAX
        s["scales"].copy_(scale[..., 0])
        y = torch.clamp(y / scale, -Q_MAX, Q_MAX)
    s["out"].copy_(y.to(s["out"].dtype))


def _norm_grad(case, s):
    g, h = _fold(case, s), s["hidden"].float()
    r = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    gw = g * s["weight"].float()
    dh = r * gw - h * (r * r * r) * (gw * h).mean(-1, keepdim=True) + s["arriving"].float()
    s["dhidden"].copy_(dh.to(s["dhidden"].dtype))
    if "dsend" in s:
        s["dsend"].copy_(dh.to(s["dsend"].dtype))
    s["dweight"].copy_((g * h * r).sum(-2))


def _to_8_bits(x, keep=False):
    """Codes and a scale for each BLOCK values; `keep`: what is above zero stays above zero."""
    x = x.view(-1, BLOCK)
    scale = torch.clamp(x.abs().amax(1), min=AMAX_MIN) / Q_MAX
    q = torch.clamp(x / scale[:, None], -Q_MAX, Q_MAX)
    if keep:
        q = torch.where(x > 0, torch.clamp(q, min=2.0 ** -9), q)
    return q.to(torch.float8_e4m3fn).view(-1), scale


def _adamw(case, s):
    lr, b1, b2 = STEP["lr"], STEP["beta1"], STEP["beta2"]
    g = s["grads"].sum(0, dtype=torch.float32) * (GRAD_SCALE * s["clip"])
    if case["states"] == "fp32":
        m, v = s["m"], s["v"]
    else:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1)
        v = v * v
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    root = v.sqrt()
    keep = (1 - lr * s["decay"])[s["tensor_of"]][:, None]
    update = lr / (1 - b1 ** STEP["step"]) * m / (root / math.sqrt(1 - b2 ** STEP["step"]) + STEP["eps"])
    p = (s["master"].view(-1, BLOCK) * keep).view(-1) - update
    s["master"].copy_(p)
    s["params"].copy_(p.to(s["params"].dtype))
    if case["states"] == "fp32":
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        q, scale = _to_8_bits(m)
        s["m"].copy_(q)
        s["m_scale"].copy_(scale)
        q, scale = _to_8_bits(root, keep=True)
        s["v"].copy_(q)
        s["v_scale"].copy_(scale)


# the operators' definitions in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    n = case["ranks"]
    total = None
    terms = s["send"][:, :, :case["cols"]] if "send" in s else s["grads"]
    for r in range(n):  # one rank at a time: 64-bit copies of all of them at once would not be small
        total = terms[r].double() if total is None else total.add_(terms[r].double())
    everyone = lambda t: t.unsqueeze(0).expand(n, *t.shape)  # noqa: E731
    if case["op"] in ("norm", "norm_grad"):
        shared = case["way"] == "all_reduce"
        if not shared:
            total = total.view(n, case["rows"], case["cols"])
        w, cols = s["weight"].double(), case["cols"]
        if case["op"] == "norm":
            h = total + s["residual"].double()
            y = h / torch.sqrt(torch.linalg.vector_norm(h, dim=-1, keepdim=True) ** 2 / cols + EPS) * w
            got = {"hidden": h}
            if case["out"] == "e4m3":
                top = torch.linalg.vector_norm(y, ord=math.inf, dim=-1)
                got["scales"] = top.clamp(min=AMAX_MIN) / Q_MAX
                got["out"] = y / got["scales"].unsqueeze(-1)
            else:
                got["out"] = y
            return {k: everyone(v) for k, v in got.items()} if shared else got
        h = s["hidden"].double()
        size = torch.sqrt(torch.linalg.vector_norm(h, dim=-1, keepdim=True) ** 2 / cols + EPS)
        unit = h / size
        inner = torch.einsum("...c,c,...c->...", total, w, unit).unsqueeze(-1) / cols
        dh = (total * w - unit * inner) / size + s["arriving"].double()
        got = {"dhidden": dh, "dweight": torch.einsum("...rc,...rc->...c", total, unit)}
        if "dsend" in s:
            got["dsend"] = dh
        return {k: everyone(v) for k, v in got.items()} if shared else got
    total.mul_(GRAD_SCALE)
    if case["op"] == "grad_norm":
        norm = float(torch.linalg.vector_norm(total))
        return torch.tensor([norm, min(1.0, MAX_NORM / (norm + 1e-6))], dtype=torch.float64)
    total.mul_(float(s["clip"].double()))
    m, v = s["m"].double(), s["v"].double()
    if case["states"] != "fp32":
        m = m * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (v * s["v_scale"].double().repeat_interleave(BLOCK)).square()
    m = STEP["beta1"] * m + (1 - STEP["beta1"]) * total
    v = STEP["beta2"] * v + (1 - STEP["beta2"]) * total.square()
    p = s["master"].double()
    p = p - STEP["lr"] * s["decay"].double()[s["tensor_of"]].repeat_interleave(BLOCK) * p
    p = p - STEP["lr"] * (m / (1 - STEP["beta1"] ** STEP["step"])) / (torch.sqrt(v / (1 - STEP["beta2"] ** STEP["step"])) + STEP["eps"])
    got = {"master": p, "params": everyone(p)}
    if case["states"] == "fp32":
        return dict(got, m=m, v=v)
    for name, x in (("m", m), ("v", v.sqrt())):
        top = x.view(-1, BLOCK).abs().amax(1).clamp(min=AMAX_MIN)
        got[name + "_scale"] = top / Q_MAX
        x = x / got[name + "_scale"].repeat_interleave(BLOCK)
        got[name] = torch.where(x > 0, x.clamp(min=2.0 ** -9), x) if name == "v" else x
    return got
