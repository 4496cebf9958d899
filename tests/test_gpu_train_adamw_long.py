"""One tensor of more than 2^30 elements, 2^32 bytes and more in 32 bits: the step and the gradients' norm reach its far end."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import megray_amd as mr  # noqa: E402
from test_gpu_train_adamw import BLOCK, TYPES, U, blocks  # noqa: E402

DEV = "cuda:0"
LENGTH = (1 << 30) + (1 << 13) + 777
# places whose values are compared, on the blocks' boundaries: the beginning, across 2^31 bytes and 2^32 bytes of 32 bits, the end
PLACES = [(0, 1024), ((1 << 29) - 512, (1 << 29) + 512), ((1 << 30) - 512, (1 << 30) + 512), ((1 << 30) + (1 << 13), LENGTH)]
STEP = dict(lr=1e-3, step=7, beta1=0.9, beta2=0.99, eps=1e-8)


@pytest.mark.parametrize("grad,param,states", [("fp32", "fp32", "fp32"), ("bf16", "bf16", "e4m3")])
def test_a_tensor_past_32_bit_offsets(grad, param, states):
    g = torch.Generator(device=DEV).manual_seed(3)
    g_type, p_type, s_type = (TYPES[k][0] for k in (grad, param, states))
    lengths = [b - a for a, b in PLACES]
    whole = {"grad": torch.zeros(LENGTH, dtype=g_type, device=DEV), "param": torch.zeros(LENGTH, dtype=p_type, device=DEV),
             "m": torch.zeros(LENGTH, dtype=s_type, device=DEV), "v": torch.zeros(LENGTH, dtype=s_type, device=DEV)}
    whole["master"] = whole["param"] if param == "fp32" else torch.zeros(LENGTH, device=DEV)
    if states == "e4m3":
        whole["m_scale"], whole["v_scale"] = (torch.zeros(blocks(LENGTH), device=DEV) for _ in range(2))
    for a, b in PLACES:
        whole["grad"][a:b] = (torch.randn(b - a, generator=g, device=DEV) * 0.1).to(g_type)
        whole["master"][a:b] = torch.randn(b - a, generator=g, device=DEV)

    def parts(name):
        per = BLOCK if name.endswith("scale") else 1
        return [whole[name][a // per:-(-b // per)] for a, b in PLACES]

    small = {name: [t.clone() for t in parts(name)] for name in whole}
    if param == "fp32":
        small["master"] = small["param"]

    def plan(lens, of):
        scales = dict(exp_avg_scales=of("m_scale"), exp_avg_sq_scales=of("v_scale")) if states == "e4m3" else {}
        return mr.AdamWPlan([of("grad")], lens, TYPES[grad][1], params=[of("param")], param_dtype=TYPES[param][1], masters=of("master"),
                            exp_avgs=of("m"), exp_avg_sqs=of("v"), state_dtype=TYPES[states][1], weight_decays=[0.1] * len(lens), **scales)

    far, near = plan([LENGTH], lambda name: [whole[name]]), plan(lengths, lambda name: small[name])
    out = torch.zeros(far.norm_floats, device=DEV)
    far.grad_norm(out, max_norm=1.0)
    far.step(**STEP)
    near.step(**STEP)
    torch.cuda.synchronize()
    norm = sum(float(t.double().square().sum()) for t in small["grad"]) ** 0.5
    assert abs(float(out[0]) / norm - 1) < 4 * U
    as_bytes = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    for name in whole:
        for k, (a, b) in enumerate(zip(parts(name), small[name])):
            assert torch.equal(as_bytes(a), as_bytes(b)), (name, k)
    # nothing else moved: zero gradients, states and parameters stay zero
    for a, b in zip([0] + [b for _, b in PLACES], [a for a, _ in PLACES] + [LENGTH]):
        for lo in range(a, b, 1 << 27):
            piece = slice(lo, min(b, lo + (1 << 27)))
            assert not bool(whole["param"][piece].any()) and not bool(as_bytes(whole["m"][piece]).any()) and not bool(as_bytes(whole["v"][piece]).any())
