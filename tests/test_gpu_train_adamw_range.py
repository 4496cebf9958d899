"""AdamW on gradients that are not finite, or whose squares leave the 32-bit range: what they reach, and what stays as the formula says."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_train_adamw import BLOCK, HYPER, Model  # noqa: E402


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan"), 1e30])
@pytest.mark.parametrize("states", ["fp32", "e4m3"])
@pytest.mark.parametrize("offset", [0, 3])
def test_gradients_without_a_finite_square(bad, states, offset):
    """One such gradient of 1000: its own state and parameter are lost with 32-bit states, its block's states with 8-bit ones; every other element
    is that of the step without it."""
    at, n = 300, 1000
    plain, hit = (Model([n], 2, 2, "fp32", "fp32", states, offset, seed=4) for _ in range(2))
    hit.grads[1].views[0][at] = bad
    for m in (plain, hit):
        m.plan().step(step=m.number, **HYPER)
    torch.cuda.synchronize()
    others = torch.arange(n, device="cuda:0") != at
    for a, b in zip([plain.master] + plain.params, [hit.master] + hit.params):
        assert torch.equal(a.views[0][others], b.views[0][others])
    if states == "fp32":
        assert torch.equal(plain.m.views[0][others], hit.m.views[0][others]) and torch.equal(plain.v.views[0][others], hit.v.views[0][others])
        assert not bool(torch.isfinite(hit.v.views[0][at]))
    else:
        block = at // BLOCK
        apart = torch.arange(n, device="cuda:0") // BLOCK != block
        for a, b in ((plain.m, hit.m), (plain.v, hit.v)):
            assert torch.equal(a.views[0].view(torch.uint8)[apart], b.views[0].view(torch.uint8)[apart])
        keep = torch.arange(hit.v_scale.views[0].numel(), device="cuda:0") != block
        for a, b in ((plain.m_scale, hit.m_scale), (plain.v_scale, hit.v_scale)):
            assert torch.equal(a.views[0][keep], b.views[0][keep])
        assert bool(torch.isnan(hit.v_scale.views[0][block])) and bool(torch.isnan(hit.v.views[0].float()[~apart]).all())
        if bad != 1e30:  # m itself is finite there
            assert bool(torch.isnan(hit.m_scale.views[0][block])) and bool(torch.isnan(hit.m.views[0].float()[~apart]).all())
    for f in hit.flats():
        assert f.intact()
