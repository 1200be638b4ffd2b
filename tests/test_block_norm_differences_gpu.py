"""block_norm's gradients against central differences of the kernel's own forward, input by
input: y, h, gamma_post, gate and gamma_pre.

Inputs and steps lie on grids that bf16 holds exactly and the residual stream is fp32, so h' is
exact to fp32 and x to its bf16 rounding.  A direction takes the sign of the gradient in about
three quarters of its elements and the opposite sign in the others, so the difference is a
share of the gradient's 1-norm of N elements, of order step N |g| / 2, which the roundings of
x (2^-9 |x| each, random, of order sqrt(N)) change by under 0.5 % for the row inputs.  The
difference's own error is of third order in the step (step^2 = 0.1 % of a row's scale and
less).  2 % of the derivative holds both; a gamma or a shared gate sums R rows into each of few
elements, where the roundings are 6 sqrt(2) 2^-9 / sqrt(3) of the 2-norm of wx x, six
deviations, on top."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

R, D = 24, 256


def _inputs(gate_shape):
    import torch
    g = torch.Generator("cuda").manual_seed(11)

    def grid(*shape, unit, most, shift=0.0):
        n = torch.randint(-most, most + 1, shape, generator=g, device="cuda")
        return (n * unit + shift).bfloat16()
    return dict(y=grid(R, D, unit=1 / 16, most=24), h=grid(R, D, unit=1 / 16, most=40).float(),
                gamma_post=grid(D, unit=1 / 32, most=12, shift=1.0),
                gate=None if gate_shape is None else grid(*gate_shape, unit=1 / 32, most=12, shift=0.75),
                gamma_pre=grid(D, unit=1 / 32, most=12, shift=1.0))


STEP = dict(y=1 / 32, h=1 / 32, gamma_post=1 / 64, gate=1 / 64, gamma_pre=1 / 64)


@pytest.mark.parametrize("gate_shape", [None, (D,), (3, D), (R, D)])
@pytest.mark.parametrize("through", ["h", "x", "both"])
def test_gradients_match_differences(cuda_device, gate_shape, through):
    import torch
    import gdn_18646_b200 as G
    s = _inputs(gate_shape)
    g = torch.Generator("cuda").manual_seed(5)
    wh = torch.randn(R, D, generator=g, device="cuda") * (through != "x")
    wx = torch.randn(R, D, generator=g, device="cuda").bfloat16() * (through != "h")

    def forward(t):
        h, x = G.block_norm(t["y"], t["h"], gamma_post=t["gamma_post"], gate=t["gate"], gamma_pre=t["gamma_pre"],
                            residual_scale=0.875)
        return h, x, float((h.double() * wh.double()).sum() + (x.double() * wx.double()).sum())
    h, x, _ = forward(s)
    grads = G.block_norm_backward(s["y"], h, wh, wx, gamma_post=s["gamma_post"], gate=s["gate"], gamma_pre=s["gamma_pre"],
                                  residual_scale=0.875)
    noise = 6 * 2 ** 0.5 * 2.0 ** -9 / 3 ** 0.5 * float((wx.double() * x.double()).norm())
    for name in ("y", "h", "gamma_post", "gate", "gamma_pre"):
        if s[name] is None or (name == "gamma_pre" and through == "h"):
            continue
        grad = grads["d" + name].double()
        for seed in range(3):
            flips = torch.from_numpy(np.random.default_rng(seed).random(tuple(grad.shape)) < 0.25).cuda()
            d = STEP[name] * torch.where(flips, -1.0, 1.0) * torch.where(grad >= 0, 1.0, -1.0)
            up, down = ((s[name].double() + k * d).to(s[name].dtype) for k in (1, -1))
            assert torch.equal(up.double() - s[name].double(), d) and torch.equal(s[name].double() - down.double(), d)
            num = forward(dict(s, **{name: up}))[2] - forward(dict(s, **{name: down}))[2]
            ana = 2 * float((grad * d).sum())
            assert abs(num - ana) <= 0.02 * abs(ana) + noise, (name, num, ana, noise)
