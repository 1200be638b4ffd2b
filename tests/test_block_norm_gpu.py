"""block_norm and its gradient against the 64-bit oracle.

Tolerances, per element: a bf16 result may be off by half a unit in its last place
(2^-8 of its value); fp32 arithmetic by a few 2^-24 of the magnitudes that enter it,
taken as 4e-6 of their sum (a row sum in pieces of 8 and a tree loses under 2e-6)."""
import numpy as np
import pytest

from oracle import attn_block_oracle as A

pytestmark = pytest.mark.gpu

BF16_HALF_ULP = 2.0 ** -8
F32 = 4e-6
F32_SUM = 1e-5          # column sums over thousands of rows in partial sums

CASES = [  # R, D, gate rows (None, 1, G, "row"), residual fp32, post, pre
    (1, 8, 1, False, True, True),
    (1, 2048, None, True, True, True),
    (3, 64, "row", False, True, True),
    (37, 256, 1, True, True, True),
    (40, 264, 4, False, True, True),
    (129, 520, 3, True, True, True),
    (8, 2048, 1, False, True, True),
    (300, 2048, 2, True, True, True),
    (17, 4096, "row", True, True, True),
    (5, 8192, 5, False, True, True),
    (9, 8184, 1, True, True, True),
    (1000, 128, None, False, True, True),
    (33, 1000, 1, False, False, True),
    (33, 1000, 11, True, True, False),
    (12, 512, "row", False, False, False),
    (2500, 72, 5, True, True, True),
]


def _inputs(R, D, gate, f32, post, pre, seed=0):
    import torch
    g = torch.Generator("cuda").manual_seed(seed + R * 31 + D)

    def rn(*s, scale=1.0, shift=0.0, dt=torch.bfloat16):
        return (torch.randn(*s, generator=g, device="cuda") * scale + shift).to(dt)
    hd = torch.float32 if f32 else torch.bfloat16
    shape = None if gate is None else (D,) if gate == 1 else (R if gate == "row" else gate, D)
    return dict(y=rn(R, D), h=rn(R, D, scale=2.0, dt=hd), gamma_post=rn(D, scale=0.1, shift=1.0) if post else None,
                gate=None if shape is None else rn(*shape, scale=0.4, shift=0.3),
                gamma_pre=rn(D, scale=0.1, shift=1.0) if pre else None, dh=rn(R, D, dt=hd), dx=rn(R, D))


def _np(t):
    return None if t is None else t.double().cpu().numpy()


def _close(got, want, tol, what):
    bad = ~(np.abs(_np(got) - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.abs(_np(got) - want)[bad].max():.3e}"


@pytest.mark.parametrize("R,D,gate,f32,post,pre", CASES)
def test_forward(cuda_device, R, D, gate, f32, post, pre):
    import torch
    import gdn_18646_b200 as G
    s = _inputs(R, D, gate, f32, post, pre)
    h, x = G.block_norm(s["y"], s["h"], gamma_post=s["gamma_post"], gate=s["gate"], gamma_pre=s["gamma_pre"],
                        residual_scale=0.8, eps=1e-5)
    wh, wx = A.block_norm(_np(s["y"]), _np(s["h"]), _np(s["gamma_post"]), _np(s["gate"]), _np(s["gamma_pre"]), 0.8, 1e-5)
    mag = np.abs(0.8 * _np(s["h"])) + np.abs(wh - 0.8 * _np(s["h"]))
    assert h.dtype == s["h"].dtype
    _close(h, wh, F32 * mag + (0 if f32 else BF16_HALF_ULP * np.abs(wh)), "h")
    if pre:
        scale = A.rms(wh, 1e-5) * np.abs(_np(s["gamma_pre"]))
        _close(x, wx, BF16_HALF_ULP * np.abs(wx) + 2 * F32 * mag * scale, "x")
    else:
        assert x is None
    # in place on the residual stream: the same bits
    h2 = s["h"].clone()
    x2 = None if x is None else torch.empty_like(x)
    G.block_norm(s["y"], h2, gamma_post=s["gamma_post"], gate=s["gate"], gamma_pre=s["gamma_pre"], residual_scale=0.8,
                 eps=1e-5, h_out=h2, x_out=x2)
    assert torch.equal(h2, h) and (x is None or torch.equal(x2, x))


@pytest.mark.parametrize("R,D,gate,f32,post,pre", CASES)
def test_backward(cuda_device, R, D, gate, f32, post, pre):
    import torch
    import gdn_18646_b200 as G
    s = _inputs(R, D, gate, f32, post, pre, seed=7)
    args = dict(gamma_post=s["gamma_post"], gate=s["gate"], gamma_pre=s["gamma_pre"], residual_scale=0.8, eps=1e-5)
    g = G.block_norm_backward(s["y"], s["h"], s["dh"], s["dx"] if pre else None, **args)
    w = A.block_norm_backward(_np(s["y"]), _np(s["h"]), _np(s["dh"]), _np(s["dx"]), _np(s["gamma_post"]), _np(s["gate"]),
                              _np(s["gamma_pre"]), 0.8, 1e-5)
    for key in ("dy", "dh", "dgate", "dgamma_post", "dgamma_pre"):
        if key not in w:
            assert g[key] is None
            continue
        bf = g[key].dtype == torch.bfloat16
        assert bf == (key == "dy" or (key == "dh" and not f32) or (key == "dgate" and (gate == "row" or gate == R)
                                                                  and s["gate"].dim() == 2))
        f = F32_SUM if key.startswith("dgamma") or key == "dgate" else 2 * F32
        _close(g[key], w[key], f * w["mag"][key] + (BF16_HALF_ULP * np.abs(w[key]) if bf else 0), key)
    again = G.block_norm_backward(s["y"], s["h"], s["dh"], s["dx"] if pre else None, **args)
    assert all(g[k] is None or torch.equal(g[k], again[k]) for k in g), "the same call gave other bits"


def test_backward_without_residual_gradient(cuda_device):
    import torch
    import gdn_18646_b200 as G
    s = _inputs(21, 512, 1, True, True, True)
    args = dict(gamma_post=s["gamma_post"], gate=s["gate"], gamma_pre=s["gamma_pre"])
    g0 = G.block_norm_backward(s["y"], s["h"], None, s["dx"], **args)
    g1 = G.block_norm_backward(s["y"], s["h"], torch.zeros_like(s["h"]), s["dx"], **args)
    assert all(torch.equal(g0[k], g1[k]) for k in g0)


def test_autograd_matches_differences_of_the_kernel(cuda_device):
    """The gradient of a scalar of both outputs along one direction, against the central
    difference of the kernel's own forward (fp32 residual stream).  bf16 inputs move by
    2^-4, exact in bf16 for these values; the difference is then good to the curvature and
    to x's bf16 rounding, together under 2 % of the derivative's scale."""
    import torch
    import gdn_18646_b200 as G
    s = _inputs(16, 256, 2, True, True, True, seed=3)
    wh, wx = torch.randn(16, 256, device="cuda"), torch.randn(16, 256, device="cuda")
    h = s["h"].clone().requires_grad_(True)
    ho, x = G.block_norm_autograd(s["y"], h, gamma_post=s["gamma_post"], gate=s["gate"], gamma_pre=s["gamma_pre"])
    ((ho * wh).sum() + (x.float() * wx).sum()).backward()
    d = torch.randn(16, 256, device="cuda") * 0.05

    def f(hh):
        a, b = G.block_norm(s["y"], hh, gamma_post=s["gamma_post"], gate=s["gate"], gamma_pre=s["gamma_pre"])
        return float((a.double() * wh).sum() + (b.double() * wx).sum())
    num = f(s["h"] + d) - f(s["h"] - d)
    ana = 2 * float((h.grad.double() * d).sum())
    scale = 2 * float((h.grad.double() * d).norm())
    assert abs(num - ana) < 0.1 * scale + 0.02 * abs(ana)


def test_autograd_all_inputs(cuda_device):
    import torch
    import gdn_18646_b200 as G
    s = _inputs(24, 320, 3, False, True, True)
    ins = [s[k].clone().requires_grad_(True) for k in ("y", "h", "gamma_post", "gate", "gamma_pre")]
    ho, x = G.block_norm_autograd(ins[0], ins[1], gamma_post=ins[2], gate=ins[3], gamma_pre=ins[4], residual_scale=0.5)
    torch.autograd.backward([ho, x], [s["dh"], s["dx"]])
    g = G.block_norm_backward(s["y"], ho.detach(), s["dh"], s["dx"], gamma_post=s["gamma_post"], gate=s["gate"],
                              gamma_pre=s["gamma_pre"], residual_scale=0.5)
    for t, k in zip(ins, ("dy", "dh", "dgamma_post", "dgate", "dgamma_pre")):
        assert t.grad.dtype == t.dtype and torch.equal(t.grad, g[k].to(t.dtype))


def test_empty_and_streams(cuda_device):
    import torch
    import gdn_18646_b200 as G
    s = _inputs(64, 1024, 1, False, True, True)
    args = dict(gamma_post=s["gamma_post"], gate=s["gate"], gamma_pre=s["gamma_pre"])
    h, x = G.block_norm(s["y"][:0], s["h"][:0], **args)
    assert h.shape == (0, 1024) and x.shape == (0, 1024)
    g = G.block_norm_backward(s["y"][:0], s["h"][:0], s["dh"][:0], s["dx"][:0], **args)
    assert all(float(g[k].abs().sum()) == 0 for k in ("dgate", "dgamma_post", "dgamma_pre"))
    want = G.block_norm(s["y"], s["h"], **args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = G.block_norm(s["y"], s["h"], **args)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(cuda_device):
    import torch
    import gdn_18646_b200 as G
    s = _inputs(6, 64, 2, False, True, True)
    y, h = s["y"], s["h"]
    for bad in (dict(gate=torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)),       # 4 does not divide 6
                dict(gate=torch.zeros(32, device="cuda", dtype=torch.bfloat16)),
                dict(gamma_pre=torch.ones(64, device="cuda")),                            # fp32 weight
                dict(gamma_post=s["gamma_post"][:32]),
                dict(h_out=torch.empty(6, 64, device="cuda"))):                           # fp32 result of a bf16 stream
        with pytest.raises(RuntimeError):
            G.block_norm(y, h, **bad)
    for a, b in ((y.float(), h), (y, h.half()), (y, h[:, :32]), (y.cpu(), h), (y[:, ::2], h[:, ::2]),
                 (y[:, :60].contiguous(), h[:, :60].contiguous())):
        with pytest.raises(RuntimeError):
            G.block_norm(a, b)
    with pytest.raises(RuntimeError):
        G.block_norm_backward(y, h, s["dh"], None, gamma_pre=s["gamma_pre"])              # dx missing
    with pytest.raises(RuntimeError):
        G.block_norm_backward(y, h, s["dh"].float(), s["dx"], gamma_pre=s["gamma_pre"])
    with pytest.raises(RuntimeError):
        G.block_norm(torch.zeros(1, 8200, device="cuda", dtype=torch.bfloat16),
                     torch.zeros(1, 8200, device="cuda", dtype=torch.bfloat16))
