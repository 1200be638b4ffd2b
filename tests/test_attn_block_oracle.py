"""The 64-bit oracle of the attention block's operators: its gradients against central
differences, its rotation against complex multiplication, and the attention's rows
against a direct evaluation (CPU only)."""
import numpy as np
import pytest

from oracle import attn_block_oracle as A


def _loss(args, w):
    h, x = A.block_norm(**args)
    return float((h * w[0]).sum() + (0.0 if x is None else (x * w[1]).sum()))


@pytest.mark.parametrize("gate_rows", [None, 1, 2, 6])
@pytest.mark.parametrize("post,pre", [(True, True), (False, True), (True, False)])
def test_block_norm_backward_matches_differences(gate_rows, post, pre):
    rng = np.random.default_rng(3)
    R, D = 6, 8
    p = dict(y=rng.standard_normal((R, D)), h=rng.standard_normal((R, D)),
             gamma_post=1 + 0.2 * rng.standard_normal(D) if post else None,
             gate=None if gate_rows is None else rng.standard_normal(D if gate_rows == 1 else (gate_rows, D)),
             gamma_pre=1 + 0.2 * rng.standard_normal(D) if pre else None, alpha=0.7, eps=1e-3)
    w = rng.standard_normal((2, R, D))
    hn, _ = A.block_norm(**p)
    g = A.block_norm_backward(p["y"], hn, w[0], w[1], p["gamma_post"], p["gate"], p["gamma_pre"], p["alpha"], p["eps"])
    for name, key in (("y", "dy"), ("h", "dh"), ("gamma_post", "dgamma_post"), ("gate", "dgate"),
                      ("gamma_pre", "dgamma_pre")):
        if p[name] is None:
            assert key not in g
            continue
        num = np.zeros_like(p[name])
        for i in np.ndindex(num.shape):
            d = 1e-5
            up, dn = (dict(p, **{name: p[name].copy()}) for _ in range(2))
            up[name][i] += d
            dn[name][i] -= d
            num[i] = (_loss(up, w) - _loss(dn, w)) / (2 * d)
        # central differences: O(d^2) truncation and 1e-16 / d rounding, both below 1e-8 here
        assert np.abs(num - g[key]).max() < 1e-7 * max(1.0, np.abs(num).max())


@pytest.mark.parametrize("style", ["half", "interleaved"])
def test_rope_is_a_rotation(style):
    rng = np.random.default_rng(4)
    T, H, D, sections = 5, 2, 24, (5, 3)
    x, pos = rng.standard_normal((T, H, D)), rng.integers(0, 1000, (2, T))
    f = 100.0 ** (-np.arange(8) / 8)
    y = A.rope(x, pos, f, sections, style)
    back = A.rope(y, pos, f, sections, style, inverse=True)
    assert np.abs(back - x).max() < 1e-12
    assert np.array_equal(y[..., 16:], x[..., 16:])
    a, b = (np.arange(8), np.arange(8) + 8) if style == "half" else (2 * np.arange(8), 2 * np.arange(8) + 1)
    z = (x[..., a] + 1j * x[..., b]) * np.exp(1j * pos[A.axis_of_pairs(sections)] * f[:, None]).T[:, None]
    assert np.abs(y[..., a] - z.real).max() < 1e-12 and np.abs(y[..., b] - z.imag).max() < 1e-12


def test_attention_rows():
    rng = np.random.default_rng(5)
    q, k, v = rng.standard_normal((4, 4, 8)), rng.standard_normal((3, 2, 8)), rng.standard_normal((3, 2, 8))
    o, lse, _ = A.attention(q, k, v, 0.3)
    assert np.all(o[0] == 0) and np.all(lse[0] == -np.inf)           # four tokens, three positions: the first sees none
    assert np.abs(o[1] - np.repeat(v[0], 2, 0)).max() < 1e-15        # one position: its value
    for h in range(4):
        s = 0.3 * k[:, h // 2] @ q[3, h]
        w = np.exp(s) / np.exp(s).sum()
        assert np.abs(o[3, h] - w @ v[:, h // 2]).max() < 1e-14
        assert abs(lse[3, h] - np.log(np.exp(s).sum())) < 1e-14
    ow, _, _ = A.attention(q, k, v, 0.3, window=1)
    assert np.abs(ow[3] - np.repeat(v[2], 2, 0)).max() < 1e-15
    on, _, _ = A.attention(q, k, v, 0.3, causal=False)
    assert np.abs(on[0] - A.attention(q[:1], k, v, 0.3)[0]).max() < 1e-15
