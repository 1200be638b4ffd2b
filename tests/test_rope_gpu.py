"""rope, rope_append and the rotation's gradient against the 64-bit oracle.

Tolerance, per element: half a bf16 unit in the last place of the exact result (2^-8 of
its value) and 4e-6 of the pair's magnitude for the fp32 sines, products and angles
(|sin, cos error| <= 2^-21 for the intrinsic, 10^-6 for the reduced angle)."""
import numpy as np
import pytest

from oracle import attn_block_oracle as A
from tests._paged import Batch

pytestmark = pytest.mark.gpu

CASES = [  # T, Hq, Hk, D, rot, sections, style, largest position
    (1, 1, 1, 64, 64, (32,), "half", 10),
    (3, 5, 1, 128, 128, (24, 20, 20), "half", 1000),
    (37, 16, 2, 128, 64, (32,), "interleaved", 100000),
    (130, 7, 7, 64, 32, (3, 13), "half", 5000),
    (5, 3, 2, 256, 128, (16, 24, 24), "interleaved", 2000),
    (64, 4, 4, 256, 256, (128,), "half", 1 << 20),
    (9, 24, 3, 128, 16, (1, 2, 2, 3), "half", 300),
    (2500, 8, 1, 64, 64, (0, 32), "interleaved", 40000),
    (2, 2, 0, 128, 128, (64,), "half", 1 << 24),
]


def _np(t):
    return t.double().cpu().numpy()


def _inv_freq(rot):
    import torch
    return (10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)).float().cuda()


def _pair_mag(x, n, style):
    """|first| + |second| of each value's pair; 0 past the rotation."""
    first, second = (slice(0, n), slice(n, 2 * n)) if style == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    m = np.zeros_like(x)
    s = np.abs(x[..., first]) + np.abs(x[..., second])
    m[..., first], m[..., second] = s, s
    return m


def _check(got, x, pos, f, sections, style, inverse=False):
    want = A.rope(_np(x), pos, _np(f), sections, style, inverse)
    tol = 2.0 ** -8 * np.abs(want) + 4e-6 * _pair_mag(_np(x), len(f), style)
    err = np.abs(_np(got) - want)
    assert (err <= tol).all(), f"worst {np.max(err - tol):.3e} beyond the tolerance"
    rest = _np(x)[..., 2 * len(f):]
    assert np.array_equal(_np(got)[..., 2 * len(f):], rest)


def _inputs(T, Hq, Hk, D, rot, sections, most, seed=0):
    import torch
    g = torch.Generator("cuda").manual_seed(seed + T)
    q = torch.randn(T, Hq, D, generator=g, device="cuda").bfloat16()
    k = torch.randn(T, Hk, D, generator=g, device="cuda").bfloat16() if Hk else None
    pos = torch.randint(0, most + 1, (len(sections), T), generator=g, device="cuda", dtype=torch.int32)
    return q, k, pos, _inv_freq(rot)


@pytest.mark.parametrize("T,Hq,Hk,D,rot,sections,style,most", CASES)
@pytest.mark.parametrize("inverse", [False, True])
def test_rope(cuda_device, T, Hq, Hk, D, rot, sections, style, most, inverse):
    import torch
    import gdn_18646_b200 as G
    q, k, pos, f = _inputs(T, Hq, Hk, D, rot, sections, most)
    qo, ko = G.rope(q, k, pos, f, sections, style=style, inverse=inverse)
    p = pos.cpu().numpy()
    _check(qo, q, p, f, sections, style, inverse)
    if Hk:
        _check(ko, k, p, f, sections, style, inverse)
        q2, k2 = q.clone(), k.clone()
        G.rope(q2, k2, pos, f, sections, style=style, inverse=inverse, q_out=q2, k_out=k2)   # in place
        assert torch.equal(q2, qo) and torch.equal(k2, ko)
    else:
        assert ko is None


def test_rope_strided_batch_and_default_sections(cuda_device):
    import torch
    import gdn_18646_b200 as G
    qkv = torch.randn(2, 11, (6 + 2 + 2) * 64, device="cuda").bfloat16()
    q, k = qkv[..., :384].unflatten(-1, (6, 64)), qkv[..., 384:512].unflatten(-1, (2, 64))
    pos = torch.arange(22, device="cuda", dtype=torch.int32)
    f = _inv_freq(64)
    qo, ko = G.rope(q, k, pos, f)
    want = G.rope(q.contiguous(), k.contiguous(), pos, f, (32,))
    assert qo.shape == (2, 11, 6, 64) and torch.equal(qo, want[0]) and torch.equal(ko, want[1])


@pytest.mark.parametrize("style", ["half", "interleaved"])
def test_gradient(cuda_device, style):
    """The rotation is linear: its gradient is the oracle's inverse rotation, and <dq, R q>
    equals <R^T dq, q> (a difference quotient of any step), up to bf16 rounding of the two."""
    import torch
    import gdn_18646_b200 as G
    q, k, pos, f = _inputs(19, 4, 2, 128, 96, (20, 28), 3000)
    q.requires_grad_(True)
    k.requires_grad_(True)
    qo, ko = G.rope_autograd(q, k, pos, f, (20, 28), style=style)
    dq, dk = torch.randn_like(qo), torch.randn_like(ko)
    torch.autograd.backward([qo, ko], [dq, dk])
    p = pos.cpu().numpy()
    _check(q.grad, dq, p, f, (20, 28), style, True)
    _check(k.grad, dk, p, f, (20, 28), style, True)
    d = torch.randn_like(q.detach())
    lhs = float((G.rope(d, None, pos, f, (20, 28), style=style)[0].double() * dq.double()).sum())
    rhs = float((q.grad.double() * d.double()).sum())
    spread = 2.0 ** -8 * float((d.double() * dq.double()).norm()) * 4    # random signs of the roundings
    assert abs(lhs - rhs) < spread


@pytest.mark.parametrize("layout,pool", [("bthd", "plain"), ("bhtd", "plain"), ("bthd", "pair"), ("bhtd", "pair")])
@pytest.mark.parametrize("lens,D,page,Hq,Hk", [
    ([(1, 1)], 64, 16, 2, 1),
    ([(1, 17), (1, 16), (1, 33)], 128, 16, 8, 2),
    ([(0, 5), (7, 7), (0, 0), (40, 100), (1, 64), (0, 3)], 128, 32, 6, 3),
    ([(65, 129)] + [(2, 2 + i) for i in range(70)], 64, 64, 4, 4),
    ([(300, 2000), (3000, 3100)], 256, 256, 3, 1),
])
def test_append(cuda_device, layout, pool, lens, D, page, Hq, Hk):
    import torch
    import gdn_18646_b200 as G
    b = Batch(lens, Hq, Hk, D, page, layout, pool, seed=5)
    k, v = (torch.randn(b.T, Hk, D, device="cuda").bfloat16() for _ in range(2))
    sections = (D // 4, D // 8, D // 8)
    pos = torch.randint(0, 5000, (3, b.T), device="cuda", dtype=torch.int32)
    f = _inv_freq(D)
    before_k, before_v = b.k.clone(), b.v.clone()
    qo = G.rope_append(b.q, k, v, pos, f, sections, b.k, b.v, b.table, b.cu, b.kv, layout=layout)
    assert G._lib.lib().gdn_check_device_error() == 0
    wq, wk = G.rope(b.q, k, pos, f, sections)
    assert torch.equal(qo, wq)
    for s, (n, kv) in enumerate(lens):
        for i in range(n):
            p = kv - n + i
            page_id, off = b.table_np[s, p // page], p % page
            at = (page_id, off) if layout == "bthd" else (page_id, slice(None), off)
            before_k[at], before_v[at] = wk[b.cu_np[s] + i], v[b.cu_np[s] + i]
    # every other element of the pool is as it was (NaN included): compare the bits
    assert torch.equal(b.k.contiguous().view(torch.int16), before_k.contiguous().view(torch.int16))
    assert torch.equal(b.v.contiguous().view(torch.int16), before_v.contiguous().view(torch.int16))


def test_append_reports_places_outside_the_cache(cuda_device):
    """A page outside the pool, a position outside the table and more tokens than positions:
    skipped on the device and reported, the other tokens written."""
    import torch
    import gdn_18646_b200 as G
    for what in ("page", "negative page", "table", "short", "offsets"):
        b = Batch([(2, 20), (1, 30)], 2, 1, 64, 16, poison=False)
        k, v = (torch.randn(b.T, 1, 64, device="cuda").bfloat16() for _ in range(2))
        pos, f = torch.zeros(1, b.T, device="cuda", dtype=torch.int32), _inv_freq(64)
        good = int(b.table_np[0, 1])
        if what == "page":
            b.table[1, 1] = b.pages
        elif what == "negative page":
            b.table[1, 1] = -5
        elif what == "table":
            b.kv[1] = 10 ** 6
        elif what == "short":
            b.kv[1] = 0
        else:
            b.cu[2] = 2
        snap = b.k.clone()
        G.rope_append(b.q, k, v, pos, f, None, b.k, b.v, b.table, b.cu, b.kv)
        assert G._lib.lib().gdn_check_device_error() == G._lib.GDN_ERR_SHAPE, what
        assert "outside the cache" in G._lib.last_error()
        assert G._lib.lib().gdn_check_device_error() == 0
        snap[good, 2:4] = k[:2]
        assert torch.equal(b.k, snap), what


def test_empty_and_refusals(cuda_device):
    import torch
    import gdn_18646_b200 as G
    q, k, pos, f = _inputs(4, 4, 2, 64, 64, (32,), 100)
    assert G.rope(q[:0], k[:0], pos[:, :0].contiguous(), f)[0].shape == (0, 4, 64)
    bad = [dict(style="other"), dict(sections=(16, 16)), dict(sections=(31,)), dict(q=q.float()), dict(q=q[..., :48]),
           dict(q=q[..., ::2]), dict(k=k[:2]), dict(positions=pos.long()), dict(positions=pos[:, :2].contiguous()),
           dict(inv_freq=f.double()), dict(inv_freq=f[:12].contiguous(), sections=(12,)), dict(q_out=q[:2]),
           dict(inv_freq=_inv_freq(128), sections=(64,)), dict(sections=(40, -8), positions=pos.repeat(2, 1))]
    for d in bad:
        args = dict(q=q, k=k, positions=pos, inv_freq=f, sections=None)
        args.update(d)
        with pytest.raises(RuntimeError):
            G.rope(**args)
    b = Batch([(4, 20)], 4, 2, 64, 16)
    v = torch.randn_like(k)
    ok = dict(q=q, k=k, v=v, positions=pos, inv_freq=f, sections=None, k_cache=b.k, v_cache=b.v, block_table=b.table,
              cu_seqlens=b.cu, kv_lens=b.kv)
    G.rope_append(**ok)
    for d in (dict(v=v[:, :1]), dict(k_cache=b.k.float(), v_cache=b.v.float()), dict(v_cache=b.v[:1]),
              dict(block_table=b.table.long()), dict(cu_seqlens=b.cu[:1]), dict(kv_lens=b.kv.long()), dict(layout="tbhd"),
              dict(k_cache=b.k[:, :12], v_cache=b.v[:, :12]), dict(k_cache=b.k[..., ::2], v_cache=b.v[..., ::2])):
        with pytest.raises(RuntimeError):
            G.rope_append(**dict(ok, **d))
    assert G._lib.lib().gdn_check_device_error() == 0
