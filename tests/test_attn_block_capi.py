"""C ABI checks of the attention block's entry points that need no GPU: bad arguments are
rejected with status codes before any CUDA call (pointers below are never dereferenced,
but for the spec and the sections, which are host memory)."""
import ctypes

import pytest

from gdn_18646_b200 import _lib

FAKE, ODD = 0x10000, 0x10002


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def fwd(**over):
    a = dict(y=FAKE, h=FAKE, hdt=0, gp=FAKE, gate=FAKE, rows=2, gq=FAKE, alpha=1.0, ho=FAKE, x=FAKE, R=6, D=64, eps=1e-6,
             stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(y=None), _lib.GDN_ERR_NULL), (dict(h=None), _lib.GDN_ERR_NULL), (dict(ho=None), _lib.GDN_ERR_NULL),
    (dict(x=None), _lib.GDN_ERR_NULL), (dict(hdt=2), _lib.GDN_ERR_DTYPE), (dict(R=-1), _lib.GDN_ERR_SHAPE),
    (dict(D=60), _lib.GDN_ERR_SHAPE), (dict(D=8200), _lib.GDN_ERR_SHAPE), (dict(D=0), _lib.GDN_ERR_SHAPE),
    (dict(rows=4), _lib.GDN_ERR_SHAPE), (dict(rows=0), _lib.GDN_ERR_SHAPE), (dict(rows=12), _lib.GDN_ERR_SHAPE),
    (dict(gp=ODD), _lib.GDN_ERR_ALIGN), (dict(gate=ODD), _lib.GDN_ERR_ALIGN), (dict(x=ODD), _lib.GDN_ERR_ALIGN),
])
def test_block_norm_fwd_rejects(lib, over, code):
    assert _lib.call_status("gdn_block_norm_fwd", *fwd(**over)) == code
    assert "gdn_block_norm_fwd" in _lib.last_error()


def bwd(**over):
    a = dict(y=FAKE, h=FAKE, hdt=1, dh=FAKE, dx=FAKE, gp=FAKE, gate=FAKE, rows=2, gq=FAKE, alpha=1.0, dy=FAKE, dho=FAKE,
             dgate=FAKE, dgdt=1, dgp=FAKE, dgq=FAKE, R=6, D=64, eps=1e-6, ws=FAKE, wsb=1 << 30, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(y=None), _lib.GDN_ERR_NULL), (dict(dx=None), _lib.GDN_ERR_NULL), (dict(dgate=None), _lib.GDN_ERR_NULL),
    (dict(dgp=None), _lib.GDN_ERR_NULL), (dict(dgq=None), _lib.GDN_ERR_NULL), (dict(dy=None), _lib.GDN_ERR_NULL),
    (dict(dgdt=0), _lib.GDN_ERR_DTYPE), (dict(dgdt=7), _lib.GDN_ERR_DTYPE), (dict(hdt=-1), _lib.GDN_ERR_DTYPE),
    (dict(rows=5), _lib.GDN_ERR_SHAPE), (dict(ws=None), _lib.GDN_ERR_SHAPE), (dict(wsb=8), _lib.GDN_ERR_SHAPE),
    (dict(dho=ODD), _lib.GDN_ERR_ALIGN), (dict(ws=ODD), _lib.GDN_ERR_ALIGN),
])
def test_block_norm_bwd_rejects(lib, over, code):
    assert _lib.call_status("gdn_block_norm_bwd", *bwd(**over)) == code


def test_block_norm_workspace(lib):
    f = lib.gdn_block_norm_bwd_workspace_bytes
    assert f(0, 64, 1) == f(6, 60, 1) == f(6, 64, 4) == f(6, 8200, 1) == f(6, 64, -1) == 0
    assert f(16384, 2048, 2) >= 4 * 2048 * 4 and f(6, 64, 6) > 0 and f(6, 64, 0) > 0


def spec(**over):
    a = dict(positions=FAKE, ld=8, inv=FAKE, sections=(24, 8), axes=2, rot=64, style=0)
    a.update(over)
    sec = (ctypes.c_int * 4)(*(a["sections"] or ()))
    s = _lib.RopeSpec(a["positions"], a["ld"], a["inv"], ctypes.cast(sec, ctypes.c_void_p) if a["sections"] else None,
                      a["axes"], a["rot"], a["style"])
    s.keep = sec
    return s


@pytest.mark.parametrize("over,code", [
    (dict(positions=None), _lib.GDN_ERR_NULL), (dict(inv=None), _lib.GDN_ERR_NULL), (dict(sections=None), _lib.GDN_ERR_NULL),
    (dict(rot=72), _lib.GDN_ERR_SHAPE), (dict(rot=0), _lib.GDN_ERR_SHAPE), (dict(rot=80), _lib.GDN_ERR_SHAPE),
    (dict(axes=0), _lib.GDN_ERR_SHAPE), (dict(axes=5), _lib.GDN_ERR_SHAPE), (dict(sections=(24, 9)), _lib.GDN_ERR_SHAPE),
    (dict(sections=(40, -8)), _lib.GDN_ERR_SHAPE), (dict(style=2), _lib.GDN_ERR_ARG), (dict(ld=4), _lib.GDN_ERR_SHAPE),
])
def test_rope_spec_rejects(lib, over, code):
    s = spec(**over)
    assert _lib.call_status("gdn_rope_fwd", FAKE, 256, FAKE, 128, FAKE, FAKE, ctypes.byref(s), 0, 8, 4, 2, 64, None) == code


@pytest.mark.parametrize("args,code", [
    ((None, 256, FAKE, 128, FAKE, FAKE), _lib.GDN_ERR_NULL), ((FAKE, 256, None, 128, FAKE, FAKE), _lib.GDN_ERR_NULL),
    ((FAKE, 256, FAKE, 128, FAKE, None), _lib.GDN_ERR_NULL), ((ODD, 256, FAKE, 128, FAKE, FAKE), _lib.GDN_ERR_ALIGN),
    ((FAKE, 260, FAKE, 128, FAKE, FAKE), _lib.GDN_ERR_ALIGN), ((FAKE, 128, FAKE, 128, FAKE, FAKE), _lib.GDN_ERR_SHAPE),
])
def test_rope_rejects(lib, args, code):
    s = spec()
    assert _lib.call_status("gdn_rope_fwd", *args, ctypes.byref(s), 0, 8, 4, 2, 64, None) == code
    assert _lib.call_status("gdn_rope_fwd", FAKE, 256, FAKE, 128, FAKE, FAKE, ctypes.byref(s), 0, 8, 4, 2, 96, None) == \
        _lib.GDN_ERR_UNSUPPORTED
    assert _lib.call_status("gdn_rope_fwd", FAKE, 256, FAKE, 128, FAKE, FAKE, None, 0, 8, 4, 2, 64, None) == _lib.GDN_ERR_NULL


def cache(**over):
    a = dict(k=FAKE, v=FAKE, table=FAKE, ld=8, ps=2048, ts=128, hs=64, pages=10, page=16, width=8, kv=2, D=64)
    a.update(over)
    return _lib.PagedCache(*a.values())


BAD_CACHES = [
    (dict(k=None), _lib.GDN_ERR_NULL), (dict(table=None), _lib.GDN_ERR_NULL), (dict(pages=0), _lib.GDN_ERR_SHAPE),
    (dict(page=24), _lib.GDN_ERR_SHAPE), (dict(page=8), _lib.GDN_ERR_SHAPE), (dict(width=0), _lib.GDN_ERR_SHAPE),
    (dict(ld=7), _lib.GDN_ERR_SHAPE), (dict(kv=0), _lib.GDN_ERR_SHAPE), (dict(ts=100), _lib.GDN_ERR_ALIGN),
    (dict(hs=0), _lib.GDN_ERR_ALIGN), (dict(v=ODD), _lib.GDN_ERR_ALIGN), (dict(width=1 << 28, ld=1 << 28), _lib.GDN_ERR_SHAPE),
    (dict(D=96), _lib.GDN_ERR_UNSUPPORTED),
]


@pytest.mark.parametrize("over,code", BAD_CACHES)
def test_paged_operators_reject_the_cache(lib, over, code):
    c, s = cache(**over), spec()
    assert _lib.call_status("gdn_rope_append", FAKE, 256, FAKE, 128, FAKE, 128, FAKE, ctypes.byref(s), ctypes.byref(c), FAKE,
                            FAKE, 2, 8, 4, None) == code
    assert _lib.call_status("gdn_paged_attn_fwd", *attn(cache=c)) == code


def attn(**over):
    a = dict(q=FAKE, q_ld=256, cache=None, cu=FAKE, kv=FAKE, out=FAKE, lse=None, B=2, T=8, Hq=4, max_q=4, max_kv=100,
             causal=1, window=0, scale=0.0, ws=FAKE, wsb=1 << 40, stream=None)
    a.update(over)
    if a["cache"] is None:
        a["cache"] = cache()
    a["cache"] = ctypes.byref(a["cache"])
    return list(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(q=None), _lib.GDN_ERR_NULL), (dict(out=None), _lib.GDN_ERR_NULL), (dict(kv=None), _lib.GDN_ERR_NULL),
    (dict(B=0), _lib.GDN_ERR_SHAPE), (dict(T=-1), _lib.GDN_ERR_SHAPE), (dict(Hq=3), _lib.GDN_ERR_SHAPE),
    (dict(Hq=130, q_ld=130 * 64), _lib.GDN_ERR_SHAPE), (dict(max_kv=129), _lib.GDN_ERR_SHAPE),
    (dict(max_q=-1), _lib.GDN_ERR_SHAPE), (dict(q_ld=128), _lib.GDN_ERR_SHAPE), (dict(window=-1), _lib.GDN_ERR_ARG),
    (dict(window=4, causal=0), _lib.GDN_ERR_ARG), (dict(q=ODD), _lib.GDN_ERR_ALIGN), (dict(q_ld=260), _lib.GDN_ERR_ALIGN),
])
def test_paged_attn_rejects(lib, over, code):
    assert _lib.call_status("gdn_paged_attn_fwd", *attn(**over)) == code
    assert "gdn_paged_attn_fwd" in _lib.last_error()


@pytest.mark.parametrize("scale", [-1.0, float("nan"), float("inf"), -float("inf")])
def test_paged_attn_rejects_scales(lib, scale):
    assert lib.gdn_paged_attn_fwd(*attn(scale=scale)) == _lib.GDN_ERR_ARG


def test_paged_attn_workspace_does_not_shrink(lib):
    """A workspace for calls up to some sizes serves every smaller one."""
    for D in (64, 128):
        for Hq, n_kv in ((1, 1), (16, 2), (48, 1), (64, 1)):
            sizes = [lib.gdn_paged_attn_workspace_bytes(4, 4096, Hq, n_kv, D, q, 65536, 0) for q in (0, 1, 2, 3, 4, 5, 8, 9, 17, 33, 64, 65, 1000)]
            assert sizes[0] > 0 and sizes == sorted(sizes) and sizes[-1] < 40e6
