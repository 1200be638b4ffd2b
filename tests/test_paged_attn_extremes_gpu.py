"""paged_attention over keys and values that are not ordinary numbers: a NaN or infinite score
that a row sees makes that row NaN and no other, wherever it lies in a tile and in either
kernel; a score of -inf weighs nothing; a value that a row does not see weighs exactly nothing,
however large.  Tolerances as in test_paged_attn_gpu.py."""
import numpy as np
import pytest

from oracle import attn_block_oracle as A
from tests._paged import Batch

pytestmark = pytest.mark.gpu

KERNELS = [  # new tokens, positions, query heads, kv heads, head dim
    (3, 300, 8, 2, 128),          # few rows
    (20, 290, 4, 2, 64),          # few rows, 64 of them
    (140, 330, 4, 2, 128),        # 128-row tiles
    (150, 300, 2, 2, 64),
]


def _np(t):
    return t.double().cpu().numpy()


def _run(b, window):
    import gdn_18646_b200 as G
    out, lse = G.paged_attention(b.q, b.k, b.v, b.table, b.cu, b.kv, max_q=b.max_q, max_kv=b.max_kv, window=window,
                                 return_lse=True)
    assert G._lib.lib().gdn_check_device_error() == 0
    return _np(out), _np(lse)


def _place(b, j):
    """(page, row) of position j of the only sequence."""
    return int(b.table_np[0, j // b.page]), j % b.page


def _sees(n, kv, window, j):
    p = kv - n + np.arange(n)
    return (p >= j) & ((p - window < j) if window else True)


def _others(b, out, lse, rows, heads, window, k=None):
    """The rows `rows` of query heads `heads` against the oracle, on finite keys."""
    k, v = b.rows(0, b.k) if k is None else k, b.rows(0, b.v)
    n, kv = b.lens[0]
    for i in rows:
        hi, lo = kv - n + i + 1, max(0, kv - n + i + 1 - window) if window else 0
        o, l, mag = A.attention(_np(b.q[i:i + 1]), k[lo:hi], v[lo:hi], b.D ** -0.5)
        for h in heads:
            assert (np.abs(out[i, h] - o[0, h]) <= (2.0 ** -7 + 1e-4) * mag[0, h]).all(), (i, h)
            assert abs(lse[i, h] - l[0, h]) <= 1e-5 * (1 + abs(l[0, h])), (i, h)


@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("n,kv,Hq,Hk,D", KERNELS)
def test_a_score_that_is_no_number(cuda_device, n, kv, Hq, Hk, D, window, what):
    b = Batch([(n, kv)], Hq, Hk, D, 16, seed=n + window, poison=False)
    group = Hq // Hk
    b.q.copy_((b.q.abs() + 0.1) if what == "inf" else b.q)      # then a key of +inf scores +inf
    for j in list(range(kv - 60, kv - 44)) + list(range(kv - 20, kv - 4)) + [kv - 1]:
        at = _place(b, j)
        kept = b.k[at][0].clone()
        b.k[at][0] = float(what)                                 # kv head 0 only
        out, lse = _run(b, window)
        b.k[at][0] = kept
        hit = _sees(n, kv, window, j)
        assert np.isnan(out[hit][:, :group]).all() and np.isnan(lse[hit][:, :group]).all(), j
        assert np.isfinite(out[~hit]).all() and np.isfinite(lse[~hit]).all(), j
        assert np.isfinite(out[:, group:]).all() and np.isfinite(lse[:, group:]).all(), j
        rest = np.flatnonzero(~hit)
        if len(rest):
            _others(b, out, lse, {int(rest[0]), int(rest[-1])}, range(group), window)


@pytest.mark.parametrize("n", [2, 130])
def test_a_row_that_sees_only_nan(cuda_device, n):
    """The first token of a prompt sees one key; a NaN there is NaN, not an empty row."""
    b = Batch([(n, n)], 2, 1, 64, 16, seed=n, poison=False)
    b.k[_place(b, 0)] = float("nan")
    out, lse = _run(b, 0)
    assert np.isnan(out).all() and np.isnan(lse).all()
    out, lse = _run(b, 1)                                        # every token sees itself only
    assert np.isnan(out[0]).all() and np.isnan(lse[0]).all()
    _others(b, out, lse, range(1, n, 7), range(2), 1)


@pytest.mark.parametrize("n,kv,Hq,Hk,D", KERNELS)
def test_scores_of_minus_infinity(cuda_device, n, kv, Hq, Hk, D):
    """Visible keys that score -inf weigh nothing: the oracle without them."""
    b = Batch([(n, kv)], Hq, Hk, D, 16, seed=7, poison=False)
    b.q.copy_(b.q.abs() + 0.1)
    gone = list(range(0, 24)) + list(range(kv - 70, kv - 40))
    for j in gone:
        b.k[_place(b, j)] = float("-inf")
    out, lse = _run(b, 0)
    k, v = b.rows(0, b.k), b.rows(0, b.v)
    for i in (0, n // 2, n - 1):
        see = [j for j in range(kv - n + i + 1) if j not in gone]
        o, l, mag = A.attention(_np(b.q[i:i + 1]), k[see], v[see], D ** -0.5)
        assert (np.abs(out[i] - o[0]) <= (2.0 ** -7 + 1e-4) * mag[0]).all()
        assert (np.abs(lse[i] - l[0]) <= 1e-5 * (1 + np.abs(l[0]))).all()


@pytest.mark.parametrize("n,Hq,D", [(140, 2, 128), (140, 2, 64), (60, 1, 64)])
def test_large_values_that_a_row_does_not_see(cuda_device, n, Hq, D):
    """Values of 1e37 that later tokens of the chunk see: a weight of 2^-125 instead of 0 on
    one of them would be 0.24 in the rows before them."""
    b = Batch([(n, n)], Hq, 1, D, 16, seed=n + D, poison=False)
    at = n - 44
    for j in range(at, at + 22):
        b.v[_place(b, j)] *= 1e37
    out, lse = _run(b, 0)
    _others(b, out, lse, range(0, n, 5), range(Hq), 0)


@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("n,kv,Hq,Hk,D", [(3, 30000, 8, 2, 128), (20, 9000, 4, 2, 64), (140, 12000, 4, 2, 128), (300, 9000, 2, 2, 64)])
def test_a_score_that_is_no_number_in_one_part_of_many(cuda_device, n, kv, Hq, Hk, D, what):
    """Items cut into parts that are joined: one part of the rows is NaN."""
    b = Batch([(n, kv)], Hq, Hk, D, 16, seed=n, poison=False)
    group = Hq // Hk
    b.q.copy_((b.q.abs() + 0.1) if what == "inf" else b.q)
    for j in (0, 700, kv // 2, kv - n - 200, kv - n // 2 - 1, kv - 1):
        at = _place(b, j)
        kept = b.k[at][0].clone()
        b.k[at][0] = float(what)
        out, lse = _run(b, 0)
        b.k[at][0] = kept
        hit = _sees(n, kv, 0, j)
        assert np.isnan(out[hit][:, :group]).all() and np.isnan(lse[hit][:, :group]).all(), j
        assert np.isfinite(out[~hit]).all() and np.isfinite(lse[~hit]).all(), j
        assert np.isfinite(out[:, group:]).all() and np.isfinite(lse[:, group:]).all(), j
    out, lse = _run(b, 0)
    _others(b, out, lse, (0, n - 1), range(Hq), 0)
