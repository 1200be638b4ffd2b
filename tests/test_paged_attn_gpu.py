"""paged_attention against the 64-bit oracle.

Tolerance, per element: the softmax's weights may be rounded to bf16 before they meet the
values (2^-8 of each, so 2^-8 A with A = softmax @ |v|), the result is rounded to bf16
(2^-8 |out| <= 2^-8 A), and fp32 scores of size s lose under 1e-5 (1 + |s|), taken as
1e-4 A: together (2^-7 + 1e-4) A.  lse: 1e-5 (1 + |lse|)."""
import numpy as np
import pytest

from oracle import attn_block_oracle as A
from tests._paged import Batch

pytestmark = pytest.mark.gpu


def _np(t):
    return t.double().cpu().numpy()


def check(b, out, lse=None, scale=None, causal=True, window=0, rows=None):
    """rows: at most so many rows of each sequence are compared (its first, last and some between)."""
    scale = scale or b.D ** -0.5
    q, got = _np(b.q), _np(out)
    gl = None if lse is None else _np(lse)
    for s, (n, kv) in enumerate(b.lens):
        if n == 0:
            continue
        k, v = b.rows(s, b.k), b.rows(s, b.v)
        pick = np.arange(n) if rows is None or n <= rows else np.unique(np.concatenate(
            [[0, n - 1], np.random.default_rng(n).integers(0, n, rows)]))
        for i in pick:
            at = b.cu_np[s] + i
            pos = kv - n + i
            hi = min(pos + 1, kv) if causal else kv
            o, l, mag = A.attention(q[at:at + 1], k[:max(hi, 0)], v[:max(hi, 0)], scale, causal and hi > 0, window)
            tol = (2.0 ** -7 + 1e-4) * mag
            err = np.abs(got[at] - o[0])
            assert (err <= tol[0]).all(), f"sequence {s} token {i}: worst {np.max(err - tol[0]):.3e} beyond the tolerance"
            if gl is not None:
                none = np.isneginf(l[0])
                assert np.array_equal(np.isneginf(gl[at]), none)
                assert (np.abs(gl[at][~none] - l[0][~none]) <= 1e-5 * (1 + np.abs(l[0][~none]))).all()


def run(b, **kw):
    import gdn_18646_b200 as G
    got = G.paged_attention(b.q, b.k, b.v, b.table, b.cu, b.kv, max_q=b.max_q, max_kv=b.max_kv, layout=b.layout, **kw)
    assert G._lib.lib().gdn_check_device_error() == 0, G._lib.last_error()
    return got


SINGLE = [  # lens, Hq, Hk, D, page
    ([(1, 1)], 1, 1, 64, 16),
    ([(1, 1), (1, 15), (1, 16), (1, 17), (1, 0)], 8, 1, 128, 16),
    ([(1, 127), (1, 128), (1, 129), (1, 255), (1, 1000)], 16, 2, 128, 32),
    ([(1, 5000), (0, 70), (1, 300)], 12, 4, 64, 64),
    ([(1, 20000)], 32, 2, 128, 128),
    ([(1, 3001)], 5, 1, 128, 256),
    ([(1, 700), (1, 3)], 64, 1, 64, 16),
    ([(2, 900), (5, 5), (1, 64), (3, 2), (4, 1500)], 6, 2, 128, 16),
    ([(1, 40 + 7 * i) for i in range(60)], 14, 2, 128, 16),
    ([(8, 2100)], 7, 7, 64, 512),
    ([(1, 64)] * 3, 40, 1, 128, 64),
]

CHUNKS = [
    ([(16, 16)], 1, 1, 64, 16),
    ([(128, 128)], 2, 2, 128, 16),
    ([(129, 129), (127, 300), (1, 77), (0, 12)], 8, 1, 128, 16),
    ([(200, 1000), (64, 64), (33, 257)], 16, 2, 128, 64),
    ([(300, 200), (5, 1)], 4, 4, 64, 32),                 # more tokens than positions: empty rows
    ([(511, 513)], 3, 1, 128, 128),
    ([(70, 70), (70, 700)], 10, 2, 64, 16),               # a group of 5
    ([(97, 2000)], 12, 2, 128, 256),                      # a group of 6
    ([(150, 150)], 64, 1, 64, 16),
    ([(40, 333), (260, 260)], 28, 4, 128, 512),           # a group of 7
    ([(50, 90)], 48, 2, 64, 32),                          # a group of 24
]


@pytest.mark.parametrize("lens,Hq,Hk,D,page", SINGLE + CHUNKS)
@pytest.mark.parametrize("layout,pool", [("bthd", "plain"), ("bhtd", "pair")])
def test_causal(cuda_device, lens, Hq, Hk, D, page, layout, pool):
    b = Batch(lens, Hq, Hk, D, page, layout, pool, seed=len(lens))
    out, lse = run(b, return_lse=True)
    check(b, out, lse, rows=24)


@pytest.mark.parametrize("window", [1, 17, 128, 1000])
@pytest.mark.parametrize("lens,Hq,Hk,D,page", [SINGLE[2], SINGLE[7], SINGLE[4], CHUNKS[2], CHUNKS[3], CHUNKS[4], CHUNKS[7]])
def test_window(cuda_device, lens, Hq, Hk, D, page, window):
    """Pages that lie before every token's window are NaN, their table entries -1."""
    b = Batch(lens, Hq, Hk, D, page, window=window, seed=window)
    out, lse = run(b, window=window, return_lse=True)
    check(b, out, lse, window=window, rows=24)


@pytest.mark.parametrize("lens,Hq,Hk,D,page", [SINGLE[2], SINGLE[7], CHUNKS[3]])
def test_windows_wider_than_the_cache(cuda_device, lens, Hq, Hk, D, page):
    import torch
    b = Batch(lens, Hq, Hk, D, page, seed=13)
    want = run(b)
    longest = max(kv for _, kv in lens)
    for window in (longest, 2 ** 31 - 1, 2 ** 40):
        assert torch.equal(run(b, window=window), want)
    check(b, run(b, window=longest - 1), window=longest - 1, rows=24)


@pytest.mark.parametrize("lens,Hq,Hk,D,page", [SINGLE[1], SINGLE[7], CHUNKS[2], CHUNKS[4], CHUNKS[6]])
def test_all_positions_and_scale(cuda_device, lens, Hq, Hk, D, page):
    b = Batch(lens, Hq, Hk, D, page, seed=2)
    out, lse = run(b, causal=False, scale=0.3, return_lse=True)
    check(b, out, lse, scale=0.3, causal=False, rows=24)


@pytest.mark.parametrize("few", [True, False])
def test_many_sequences(cuda_device, few):
    """More sequences than a CTA has threads, many of them without tokens or positions."""
    rng = np.random.default_rng(17)
    lens = [(int(rng.integers(0, 3 if few else 24)), int(rng.integers(0, 90))) for _ in range(700)] + [(1, 1500), (2, 0), (0, 700)]
    b = Batch(lens, 6, 2, 64, 16, seed=21)
    out, lse = run(b, return_lse=True)
    check(b, out, lse)
    b = Batch([(n, 0) for n, _ in lens[:50]], 6, 2, 64, 16, seed=22)          # nothing anywhere
    out, lse = run(b, return_lse=True)
    assert float(out.abs().max()) == 0 and bool((lse == -np.inf).all())


@pytest.mark.parametrize("seed", range(16))
def test_random_batches(cuda_device, seed):
    rng = np.random.default_rng(100 + seed)
    G, Hk, D = int(rng.choice([1, 2, 3, 5, 8, 13, 32, 64])), int(rng.choice([1, 2, 3])), int(rng.choice([64, 128]))
    most = int(rng.choice([1, 4, 40, 300]))
    lens = []
    for _ in range(int(rng.integers(1, 9))):
        n = int(rng.integers(0, most + 1))
        lens.append((n, max(0, n + int(rng.integers(-2, 1200)) if rng.random() < 0.8 else int(rng.integers(0, 40)))))
    lens.append((most, most + int(rng.integers(0, 3000))))
    window = int(rng.choice([0, 0, 1, 63, 128, 500]))
    b = Batch(lens, G * Hk, Hk, D, int(rng.choice([16, 32, 128, 512])), str(rng.choice(["bthd", "bhtd"])),
              str(rng.choice(["plain", "pair"])), window=window, seed=seed)
    out, lse = run(b, window=window, return_lse=True)
    check(b, out, lse, window=window, rows=10)


def test_large_scores(cuda_device):
    """Scores of several hundred: the running maximum keeps the exponentials finite, and a
    maximum that keeps growing along the cache is followed."""
    import torch
    for lens, Hq, Hk in (([(1, 2000), (2, 600)], 8, 2), ([(140, 900)], 4, 2)):
        b = Batch(lens, Hq, Hk, 128, 16, seed=9, poison=False)
        b.q *= 8
        ramp = torch.linspace(0.1, 6, b.k.shape[0] * 16, device="cuda").view(b.k.shape[0], 16, 1, 1)
        b.k.copy_((b.k.float() * ramp).bfloat16())
        out, lse = run(b, return_lse=True)
        check(b, out, lse, rows=24)


def test_infinite_scores_of_masked_keys(cuda_device):
    """Infinities of either sign in the keys and values of positions that nobody sees."""
    import torch
    b = Batch([(1, 50), (130, 180)], 4, 2, 64, 16, seed=4)
    b.k[torch.isnan(b.k)] = float("inf")
    b.v[torch.isnan(b.v)] = float("-inf")
    out, lse = run(b, return_lse=True)
    check(b, out, lse, rows=24)


@pytest.mark.parametrize("lens", [[(1, 6000), (1, 20)], [(700, 6000)]])
def test_same_bits_again_and_on_another_stream(cuda_device, lens):
    import torch
    b = Batch(lens, 16, 2, 128, 32, seed=6)
    want, lse = run(b, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, lse2 = run(b, return_lse=True)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, lse2)


def test_generous_bounds_and_defaults(cuda_device):
    """max_q and max_kv only size the launch: bounds far above the lengths give the same
    result up to the split of the sums; without them they are taken from the batch."""
    import gdn_18646_b200 as G
    for lens in ([(1, 900), (1, 40)], [(90, 200), (3, 70)]):
        b = Batch(lens, 8, 2, 128, 16, seed=8)
        for kw in (dict(max_q=b.max_q + 100, max_kv=b.table.shape[1] * 16), dict()):
            out, lse = G.paged_attention(b.q, b.k, b.v, b.table, b.cu, b.kv, return_lse=True, **kw)
            assert G._lib.lib().gdn_check_device_error() == 0
            check(b, out, lse, rows=24)


def test_strided_queries_and_given_buffers(cuda_device):
    import torch
    import gdn_18646_b200 as G
    for lens in ([(1, 500), (1, 77)], [(150, 400)]):
        b = Batch(lens, 8, 2, 128, 16, seed=3)
        wide = torch.randn(b.T, 12, 128, device="cuda").bfloat16()
        wide[:, :8] = b.q
        n = G.paged_attention_workspace(2, b.T, 8, 2, 128, b.max_q, b.max_kv)
        ws = torch.full((n + 64,), 0xFF, dtype=torch.uint8, device="cuda")
        out = torch.full_like(b.q, float("nan"))
        kw = dict(max_q=b.max_q, max_kv=b.max_kv)
        got = G.paged_attention(wide[:, :8], b.k, b.v, b.table, b.cu, b.kv, out=out, workspace=ws, **kw)
        assert got is out and torch.equal(out, run(b))
        assert bool((ws[n:] == 0xFF).all())


def test_captured_in_a_graph_with_growing_lengths(cuda_device):
    """Lengths are read on the device: one captured step serves every length up to max_kv."""
    import torch
    import gdn_18646_b200 as G
    b = Batch([(1, 4000), (1, 4000)], 16, 2, 128, 16, seed=1, poison=False)
    run(b)
    out = torch.empty_like(b.q)
    ws = torch.empty(max(1, G.paged_attention_workspace(2, 2, 16, 2, 128, 1, 4000)), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        G.paged_attention(b.q, b.k, b.v, b.table, b.cu, b.kv, max_q=1, max_kv=4000, out=out, workspace=ws)
    for lens in ([(1, 1), (1, 4000)], [(1, 130), (1, 2049)], [(1, 0), (1, 7)]):
        b.kv.copy_(torch.tensor([kv for _, kv in lens], dtype=torch.int32))
        b.lens = lens
        g.replay()
        torch.cuda.synchronize()
        check(b, out)


def test_a_cache_past_32_bit_offsets(cuda_device):
    """Pages whose element offsets exceed 2^31 (a pool of 4.8 GB per side)."""
    import torch
    import gdn_18646_b200 as G
    page, Hk, D = 64, 8, 128
    pages = (1 << 31) // (page * Hk * D) + 4000
    pool = torch.empty(pages, page, Hk, D, dtype=torch.bfloat16, device="cuda")
    for lens in ([(1, 150), (1, 90)], [(80, 150)]):
        b = Batch(lens, 16, Hk, D, page, seed=12, poison=False)
        pool[-b.pages:].copy_(b.k)
        vpool = torch.empty_like(pool)
        vpool[-b.pages:].copy_(b.v)
        table = torch.where(b.table < b.pages, b.table + (pages - b.pages), b.table)
        out = G.paged_attention(b.q, pool, vpool, table, b.cu, b.kv, max_q=b.max_q, max_kv=b.max_kv)
        assert G._lib.lib().gdn_check_device_error() == 0
        assert torch.equal(out, run(b))
        del vpool


def test_reports_pages_and_lengths_outside(cuda_device):
    import torch
    import gdn_18646_b200 as G
    for lens in ([(1, 40), (1, 60)], [(140, 200), (1, 60)]):
        for what in ("page", "kv", "q", "offsets"):
            b = Batch(lens, 4, 2, 128, 16, poison=False)
            kw = dict(max_q=b.max_q, max_kv=b.max_kv)
            if what == "page":
                b.table[0, 1] = b.pages + 7
            elif what == "kv":
                kw["max_kv"] = 48
            elif what == "q":
                b.cu[1] = b.cu[1] - 1
                b.cu[2] = b.cu[2] + 1
            else:
                b.cu[1] = -3
            G.paged_attention(b.q, b.k, b.v, b.table, b.cu, b.kv, **kw)
            assert G._lib.lib().gdn_check_device_error() == G._lib.GDN_ERR_SHAPE, what
            assert G._lib.lib().gdn_check_device_error() == 0


def test_refusals(cuda_device):
    import torch
    import gdn_18646_b200 as G
    b = Batch([(2, 20)], 4, 2, 64, 16)
    ok = dict(q=b.q, k_cache=b.k, v_cache=b.v, block_table=b.table, cu_seqlens=b.cu, kv_lens=b.kv, max_q=2, max_kv=20)
    G.paged_attention(**ok)
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    for d in (dict(q=b.q.float()), dict(q=z(2, 3, 64)), dict(q=z(2, 4, 128)), dict(q=z(2, 130, 64)), dict(window=-1),
              dict(window=8, causal=False), dict(max_kv=10 ** 6), dict(max_q=-1), dict(k_cache=b.k[:, :8], v_cache=b.v[:, :8]),
              dict(k_cache=z(4, 24, 2, 64), v_cache=z(4, 24, 2, 64)), dict(q=z(2, 4, 32), k_cache=z(4, 16, 2, 32), v_cache=z(4, 16, 2, 32)),
              dict(block_table=b.table[0]), dict(cu_seqlens=b.cu.long()), dict(kv_lens=b.kv.cpu()), dict(layout="x"),
              dict(out=b.q[:1]), dict(workspace=torch.zeros(4, device="cuda"))):
        with pytest.raises(RuntimeError):
            G.paged_attention(**dict(ok, **d))


@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (128, 128)])
@pytest.mark.parametrize("n,group", [(1, 9), (2, 8), (3, 8), (1, 31), (8, 4), (11, 3), (3, 16), (5, 10), (64, 1), (1, 63), (9, 7), (2, 32)])
def test_row_counts_of_few_rows(cuda_device, n, group, D, page):
    """Up to 64 rows of an item, most of them not a multiple of eight; short and cut sequences,
    an empty one, one with more tokens than positions, and a window that starts inside a tile."""
    lens = [(n, 3300), (n, 130), (0, 50), (max(1, n - 1), n + 1), (n, max(0, n - 2)), (1, 0)]
    b = Batch(lens, 2 * group, 2, D, page, seed=n + group)
    out, lse = run(b, return_lse=True)
    check(b, out, lse, rows=8)
    b = Batch(lens, 2 * group, 2, D, page, window=201, seed=n + group)
    out, lse = run(b, window=201, return_lse=True)
    check(b, out, lse, window=201, rows=8)
    b = Batch(lens, 2 * group, 2, D, page, seed=n + group)      # without a window: its pages are not poisoned
    out = run(b, causal=False)
    check(b, out, causal=False, rows=2)


@pytest.mark.parametrize("lens,Hq,Hk,D,page", [
    ([(70, 30000)], 2, 1, 128, 64),                       # an item in nearly as many parts as there are CTAs
    ([(5, 60000)], 13, 1, 64, 256),                       # 65 rows
    ([(9, 40000)], 7, 1, 128, 16),                        # 63 rows
    ([(140, 9000), (3, 12000)], 6, 3, 128, 32),
    ([(300, 700 + 60 * i) for i in range(20)], 12, 3, 128, 64),
    ([(130, 500 + 40 * i) for i in range(32)], 8, 4, 64, 16),
])
def test_items_cut_into_parts(cuda_device, lens, Hq, Hk, D, page):
    b = Batch(lens, Hq, Hk, D, page, seed=31)
    out, lse = run(b, return_lse=True)
    check(b, out, lse, rows=6)
