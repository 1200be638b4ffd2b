"""paged_attention at the ends of its integers: tables that reach 2^31 positions."""
import pytest

from tests._paged import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 140])
def test_sequences_near_2_to_31_positions(cuda_device, n):
    """A length past 2^31 - 512 is reported and left out; the other sequence is served."""
    import torch
    import gdn_18646_b200 as G
    b = Batch([(n, n + 20), (n, n + 300)], 4, 2, 64, 16, seed=n, poison=False)
    width = 0x7FFFFFFF // 16
    table = torch.zeros(2, width, dtype=torch.int32, device="cuda")
    table[:, :b.table.shape[1]] = torch.where(b.table < b.pages, b.table, 0)
    want = G.paged_attention(b.q, b.k, b.v, b.table, b.cu, b.kv, max_q=n, max_kv=b.max_kv)
    assert G._lib.lib().gdn_check_device_error() == 0
    out = G.paged_attention(b.q, b.k, b.v, table, b.cu, b.kv, max_q=n)          # max_kv: the table's width
    assert G._lib.lib().gdn_check_device_error() == 0
    tol = 2.0 ** -7 * float(want.float().abs().max())                            # split otherwise: roundings of bf16
    assert float((out.float() - want.float()).abs().max()) <= tol
    for kv in (width * 16, 0x7FFFFFFF - 500):
        b.kv[0] = kv
        out = torch.full_like(b.q, float("nan"))
        G.paged_attention(b.q, b.k, b.v, table, b.cu, b.kv, max_q=n, out=out)
        assert G._lib.lib().gdn_check_device_error() == G._lib.GDN_ERR_SHAPE
        assert bool(torch.isnan(out[:n]).all())
        assert float((out[n:].float() - want[n:].float()).abs().max()) <= tol
