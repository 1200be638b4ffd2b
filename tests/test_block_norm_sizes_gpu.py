"""block_norm and its gradient at the ends of their ranges; tolerances and the comparison with
the 64-bit oracle as in test_block_norm_gpu.py."""
import pytest

from tests import test_block_norm_gpu as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,D,gate", [(140000, 8, 70000), (131066, 8, 65533), (131068, 8, 65534)])
def test_many_shared_gate_rows(cuda_device, R, D, gate):
    """More gate rows with a summed gradient than the y extent of a grid."""
    T.test_forward(cuda_device, R, D, gate, False, True, True)
    T.test_backward(cuda_device, R, D, gate, False, True, True)


def test_many_shared_gate_rows_of_wide_rows(cuda_device):
    """The rows of a gate row are summed by themselves: halves of the batch give the same bits."""
    import torch
    import gdn_18646_b200 as G
    s = T._inputs(132000, 264, 66000, False, True, True)
    w = dict(gamma_post=s["gamma_post"], gamma_pre=s["gamma_pre"])
    whole = G.block_norm_backward(s["y"], s["h"], s["dh"], s["dx"], gate=s["gate"], **w)
    for a, b in ((0, 33000), (33000, 66000)):
        r = slice(2 * a, 2 * b)
        part = G.block_norm_backward(s["y"][r], s["h"][r], s["dh"][r], s["dx"][r], gate=s["gate"][a:b], **w)
        assert torch.equal(part["dgate"], whole["dgate"][a:b]) and torch.equal(part["dy"], whole["dy"][r])


@pytest.mark.parametrize("D", [64, 512, 4096, 4104])
@pytest.mark.parametrize("gate", [1, "row"])
@pytest.mark.parametrize("f32", [False, True])
def test_infinities_where_no_norm_looks(cuda_device, D, gate, f32):
    """Without gamma_pre no gradient depends on h', without gamma_post dy does not depend on y:
    infinities and NaN there leave them as they are."""
    import torch
    import gdn_18646_b200 as G
    s = T._inputs(7, D, gate, f32, False, False)
    clean = G.block_norm_backward(s["y"], s["h"], s["dh"], gate=s["gate"])
    bad_h = s["h"].clone()
    bad_h[2, 5], bad_h[3, 0], bad_h[6] = float("inf"), float("nan"), float("-inf")
    got = G.block_norm_backward(s["y"], bad_h, s["dh"], gate=s["gate"])
    assert all(clean[k] is None or torch.equal(got[k], clean[k]) for k in clean)
    bad_y = s["y"].clone()
    bad_y[1, 3], bad_y[4, 7] = float("inf"), float("nan")
    got = G.block_norm_backward(bad_y, bad_h, s["dh"], gate=s["gate"])
    assert torch.equal(got["dy"], clean["dy"]) and torch.equal(got["dh"], clean["dh"])
    s = T._inputs(7, D, gate, f32, True, False)
    clean = G.block_norm_backward(s["y"], s["h"], s["dh"], gate=s["gate"], gamma_post=s["gamma_post"])
    got = G.block_norm_backward(s["y"], bad_h, s["dh"], gate=s["gate"], gamma_post=s["gamma_post"])
    assert all(clean[k] is None or torch.equal(got[k], clean[k]) for k in clean)


@pytest.mark.parametrize("R,D,gate,f32", [
    (200, 8192, "row", True),          # a ring of one stage, several rows a CTA
    (200, 8192, "row", False),
    (301, 8192, 1, True),
    (333, 5120, 3, True),
    (320, 7168, 4, False),
    (150, 4104, "row", True),
])
def test_wide_rows(cuda_device, R, D, gate, f32):
    """Rows above 4096 columns, more of them than CTAs."""
    T.test_forward(cuda_device, R, D, gate, f32, True, True)
    T.test_backward(cuda_device, R, D, gate, f32, True, True)
