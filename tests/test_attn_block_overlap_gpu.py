"""The attention block's kernels that launch early under gdn_set_launch_overlap: what the
kernel just before them writes (the gate, the block's output, the residual stream, the
queries) is read only after that kernel is done.  Every call is compared bit by bit with the
same calls without overlap; the buffers in between hold NaN before each round, so an early
read shows."""
import pytest

from tests._paged import Batch

pytestmark = pytest.mark.gpu


def _overlapped(on, body):
    from gdn_18646_b200 import _lib
    _lib.lib().gdn_set_launch_overlap(1 if on else 0)
    try:
        body()
    finally:
        _lib.lib().gdn_set_launch_overlap(0)


def _same_with_overlap(poison, body, result, inputs):
    """``body`` launches the kernels, ``poison`` overwrites what they write to each other,
    ``inputs(i)`` sets the i-th round's inputs: eager and captured, overlap on against off."""
    import torch
    want = []
    for i in range(4):
        inputs(i)
        poison()
        _overlapped(False, body)
        want.append([t.clone() for t in result()])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            _overlapped(True, body)
    torch.cuda.current_stream().wait_stream(side)
    for go in (lambda: _overlapped(True, body), graph.replay):
        for i in list(range(4)) * 5:
            inputs(i)
            poison()
            go()
            torch.cuda.synchronize()
            assert all(bool(torch.isfinite(t.float()).all()) for t in result())
            assert all(torch.equal(a, b) for a, b in zip(result(), want[i]))


@pytest.mark.parametrize("D", [128, 1024, 4096])
@pytest.mark.parametrize("R,two_dim", [(1, True), (1, False), (24, True), (24, False)])
def test_gate_of_the_kernel_before(cuda_device, R, two_dim, D):
    """One gate row for all rows, computed by a projection right before."""
    import torch
    import gdn_18646_b200 as G
    g = torch.Generator("cuda").manual_seed(D + R)
    rn = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).bfloat16()  # noqa: E731
    xs = [rn(1, 1024) for _ in range(4)]
    x, W, y, h0 = torch.empty_like(xs[0]), rn(D, 1024, scale=0.03), rn(R, D), rn(R, D)
    gp, gq = rn(D), rn(D)
    gate, h, out = torch.empty(1, D, device="cuda").bfloat16(), torch.empty_like(h0), torch.empty_like(y)

    def body():
        G.decode_proj(x, [dict(W=W, out=gate)])
        G.block_norm(y, h0, gamma_post=gp, gate=gate if two_dim else gate[0], gamma_pre=gq, h_out=h, x_out=out)
    _same_with_overlap(lambda: [t.fill_(float("nan")) for t in (gate, h, out)], body, lambda: (gate, h, out),
                       lambda i: x.copy_(xs[i]))


def test_block_output_and_row_gates_of_the_kernel_before(cuda_device):
    """y and a gate row per token from one projection; the norm's result feeds the next one."""
    import torch
    import gdn_18646_b200 as G
    g = torch.Generator("cuda").manual_seed(5)
    rn = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).bfloat16()  # noqa: E731
    B, D = 6, 1024
    xs = [rn(B, D) for _ in range(4)]
    x, Wy, Wg, Wn, h0 = torch.empty_like(xs[0]), rn(D, D, scale=0.03), rn(D, D, scale=0.03), rn(D, D, scale=0.03), rn(B, D)
    gp, gq = rn(D), rn(D)
    y, gate, h, xn, z = (torch.empty(B, D, device="cuda").bfloat16() for _ in range(5))

    def body():
        G.decode_proj(x, [dict(W=Wy, out=y), dict(W=Wg, out=gate)])
        G.block_norm(y, h0, gamma_post=gp, gate=gate, gamma_pre=gq, h_out=h, x_out=xn)
        G.decode_proj(xn, [dict(W=Wn, out=z)])
        G.block_norm(z, h, gamma_post=gp, gate=gate[0], gamma_pre=gq, h_out=h, x_out=xn)
    _same_with_overlap(lambda: [t.fill_(float("nan")) for t in (y, gate, h, xn, z)], body, lambda: (h, xn, z),
                       lambda i: x.copy_(xs[i]))


@pytest.mark.parametrize("lens", [[(1, 700), (1, 90)], [(1, 9000), (1, 33)], [(3, 5000), (2, 40)]])
def test_attention_of_few_rows_after_a_projection(cuda_device, lens):
    """q straight from a projection, and the attention's output straight into one; items that
    stay whole and items that are cut."""
    import torch
    import gdn_18646_b200 as G
    b = Batch(lens, 8, 2, 64, 16, seed=3, poison=False)
    g = torch.Generator("cuda").manual_seed(9)
    rn = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).bfloat16()  # noqa: E731
    xs = [rn(b.T, 512) for _ in range(4)]
    x, Wq, Wo = torch.empty_like(xs[0]), rn(512, 512, scale=0.05), rn(512, 512, scale=0.05)
    q, o, z = (torch.empty(b.T, 512, device="cuda").bfloat16() for _ in range(3))
    ws = torch.empty(G.paged_attention_workspace(2, b.T, 8, 2, 64, b.max_q, b.max_kv), dtype=torch.uint8, device="cuda")

    def body():
        G.decode_proj(x, [dict(W=Wq, out=q)])
        G.paged_attention(q.view(b.T, 8, 64), b.k, b.v, b.table, b.cu, b.kv, max_q=b.max_q, max_kv=b.max_kv,
                          out=o.view(b.T, 8, 64), workspace=ws)
        G.decode_proj(o, [dict(W=Wo, out=z)])
    _same_with_overlap(lambda: [t.fill_(float("nan")) for t in (q, o, z)], body, lambda: (q, o, z), lambda i: x.copy_(xs[i]))
    assert G._lib.lib().gdn_check_device_error() == 0
