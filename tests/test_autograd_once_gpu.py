"""The gradients of the autograd ops come from kernels: a second derivative is an error, not
a number without their share.  Also the wrappers with inputs left out."""
import pytest

pytestmark = pytest.mark.gpu


def _refuses(outs, ins):
    """Also where the loss has a second derivative of its own beside the refused one."""
    import torch
    want = torch.autograd.grad(sum((o.float() ** 2).sum() for o in outs), ins, retain_graph=True)
    first = torch.autograd.grad(sum((o.float() ** 2).sum() for o in outs), ins, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, want))
    loss = sum((g.float() ** 2).sum() for g in first) + sum((t.float() ** 3).sum() for t in ins)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(loss, ins, retain_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        loss.backward()


def test_block_norm(cuda_device):
    import torch
    import gdn_18646_b200 as G
    y, h = (torch.randn(6, 64, device="cuda").bfloat16().requires_grad_(True) for _ in range(2))
    w = torch.ones(64, device="cuda").bfloat16()
    _refuses(G.block_norm_autograd(y, h, gamma_post=w, gate=w, gamma_pre=w), [y, h])


def test_rope(cuda_device):
    import torch
    import gdn_18646_b200 as G
    q, k = (torch.randn(5, 2, 64, device="cuda").bfloat16().requires_grad_(True) for _ in range(2))
    pos, f = torch.arange(5, device="cuda", dtype=torch.int32), torch.ones(32, device="cuda")
    _refuses(G.rope_autograd(q, k, pos, f), [q, k])


def test_prefill(cuda_device):
    import torch
    from gdn_18646_b200 import ops
    q, k, v = ((torch.randn(1, 2, 96, 64, device="cuda") * 0.1).bfloat16().requires_grad_(True) for _ in range(3))
    a, b = (torch.randn(1, 2, 96, device="cuda") for _ in range(2))
    o, S = ops.prefill_autograd(q, k, v, torch.zeros(2, device="cuda"), a, b, torch.zeros(2, device="cuda"),
                                torch.zeros(1, 2, 64, 64, device="cuda"))
    _refuses((o, S), [q, k, v])


@pytest.mark.parametrize("post,gate,pre", [(False, None, True), (True, None, False), (False, 1, False), (False, 3, True),
                                           (True, "row", False), (False, None, False), (True, 1, True)])
@pytest.mark.parametrize("f32", [False, True])
def test_block_norm_with_inputs_left_out(cuda_device, post, gate, pre, f32):
    """Every combination of absent gammas and gate through autograd: the gradients of
    block_norm_backward, None where there is no input, the other output's gradient taken as 0."""
    import torch
    import gdn_18646_b200 as G
    R, D = 12, 128
    g = torch.Generator("cuda").manual_seed(3)
    rn = lambda *s, dt=torch.bfloat16: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    y, h = rn(R, D).requires_grad_(True), rn(R, D, dt=torch.float32 if f32 else torch.bfloat16).requires_grad_(True)
    opt = dict(gamma_post=rn(D) if post else None, gamma_pre=rn(D) if pre else None,
               gate=None if gate is None else rn(D) if gate == 1 else rn(R if gate == "row" else gate, D))
    ins = dict(y=y, h=h, **{k: t.requires_grad_(True) for k, t in opt.items() if t is not None})
    dh, dx = rn(R, D, dt=h.dtype), rn(R, D)
    for use_h, use_x in ((True, pre), (True, False), (False, pre)):
        if not (use_h or use_x):
            continue
        ho, x = G.block_norm_autograd(y, h, residual_scale=0.7, **opt)
        assert (x is None) == (not pre)
        outs = ([ho] if use_h else []) + ([x] if use_x else [])
        got = dict(zip(ins, torch.autograd.grad(outs, list(ins.values()), ([dh] if use_h else []) + ([dx] if use_x else []))))
        want = G.block_norm_backward(y.detach(), ho.detach(), dh if use_h else None,
                                     (dx if use_x else torch.zeros_like(dx)) if pre else None, residual_scale=0.7,
                                     **{k: None if t is None else t.detach() for k, t in opt.items()})
        for name, t in got.items():
            assert torch.equal(t, want[{"y": "dy", "h": "dh"}.get(name, "d" + name)].to(t.dtype)), name


def test_rope_of_queries_alone(cuda_device):
    import torch
    import gdn_18646_b200 as G
    q = torch.randn(5, 2, 64, device="cuda").bfloat16().requires_grad_(True)
    pos, f = torch.arange(5, device="cuda", dtype=torch.int32), torch.full((32,), 0.3, device="cuda")
    qo, ko = G.rope_autograd(q, None, pos, f)
    assert ko is None
    d = torch.randn_like(qo)
    (dq,) = torch.autograd.grad(qo, q, d)
    assert torch.equal(dq, G.rope(d, None, pos, f, inverse=True)[0])
