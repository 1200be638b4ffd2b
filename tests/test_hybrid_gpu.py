"""The hybrid stack that runs block_norm, rope_append and paged_attention together: the
attention layer against a plain fp32 restatement, chunked prefill and decode steps against
one whole prefill, and the GDN layer's ``normed`` switch."""
import pytest

pytestmark = pytest.mark.gpu


def _rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def _plain_attention(layer, x, window):
    """The layer on whole prompts in fp32 from its bf16 weights, bf16 where the kernels store."""
    import torch
    c, w = layer.cfg, {k: v.float() for k, v in layer.w.items()}
    B, T, _ = x.shape
    q, k, v = ((x.float() @ w[n].t()).bfloat16().float() for n in ("W_q", "W_k", "W_v"))
    q, k, v = q.view(B, T, c.n_q, c.head_dim), k.view(B, T, c.n_kv, c.head_dim), v.view(B, T, c.n_kv, c.head_dim)
    n = sum(c.sections)
    ang = torch.arange(T, device=x.device, dtype=torch.float64)[:, None] * layer.inv_freq.double()
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]

    def turn(t):
        a, b, rest = t[..., :n], t[..., n:2 * n], t[..., 2 * n:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).bfloat16().float()
    q, k = turn(q), turn(k)
    G = c.n_q // c.n_kv
    k, v = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) * c.head_dim ** -0.5
    i = torch.arange(T, device=x.device)
    hide = i[None, :] > i[:, None]
    if window:
        hide |= i[None, :] <= i[:, None] - window
    o = torch.einsum("bhij,bjhd->bihd", s.masked_fill(hide, float("-inf")).softmax(-1), v).bfloat16().float()
    return o.reshape(B, T, -1) @ w["W_o"].t()


@pytest.mark.parametrize("cfg", [dict(), dict(n_q=8, n_kv=4, head_dim=64, sections=(16, 8, 8), window=37),
                                 dict(n_q=12, n_kv=2, head_dim=64, sections=(16,))])
def test_attention_layer(cuda_device, cfg):
    """bf16 rounding of q, k, v, the weights of the softmax and o: under 1 % of the norm."""
    import torch
    from gdn_18646_b200 import hybrid as H
    c = H.AttentionConfig(hidden=512, **cfg)
    layer = H.AttentionLayer(H.make_attention_weights(c, seed=3), c)
    x = torch.randn(3, 150, 512, device="cuda").bfloat16()
    kv = H.PagedKV(c, 3, pages=40, page_size=16, max_len=160)
    y = layer.forward(x, kv)
    want = _plain_attention(layer, x, c.window)
    assert _rel(y, want) < 1e-2
    # the same tokens in chunks, the last ones one by one
    kv2 = H.PagedKV(c, 3, pages=40, page_size=16, max_len=160)
    parts = [layer.forward(x[:, a:b].contiguous(), kv2) for a, b in ((0, 64), (64, 129), (129, 146))]
    parts += [layer.forward(x[:, t:t + 1].contiguous(), kv2) for t in range(146, 150)]
    assert kv2.lens.tolist() == [150] * 3 and _rel(torch.cat(parts, 1), want) < 1e-2


def test_many_sequences_decode(cuda_device):
    """More sequences than the streaming projection takes (8): the GEMM path, single tokens."""
    import torch
    from gdn_18646_b200 import hybrid as H
    c = H.AttentionConfig(hidden=512, n_q=8, n_kv=2, head_dim=64, sections=(32,))
    layer = H.AttentionLayer(H.make_attention_weights(c, seed=4), c)
    x = torch.randn(20, 9, 512, device="cuda").bfloat16()
    kv = H.PagedKV(c, 20, pages=20, page_size=16)
    parts = [layer.forward(x[:, t:t + 1].contiguous(), kv) for t in range(9)]
    assert _rel(torch.cat(parts, 1), _plain_attention(layer, x, 0)) < 1e-2
    with pytest.raises(RuntimeError):
        layer.forward(torch.randn(20, 9, 512, device="cuda").bfloat16(), kv)     # no page left


def test_stack_chunks_and_decode_match_whole_prefill(cuda_device):
    """Same tokens in two chunks and single steps; the layers' bf16 activations differ by
    roundings that four layers and the norms carry on: a few bf16 units, under 3 %."""
    import torch
    from gdn_18646_b200 import hybrid as H
    stack = H.make_stack(512, "GAGA", residual_scale=0.9)
    x = torch.randn(2, 200, 512, device="cuda").bfloat16()
    whole = stack.forward(x, stack.init_state(2, pages=64, page_size=32))
    assert bool(torch.isfinite(whole.float()).all())
    st = stack.init_state(2, pages=64, page_size=32)
    parts = [stack.forward(x[:, a:b].contiguous(), st) for a, b in ((0, 130), (130, 196))]
    parts += [stack.forward(x[:, t:t + 1].contiguous(), st) for t in range(196, 200)]
    assert _rel(torch.cat(parts, 1), whole) < 3e-2


def test_normed_switch_of_the_gdn_layer(cuda_device):
    import torch
    from gdn_18646_b200 import ops
    from gdn_18646_b200.layer import GDNConfig, GDNLayer, make_weights
    cfg = GDNConfig(hidden=512, n_qk=8, n_v=16, dk=64, dv=64)
    layer = GDNLayer(make_weights(cfg), cfg)
    x = torch.randn(2, 70, 512, device="cuda").bfloat16()
    y, st = layer.prefill(x)
    xn = ops.rmsnorm(x, layer.w["norm_gamma"], cfg.eps)
    yn, stn = layer.prefill(xn, normed=True)
    assert torch.equal(y, yn) and all(torch.equal(st[k], stn[k]) for k in st)
    one = torch.randn(2, 1, 512, device="cuda").bfloat16()
    d, _ = layer.decode(one, {k: v.clone() for k, v in st.items()})
    dn, _ = layer.decode(ops.rmsnorm(one, layer.w["norm_gamma"], cfg.eps), {k: v.clone() for k, v in st.items()}, normed=True)
    assert _rel(dn, d) < 1e-2


def test_example_runs(cuda_device, capsys):
    from gdn_18646_b200 import hybrid
    hybrid.main()
    out = capsys.readouterr().out
    assert "16 decode steps" in out and "cache lengths [528, 528]" in out
