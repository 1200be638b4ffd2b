"""What an attention layer or a stack refuses leaves its caches as they were."""
import pytest
import torch

from gdn_18646_b200 import hybrid as H


def _layer(device):
    c = H.AttentionConfig(hidden=256, n_q=4, n_kv=2, head_dim=64, sections=(16, 16))
    return c, H.AttentionLayer(H.make_attention_weights(c, device=device), c)


def _state(kv):
    return list(kv.host_lens), kv.lens.tolist(), list(kv.free), kv.table.tolist()


@pytest.mark.parametrize("B,T", [(3, 4), (1, 4), (2, 0), (2, 100)])
def test_a_layer_refuses_batches_and_lengths(B, T):
    c, layer = _layer("cpu")
    kv = H.PagedKV(c, 2, pages=4, page_size=16, device="cpu")
    kv.grow(3)
    before = _state(kv)
    with pytest.raises(RuntimeError, match="PagedKV|at least one token"):
        layer.forward(torch.zeros(B, T, 256).bfloat16(), kv)
    assert _state(kv) == before


@pytest.mark.gpu
def test_a_layer_refuses_inputs(cuda_device):
    c, layer = _layer("cuda")
    kv = H.PagedKV(c, 2, pages=4, page_size=16)
    x = torch.randn(2, 5, 256, device="cuda").bfloat16()
    layer.forward(x, kv)
    before = _state(kv)
    pos = torch.zeros(2, 10, dtype=torch.int32, device="cuda")
    for bad in (dict(x=x.float()), dict(x=x[..., :128].contiguous()), dict(x=x, positions=pos.long()),
                dict(x=x, positions=pos.t().contiguous()), dict(x=x, positions=pos[:, :5].contiguous())):
        with pytest.raises(RuntimeError):
            layer.forward(bad["x"], kv, bad.get("positions"))
        assert _state(kv) == before
    layer.forward(x, kv, pos)
    assert kv.lens.tolist() == [10, 10]


@pytest.mark.gpu
def test_a_stack_refuses_before_its_first_layer(cuda_device):
    """The second attention layer's cache is full: the first one's stays as it was, and the same
    tokens give the same result once there is room."""
    stack = H.make_stack(512, "AGA")
    x = torch.randn(2, 40, 512, device="cuda").bfloat16()
    want = stack.forward(x, stack.init_state(2, pages=8, page_size=16))
    states = stack.init_state(2, pages=8, page_size=16)
    full = H.PagedKV(stack.layers[2].cfg, 2, pages=4, page_size=16)
    with pytest.raises(RuntimeError, match="pages"):
        stack.forward(x, [states[0], None, full])
    assert states[0].host_lens == [0, 0] and states[0].lens.tolist() == [0, 0] and len(states[0].free) == 8
    assert torch.equal(stack.forward(x, states), want)
