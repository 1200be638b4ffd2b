"""Hybrid stacks: Gated DeltaNet layers with softmax-attention layers between them, on one
residual stream.

    h, x -> block (GDNLayer or AttentionLayer on x) -> y
         -> block_norm: h' = residual_scale h + gate RMSNorm(y), x' = RMSNorm(h') for the next block

``AttentionLayer``: q|k|v projections in one launch, ``rope_append`` (rotary positions with
several axes, keys and values into the paged cache), ``paged_attention``, output projection;
the same four steps for a chunk of a prompt and for single tokens.  ``PagedKV``: the cache
of one attention layer for a batch of sequences.  ``HybridStack``: layers, their states and
caches, and the norms between them.

    python -m gdn_18646_b200.hybrid            # a small stack: two chunks of a prompt, then decode steps
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ops
from .layer import GDNConfig, GDNLayer, make_weights


@dataclass
class AttentionConfig:
    hidden: int = 2048
    n_q: int = 16
    n_kv: int = 2
    head_dim: int = 128
    sections: tuple = (64,)     # rotated pairs per position axis; 2 * sum <= head_dim values are turned
    theta: float = 10000.0
    style: str = "half"
    window: int = 0

    @property
    def q_dim(self):
        return self.n_q * self.head_dim

    @property
    def kv_dim(self):
        return self.n_kv * self.head_dim

    def inv_freq(self, device="cuda"):
        n = sum(self.sections)
        return (self.theta ** (-torch.arange(n, dtype=torch.float64, device=device) / n)).float()


def make_attention_weights(cfg: AttentionConfig, device="cuda", seed=0, std=0.02):
    """Random weights (bf16 ~N(0, std)) of an attention layer."""
    g = torch.Generator(device=device).manual_seed(seed)

    def w(*shape):
        return (torch.randn(*shape, generator=g, device=device) * std).bfloat16()
    return dict(W_q=w(cfg.q_dim, cfg.hidden), W_k=w(cfg.kv_dim, cfg.hidden), W_v=w(cfg.kv_dim, cfg.hidden),
                W_o=w(cfg.hidden, cfg.q_dim))


class PagedKV:
    """The paged cache of one attention layer for B sequences: a pool of pages, the block
    table and the lengths on the device; pages are handed out as the sequences grow."""

    def __init__(self, cfg: AttentionConfig, B: int, pages: int, page_size: int = 64, max_len: int | None = None,
                 device="cuda"):
        self.page_size, self.pages = page_size, pages
        width = pages if max_len is None else -(-max_len // page_size)
        pool = torch.zeros(pages, 2, page_size, cfg.n_kv, cfg.head_dim, dtype=torch.bfloat16, device=device)
        self.k, self.v = pool[:, 0], pool[:, 1]
        self.table = torch.zeros(B, width, dtype=torch.int32, device=device)
        self.lens = torch.zeros(B, dtype=torch.int32, device=device)
        self.host_lens = [0] * B
        self.free = list(range(pages - 1, -1, -1))

    def room(self, B: int, n: int):
        """Pages that the sequences have, and need with n more tokens each; raises, with nothing
        changed, where this is not the cache of B sequences or the pages do not suffice."""
        if B != len(self.host_lens) or n < 0:
            raise RuntimeError(f"PagedKV: {n} tokens of {B} sequences for a cache of {len(self.host_lens)} sequences")
        need = [-(-(m + n) // self.page_size) for m in self.host_lens]
        have = [-(-m // self.page_size) for m in self.host_lens]
        if sum(need) - sum(have) > len(self.free) or max(need) > self.table.shape[1]:
            raise RuntimeError(f"PagedKV: {n} more tokens need {sum(need) - sum(have)} pages, {len(self.free)} are free, "
                               f"at most {self.table.shape[1]} per sequence")
        return have, need

    def grow(self, n: int):
        """Room for n more tokens of every sequence, counted as theirs from now on."""
        have, need = self.room(len(self.host_lens), n)
        for b, (lo, hi) in enumerate(zip(have, need)):
            if hi > lo:
                mine = [self.free.pop() for _ in range(hi - lo)]
                self.table[b, lo:hi] = torch.tensor(mine, dtype=torch.int32)
        self.host_lens = [m + n for m in self.host_lens]
        self.lens += n


class AttentionLayer:
    """Softmax attention over a paged cache; every step is a libgdn_b200 kernel."""

    def __init__(self, weights: dict, cfg: AttentionConfig | None = None):
        self.w = weights
        self.cfg = cfg or AttentionConfig()
        self.inv_freq = self.cfg.inv_freq(weights["W_q"].device)

    @torch.no_grad()
    def forward(self, x: torch.Tensor, kv: PagedKV, positions: torch.Tensor | None = None):
        """x [B,T,D] bf16 (normed): the next T tokens of every sequence of ``kv``, a chunk of
        the prompts or one decode step.  ``positions`` int32 [axes, B * T] (default: the
        place in the sequence, on every axis).  Returns y [B,T,D] bf16."""
        c, w = self.cfg, self.w
        B, T, D = x.shape
        if T < 1:
            raise RuntimeError("x must hold at least one token of every sequence")
        start = list(kv.host_lens)
        kv.room(B, T)                                  # tokens count as the cache's only once nothing can refuse them
        if positions is None:
            positions = (torch.arange(T, device=x.device, dtype=torch.int32) +
                         torch.tensor(start, dtype=torch.int32, device=x.device)[:, None]).reshape(1, -1) \
                .expand(len(c.sections), -1).contiguous()
        cu = torch.arange(0, B * T + 1, T, dtype=torch.int32, device=x.device)
        seg = [dict(W=w["W_q"]), dict(W=w["W_k"]), dict(W=w["W_v"])]
        if T == 1 and B <= 8:                          # a decode step streams the weights once
            q, k, v = ops.decode_proj(x.reshape(B, D), seg)
        else:
            q, k, v = ops.proj_multi(x.reshape(1, B * T, D), seg)
        ops._rope_spec(positions, self.inv_freq, c.sections, c.style, B * T)
        kv.grow(T)
        q = ops.rope_append(q.view(B * T, c.n_q, c.head_dim), k.view(B * T, c.n_kv, c.head_dim),
                            v.view(B * T, c.n_kv, c.head_dim), positions, self.inv_freq, c.sections, kv.k, kv.v, kv.table, cu,
                            kv.lens, style=c.style)
        o = ops.paged_attention(q, kv.k, kv.v, kv.table, cu, kv.lens, max_q=T, max_kv=max(kv.host_lens), window=c.window)
        if T == 1 and B <= 8:
            (y,) = ops.decode_proj(o.view(B, c.q_dim), [dict(W=w["W_o"])])
        else:
            (y,) = ops.proj_multi(o.view(1, B * T, c.q_dim), [dict(W=w["W_o"])])
        return y.view(B, T, D)


class HybridStack:
    """Layers on one residual stream.  ``layers``: GDNLayer and AttentionLayer objects;
    ``norms``: per layer a dict of gamma_pre (the layer's input norm), gamma_post and gate
    (both may be None) [D] bf16; ``norm_out`` [D] bf16: the norm after the last layer.  The
    residual stream is fp32."""

    def __init__(self, layers, norms, norm_out, residual_scale: float = 1.0, eps: float = 1e-6):
        self.layers, self.norms, self.norm_out = list(layers), list(norms), norm_out
        self.residual_scale, self.eps = residual_scale, eps

    def init_state(self, B: int, pages: int, page_size: int = 64, device="cuda"):
        """Empty per-layer states: None for a GDN layer, a PagedKV for an attention layer."""
        return [PagedKV(m.cfg, B, pages, page_size, device=device) if isinstance(m, AttentionLayer) else None
                for m in self.layers]

    @torch.no_grad()
    def forward(self, x: torch.Tensor, states: list):
        """x [B,T,D] bf16, the next T tokens' embeddings; ``states`` is updated (not if a cache
        has no room for them).  Returns the normed residual stream [B,T,D] bf16 after the last
        layer."""
        for s in states:
            if isinstance(s, PagedKV):
                s.room(x.shape[0], x.shape[1])
        h = x.float()
        xn = ops.rmsnorm(x, self.norms[0]["gamma_pre"], self.eps)
        for i, m in enumerate(self.layers):
            if isinstance(m, AttentionLayer):
                y = m.forward(xn, states[i])
            elif x.shape[1] == 1 and states[i] is not None and x.shape[0] <= 8:
                y, states[i] = m.decode(xn, states[i], states[i], normed=True)
            else:
                y, states[i] = m.prefill(xn, states[i], normed=True)
            gamma_next = self.norms[i + 1]["gamma_pre"] if i + 1 < len(self.layers) else self.norm_out
            n = self.norms[i]
            h, xn = ops.block_norm(y, h, gamma_post=n.get("gamma_post"), gate=n.get("gate"), gamma_pre=gamma_next,
                                   residual_scale=self.residual_scale, eps=self.eps, h_out=h)
        return xn


def make_stack(hidden=512, kinds="GGGA", device="cuda", seed=0, residual_scale=1.0, attention=None, gdn=None) -> HybridStack:
    """A random stack: one layer per letter, G a GDN layer, A an attention layer."""
    gdn = gdn or GDNConfig(hidden=hidden, n_qk=8, n_v=16, dk=64, dv=64)
    attention = attention or AttentionConfig(hidden=hidden, n_q=hidden // 64, n_kv=hidden // 256, head_dim=64, sections=(16, 8, 8))
    g = torch.Generator(device=device).manual_seed(seed + 1000)

    def vec(shift, scale):
        return (torch.randn(hidden, generator=g, device=device) * scale + shift).bfloat16()
    layers = [AttentionLayer(make_attention_weights(attention, device, seed + i), attention) if kind == "A" else
              GDNLayer(make_weights(gdn, device, seed + i), gdn) for i, kind in enumerate(kinds)]
    norms = [dict(gamma_pre=vec(1, 0.1), gamma_post=vec(1, 0.1), gate=vec(0.5, 0.1)) for _ in kinds]
    return HybridStack(layers, norms, vec(1, 0.1), residual_scale)


def main():
    B, chunks, steps, hidden = 2, (300, 212), 16, 512
    stack = make_stack(hidden)
    states = stack.init_state(B, pages=64, page_size=32)
    for n in chunks:
        y = stack.forward(torch.randn(B, n, hidden, device="cuda").bfloat16(), states)
        print(f"chunk of {n} tokens: out {tuple(y.shape)}, rms {y.float().square().mean().sqrt().item():.3f}")
    for _ in range(steps):
        y = stack.forward(y[:, -1:].contiguous(), states)
    torch.cuda.synchronize()
    kv = next(s for s in states if isinstance(s, PagedKV))
    print(f"{steps} decode steps: out {tuple(y.shape)}, rms {y.float().square().mean().sqrt().item():.3f}, "
          f"cache lengths {kv.lens.tolist()}")


if __name__ == "__main__":
    main()
