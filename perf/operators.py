"""Timed cases of the attention block's operators: the norms around a block with its gate and
residual scale (forward and backward), rotary positions with several axes (with the append to a
paged cache, and the gradient), and attention of new tokens over the paged cache.

``run`` computes an operator with elementary torch operations in fp32, or with ``own`` true
through the package's entry points.  Lengths are a function of the case, values of the seed.
"""
import math
import random

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the hot loop of serving one user: a single token, a short context
        dict(name="attn_decode_one", op="attn", batch=1, q=1, kv=1000, ragged=False, heads=16, kv_heads=2, dim=128,
             page=16, window=0, layout="bthd", lse=False),
        # a full serving batch, every sequence at another length
        dict(name="attn_decode_batch", op="attn", batch=256, q=1, kv=8192, ragged=True, heads=16, kv_heads=2, dim=128,
             page=16, window=0, layout="bthd", lse=False),
        # one token over a long document: the length is all there is to split
        dict(name="attn_decode_long", op="attn", batch=2, q=1, kv=131072, ragged=True, heads=32, kv_heads=4, dim=128,
             page=64, window=0, layout="bhtd", lse=False),
        # chunked prefill: the last chunk of a long prompt
        dict(name="attn_chunk_long", op="attn", batch=1, q=2048, kv=32768, ragged=False, heads=16, kv_heads=2, dim=128,
             page=64, window=0, layout="bthd", lse=False),
        # whole prompts at once into an empty cache, one key head per four query heads
        dict(name="attn_prompts", op="attn", batch=2, q=8192, kv=8192, ragged=True, heads=16, kv_heads=4, dim=128,
             page=128, window=0, layout="bhtd", lse=True),
        # a mixed step: short odd chunks and single tokens, sliding window, narrow heads
        dict(name="attn_mixed_window", op="attn", batch=24, q=301, kv=5003, ragged=True, heads=12, kv_heads=4, dim=64,
             page=32, window=1000, layout="bthd", lse=False),
        # the append of one decode step
        dict(name="rope_append_step", op="rope_append", batch=8, q=1, kv=777, ragged=True, heads=16, kv_heads=2, dim=128,
             page=16, axes=3, rot=128, style="half", layout="bthd"),
        # the append of two long image-and-text chunks
        dict(name="rope_append_chunk", op="rope_append", batch=2, q=8192, kv=16384, ragged=True, heads=16, kv_heads=2,
             dim=128, page=64, axes=3, rot=128, style="half", layout="bthd"),
        # the gradient of the rotation in a training step, partial rotary width
        dict(name="rope_grad", op="rope", tokens=16384, heads=16, kv_heads=16, dim=128, axes=1, rot=64,
             style="interleaved", inverse=True),
        # between two blocks of one decode step
        dict(name="norm_step", op="norm_fwd", rows=8, width=2048, groups=0, f32=False),
        # between two blocks of a prefill of 2 x 8192 tokens, one gate per channel
        dict(name="norm_prefill", op="norm_fwd", rows=16384, width=2048, groups=1, f32=False),
        # the same in training, one gate row per sequence, residual stream in fp32
        dict(name="norm_grad", op="norm_bwd", rows=16384, width=2048, groups=2, f32=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "rope_append", "rope", "norm_fwd", "norm_bwd"])
    if op == "norm_fwd" or op == "norm_bwd":
        width = 8 * (2 * _log(rng, 4, 255) + 1)     # odd multiples of a 16-byte piece of a row
        rows = min(_log(rng, 1, 16384), 16384 * 2048 // width)
        groups = rng.choice([0, 1, 3, rows])        # no gate, one row of it, one per sequence, one per token
        if groups == 3:
            rows = 3 * max(1, rows // 3)
        return dict(op=op, rows=rows, width=width, groups=groups, f32=rng.random() < 0.5)
    group, kv_heads = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 16]), rng.choice([1, 2, 3, 4, 8])
    heads = group * kv_heads
    dim = rng.choice([64, 128])
    if op == "rope":
        axes, rot = rng.choice([1, 2, 3]), rng.choice([dim, dim // 2])
        tokens = min(_log(rng, 1, 16384), 16384 * 32 * 128 // ((heads + kv_heads) * dim))
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, axes=axes, rot=rot,
                    style=rng.choice(["half", "interleaved"]), inverse=rng.random() < 0.5)
    page, layout = rng.choice([16, 32, 64, 128, 256]), rng.choice(["bthd", "bhtd"])
    if op == "rope_append":
        axes, rot = rng.choice([1, 2, 3]), rng.choice([dim, dim // 2])
        batch, q = _log(rng, 1, 64), _log(rng, 1, 8192)
        q = max(1, min(q, 16384 * 20 * 128 // ((heads + 2 * kv_heads) * dim * batch)))
        return dict(op=op, batch=batch, q=q, kv=q + rng.randrange(0, 2000), ragged=rng.random() < 0.7, heads=heads,
                    kv_heads=kv_heads, dim=dim, page=page, axes=axes, rot=rot,
                    style=rng.choice(["half", "interleaved"]), layout=layout)
    window = rng.choice([0, 0, _log(rng, 16, 4096)])
    if rng.random() < 0.5:                          # single tokens, or a few drafted ones
        batch, q, kv = _log(rng, 1, 256), rng.choice([1, 1, 1, 2, 5]), _log(rng, 1, 65536)
        kv = max(q, min(kv, 2 ** 21 * 128 * 2 // (batch * kv_heads * dim)))
    else:                                           # chunks
        batch, q = _log(rng, 1, 32), _log(rng, 8, 8192)
        kv = q + rng.choice([0, _log(rng, 1, 32768)])
        kv = max(q, min(kv, 2 ** 21 * 128 * 2 // (batch * kv_heads * dim)))
        most = 10 ** 9 // (heads * batch)           # query-key pairs of one head and sequence
        q = max(1, min(q, most // kv, 2 ** 25 // (heads * batch * dim)))
    return dict(op="attn", batch=batch, q=q, kv=kv, ragged=rng.random() < 0.7, heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, window=window, layout=layout, lse=rng.random() < 0.3)


def _lengths(c):
    """(new tokens, cache length with them) of every sequence.  Ragged: the first sequence has the
    full lengths, the others anything from one token up."""
    b, q, kv = c["batch"], c["q"], c["kv"]
    if not c["ragged"]:
        return [q] * b, [kv] * b
    r = random.Random(b * 1000003 + q * 1009 + kv)
    qs = [q] + [r.randint(1, q) for _ in range(b - 1)]
    kvs = [kv] + [r.randint(n, n + kv - q) if kv > q else n for n in qs[1:]]
    return qs, kvs


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=BF16, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def _paging(c, g):
    """cu_seqlens, kv_lens and a block table over shuffled pages (the pool has a few to spare)."""
    qs, kvs = _lengths(c)
    page = c["page"]
    need = [-(-n // page) for n in kvs]
    width, total = max(need), sum(need)
    pool = total + 3
    perm = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    starts = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    at = starts[:, None] + torch.arange(width, device="cuda")
    used = torch.arange(width, device="cuda") < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(used, perm[at.clamp(max=pool - 1)], torch.zeros_like(perm[:1]))
    cu = torch.tensor([0] + [sum(qs[:i + 1]) for i in range(len(qs))], dtype=torch.int32, device="cuda")
    return dict(cu_seqlens=cu, kv_lens=torch.tensor(kvs, dtype=torch.int32, device="cuda"), block_table=table,
                pool=pool, total=sum(qs), max_q=max(qs), max_kv=max(kvs))


def _pool_shape(c, pool):
    return (pool, c["page"], c["kv_heads"], c["dim"]) if c["layout"] == "bthd" else \
        (pool, c["kv_heads"], c["page"], c["dim"])


def _axis_positions(first, n, axes):
    """Positions [axes, n] of tokens first..first+n: a text index, and row and column within
    a grid of 24 columns for the image axes."""
    t = torch.arange(first, first + n, device="cuda", dtype=torch.int32)
    return [t, t // 24, t % 24][:axes]


def _rotary(c):
    pairs, axes = c["rot"] // 2, c["axes"]
    sections = [pairs - (axes - 1) * (3 * pairs // 8 if axes == 3 else pairs // 2)] + \
        [3 * pairs // 8 if axes == 3 else pairs // 2] * (axes - 1)
    inv_freq = (10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)).to(F32)
    return tuple(sections), inv_freq


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(c=c)
    if c["op"] in ("norm_fwd", "norm_bwd"):
        R, D, G = c["rows"], c["width"], c["groups"]
        hd = F32 if c["f32"] else BF16
        s.update(y=_randn(g, R, D), h=_randn(g, R, D, dtype=hd, scale=2.0),
                 gamma_post=_randn(g, D, scale=0.1, shift=1.0), gamma_pre=_randn(g, D, scale=0.1, shift=1.0),
                 gate=None if G == 0 else _randn(g, D, scale=0.3, shift=0.5) if G == 1 else
                 _randn(g, G, D, scale=0.3, shift=0.5), alpha=0.9, eps=1e-6)
        if c["op"] == "norm_bwd":
            s.update(dx=_randn(g, R, D), dh=_randn(g, R, D, dtype=hd))
        return s
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "rope":
        sections, inv_freq = _rotary(c)
        s.update(q=_randn(g, c["tokens"], H, D), k=_randn(g, c["tokens"], Hk, D), sections=sections, inv_freq=inv_freq,
                 positions=torch.stack(_axis_positions(seed % 97, c["tokens"], c["axes"])))
        return s
    s.update(_paging(c, g))
    shape = _pool_shape(c, s["pool"])
    s.update(k_cache=_randn(g, *shape), v_cache=_randn(g, *shape), q=_randn(g, s["total"], H, D))
    if c["op"] == "rope_append":
        sections, inv_freq = _rotary(c)
        qs, kvs = _lengths(c)
        per = [_axis_positions(kv - n, n, c["axes"]) for n, kv in zip(qs, kvs)]
        s.update(k=_randn(g, s["total"], Hk, D), v=_randn(g, s["total"], Hk, D), sections=sections, inv_freq=inv_freq,
                 positions=torch.stack([torch.cat([p[a] for p in per]) for a in range(c["axes"])]))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    import gdn_18646_b200 as G
    c = s["c"]
    if c["op"] == "norm_fwd":
        h, x = G.block_norm(s["y"], s["h"], gamma_post=s["gamma_post"], gate=s["gate"], gamma_pre=s["gamma_pre"],
                            residual_scale=s["alpha"], eps=s["eps"])
        return dict(h=h, x=x)
    if c["op"] == "norm_bwd":
        g = G.block_norm_backward(s["y"], s["h"], s["dh"], s["dx"], gamma_post=s["gamma_post"], gate=s["gate"],
                                  gamma_pre=s["gamma_pre"], residual_scale=s["alpha"], eps=s["eps"])
        return g if s["gate"] is not None else {k: v for k, v in g.items() if k != "dgate"}
    if c["op"] == "rope":
        q, k = G.rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"], style=c["style"],
                      inverse=c["inverse"])
        return dict(q=q, k=k)
    if c["op"] == "rope_append":
        q = G.rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["sections"], s["k_cache"],
                          s["v_cache"], s["block_table"], s["cu_seqlens"], s["kv_lens"], style=c["style"],
                          layout=c["layout"])
        return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])
    o = G.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["cu_seqlens"], s["kv_lens"],
                          max_q=s["max_q"], max_kv=s["max_kv"], window=c["window"], layout=c["layout"],
                          return_lse=c["lse"])
    return dict(out=o[0], lse=o[1]) if c["lse"] else dict(out=o)


def _rows_of_gate(gate, R):
    """The gate as fp32 rows that broadcast over, or match, the R rows."""
    g = gate.float()
    return g if g.dim() == 1 else g.repeat_interleave(R // g.shape[0], 0)


def _plain_norm_fwd(s):
    y, h, eps = s["y"].float(), s["h"].float(), s["eps"]
    u = y * (y.square().mean(-1, keepdim=True) + eps).rsqrt() * s["gamma_post"].float()
    if s["gate"] is not None:
        u = u * _rows_of_gate(s["gate"], y.shape[0])
    hn = s["alpha"] * h + u
    x = hn * (hn.square().mean(-1, keepdim=True) + eps).rsqrt() * s["gamma_pre"].float()
    return dict(h=hn.to(s["h"].dtype), x=x.to(BF16))


def _plain_norm_bwd(s):
    y, h, eps = s["y"].float(), s["h"].float(), s["eps"]
    dx, dh = s["dx"].float(), s["dh"].float()
    gp, gq = s["gamma_post"].float(), s["gamma_pre"].float()
    r2 = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    n2 = h * r2
    g2 = dx * gq
    dt = dh + r2 * (g2 - n2 * (g2 * n2).mean(-1, keepdim=True))
    r1 = (y.square().mean(-1, keepdim=True) + eps).rsqrt()
    n1 = y * r1
    du = dt
    out = {}
    gate = s["gate"]
    if gate is not None:
        du = dt * _rows_of_gate(gate, y.shape[0])
        dg = dt * n1 * gp
        if gate.dim() == 1:
            out["dgate"] = dg.sum(0)
        elif gate.shape[0] == y.shape[0]:
            out["dgate"] = dg.to(BF16)
        else:
            out["dgate"] = dg.view(gate.shape[0], -1, dg.shape[1]).sum(1)
    g1 = du * gp
    dy = r1 * (g1 - n1 * (g1 * n1).mean(-1, keepdim=True))
    out.update(dy=dy.to(BF16), dh=(s["alpha"] * dt).to(s["h"].dtype), dgamma_post=(du * n1).sum(0),
               dgamma_pre=(dx * n2).sum(0))
    return out


def _axis_of_pair(sections):
    return [a for a, n in enumerate(sections) for _ in range(n)]


def _plain_rotate(x, cos, sin, style):
    """Rotates the first 2 * cos.shape[1] values of every head of x [T, H, D]; fp32."""
    x = x.float()
    n = cos.shape[1]
    c, s = cos[:, None, :], sin[:, None, :]
    rot, rest = x[..., :2 * n], x[..., 2 * n:]
    if style == "half":
        a, b = rot[..., :n], rot[..., n:]
        return torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    a, b = rot[..., 0::2], rot[..., 1::2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), rest], -1)


def _plain_angles(s):
    axis = torch.tensor(_axis_of_pair(s["sections"]), device="cuda")
    ang = s["positions"][axis].t().float() * s["inv_freq"]
    return ang.cos(), ang.sin()


def _plain_rope(s):
    cos, sin = _plain_angles(s)
    if s["c"]["inverse"]:
        sin = -sin
    return dict(q=_plain_rotate(s["q"], cos, sin, s["c"]["style"]).to(BF16),
                k=_plain_rotate(s["k"], cos, sin, s["c"]["style"]).to(BF16))


def _plain_append(s):
    c = s["c"]
    cos, sin = _plain_angles(s)
    q, k = (_plain_rotate(s[n], cos, sin, c["style"]).to(BF16) for n in ("q", "k"))
    cu, lens = s["cu_seqlens"].long(), s["kv_lens"].long()
    tok = torch.arange(s["total"], device="cuda")
    b = torch.searchsorted(cu[1:], tok, right=True)
    pos = lens[b] - (cu[b + 1] - cu[b]) + tok - cu[b]
    page, off = s["block_table"][b, pos // c["page"]].long(), pos % c["page"]
    if c["layout"] == "bthd":
        s["k_cache"][page, off] = k
        s["v_cache"][page, off] = s["v"]
    else:
        s["k_cache"][page, :, off] = k
        s["v_cache"][page, :, off] = s["v"]
    return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_attn(s):
    c = s["c"]
    H, Hk, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    G = H // Hk
    cu, lens = s["cu_seqlens"].long(), s["kv_lens"].long()
    B, Lq, Lk, T = lens.numel(), s["max_q"], s["max_kv"], s["total"]
    iq, jk = torch.arange(Lq, device="cuda"), torch.arange(Lk, device="cuda")
    nq = cu[1:] - cu[:-1]
    real = iq < nq[:, None]                                                     # [B, Lq]
    tok = (cu[:-1, None] + iq).clamp(max=T - 1)
    q = s["q"][tok].float().view(B, Lq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Lq, D)
    pg, off = s["block_table"][:, jk // page].long(), (jk % page).expand(B, Lk)
    inside = jk < lens[:, None]                                                 # [B, Lk]

    def rows(cache):
        x = cache[pg, off] if c["layout"] == "bthd" else cache[pg, :, off]      # [B, Lk, Hk, D]
        return torch.where(inside[:, :, None, None], x, torch.zeros((), dtype=x.dtype, device="cuda")) \
            .permute(0, 2, 1, 3).float()

    pos = (lens - nq)[:, None] + iq                                             # [B, Lq]
    see = inside[:, None, :] & (jk <= pos[:, :, None])
    if c["window"]:
        see &= jk > pos[:, :, None] - c["window"]
    sc = (q @ rows(s["k_cache"]).transpose(-1, -2)).mul_(1.0 / math.sqrt(D)).view(B, Hk, G, Lq, Lk)
    sc.masked_fill_(~see[:, None, None], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = sc.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p.view(B, Hk, G * Lq, Lk) @ rows(s["v_cache"])).view(B, Hk, G, Lq, D)
    o = torch.where(l > 0, o / l, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(B, Lq, H, D)[real].to(BF16)
    if not c["lse"]:
        return dict(out=o)
    lse = (m + l.log())[..., 0].permute(0, 3, 1, 2).reshape(B, Lq, H)[real]
    return dict(out=o, lse=lse)


def _run_plain(s):
    return dict(norm_fwd=_plain_norm_fwd, norm_bwd=_plain_norm_bwd, rope=_plain_rope, rope_append=_plain_append,
                attn=_plain_attn)[s["c"]["op"]](s)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] in ("norm_fwd", "norm_bwd"):
        return _exact_norm(s, c)
    if c["op"] == "attn":
        return _exact_attn(s, c)
    # rotation as the product with e^{i angle}
    ax = torch.tensor(_axis_of_pair(s["sections"]), device="cuda")
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[ax] * s["inv_freq"].double()[:, None]).t()[:, None, :]
    if c.get("inverse"):
        turn = turn.conj()

    def rotated(x):
        x, n = x.double(), c["rot"] // 2
        first, second = (slice(0, n), slice(n, 2 * n)) if c["style"] == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
        z = torch.complex(x[..., first], x[..., second]) * turn
        out = x.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out

    if c["op"] == "rope":
        return dict(q=rotated(s["q"]), k=rotated(s["k"]))
    kc, vc, k, v = s["k_cache"].double(), s["v_cache"].double(), rotated(s["k"]), s["v"].double()
    if c["layout"] == "bhtd":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    at = 0
    for b, (n, kv) in enumerate(zip(*_lengths(c))):
        pos = torch.arange(kv - n, kv, device="cuda")
        flat = s["block_table"][b].long()[pos // c["page"]], pos % c["page"]
        kc[flat], vc[flat] = k[at:at + n], v[at:at + n]
        at += n
    if c["layout"] == "bhtd":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    return dict(q=rotated(s["q"]), k_cache=kc.contiguous(), v_cache=vc.contiguous())


def _exact_norm(s, c):
    """By autograd in 64 bits for the gradients: the forward is written down once."""
    R, D = s["y"].shape
    want = c["op"] == "norm_bwd"
    y, gp, gq = (s[n].double().requires_grad_(want) for n in ("y", "gamma_post", "gamma_pre"))
    gate = None if s["gate"] is None else s["gate"].double().requires_grad_(want)
    u = y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + s["eps"]) * gp
    if gate is not None:
        u = (u.view(1 if gate.dim() == 1 else gate.shape[0], -1, D) * gate.view(-1, 1, D)).view(R, D)
    if not want:
        hn = s["alpha"] * s["h"].double() + u
    else:                                   # h is the stored sum: du flows through it as through a leaf
        hn = s["h"].double().requires_grad_(True)
    x = hn / torch.sqrt((hn * hn).sum(-1, keepdim=True) / D + s["eps"]) * gq
    if not want:
        return dict(h=hn, x=x)
    dt, dgq = torch.autograd.grad(x, [hn, gq], s["dx"].double())
    dt = dt + s["dh"].double()
    g = torch.autograd.grad(u, [y, gp] + ([] if gate is None else [gate]), dt)
    out = dict(dy=g[0], dh=s["alpha"] * dt, dgamma_post=g[1], dgamma_pre=dgq)
    if gate is not None:
        out["dgate"] = g[2]
    return out


def _exact_attn(s, c):
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    G = H // Hk
    out, lse = [], []
    at = 0
    for b, (n, kv) in enumerate(zip(*_lengths(c))):
        pages = s["block_table"][b, :-(-kv // c["page"])].long()
        o_b = torch.empty(n, H, D, dtype=torch.float64, device="cuda")
        l_b = torch.empty(n, H, dtype=torch.float64, device="cuda")
        i, j = torch.arange(kv - n, kv, device="cuda")[:, None], torch.arange(kv, device="cuda")
        hide = j > i
        if c["window"]:
            hide |= j <= i - c["window"]
        for h in range(Hk):
            if c["layout"] == "bthd":
                K, V = (t[pages, :, h].reshape(-1, D)[:kv].double() for t in (s["k_cache"], s["v_cache"]))
            else:
                K, V = (t[pages, h].reshape(-1, D)[:kv].double() for t in (s["k_cache"], s["v_cache"]))
            for r in range(h * G, (h + 1) * G):
                S = (s["q"][at:at + n, r].double() @ K.t() / math.sqrt(D)).masked_fill(hide, -math.inf)
                l_b[:, r] = torch.logsumexp(S, -1)
                o_b[:, r] = torch.softmax(S, -1) @ V
        out.append(o_b)
        lse.append(l_b)
        at += n
    out = dict(out=torch.cat(out))
    if c["lse"]:
        out["lse"] = torch.cat(lse)
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] in ("norm_fwd", "norm_bwd"):
        R, D, G, hb = c["rows"], c["width"], c["groups"], 4 if c["f32"] else 2
        gate = (D if G == 1 else G * D) * 2
        if c["op"] == "norm_fwd":
            return dict(bytes=R * D * (2 + hb + hb + 2) + gate + 4 * D, flops=12 * R * D)
        dgate = 0 if G == 0 else G * D * (2 if G == R and G > 1 else 4)
        return dict(bytes=R * D * (2 + hb + hb + 2 + 2 + hb) + gate + dgate + 12 * D, flops=30 * R * D)
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "rope":
        T = c["tokens"]
        return dict(bytes=T * (H + Hk) * D * 4 + T * c["axes"] * 4, flops=3 * T * (H + Hk) * c["rot"])
    qs, kvs = _lengths(c)
    T = sum(qs)
    if c["op"] == "rope_append":
        return dict(bytes=T * (H + 2 * Hk) * D * 4 + T * c["axes"] * 4, flops=3 * T * (H + Hk) * c["rot"])
    W = c["window"]
    pairs = keys = 0
    for n, kv in zip(qs, kvs):
        if W:                               # token at position p sees min(p + 1, W) keys
            full = max(0, kv - max(kv - n, W - 1))
            short = n - full
            pairs += full * W + short * (kv - n + 1) + short * (short - 1) // 2
            keys += min(kv, n + W - 1)
        else:
            pairs += n * (kv - n) + n * (n + 1) // 2
            keys += kv
    return dict(bytes=2 * T * H * D * 2 + 2 * keys * Hk * D * 2, flops=4 * pairs * H * D)
