"""Builds packed batches over a paged cache for the tests: shuffled pages, NaN in every
place that no token sees, block-table entries that must not be used set to garbage."""
import numpy as np

GARBAGE = 0x7FFFFFFF


class Batch:
    """lens: (new tokens, cache length) per sequence.  ``layout`` "bthd" | "bhtd";
    ``pool``: "plain", or "pair" (k and v halves of one [pages, 2, ...] pool, so strided)."""

    def __init__(self, lens, Hq, Hk, D, page, layout="bthd", pool="plain", window=0, causal=True, seed=0, poison=True):
        import torch
        rng = np.random.default_rng(seed)
        g = torch.Generator("cuda").manual_seed(seed)
        self.lens, self.Hq, self.Hk, self.D, self.page, self.layout = lens, Hq, Hk, D, page, layout
        need = [-(-kv // page) for _, kv in lens]
        width, pages = max(max(need), 1) + 1, sum(need) + 2
        shape = (page, Hk, D) if layout == "bthd" else (Hk, page, D)
        if pool == "pair":
            both = torch.randn(pages, 2, *shape, generator=g, device="cuda").bfloat16()
            self.k, self.v = both[:, 0], both[:, 1]
        else:
            self.k, self.v = (torch.randn(pages, *shape, generator=g, device="cuda").bfloat16() for _ in range(2))
        perm = rng.permutation(pages)
        table = np.full((len(lens), width), GARBAGE, np.int32)
        at = 0
        hide = np.ones((pages, page), bool)                       # positions that nobody sees
        for b, (n, kv) in enumerate(lens):
            mine = perm[at:at + need[b]]
            at += need[b]
            table[b, :need[b]] = mine
            first = max(0, kv - n + 1 - window) if window else 0  # what the first token sees
            if n == 0:
                first = kv
            pos = np.arange(first, kv)
            hide[mine[pos // page], pos % page] = False
            if poison and window:
                table[b, :first // page] = -1
        self.table_np, self.pages = table, pages
        if poison:
            mask = torch.from_numpy(hide).cuda()
            for t in (self.k, self.v):
                if layout == "bthd":
                    t[mask] = float("nan")
                else:
                    t.transpose(1, 2)[mask] = float("nan")
        self.table = torch.from_numpy(table).cuda()
        q_lens = [n for n, _ in lens]
        self.cu_np = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        self.cu = torch.from_numpy(self.cu_np).cuda()
        self.kv = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")
        self.T, self.max_q, self.max_kv = int(self.cu_np[-1]), max(q_lens), max(kv for _, kv in lens)
        self.q = torch.randn(self.T, Hq, D, generator=g, device="cuda").bfloat16()

    def rows(self, b, cache):
        """The cached rows of sequence b, [kv, Hk, D] (numpy float64; rows of unused pages NaN)."""
        kv = self.lens[b][1]
        x = cache if self.layout == "bthd" else cache.transpose(1, 2)
        pages = self.table_np[b, :-(-kv // self.page)]
        out = np.full((len(pages), self.page, self.Hk, self.D), np.nan)
        use = np.flatnonzero((pages >= 0) & (pages < self.pages))
        if len(use):
            out[use] = x[pages[use].tolist()].double().cpu().numpy()
        return out.reshape(-1, self.Hk, self.D)[:kv]
