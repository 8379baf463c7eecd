"""Inputs of the paged cache's tests: caches whose unseen rows hold NaN."""

from __future__ import annotations

import numpy as np
import torch

from oracle import paged as opaged


class Batch:
    """A paged cache with `lengths[r]` rows (the last `counts[r]` of them this
    step's) per request, and a prefix of `prefix` rows; every cache row that
    belongs to nobody and, with a window, every row that no query sees, holds
    NaN, and table entries that name no block hold nonsense."""

    def __init__(self, lengths, counts, heads, kv_heads, *, dim=128, dtype=torch.bfloat16, block=16, window=0, sinks=0,
                 causal=True, prefix=0, layout="heads", pad=0, seed=0, width=None, scale=None, device="cuda",
                 spare=3):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.window, self.sinks, self.causal, self.prefix = window, sinks, causal, prefix
        self.block, self.dtype = block, dtype
        self.scale = dim ** -0.5 if scale is None else scale
        need = [-(-int(n) // block) for n in lengths]
        front = -(-prefix // block)
        N = sum(need) + front + spare
        order = rng.permutation(N)
        M = max(max(need), 1) + 2 if width is None else width
        tables = np.full((len(lengths), M), 0x7FFFFFF0, np.int64)
        at = front
        live = np.zeros((N, block), bool)
        for r, (n, c) in enumerate(zip(need, counts)):
            tables[r, :n] = order[at:at + n]
            at += n
            seen = np.zeros(n * block, bool)
            total = int(lengths[r])
            if c > 0:
                lo = max(0, total - c - window + 1) if window else 0
                seen[lo:total] = True
                seen[:min(sinks, total) if window else 0] = True
            live[tables[r, :n]] = seen.reshape(n, block)
            if window:  # blocks that no query sees may belong to someone else by now
                gone = ~seen.reshape(n, block).any(1)
                tables[r, :n][gone] = -7
        self.prefix_blocks = order[:front]
        flat = np.zeros(front * block, bool)
        flat[:prefix] = True
        live[order[:front]] = flat.reshape(front, block)
        T = int(sum(counts)) + pad
        self.q = torch.randn((T, heads, dim), generator=gen).to(dtype)
        shape = (N, kv_heads, block, dim)
        nan = torch.full(shape, float("nan"))
        mask = torch.from_numpy(live)[:, None, :, None]
        self.k = torch.where(mask, torch.randn(shape, generator=gen), nan).to(dtype)
        self.v = torch.where(mask, torch.randn(shape, generator=gen), nan).to(dtype)
        self.tables = tables
        self.lengths = np.array(lengths, np.int32)
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.layout, self.device = layout, device

    def _cache(self, t):
        if self.layout == "tokens":
            return t.transpose(1, 2).contiguous().to(self.device).transpose(1, 2)
        if self.layout == "gaps":  # every stride larger than the rows need
            n, h, b, d = t.shape
            big = torch.full((n + 1, h + 2, b + 1, d + 8), float("nan"), dtype=t.dtype, device=self.device)
            big[:n, 1:h + 1, :b, :d] = t.to(self.device)
            return big[:n, 1:h + 1, :b, :d]
        return t.to(self.device)

    def kwargs(self):
        i32 = lambda a: torch.from_numpy(np.asarray(a).astype(np.int32)).to(self.device)  # noqa: E731
        a = dict(q=self.q.to(self.device), k_cache=self._cache(self.k), v_cache=self._cache(self.v),
                 block_tables=i32(self.tables), lengths=i32(self.lengths), query_starts=i32(self.starts),
                 softmax_scale=self.scale, causal=self.causal)
        if self.prefix or not self.window and self.prefix_blocks.size:
            a.update(prefix_blocks=i32(self.prefix_blocks), prefix_length=self.prefix)
        elif self.window or self.sinks:
            a.update(window=self.window, sinks=self.sinks)
        return a

    def expected(self):
        f = lambda t: t.double().numpy()  # noqa: E731
        tables = np.where((self.tables < 0) | (self.tables >= self.k.shape[0]), 0, self.tables)
        half = torch.finfo(self.dtype).eps / 2
        return opaged.attention(f(self.q), f(self.k), f(self.v), tables, self.lengths, self.starts, self.scale, half,
                                self.window, self.sinks, self.causal, self.prefix_blocks, self.prefix)

    def check(self, out, lse=None, rows=None):
        ref, rlse, tol, ltol = self.expected()
        T, H, D = self.q.shape
        got = out.double().cpu().numpy().reshape(T, H, D)
        rows = slice(None) if rows is None else rows
        with np.errstate(invalid="ignore"):
            bad = ~(np.abs(got - ref) <= tol)[rows]
        assert not bad.any(), f"{bad.sum()} of {bad.size}, worst {np.nanmax(np.abs(got - ref)[rows] - tol[rows]):.3g} over"
        if lse is not None:
            l = lse.double().cpu().numpy()
            with np.errstate(invalid="ignore"):
                ok = (np.abs(l - rlse) <= ltol) | (l == rlse)
            assert ok[:, rows].all(), f"lse off by {np.nanmax(np.abs(l - rlse)[:, rows]):.3g}"
