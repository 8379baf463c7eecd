"""The paged cache's tables and append against a Python free list, and whole steps together."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from heatkv_amd import append_paged_kv, build_paged_tables, paged_shared_prefix_attention, paged_window_attention
from oracle import paged as opaged

pytestmark = pytest.mark.gpu


class State:
    """A cache's bookkeeping on the host, and what the operator is given."""

    def __init__(self, requests, width, blocks, block, seed=0, ring=None):
        rng = np.random.default_rng(seed)
        self.tables = np.full((requests, width), -1, np.int32)
        self.lengths = np.zeros(requests, np.int32)
        size = blocks if ring is None else ring
        self.ring = np.full(size, -9, np.int32)
        first = int(rng.integers(size))
        self.ring[(first + np.arange(blocks)) % size] = rng.permutation(blocks)
        self.range = np.array([first, blocks], np.int32)
        self.block = block

    def step(self, counts, num_tokens, window=0, sinks=0, in_place=False, device="cuda", stride=None):
        """One step on both sides, compared; the host's becomes the state."""
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(device)  # noqa: E731
        tables = t(self.tables)
        if stride is not None:
            wide = torch.full((tables.shape[0], stride), -3, dtype=torch.int32, device=device)
            wide[:, :tables.shape[1]] = tables
            tables = wide[:, :tables.shape[1]]
        ring, lengths, rng = t(self.ring), t(self.lengths), t(self.range)
        got = build_paged_tables(block_tables=tables, lengths=lengths, new_counts=t(counts), free_blocks=ring,
                                 free_range=rng, num_tokens=num_tokens, block_size=self.block, window=window,
                                 sinks=sinks, in_place=in_place)
        want = opaged.build_tables(self.tables, self.lengths, counts, self.ring, self.range, num_tokens, self.block,
                                   window, sinks)
        for g, w in zip((tables, ring, got.slot_map, got.query_starts, got.lengths, got.free_range, got.status), want):
            np.testing.assert_array_equal(g.cpu().numpy(), np.asarray(w).reshape(g.shape))
        assert (got.lengths is lengths) == in_place and (got.free_range is rng) == in_place
        if not in_place:
            assert torch.equal(lengths, t(self.lengths)) and torch.equal(rng, t(self.range))
        self.tables, self.ring, _, _, self.lengths, self.range, status = want
        return status


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 0), (20, 5), (1, 0), (64, 64)])
@pytest.mark.parametrize("block", [1, 4, 16])
def test_steps_of_a_batch(device, window, sinks, block):
    """Prompts, single tokens, idle and ended requests, for many steps."""
    rng = np.random.default_rng(window + 7 * block)
    s = State(9, 200 // block + 1, 1500 // block, block, seed=block)
    for i in range(40):
        counts = rng.choice([0, 1, 1, 1, 2, 9], 9)
        counts[rng.integers(9)] = rng.integers(0, 60)
        counts = np.where((s.lengths > 100) | (rng.random(9) < 0.04), -1, counts)
        total = int(np.maximum(counts, 0).sum())
        assert s.step(counts, total + int(rng.integers(3)), window, sinks, in_place=bool(i % 2)) == 0


@pytest.mark.parametrize("requests", [1, 63, 64, 65, 1000, 1024, 1025, 4096])
@pytest.mark.parametrize("most", [1, 40])
def test_request_counts(device, requests, most):
    rng = np.random.default_rng(requests)
    s = State(requests, 12, 12 * requests + 1, 8, seed=1)
    for _ in range(3):
        counts = rng.integers(0, most + 1, requests)
        counts = np.where(s.lengths + counts > 96, -1, counts)
        assert s.step(counts, int(np.maximum(counts, 0).sum()) + 3, stride=15) == 0


def test_one_long_prompt(device):
    s = State(3, 8192, 9000, 16)
    assert s.step([0, 100000, 1], 100001) == 0
    assert s.step([-1, 1, 1], 5000) == 0


def test_ring_larger_than_its_blocks(device):
    s = State(2, 4, 8, 4, ring=37)
    for counts in ([9, 3], [1, -1], [-1, 12], [4, 1], [9, -1]):
        assert s.step(counts, 21) == 0


@pytest.mark.parametrize("counts,tokens,status", [
    ([20, 20, 20], 60, 1), ([40, 0, 0], 60, 2 | 1), ([5, 5, 5], 14, 4), ([33, 0, -1], 20, 2 | 4),
    ([2**31 - 1, 2**31 - 1, 2**31 - 1], 60, 7)])
def test_refused_steps_change_nothing(device, counts, tokens, status):
    s = State(3, 8, 12, 4)
    assert s.step([7, 1, 4], 12) == 0
    assert s.step(counts, tokens, in_place=True) == status
    assert s.step([1, 1, -1], 12) == 0


@pytest.mark.parametrize("requests", [2, 600])
def test_prompt_longer_than_its_window_on_a_full_ring(device, requests):
    """Blocks popped and pushed in one step, on a ring without room for both."""
    s = State(requests, 64, 20 + requests, 4)
    counts = np.zeros(requests, int)
    counts[0] = 70
    assert s.step(counts, 70, window=8, sinks=3) == 0
    counts[:] = 1
    assert s.step(counts, requests, window=8, sinks=3, in_place=True) == 0
    counts[0], counts[1] = -1, 75
    assert s.step(counts, 2 * requests + 75, window=8, sinks=3) == 0


def test_blocks_that_the_ring_has_no_room_for(device):
    s = State(2, 8, 4, 4)
    s.tables[0, :6], s.lengths[0] = np.arange(6), 22
    assert s.step([-1, 3], 5) == 8
    assert s.step([-1, 3], 5, in_place=True) == 8


def test_no_requests_no_tokens(device):
    s = State(2, 4, 8, 4)
    assert s.step([0, 0], 0) == 0
    assert s.step([0, 0], 5) == 0
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    got = build_paged_tables(block_tables=torch.zeros((0, 4), dtype=torch.int32, device=device), lengths=i32(),
                             new_counts=i32(), free_blocks=i32(), free_range=i32(0, 0), num_tokens=3, block_size=16)
    assert got.slot_map.tolist() == [-1] * 3 and got.query_starts.tolist() == [0] and got.status.item() == 0


@pytest.mark.parametrize("kv_heads,dim,dtype,layout,tokens", [
    (1, 128, torch.bfloat16, "heads", 1), (4, 128, torch.float16, "tokens", 77), (3, 64, torch.bfloat16, "heads", 1000),
    (5, 64, torch.float16, "odd", 33), (2, 128, torch.bfloat16, "view", 19)])
def test_append(device, kv_heads, dim, dtype, layout, tokens):
    gen = torch.Generator(device=device).manual_seed(3)
    block, n = 8, tokens // 8 + 9
    shape = (n, kv_heads, block, dim)

    def cache():
        if layout == "tokens":
            return torch.randn((n, block, kv_heads, dim), generator=gen, device=device).to(dtype).transpose(1, 2)
        if layout == "odd":  # rows that do not start on 16-byte boundaries
            return torch.randn((n, kv_heads, block, dim + 3), generator=gen, device=device).to(dtype)[..., 1:dim + 1]
        return torch.randn(shape, generator=gen, device=device).to(dtype)

    kc, vc = cache(), cache()
    if layout == "view":
        qkv = torch.randn((tokens, 5 * kv_heads, dim), generator=gen, device=device).to(dtype)
        k, v = qkv[:, kv_heads:2 * kv_heads], qkv[:, -kv_heads:]
    else:
        k, v = (torch.randn((tokens, kv_heads, dim), generator=gen, device=device).to(dtype) for _ in range(2))
    slots = torch.randperm(n * block, generator=gen, device=device)[:tokens]
    slots[::5] = -1
    if tokens > 2:
        slots[2] = n * block  # outside the cache: skipped
    want_k, want_v = kc.clone(), vc.clone()
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < n * block:
            want_k[slot // block, :, slot % block] = k[t]
            want_v[slot // block, :, slot % block] = v[t]
    got = append_paged_kv(k=k, v=v, k_cache=kc, v_cache=vc, slot_map=slots)
    assert got[0] is kc and got[1] is vc
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_append_past_32_bits(device):
    n, block, dim = 2**32 // (16 * 128) + 4, 16, 128
    kc = torch.empty((n, 1, block, dim), dtype=torch.bfloat16, device=device)
    vc = torch.empty_like(kc)
    k = torch.randn((3, 1, dim), device=device).to(torch.bfloat16)
    slots = torch.tensor([n * block - 1, (n - 2) * block, 5], device=device)
    append_paged_kv(k=k, v=-k, k_cache=kc, v_cache=vc, slot_map=slots)
    assert torch.equal(kc[n - 1, 0, block - 1], k[0, 0]) and torch.equal(vc[n - 2, 0, 0], -k[1, 0])
    assert torch.equal(kc[0, 0, 5], k[2, 0])
