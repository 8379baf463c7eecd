"""The paged cache's operators together: serving steps, HIP graphs, streams, and the native call path."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from heatkv_amd import (_lib, append_paged_kv, build_paged_tables, paged_shared_prefix_attention,
                        paged_window_attention)
from oracle import paged as opaged
from paged_support import Batch

pytestmark = pytest.mark.gpu


class Server:
    """A paged cache and what its requests hold, on the host too (rows in 64 bits)."""

    def __init__(self, device, requests, blocks, block, heads, kv_heads, dim, dtype, width, window=0, sinks=0, seed=0):
        self.device, self.block, self.dtype, self.window, self.sinks = device, block, dtype, window, sinks
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        shape = (blocks, kv_heads, block, dim)
        self.k = torch.full(shape, float("nan"), dtype=dtype, device=device)
        self.v = torch.full(shape, float("nan"), dtype=dtype, device=device)
        i32 = lambda a: torch.as_tensor(a, dtype=torch.int32).to(device)  # noqa: E731
        self.tables = i32(np.full((requests, width), -1))
        self.lengths = i32(np.zeros(requests))
        self.ring = i32(np.random.default_rng(seed).permutation(blocks))
        self.range = i32([0, blocks])
        self.gen = torch.Generator(device=device).manual_seed(seed)
        self.rows = [[] for _ in range(requests)]  # (k, v) of each row, host

    def rand(self, *shape):
        return torch.randn(shape, generator=self.gen, device=self.device).to(self.dtype)

    def launch(self, counts, q, k, v, tokens):
        """One step as a program runs it; the state is updated in place."""
        step = build_paged_tables(block_tables=self.tables, lengths=self.lengths, new_counts=counts,
                                  free_blocks=self.ring, free_range=self.range, num_tokens=tokens,
                                  block_size=self.block, window=self.window, sinks=self.sinks, in_place=True)
        append_paged_kv(k=k, v=v, k_cache=self.k, v_cache=self.v, slot_map=step.slot_map)
        out = paged_window_attention(q=q, k_cache=self.k, v_cache=self.v, block_tables=self.tables,
                                     lengths=self.lengths, query_starts=step.query_starts,
                                     softmax_scale=self.dim ** -0.5, window=self.window, sinks=self.sinks)
        return out, step.status

    def state(self):
        return [t.clone() for t in (self.k, self.v, self.tables, self.lengths, self.ring, self.range)]

    def restore(self, state):
        for mine, was in zip((self.k, self.v, self.tables, self.lengths, self.ring, self.range), state):
            mine.copy_(was)

    def check(self, counts, q, k, v, out):
        """The step's output against attention over the host's rows."""
        at = 0
        for r, n in enumerate(counts):
            if n < 0:
                self.rows[r] = []
            for i in range(max(n, 0)):
                self.rows[r].append((k[at + i].double().cpu().numpy(), v[at + i].double().cpu().numpy()))
            if n > 0:
                K, V = (np.stack([row[x] for row in self.rows[r]])[None].transpose(0, 2, 1, 3) for x in (0, 1))
                ref, _, tol, _ = opaged.attention(
                    q[at:at + n].double().cpu().numpy(), K, V, np.zeros((1, 1), int), [len(self.rows[r])], [0, n],
                    self.dim ** -0.5, torch.finfo(self.dtype).eps / 2, self.window, self.sinks)
                got = out[at:at + n].double().cpu().numpy().reshape(ref.shape)
                assert (np.abs(got - ref) <= tol).all(), f"request {r}"
                at += n
        assert (out[at:] == 0).all()


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 0), (40, 9)])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(4, 2, 128, torch.bfloat16), (3, 3, 64, torch.float16)])
def test_serving_steps(device, window, sinks, heads, kv_heads, dim, dtype):
    """Prompts, single tokens, idle, ended and reused requests over many steps."""
    rng = np.random.default_rng(window + heads)
    s = Server(device, 5, 60, 16, heads, kv_heads, dim, dtype, 16, window, sinks)
    for i in range(25):
        counts = [int(rng.choice([0, 1, 1, 1, 3])) for _ in range(5)]
        for r in range(5):
            if len(s.rows[r]) > 150 or (s.rows[r] and rng.random() < 0.05):
                counts[r] = -1
            elif not s.rows[r]:
                counts[r] = int(rng.integers(0, 100))
        total = sum(max(n, 0) for n in counts)
        tokens = total + int(rng.integers(0, 4))
        q, k, v = s.rand(tokens, heads, dim), s.rand(tokens, kv_heads, dim), s.rand(tokens, kv_heads, dim)
        out, status = s.launch(torch.tensor(counts, dtype=torch.int32, device=device), q, k, v, tokens)
        assert status.item() == 0
        s.check(counts, q, k, v, out)


def test_a_refused_step_leaves_the_cache(device):
    s = Server(device, 2, 4, 16, 2, 2, 128, torch.bfloat16, 8)
    q, k, v = s.rand(40, 2, 128), s.rand(40, 2, 128), s.rand(40, 2, 128)
    counts = lambda *c: torch.tensor(c, dtype=torch.int32, device=device)  # noqa: E731
    out, status = s.launch(counts(30, 10), q, k, v, 40)
    assert status.item() == 0
    s.check([30, 10], q, k, v, out)
    before = s.state()
    out, status = s.launch(counts(30, 10), q, k, v, 40)
    assert status.item() == 1 and (out == 0).all()
    for a, b in zip(before, s.state()):
        assert torch.equal(torch.nan_to_num(a.float(), 7.0), torch.nan_to_num(b.float(), 7.0))


@pytest.mark.parametrize("held", [5, 900, 3000])
def test_captured_steps(device, held):
    """A step in a HIP graph, replayed with other work and waits between, is the eager step each time."""
    s = Server(device, 3, 3 * (held // 16 + 4), 16, 8, 2, 128, torch.bfloat16, held // 16 + 4)
    big = 3 * held
    one = lambda n: torch.full((3,), n, dtype=torch.int32, device=device)  # noqa: E731
    s.launch(one(held), s.rand(big, 8, 128), s.rand(big, 2, 128), s.rand(big, 2, 128), big)
    q, k, v, counts = s.rand(4, 8, 128), s.rand(4, 2, 128), s.rand(4, 2, 128), one(1)
    start = s.state()
    want = []
    inputs = [[s.rand(*t.shape) for t in (q, k, v)] for _ in range(5)]
    for new in inputs:
        for t, x in zip((q, k, v), new):
            t.copy_(x)
        want.append(s.launch(counts, q, k, v, 4)[0].clone())
    s.restore(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, status = s.launch(counts, q, k, v, 4)
    s.restore(start)
    for i, new in enumerate(inputs):
        for t, x in zip((q, k, v), new):
            t.copy_(x)
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        other = torch.randn((64, 64), device=device)
        assert torch.isfinite(other @ other).all()
        assert torch.equal(out, want[i]) and status.item() == 0


def _cut(device, seed):
    """A call whose tiles are cut and joined."""
    b = Batch([4000 + 100 * seed, 700], [1, 1], 8, 2, seed=seed)
    return b.kwargs()


def test_graphs_and_streams_do_not_share_state(device):
    """Two captured graphs, and eager calls on two streams, with cut tiles in flight together."""
    calls = [_cut(device, i) for i in range(4)]
    want = [paged_window_attention(**c) for c in calls]
    graphs = []
    for c in calls[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = paged_window_attention(**c)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(5):
        outs = [None] * 4
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                if i < 2:
                    graphs[i][0].replay()
                    outs[i] = graphs[i][1]
                else:
                    for _ in range(3):
                        outs[i] = paged_window_attention(**calls[i])
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_counters_are_left_zero(device):
    for i in range(3):
        paged_window_attention(**_cut(device, i))
    torch.cuda.synchronize()
    assert _lib._paged_counters
    for buf in _lib._paged_counters.values():
        assert not buf.any()


def test_native_path_gives_the_same(device):
    """The extension's calls and the Python bodies launch the same."""
    native = _lib.op_call
    if native is None:
        pytest.skip("heatkv_amd/_op_call.so not built")
    prefix = Batch([30, 7], [2, 1], 8, 2, prefix=900, pad=2)

    def run():
        s = Server(device, 3, 40, 16, 4, 2, 128, torch.bfloat16, 12, window=50, sinks=3)
        counts = torch.tensor([70, 3, 0], dtype=torch.int32, device=device)
        q, k, v = s.rand(75, 4, 128), s.rand(75, 2, 128), s.rand(75, 2, 128)
        out, status = s.launch(counts, q, k, v, 75)
        mine = torch.full_like(out, 3.0)
        cut = _cut(device, 1)
        got = [out, status, *s.state(), *paged_shared_prefix_attention(**prefix.kwargs(), return_lse=True),
               *paged_window_attention(**cut, return_lse=True)]
        step = build_paged_tables(block_tables=s.tables, lengths=s.lengths, new_counts=counts, free_blocks=s.ring,
                                  free_range=s.range, num_tokens=80, block_size=16)
        back = paged_window_attention(q=q, k_cache=s.k, v_cache=s.v, block_tables=s.tables, lengths=step.lengths,
                                      query_starts=step.query_starts, softmax_scale=0.1, causal=False, out=mine)
        assert back is mine
        return got + list(step) + [mine]

    run()  # the first call on a stream makes its counters
    fast = run()
    try:
        _lib.op_call = None
        slow = run()
    finally:
        _lib.op_call = native
    for a, b in zip(fast, slow):
        assert a.dtype == b.dtype and a.shape == b.shape
        assert torch.equal(torch.nan_to_num(a.float(), 7.0), torch.nan_to_num(b.float(), 7.0))


def test_inputs_that_require_a_gradient(device):
    a = Batch([20], [1], 2, 2).kwargs()
    a["q"].requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_window_attention(**a)
    with torch.no_grad():
        out = paged_window_attention(**a)
    assert not out.requires_grad
    with pytest.raises(RuntimeError, match="no gradient"):
        append_paged_kv(k=torch.zeros((1, 2, 128), dtype=torch.bfloat16, device=device, requires_grad=True),
                        v=torch.zeros((1, 2, 128), dtype=torch.bfloat16, device=device), k_cache=a["k_cache"],
                        v_cache=a["v_cache"], slot_map=torch.tensor([-1], device=device))


def test_unaligned_cache_is_refused(device):
    a = Batch([20], [1], 2, 2).kwargs()
    c = torch.zeros(a["k_cache"].numel() + 1, dtype=torch.bfloat16, device=device)[1:].view_as(a["k_cache"])
    with pytest.raises(ValueError, match="16-byte"):
        paged_window_attention(**{**a, "k_cache": c})


@pytest.mark.parametrize("prefix", [0, 1500])
def test_captured_with_many_requests(device, prefix):
    """More requests than a wave plans: a graph follows lengths and starts that change between replays."""
    n = 150
    rng = np.random.default_rng(5)
    counts = np.ones(n, np.int64)
    b = Batch(rng.integers(100, 400, n), counts, 8, 2, prefix=prefix)
    a = b.kwargs()
    a["k_cache"], a["v_cache"] = (torch.nan_to_num(a[x]) for x in ("k_cache", "v_cache"))
    fn = paged_shared_prefix_attention if prefix else paged_window_attention
    fn(**a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn(**a)
    for i in range(4):
        keep = rng.integers(0, 3, n)  # tokens of each request, as many of them as there is room for
        starts = np.minimum(np.concatenate([[0], np.cumsum(keep)]), n).astype(np.int32)
        a["query_starts"].copy_(torch.from_numpy(starts))
        a["lengths"].copy_(torch.from_numpy(rng.integers(2, 100, n).astype(np.int32)))
        want = fn(**a)
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        assert torch.equal(out, want)
