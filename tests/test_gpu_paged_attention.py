"""The paged attentions against softmax attention in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from heatkv_amd import paged_shared_prefix_attention, paged_window_attention
from paged_support import Batch

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16

# (name, lengths, counts, heads, kv_heads, options)
WINDOW = [
    ("one_row", [1], [1], 1, 1, {}),
    ("single_tokens", [1, 17, 64, 65, 300, 1025], [1] * 6, 8, 2, {}),
    ("single_tokens_mha", [5, 700], [1, 1], 16, 16, dict(dtype=FP)),
    ("single_tokens_d64", [129, 63, 2], [1, 1, 1], 6, 2, dict(dim=64)),
    ("group_of_16", [333, 90], [1, 1], 32, 2, {}),
    ("group_of_17", [333, 90], [1, 1], 17, 1, {}),
    ("group_of_5_d64", [200, 131], [3, 2], 10, 2, dict(dim=64, dtype=FP)),
    ("few_tokens", [40, 5, 260], [4, 5, 3], 4, 2, {}),
    ("idle_and_empty", [0, 70, 33, 0], [0, 1, 0, 0], 4, 4, {}),
    ("prompt", [200], [200], 4, 2, {}),
    ("prompt_behind_rows", [511, 130], [200, 129], 4, 1, {}),
    ("prompt_d64", [321], [321], 2, 2, dict(dim=64)),
    ("mixed", [500, 77, 1, 260, 900], [1, 77, 1, 130, 1], 8, 4, dict(pad=5)),
    ("scale_not_causal", [300, 164], [100, 64], 4, 4, dict(causal=False)),
    ("tokens_not_causal", [300, 164], [2, 1], 4, 4, dict(causal=False)),
    ("window", [1000, 300, 90], [1, 1, 1], 8, 2, dict(window=100)),
    ("window_sinks", [1000, 300, 90], [1, 1, 1], 8, 2, dict(window=100, sinks=21)),
    ("window_of_one", [200, 65], [1, 3], 4, 4, dict(window=1)),
    ("window_of_one_sink", [200, 65], [1, 3], 4, 4, dict(window=1, sinks=1)),
    ("window_prompt", [700], [700], 4, 2, dict(window=97, sinks=5)),
    ("window_prompt_wide_sinks", [600, 333], [310, 333], 2, 1, dict(window=64, sinks=200)),
    ("window_not_causal", [400], [150], 2, 2, dict(window=50, sinks=3, causal=False)),
    ("window_64_aligned", [640], [256], 2, 2, dict(window=64, sinks=64, dtype=FP)),
    ("sinks_beyond", [50, 500], [50, 1], 2, 2, dict(window=10, sinks=1000)),
    ("block_1", [70, 9], [1, 9], 2, 1, dict(block=1)),
    ("block_8", [300, 64], [1, 40], 4, 2, dict(block=8, window=77, sinks=9)),
    ("block_64", [300, 64, 65], [1, 1, 2], 4, 2, dict(block=64)),
    ("block_256", [300, 600], [1, 200], 4, 2, dict(block=256)),
    ("tokens_layout", [300, 77], [1, 50], 4, 2, dict(layout="tokens")),
    ("gaps_layout", [300, 77], [1, 50], 4, 2, dict(layout="gaps", dim=64)),
    ("negative_scale", [300, 40], [1, 40], 2, 2, dict(scale=-0.3)),
    ("zero_scale", [300, 40], [1, 40], 2, 2, dict(scale=0.0)),
    ("steep_scale", [900, 200], [1, 200], 4, 4, dict(scale=4.0)),
    ("long", [9000, 4100], [1, 1], 8, 1, {}),
    ("long_prompt_part", [5000], [130], 4, 1, {}),
    ("many_requests", [3 + 7 * i % 150 for i in range(300)], [1] * 300, 2, 1, {}),
    ("many_ragged", [1 + 37 * i % 190 for i in range(90)], [min(1 + 37 * i % 190, 1 + i % 9) for i in range(90)], 3, 1,
     dict(pad=11)),
]

PREFIX = [
    ("one_prefix_row", [1], [1], 1, 1, dict(prefix=1)),
    ("single_tokens", [5, 40, 1, 90], [1] * 4, 8, 2, dict(prefix=300)),
    ("single_tokens_d64", [5, 40], [1, 1], 4, 4, dict(prefix=521, dim=64, dtype=FP)),
    ("no_own_rows_seen", [3, 0, 60], [1, 0, 2], 4, 2, dict(prefix=77)),
    ("many_requests", [1 + i % 30 for i in range(70)], [1] * 70, 8, 2, dict(prefix=700)),
    ("few_tokens", [9, 60, 30], [3, 4, 1], 4, 2, dict(prefix=200, pad=3)),
    ("scales", [100, 100], [64, 64], 4, 4, dict(prefix=421, causal=False)),
    ("prompts", [200, 33], [150, 33], 4, 2, dict(prefix=130, block=32)),
    ("long_prefix", [33, 7], [1, 1], 16, 2, dict(prefix=9001)),
    ("tokens_layout", [33, 70], [1, 5], 4, 2, dict(prefix=190, layout="tokens")),
]


def _ids(cases):
    return [c[0] for c in cases]


@pytest.mark.parametrize("name,lengths,counts,heads,kv_heads,options", WINDOW, ids=_ids(WINDOW))
def test_window_attention(device, name, lengths, counts, heads, kv_heads, options):
    b = Batch(lengths, counts, heads, kv_heads, **options)
    out, lse = paged_window_attention(**b.kwargs(), return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("name,lengths,counts,heads,kv_heads,options", PREFIX, ids=_ids(PREFIX))
def test_shared_prefix_attention(device, name, lengths, counts, heads, kv_heads, options):
    b = Batch(lengths, counts, heads, kv_heads, **options)
    out, lse = paged_shared_prefix_attention(**b.kwargs(), return_lse=True)
    b.check(out, lse)


def test_empty_prefix_is_the_window_attention(device):
    b = Batch([70, 9], [1, 2], 4, 2)
    a = b.kwargs()
    out = paged_shared_prefix_attention(**a, prefix_blocks=torch.zeros(0, dtype=torch.int32, device=device),
                                        prefix_length=0)
    assert torch.equal(out, paged_window_attention(**a))


@pytest.mark.parametrize("counts", [[1, 1], [40, 33]])
def test_rows_behind_the_last_request(device, counts):
    """Zeros (-inf) in a new output; untouched in the caller's."""
    b = Batch([100, 64], counts, 4, 2, pad=70)
    n = sum(counts)
    out, lse = paged_window_attention(**b.kwargs(), return_lse=True)
    assert (out[n:] == 0).all() and (lse[:, n:] == -float("inf")).all()
    mine = torch.full_like(out, 7.0)
    assert paged_window_attention(**b.kwargs(), out=mine) is mine
    assert (mine[n:] == 7).all() and torch.equal(mine[:n], out[:n])


def test_no_tokens_and_no_requests(device):
    b = Batch([64, 3], [0, 0], 4, 2)
    assert tuple(paged_window_attention(**b.kwargs()).shape) == (0, 512)
    a = Batch([64], [1], 4, 2, pad=2).kwargs()
    a.update(block_tables=a["block_tables"][:0], lengths=a["lengths"][:0], query_starts=a["query_starts"][:1])
    out = paged_window_attention(**a)
    assert (out == 0).all()


@pytest.mark.parametrize("counts,group", [([1, 1], 4), ([40, 90], 2), ([5, 3], 1)])
def test_queries_before_the_first_row(device, counts, group):
    """More queries than rows (a step that was refused): the first ones see nothing."""
    b = Batch([40, 90], counts, 2 * group, 2)
    b.lengths = np.array([0, counts[1] - 1], np.int32)
    out, lse = paged_window_attention(**b.kwargs(), return_lse=True)
    b.check(out, lse)
    assert (out[:counts[0] + 1] == 0).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("counts", [[1, 1], [7, 2], [150, 70]])
def test_unseen_values_have_no_effect(device, value, counts):
    """A query's result does not depend on rows behind it, whatever they hold,
    and those that see a NaN or infinity show it."""
    b = Batch([200, 70], counts, 4, 2)
    out = paged_window_attention(**b.kwargs())
    n0, last = counts[0], 200 - 1
    row, off = b.tables[0, last // b.block], last % b.block
    b.v[row, :, off, 3] = value
    b.v[row, 0, off, 77] = value
    got = paged_window_attention(**b.kwargs())
    assert torch.equal(got[:n0 - 1], out[:n0 - 1]) and torch.equal(got[n0:], out[n0:])
    want = b.expected()[0][n0 - 1].reshape(-1)
    np.testing.assert_array_equal(np.isfinite(want), np.isfinite(got[n0 - 1].double().cpu().numpy()))
    b.k[row, 1, off, 5] = float("nan")
    got = paged_window_attention(**b.kwargs())
    assert torch.equal(got[:n0 - 1], out[:n0 - 1]) and torch.equal(got[n0:], out[n0:])
    assert torch.isnan(got[n0 - 1, 256:]).all()


@pytest.mark.parametrize("counts", [[1, 1], [100, 3]])
def test_strided_and_unaligned_queries(device, counts):
    b = Batch([150, 64], counts, 4, 2)
    a = b.kwargs()
    out = paged_window_attention(**a)
    q = a["q"]
    qkv = torch.zeros((q.shape[0], 12, 128), dtype=q.dtype, device=device)
    qkv[:, 4:8] = q
    a["q"] = qkv[:, 4:8]
    assert torch.equal(paged_window_attention(**a), out)
    flat = torch.zeros(q.numel() + 1, dtype=q.dtype, device=device)
    flat[1:] = q.flatten()
    a["q"] = flat[1:].view_as(q)
    assert torch.equal(paged_window_attention(**a), out)


def test_repeated_calls_are_identical(device):
    for b in (Batch([4000, 900, 77], [1, 1, 1], 8, 2), Batch([900], [400], 4, 1),
              Batch([30, 60], [1, 1], 8, 2, prefix=3000)):
        fn = paged_shared_prefix_attention if b.prefix else paged_window_attention
        first = fn(**b.kwargs(), return_lse=True)
        for _ in range(3):
            again = fn(**b.kwargs(), return_lse=True)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_blocks_outside_the_cache_are_not_read(device):
    """Ids past the cache's end stand for block 0 (no access outside the cache)."""
    for counts in ([1, 1], [40, 20]):
        b = Batch([100, 64], counts, 4, 2)
        a = b.kwargs()
        bad = a["block_tables"].clone()
        zero = bad.clone()
        bad[0, 1], bad[1, 0], zero[0, 1], zero[1, 0] = 0x7FFFFFFF, -1, 0, 0
        a["k_cache"] = torch.nan_to_num(a["k_cache"])
        a["v_cache"] = torch.nan_to_num(a["v_cache"])
        got = paged_window_attention(**{**a, "block_tables": bad})
        assert torch.equal(got, paged_window_attention(**{**a, "block_tables": zero}))


@pytest.mark.parametrize("counts", [[1, 1], [70, 130]])
def test_offsets_past_32_bits(device, counts):
    """Blocks whose element offsets need more than 32 bits."""
    b = Batch([300, 200], counts, 4, 2, block=32)
    a = b.kwargs()
    want = paged_window_attention(**a)
    n, hk, block, d = b.k.shape
    big = 2**32 // (hk * block * d) + n + 1
    for name in ("k_cache", "v_cache"):
        cache = torch.empty((big, hk, block, d), dtype=b.dtype, device=device)
        cache[big - n:] = a[name]
        a[name] = cache
    a["block_tables"] = torch.where((a["block_tables"] >= 0) & (a["block_tables"] < n),
                                    a["block_tables"] + (big - n), a["block_tables"])
    assert torch.equal(paged_window_attention(**a), want)


@pytest.mark.parametrize("counts", [[1, 1, 2], [60, 3, 40]])
def test_the_widest_windows(device, counts):
    """A window (and sinks) up to 2^31 - 1 is no window."""
    b = Batch([300, 40, 90], counts, 4, 2)
    want = paged_window_attention(**b.kwargs())
    for window, sinks in ((2**31 - 1, 0), (2**31 - 1, 2**31 - 1), (1, 2**31 - 1), (300, 0)):
        assert torch.equal(paged_window_attention(**b.kwargs(), window=window, sinks=sinks), want)


@pytest.mark.parametrize("counts", [[1, 1, 1], [50, 1, 130]])
@pytest.mark.parametrize("prefix", [0, 2500])
def test_a_part_of_a_batch(device, counts, prefix):
    """Requests 1 and 2 of three: the tokens of request 0 are not theirs."""
    b = Batch([5000, 700, 300], counts, 8, 2, prefix=prefix)
    fn = paged_shared_prefix_attention if prefix else paged_window_attention
    a = b.kwargs()
    whole, lse = fn(**a, return_lse=True)
    a.update(block_tables=a["block_tables"][1:], lengths=a["lengths"][1:], query_starts=a["query_starts"][1:])
    n = counts[0]
    out, l = fn(**a, return_lse=True)
    b.check(out, l, slice(n, None))
    assert (out[:n] == 0).all() and (l[:, :n] == -float("inf")).all()
    mine = torch.full_like(out, 5.0)
    fn(**a, out=mine)
    assert (mine[:n] == 5).all() and torch.equal(mine[n:], out[n:])


@pytest.mark.parametrize("prefix", [0, 2500])
def test_query_starts_out_of_order(device, prefix):
    """Starts that are not ascending (a caller's mistake) stay within every buffer:
    what comes out is of no meaning, and the calls after it are as before."""
    b = Batch([5000, 700, 300], [40, 2, 90], 8, 2, prefix=prefix)
    fn = paged_shared_prefix_attention if prefix else paged_window_attention
    a = b.kwargs()
    want = fn(**a)
    for starts in ([0, 132, 0, 132], [132, 0, 132, 0], [-5, 9000, 7, -1]):
        fn(**{**a, "query_starts": torch.tensor(starts, dtype=torch.int32, device=device)})
    assert torch.equal(fn(**a), want)


@pytest.mark.parametrize("requests,prefix", [(65, 0), (65, 700), (200, 0), (1024, 0), (1025, 0), (1500, 90), (4096, 0)])
def test_many_requests(device, requests, prefix):
    """More requests than a wave plans: none, one and several tokens each, lengths from 0, one long request."""
    rng = np.random.default_rng(requests)
    counts = rng.choice([0, 1, 1, 1, 2, 9], requests)
    lengths = counts + rng.integers(0, 60, requests)
    lengths[counts == 0] -= rng.integers(0, 2, int((counts == 0).sum())) * lengths[counts == 0]
    lengths[requests // 2] += 1500
    counts[0] = 0
    b = Batch(lengths, counts, 4, 2, dim=64, prefix=prefix, pad=3)
    fn = paged_shared_prefix_attention if prefix else paged_window_attention
    out, l = fn(**b.kwargs(), return_lse=True)
    b.check(out, l)


def test_many_prompts(device):
    """Several 128-row tiles each, cut and whole, for more requests than a wave plans."""
    rng = np.random.default_rng(3)
    counts = rng.integers(30, 130, 70)
    lengths = counts + rng.integers(0, 40, 70)
    lengths[[0, 69]] += 900
    b = Batch(lengths, counts, 8, 2, dim=64, window=200, sinks=5)
    out, l = paged_window_attention(**b.kwargs(), return_lse=True)
    b.check(out, l)


@pytest.mark.parametrize("prefix", [0, 2500])
def test_many_query_starts_out_of_order(device, prefix):
    counts = [2] * 100
    b = Batch([300] * 100, counts, 8, 2, prefix=prefix)
    fn = paged_shared_prefix_attention if prefix else paged_window_attention
    a = b.kwargs()
    want = fn(**a)
    up_down = torch.tensor([0, 200], dtype=torch.int32, device=device).repeat(51)[:101].contiguous()
    for starts in (up_down, 200 - up_down, torch.full_like(up_down, -7), up_down * 10**6):
        fn(**{**a, "query_starts": starts})
    assert torch.equal(fn(**a), want)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("requests", [95, 131])
def test_prefix_with_many_tiles(device, requests, dim):
    """More of the requests' own tiles than CUs beside a prefix in 128-row tiles; an odd number of them."""
    rng = np.random.default_rng(requests)
    counts = rng.choice([0, 1, 1, 1, 2, 7], requests)
    lengths = counts + rng.integers(0, 200, requests)
    lengths[-1] += 1200
    b = Batch(lengths, counts, 6, 3, dim=dim, prefix=1500, pad=5)
    out, l = paged_shared_prefix_attention(**b.kwargs(), return_lse=True)
    b.check(out, l)
