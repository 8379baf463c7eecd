"""The paged cache's operators in plain numpy: a Python free list, and softmax
attention in 64 bits with the error bound of a 16-bit kernel.

Test infrastructure only; nothing in heatkv_amd imports it.
"""

from __future__ import annotations

import numpy as np


def build_tables(tables, lengths, new_counts, ring, ring_range, num_tokens, block, window=0, sinks=0):
    """(tables, ring, slot_map, query_starts, lengths, range, status) after one step; inputs untouched."""
    tables, ring = np.array(tables), np.array(ring)
    R, M = tables.shape
    first, free = (int(x) for x in ring_range)
    N = len(ring)
    blocks_of = lambda rows: -(-rows // block)  # noqa: E731
    fresh = [max(0, int(n)) for n in new_counts]
    take = [blocks_of(int(l) + n) - blocks_of(int(l)) for l, n in zip(lengths, fresh)]
    status = 0
    if sum(take) > free:
        status |= 1
    if any(blocks_of(int(l) + n) > M for l, n in zip(lengths, fresh)):
        status |= 2
    if sum(fresh) > num_tokens:
        status |= 4
    slots = np.full(num_tokens, -1, np.int64)
    given = np.array(tables), np.array(ring)
    if status:
        return (tables, ring, slots, np.zeros(R + 1, np.int32), np.array(lengths, np.int32),
                np.array(ring_range, np.int32), status)
    popped, pushed, token, starts, after = 0, [], 0, [0], []
    for r in range(R):
        held, n = int(lengths[r]), fresh[r]
        for j in range(blocks_of(held), blocks_of(held) + take[r]):
            tables[r, j] = ring[(first + popped) % N]
            popped += 1
        for row in range(held, held + n):
            slots[token] = int(tables[r, row // block]) * block + row % block
            token += 1
        starts.append(token)
        after.append(0 if new_counts[r] < 0 else held + n)

        def needed(j, rows):
            """Whether a token at position `rows` or later sees a row of block j."""
            if window == 0:
                return True
            return j < blocks_of(sinks) or (j + 1) * block > rows - window + 1

        if new_counts[r] < 0:
            pushed += [tables[r, j] for j in range(blocks_of(held)) if needed(j, held)]
        else:
            pushed += [tables[r, j] for j in range(blocks_of(held + n)) if needed(j, held) and not needed(j, held + n)]
    if free - popped + len(pushed) > N:  # more than the ring has room for
        return (*given, np.full(num_tokens, -1, np.int64), np.zeros(R + 1, np.int32), np.array(lengths, np.int32),
                np.array(ring_range, np.int32), 8)
    for i, b in enumerate(pushed):
        ring[(first + free + i) % N] = b
    new_range = np.array([(first + popped) % N if N else 0, free - popped + len(pushed)], np.int32)
    return tables, ring, slots, np.array(starts, np.int32), np.array(after, np.int32), new_range, 0


def rows_of(cache, blocks, rows):
    """The first `rows` rows of `blocks`, [kv_heads, rows, D] in 64 bits."""
    n = -(-rows // cache.shape[2])
    got = cache[np.asarray(blocks[:n], np.int64)].astype(np.float64)
    return np.moveaxis(got, 1, 0).reshape(cache.shape[1], n * cache.shape[2], cache.shape[3])[:, :rows]


def attention(q, k_cache, v_cache, tables, lengths, starts, scale, half_step, window=0, sinks=0, causal=True,
              prefix_blocks=None, prefix_len=0):
    """(out [T, H, D], lse [H, T], out bound, lse bound) of the paged attentions.

    ``half_step``: the largest relative rounding error of q's type.  A kernel
    rounds each weight p to that type for the product with V and the result
    once, and works in 32 bits otherwise: with A = sum p |v| / sum p,
    |error| <= half_step (A + |out|) + e A with e the relative error of p / sum p in
    32 bits, twice the score's absolute error (its D products accumulated, at
    most D + 8 roundings of sum |q k|) plus the roundings of exp2 and of the
    sum over the keys.  Rows that see nothing: 0 and -inf, held exactly."""
    T, H, D = q.shape
    hk = k_cache.shape[1]
    group = H // hk
    out = np.zeros((T, H, D))
    tol = np.zeros((T, H, D))
    lse = np.full((H, T), -np.inf)
    lse_tol = np.zeros((H, T))
    ulp = 2.0 ** -24
    for r in range(len(lengths)):
        n, total = int(starts[r + 1] - starts[r]), int(lengths[r])
        if n == 0:
            continue
        K, V = rows_of(k_cache, tables[r], total), rows_of(v_cache, tables[r], total)
        if prefix_len:
            K = np.concatenate([rows_of(k_cache, prefix_blocks, prefix_len), K], 1)
            V = np.concatenate([rows_of(v_cache, prefix_blocks, prefix_len), V], 1)
        for i in range(n):
            t, pos = int(starts[r]) + i, total - n + i
            j = np.arange(total)
            seen = (j <= pos) if causal else np.full(total, pos >= 0)
            if window:
                seen = seen & ((j > pos - window) | (j < sinks))
            seen = np.concatenate([np.ones(prefix_len, bool), seen])
            if not seen.any():
                continue
            for h in range(H):
                k, v = K[h // group][seen], V[h // group][seen]
                qq = q[t, h].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = k @ qq * scale
                    m = s.max()
                    p = np.exp(s - m)
                    total_p = p.sum()
                    out[t, h] = p @ v / total_p
                    A = p @ np.abs(v) / total_p
                    lse[h, t] = m + np.log(total_p)
                    e_s = (D + 8) * ulp * (np.abs(k) @ np.abs(qq)).max() * abs(scale) + 4 * ulp * np.abs(s).max()
                e = 2 * e_s + (len(s) + 16) * ulp
                tol[t, h] = half_step * (A + np.abs(out[t, h])) + e * A + 1e-30
                lse_tol[h, t] = e + 8 * ulp * (abs(lse[h, t]) + 1)
    return out, lse, tol, lse_tol
