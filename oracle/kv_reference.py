"""CPU oracle for the cache operators of include/kv_cache.h -- test
infrastructure only, never on the product path.

Norm over each head, position rotation, append to the paged caches, the 4-bit
form and the attention over it, in float64 numpy on the bf16 inputs widened
exactly. No reference counterpart (the reference fills its caches with torch
and has no compressed cache); the 4-bit element and scale formats are those of
the OCP Microscaling specification (E2M1, E8M0).

How it is pinned (tests/test_kv_cache_oracle.py): worked examples of the
rotation and of the 4-bit codes, the rotation's invariants (lengths of pairs,
scores that depend on distances alone), torch's rounding, a second way to the
nearest code, the byte layout of one element at a time, attention against
oracle.reference on the decoded values.
"""

import numpy as np

D = 128
TILE = 16
TILE_BYTES = 2176
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def places(T, seq_lens, cu_seqlens=None):
    """[(request, position) or None for padding] of every row."""
    B = len(seq_lens)
    out = [None] * T
    for b in range(B):
        first, last = (b, b + 1) if cu_seqlens is None else (cu_seqlens[b], cu_seqlens[b + 1])
        for t in range(first, min(last, T)):
            pos = int(seq_lens[b]) - (last - t)
            if pos >= 0:
                out[t] = (b, pos)
    return out


def slots(where, block_table, num_blocks, block_size):
    """[(block, slot) or None] of every place."""
    out = []
    for p in where:
        out.append(None)
        if p is None or p[1] // block_size >= block_table.shape[1]:
            continue
        blk = int(block_table[p[0], p[1] // block_size])
        if 0 <= blk < num_blocks:
            out[-1] = (blk, p[1] % block_size)
    return out


def norm(x, weight, eps):
    """x [..., dims] / sqrt(mean(x^2) + eps) * weight (None: x)."""
    x = np.asarray(x, dtype=np.float64)
    if weight is None:
        return x
    return x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * np.asarray(weight, np.float64)


def rotate(x, cos_sin, interleaved):
    """x [T, heads, dims] turned by the rows cos_sin [T, rotary_dim]."""
    x = np.array(x, dtype=np.float64)
    rot = cos_sin.shape[-1]
    h = rot // 2
    for i in range(h):
        p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
        c, s = cos_sin[:, None, i].astype(np.float64), cos_sin[:, None, h + i].astype(np.float64)
        a, b = x[..., p].copy(), x[..., q].copy()
        x[..., p], x[..., q] = a * c - b * s, b * c + a * s
    return x


def turn_rows(cos_sin, positions):
    """The table's rows at `positions`; NaN outside the table."""
    out = np.full((len(positions), cos_sin.shape[1]), np.nan)
    for t, p in enumerate(positions):
        if 0 <= p < cos_sin.shape[0]:
            out[t] = cos_sin[p]
    return out


def mxfp4_encode(x):
    """x [..., 128] -> codes [..., 128] (0..15) and scale bytes [..., 4]."""
    x = np.asarray(x, dtype=np.float64)
    g = x.reshape(x.shape[:-1] + (4, 32))
    top = np.abs(g).max(axis=-1)
    finite = np.isfinite(g).all(axis=-1)
    # The smallest exponent, from -126 up, that leaves at most 7.
    ok = np.where(finite, top, 0.0)
    exact = np.frexp(np.where(ok > 0, ok, 1.0))[1] - 4  # a start below the answer
    scale = np.where(ok > 0, np.maximum(exact + 127, 1), 1)
    for _ in range(4):
        scale = np.where(ok > 7.0 * np.ldexp(1.0, scale - 127), scale + 1, scale)
    y = np.abs(np.ldexp(np.where(finite[..., None], g, 0.0), (127 - scale)[..., None]))
    dist = np.abs(y[..., None] - GRID)
    # Nearest; at a tie the even index.
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])
    code = order[np.argmin(dist[..., order], axis=-1)]
    code = np.where(finite[..., None], code + 8 * np.signbit(g), 0)
    scale = np.where(finite, scale, 255)
    return code.reshape(x.shape).astype(np.uint8), scale.astype(np.uint8)


def mxfp4_decode(codes, scales):
    """The values that codes [..., 128] and scale bytes [..., 4] stand for."""
    mag = GRID[codes & 7] * np.where(codes > 7, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return mag * np.repeat(s, 32, axis=-1)


def tile_offsets(r, d):
    """(key code byte, value code byte, key scale byte, value scale byte) of token r, dim d."""
    return ((d // 32) * 256 + r * 16 + (d % 32) // 2,
            1024 + (r // 4) * 256 + (d // 8) * 16 + (r % 4) * 4 + (d % 8) // 2,
            2048 + (d // 32) * 16 + r,
            2112 + (r // 4) * 16 + (d // 32) * 4 + r % 4)


def mxfp4_store(cache, block, slot, head, k, v):
    """Put one token's 128 key and value numbers into the byte array."""
    tile = cache[block, head, slot // TILE]
    r = slot % TILE
    for x, code_at, scale_at in ((k, 0, 2), (v, 1, 3)):
        code, scale = mxfp4_encode(x)
        for d in range(D):
            at = tile_offsets(r, d)
            old = int(tile[at[code_at]])
            tile[at[code_at]] = (old & 0x0F) | (int(code[d]) << 4) if d % 2 else \
                (old & 0xF0) | int(code[d])
            tile[at[scale_at]] = scale[d // 32]


def mxfp4_load(cache, block, slot, head):
    """(keys [128], values [128]) of one token."""
    tile = cache[block, head, slot // TILE]
    r = slot % TILE
    at = np.array([tile_offsets(r, d) for d in range(D)])
    nib = 4 * (np.arange(D) % 2)
    out = []
    for code_at, scale_at in ((0, 2), (1, 3)):
        codes = (tile[at[:, code_at]] >> nib) & 15
        out.append(mxfp4_decode(codes, tile[at[::32, scale_at]]))
    return out


def mxfp4_rows(cache, block_table_row, n, head):
    """Keys and values [n, 128] of a request's first n tokens, with a mask of those in blocks of
    the cache."""
    num_blocks, bs = cache.shape[0], cache.shape[2] * TILE
    k, v, live = np.zeros((n, D)), np.zeros((n, D)), np.zeros(n, dtype=bool)
    for lb in range((n + bs - 1) // bs):
        blk = int(block_table_row[lb])
        if not 0 <= blk < num_blocks:
            continue
        m = min(bs, n - lb * bs)
        tiles = cache[blk, head]  # [tiles, bytes]
        r, d = np.meshgrid(np.arange(bs), np.arange(D), indexing="ij")
        at = tile_offsets(r % TILE, d)
        nib = 4 * (d % 2)
        for out, c, s in ((k, 0, 2), (v, 1, 3)):
            codes = (tiles[r // TILE, at[c]] >> nib) & 15
            scales = tiles[r // TILE, at[s]][:, ::32]
            out[lb * bs:lb * bs + m] = mxfp4_decode(codes, scales)[:m]
        live[lb * bs:lb * bs + m] = True
    return k, v, live


def mxfp4_attention(q, cache, block_table, seq_lens, scale):
    """out [B, Hq, 128] in float64, and for each row what its error can lean on: the sum of
    weight times |value|, the largest sum of |q k| times |scale| of a key, and the number of
    keys."""
    q = np.asarray(q, dtype=np.float64)
    B, Hq, _ = q.shape
    Hkv = cache.shape[1]
    G = Hq // Hkv
    out, mass = np.zeros((B, Hq, D)), np.zeros((B, Hq, D))
    reach, count = np.zeros((B, Hq)), np.zeros((B, Hq))
    cap = block_table.shape[1] * cache.shape[2] * TILE
    for b in range(B):
        n = min(max(int(seq_lens[b]), 0), cap)
        for kv in range(Hkv):
            k, v, live = mxfp4_rows(cache, block_table[b], n, kv)
            k, v = k[live], v[live]
            if not len(k):
                continue
            for h in range(kv * G, (kv + 1) * G):
                s = k @ q[b, h] * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[b, h], mass[b, h] = w @ v, w @ np.abs(v)
                reach[b, h] = (np.abs(k) @ np.abs(q[b, h])).max() * abs(scale)
                count[b, h] = len(k)
    return out, mass, reach, count
