"""CPU tests that pin oracle/kv_reference.py, what the cache operators are compared with."""

import numpy as np
import pytest
import torch

from oracle import kv_reference as kv
from oracle import reference as ref


def test_places_by_hand():
    assert kv.places(3, [5, 0, 1]) == [(0, 4), None, (2, 0)]
    # Rows 0-1 of request 0 (length 4), none of 1, 2-4 of request 2 (length 2: one has no place).
    assert kv.places(6, [4, 9, 2], [0, 2, 2, 5]) == [(0, 2), (0, 3), None, (2, 0), (2, 1), None]


def test_slots_leave_out_what_the_cache_lacks():
    table = np.array([[3, -1], [7, 0]])
    where = [(0, 0), (0, 16), (1, 5), (1, 31), (1, 32), None]
    assert kv.slots(where, table, 5, 16) == [(3, 0), None, None, (0, 15), None, None]


def test_rotation_by_hand():
    # A quarter turn of the pair (1, 0) is (0, 1).
    x = np.zeros((1, 1, 128))
    x[0, 0, 0] = 1.0
    quarter = np.zeros((1, 16))
    quarter[0, 8:] = 1.0  # cos 0, sin 1
    y = kv.rotate(x, quarter, False)
    assert y[0, 0, 0] == 0 and y[0, 0, 8] == 1 and np.count_nonzero(y) == 1
    y = kv.rotate(x, quarter, True)
    assert y[0, 0, 0] == 0 and y[0, 0, 1] == 1 and np.count_nonzero(y) == 1
    x[0, 0, 20] = 5.0  # past rotary_dim: stays
    assert kv.rotate(x, quarter, True)[0, 0, 20] == 5.0


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_makes_scores_of_distances(interleaved):
    rng = np.random.default_rng(0)
    ang = np.arange(50)[:, None] * 0.3 ** np.arange(32)
    table = np.concatenate([np.cos(ang), np.sin(ang)], axis=1)
    q, k = rng.normal(size=(2, 1, 1, 128))
    score = lambda i, j: float((kv.rotate(q, table[i:i + 1], interleaved)  # noqa: E731
                                * kv.rotate(k, table[j:j + 1], interleaved)).sum())
    assert abs(score(30, 10) - score(45, 25)) < 1e-9
    assert abs(score(30, 10) - score(30, 11)) > 1e-3


def test_norm_has_unit_mean_square():
    x = np.random.default_rng(1).normal(size=(3, 128)) * 7
    assert np.allclose((kv.norm(x, np.ones(128), 0.0) ** 2).mean(-1), 1.0)
    assert kv.norm(x, None, 0.0) is not None and np.array_equal(kv.norm(x, None, 0.0), x)


def test_codes_by_hand():
    x = np.zeros(128)
    x[:9] = [6.0, 0.25, 0.26, 0.75, 1.25, 2.5, 3.5, 5.0, -0.5]
    codes, scales = kv.mxfp4_encode(x)
    # Ties: 0.25 -> 0, 0.75 -> 1, 1.25 -> 1, 2.5 -> 2, 3.5 -> 4, 5 -> 4.
    assert list(codes[:9]) == [7, 0, 1, 2, 2, 4, 6, 6, 9]
    assert list(scales) == [127, 1, 1, 1]
    # 7 rounds to 6 at scale 1; beyond it the scale doubles.
    for top, scale, code in ((7.0, 127, 7), (7.001, 128, 6), (8.0, 128, 6), (3.5, 126, 7),
                             (3.501, 127, 6), (4.0, 127, 6)):
        x = np.zeros(128)
        x[40] = top
        codes, scales = kv.mxfp4_encode(x)
        assert (scales[1], codes[40]) == (scale, code), top


def test_codes_of_what_is_not_finite():
    for bad in (np.nan, np.inf, -np.inf):
        x = np.ones(128)
        x[70] = bad
        codes, scales = kv.mxfp4_encode(x)
        assert list(scales) == [125, 125, 255, 125] and not codes[64:96].any()
        y = kv.mxfp4_decode(codes, scales)
        assert np.isnan(y[64:96]).all() and (np.delete(y, range(64, 96)) == 1.0).all()


def test_codes_against_bisection():
    """The nearest value by another way: the midpoints between neighbours."""
    rng = np.random.default_rng(2)
    x = rng.normal(size=(200, 128)) * np.exp(rng.normal(size=(200, 1)) * 20)
    codes, scales = kv.mxfp4_encode(x)
    y = np.ldexp(np.abs(x).reshape(200, 4, 32), 127 - scales.astype(int)[..., None])
    assert (y.max(-1) <= 7).all() and (y.max(-1) > 3.5).all()
    mids = (kv.GRID[1:] + kv.GRID[:-1]) / 2
    want = np.searchsorted(mids, y).reshape(200, 128)
    assert np.array_equal(codes & 7, want) and np.array_equal(codes > 7, x < 0)
    # An element is off by half a step of its grid interval, at most 1 of [.., 7].
    err = np.abs(kv.mxfp4_decode(codes, scales) - x).reshape(200, 4, 32)
    step = np.where(y < 2, 0.25, np.where(y < 4, 0.5, 1.0))
    assert (err <= np.ldexp(step, scales.astype(int)[..., None] - 127)).all()


def test_every_decoded_value_is_bf16():
    codes = np.tile(np.arange(16, dtype=np.uint8), 8)
    for s in (1, 2, 100, 127, 250):
        y = kv.mxfp4_decode(codes, np.full(4, s, np.uint8))
        assert np.array_equal(torch.from_numpy(y).bfloat16().double().numpy(), y)


def test_layout_one_element_at_a_time():
    """Every byte of a tile belongs to one thing, and comes back from where it was put."""
    seen = np.zeros(kv.TILE_BYTES, dtype=int)
    for r in range(16):
        for d in range(128):
            at = kv.tile_offsets(r, d)
            seen[at[0]] += 1
            seen[at[1]] += 1
            if d % 32 == 0:
                seen[at[2]] += 2
                seen[at[3]] += 2
    assert (seen == 2).all()
    rng = np.random.default_rng(3)
    cache = rng.integers(0, 256, (3, 2, 2, kv.TILE_BYTES)).astype(np.uint8)
    k, v = rng.normal(size=(2, 128))
    before = cache.copy()
    kv.mxfp4_store(cache, 1, 21, 1, k, v)
    got_k, got_v = kv.mxfp4_load(cache, 1, 21, 1)
    assert np.array_equal(got_k, kv.mxfp4_decode(*kv.mxfp4_encode(k)))
    assert np.array_equal(got_v, kv.mxfp4_decode(*kv.mxfp4_encode(v)))
    changed = np.zeros_like(cache, dtype=bool)
    changed[1, 1, 1] = before[1, 1, 1] != cache[1, 1, 1]
    assert np.array_equal(before != cache, changed)
    assert (before != cache).sum() <= 136
    kk, vv, live = kv.mxfp4_rows(cache, [1], 22, 1)
    assert live.all() and np.array_equal(kk[21], got_k) and np.array_equal(vv[21], got_v)


def test_attention_against_the_bf16_oracle():
    rng = np.random.default_rng(4)
    cache = rng.integers(0, 256, (6, 2, 1, kv.TILE_BYTES)).astype(np.uint8)
    cache[..., 2048:] = rng.integers(120, 130, (6, 2, 1, 128))
    table, lens = np.array([[4, 1, 0], [2, 5, -1]]), [37, 20]
    q = torch.from_numpy(rng.normal(size=(2, 8, 128))).bfloat16()
    got, mass, reach, count = kv.mxfp4_attention(q.double().numpy(), cache, table, lens, 0.1)
    k = np.zeros((6, 16, 2, 128), dtype=np.float32)
    v = np.zeros_like(k)
    for blk in range(6):
        for h in range(2):
            kk, vv, _ = kv.mxfp4_rows(cache, [blk], 16, h)
            k[blk, :, h], v[blk, :, h] = kk, vv
    want = ref.attention_ref(q.float().numpy(), k, v, table, lens, 0.1)
    assert np.allclose(got, want, atol=1e-5 * np.abs(v).max(), rtol=1e-5)
    assert (count == np.array(lens)[:, None]).all() and (np.abs(got) <= mass + 1e-9).all()
    assert (reach > 0).all()


def test_attention_without_keys_is_zero():
    cache = np.zeros((2, 1, 1, kv.TILE_BYTES), dtype=np.uint8)
    q = np.ones((3, 2, 128))
    out, _, _, count = kv.mxfp4_attention(q, cache, np.array([[0], [-1], [9]]), [0, 16, 16], 1.0)
    assert not out.any() and not count.any()
