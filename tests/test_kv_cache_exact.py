"""How exact the attention over the 4-bit cache is, beyond what the output's rounding
hides (tests/test_kv_cache.py has the tolerances of arbitrary inputs).

The inputs make the scores exact in fp32: queries are small integers times a power
of two, keys multiples of a quantum, so that every product and sum of a score is a
multiple of one quantum and fits 24 bits, whatever the order of the sum. What is
left, for requests of up to 4 tokens and scores whose differences stay below 2^A in
the exponent, relative to the sum of weight times |value|:
  a weight: the scale times log2(e) (two roundings, 2^-23) and the fma (2^-24), times
    A ln 2, and the exponential, 2^-23 (the maximum's rounding is common to all);
    for numerator and denominator both;
  the sums: a weight in up to 3 parts whose products are exact, 12 additions and 2
    between columns, 2^-23 each, for both;
  quotient and product: 2 * 2^-23.
The output is then rounded to the nearest bf16 value: half its own step."""

import math

import numpy as np
import pytest
import torch

import kv_cache
from oracle import kv_reference as ref

D = 128
A = 4.0


def tolerance(a):
    return (2 * (1.5 * a * math.log(2) + 1) + 2 * 14 + 2) * 2.0 ** -23


TOL = tolerance(A)


def half_step(x):
    """Half the distance of the bf16 values around |x| (normal ones)."""
    return 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -126))) - 8)


def check_exact(got, want, mass, tol=TOL, under=0.0):
    over = tol * mass + under
    bad = ~(np.abs(got - want) <= half_step(np.abs(want) + over) + over)
    assert not bad.any(), f"{bad.sum()} of {bad.size}"


def most_difference(q, cache, table, lens):
    G = q.shape[1] // cache.shape[1]
    most = 0.0
    for b, n in enumerate(lens):
        for h in range(q.shape[1]):
            s = ref.mxfp4_rows(cache, table[b], n, h // G)[0] @ q[b, h]
            most = max(most, s.max() - s.min())
    return most


def fitting(q, cache, table, lens):
    """A power of two as scale."""
    return 2.0 ** math.floor(math.log2(A / (most_difference(q, cache, table, lens)
                                            * math.log2(math.e))))


def exact_inputs(seed, B, Hq, Hkv, bs=16):
    """Requests of 2 to 4 tokens: (q [B, Hq, 128] float64, cache, table, lengths, scale)."""
    rng = np.random.default_rng(seed)
    cache = rng.integers(0, 256, (B, Hkv, bs // 16, 2176), dtype=np.uint8)
    cache[..., 2048:2112] = rng.integers(126, 129, (B, Hkv, bs // 16, 64), dtype=np.uint8)
    cache[..., 2112:] = rng.integers(120, 134, (B, Hkv, bs // 16, 64), dtype=np.uint8)
    q = rng.integers(-8, 9, (B, Hq, D)).astype(np.float64)
    lens = [2 + b % 3 for b in range(B)]
    table = np.arange(B)[:, None].astype(np.int32)
    # Scores: multiples of 0.25 below 128 * 8 * 12; their differences times scale and
    # log2(e) below A.
    return q, cache, table, lens, fitting(q, cache, table, lens)


def model(q, cache, table, lens, scale, parts, heads_per_kv):
    """The attention with fp32 weights cut to `parts` (how many bits each keeps; None: whole),
    rounded to bf16."""
    B, Hq, _ = q.shape
    out = np.zeros((B, Hq, D))
    for b in range(B):
        for h in range(Hq):
            k, v, _ = ref.mxfp4_rows(cache, table[b], lens[b], h // heads_per_kv)
            s = k @ q[b, h] * scale
            w = np.exp(s - s.max()).astype(np.float32)
            if parts is not None:
                rest, total = w.copy(), np.zeros(len(w))
                for _ in range(parts):
                    p = (rest.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
                    total, rest = total + p, rest - p
                w = total
            out[b, h] = (w.astype(np.float64) @ v) / w.astype(np.float64).sum()
    return torch.from_numpy(out).bfloat16().double().numpy()


def test_the_check_tells_weights_of_fewer_bits():
    q, cache, table, lens, scale = exact_inputs(0, 24, 8, 2)
    want, mass, _, _ = ref.mxfp4_attention(q, cache, table, lens, scale)
    for parts in (None, 3):
        check_exact(model(q, cache, table, lens, scale, parts, 4), want, mass)
    for got in (model(q, cache, table, lens, scale, 2, 4), model(q, cache, table, lens, scale, 1, 4),
                np.zeros_like(want), 2 * want):
        with pytest.raises(AssertionError):
            check_exact(got, want, mass)


def run(gpu, q, cache, table, lens, scale, **how):
    assert np.array_equal(torch.from_numpy(q).bfloat16().double().numpy(), q)
    return run_any(gpu, q, cache, table, lens, scale, **how)


def run_any(gpu, q, cache, table, lens, scale, **how):
    qt = torch.from_numpy(q).bfloat16()
    index = lambda x: torch.as_tensor(np.asarray(x), dtype=torch.int32).to(gpu)  # noqa: E731
    out = kv_cache.gqa_decode_mxfp4(qt.to(gpu), torch.from_numpy(cache).to(gpu), index(table),
                                    index(lens), scale, **how)
    return out.double().cpu().numpy()


GROUPS = [(2, 2), (8, 2), (4, 1), (5, 1), (16, 2), (9, 1), (32, 2), (20, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", GROUPS)
def test_weights_keep_their_24_bits(gpu, Hq, Hkv):
    q, cache, table, lens, scale = exact_inputs(Hq, 48, Hq, Hkv)
    want, mass, _, _ = ref.mxfp4_attention(q, cache, table, lens, scale)
    for how in ({}, {"num_workgroups": 5}):
        check_exact(run(gpu, q, cache, table, lens, scale, **how), want, mass)


# Rounding errors that spread evenly over half a step, 2^-8 of a value at most: 2^-8 / sqrt(3)
# of the outputs in the 2-norm (less, as values lie all over a step's binade).
NORM = 2.0 ** -8 / math.sqrt(3)


def ordinary_inputs(seed, lens, Hq, Hkv, bs=16):
    """Normal queries over random codes, scores of a few units: (q, cache, table, scale)."""
    rng = np.random.default_rng(seed)
    blocks = [-(-n // bs) for n in lens]
    cache = rng.integers(0, 256, (sum(blocks), Hkv, bs // 16, 2176), dtype=np.uint8)
    cache[..., 2048:] = rng.integers(125, 128, cache[..., 2048:].shape, dtype=np.uint8)
    table = np.full((len(lens), max(blocks)), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = np.arange(at, at + n)
        at += n
    q = torch.from_numpy(rng.normal(size=(len(lens), Hq, D))).bfloat16().double().numpy()
    return q, cache, table, D ** -0.5


def off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


def test_the_norm_tells_mistakes():
    lens = [300, 77]
    q, cache, table, scale = ordinary_inputs(3, lens, 4, 1)
    want, _, _, _ = ref.mxfp4_attention(q, cache, table, lens, scale)
    assert off(model(q, cache, table, lens, scale, None, 4), want) < NORM
    for got in (model(q, cache, table, lens, scale, 1, 4), np.zeros_like(want), 2 * want):
        assert off(got, want) > NORM


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", GROUPS)
def test_ordinary_batches(gpu, Hq, Hkv):
    lens = [2000, 1, 333, 640, 77, 0, 1500]
    q, cache, table, scale = ordinary_inputs(Hq, lens, Hq, Hkv)
    want, _, _, _ = ref.mxfp4_attention(q, cache, table, lens, scale)
    for how in ({}, {"num_workgroups": 37}):
        assert off(run(gpu, q, cache, table, lens, scale, **how), want) < NORM


def silence(cache, dims):
    """Keys of all tokens zero in these dims (of either sign)."""
    for r in range(16):
        for d in dims:
            at = ref.tile_offsets(r, d)[0]
            cache[..., at] &= 0xF7 if d % 2 == 0 else 0x7F
            cache[..., at] &= 0xF8 if d % 2 == 0 else 0x8F


@pytest.mark.gpu
@pytest.mark.parametrize("times", [0.0, -1.0, 16.0, -64.0, 1024.0])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (8, 1), (16, 1)])
def test_exact_scores_under_other_scales(gpu, Hq, Hkv, times):
    """No softmax at all, the smallest score first, one key taking nearly all. There a weight,
    relative to the largest one, can lie below fp32's smallest normal number, 2^-126, and count as
    0, and so can its second and third part and their products: 4 * 2^-126 of the largest |value|
    for each of up to 4 keys (all that is left where the largest weight's value is 0)."""
    q, cache, table, lens, scale = exact_inputs(Hq, 48, Hq, Hkv)
    want, mass, _, _ = ref.mxfp4_attention(q, cache, table, lens, scale * times)
    largest = 6.0 * 2.0 ** (cache[..., 2112:].max() - 127.0)
    check_exact(run(gpu, q, cache, table, lens, scale * times), want, mass,
                tolerance(A * max(abs(times), 1.0)), 4 * 4 * 2.0 ** -126 * largest)


@pytest.mark.gpu
@pytest.mark.parametrize("loud", [2.0 ** 8, 2.0 ** 12, 2.0 ** 30, 2.0 ** 100])
@pytest.mark.parametrize("Hq,Hkv", GROUPS)
def test_quiet_dims_beside_loud_ones(gpu, Hq, Hkv, loud):
    """Queries with a few dims many times the others, which keys that are zero there take out of
    the score: what the other dims say is not lost."""
    q, cache, table, lens, _ = exact_inputs(Hq, 24, Hq, Hkv)
    dims = [3, 40, 41, 127]
    silence(cache, dims)
    rng = np.random.default_rng(1)
    q[..., dims] = rng.integers(4, 9, q[..., dims].shape) * loud
    q[::3, ::2, dims] = 1.0  # and heads without, beside them
    scale = 2.0 ** -9
    want, mass, _, _ = ref.mxfp4_attention(q, cache, table, lens, scale)
    assert most_difference(q, cache, table, lens) * scale * math.log2(math.e) <= A
    check_exact(run(gpu, q, cache, table, lens, scale), want, mass)


@pytest.mark.gpu
@pytest.mark.parametrize("loud", [2.0 ** 8, 2.0 ** 10])
@pytest.mark.parametrize("Hq,Hkv", GROUPS)
def test_sums_of_loud_and_quiet_dims(gpu, Hq, Hkv, loud):
    """The same with keys that are not zero there: the sum has all its terms. (4 terms of up to
    8 * 12 * 2^10 and 124 of up to 96, in steps of 0.25: 21 bits.)"""
    q, cache, table, lens, _ = exact_inputs(Hq, 24, Hq, Hkv)
    dims = [3, 40, 41, 127]
    rng = np.random.default_rng(1)
    q[..., dims] = rng.integers(4, 9, q[..., dims].shape) * loud
    scale = fitting(q, cache, table, lens)
    want, mass, _, _ = ref.mxfp4_attention(q, cache, table, lens, scale)
    check_exact(run(gpu, q, cache, table, lens, scale), want, mass)


@pytest.mark.gpu
@pytest.mark.parametrize("keys,at", [((0, 4), 124), ((4, 7), 122), ((100, 103), 26),
                                     ((246, 250), -121),
                                     ((252, 255), -126)])
@pytest.mark.parametrize("tiny", [False, True])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (8, 1), (16, 1)])
def test_far_scales(gpu, Hq, Hkv, keys, at, tiny):
    """Keys of very small and very large scales under queries of the opposite size; slots behind
    the last token hold anything. With `tiny`, an element far below its head's largest too."""
    rng = np.random.default_rng(2)
    q, cache, table, lens, _ = exact_inputs(Hq, 24, Hq, Hkv)
    cache[..., 2048:2112] = rng.integers(*keys, cache[..., 2048:2112].shape)
    for b, n in enumerate(lens):
        for r in range(n, 16):
            cache[b, :, 0, [2048 + g * 16 + r for g in range(4)]] = rng.integers(0, 256, (4, Hkv))
            cache[b, :, 0, [2112 + r // 4 * 16 + g * 4 + r % 4 for g in range(4)]] = 255
    q *= 2.0 ** at
    if tiny:
        silence(cache, [64])
        q[..., 64] = 2.0 ** -133
    scale = 2.0 ** -10
    assert most_difference(q, cache, table, lens) * scale * math.log2(math.e) <= A
    want, mass, _, _ = ref.mxfp4_attention(q, cache, table, lens, scale)
    check_exact(run(gpu, q, cache, table, lens, scale), want, mass)


@pytest.mark.gpu
@pytest.mark.parametrize("keys,at", [((126, 129), 0), ((252, 255), -126)])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (8, 1), (16, 1)])
def test_queries_that_are_not_finite(gpu, Hq, Hkv, keys, at):
    """NaN for the head of an infinity or NaN, whatever the keys' scales and signs; for no other."""
    rng = np.random.default_rng(4)
    q, cache, table, lens, _ = exact_inputs(Hq, 24, Hq, Hkv)
    cache[..., 2048:2112] = rng.integers(*keys, cache[..., 2048:2112].shape)
    cache[5:, ..., :1024] = 0x33  # keys of one sign: scores of one infinity
    q *= 2.0 ** at
    bad = np.zeros(q.shape[:2], dtype=bool)
    for b, h, d, x in ((0, 1, 77, np.nan), (3, 0, 3, np.inf), (7, Hq - 1, 127, -np.inf),
                       (8, 2, 31, np.inf)):
        q[b, h, d], bad[b, h] = x, True
    got = torch.from_numpy(run_any(gpu, q, cache, table, lens, 2.0 ** -10))
    assert torch.isnan(got[torch.from_numpy(bad)]).all()
    assert torch.isfinite(got[torch.from_numpy(~bad)]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Hq", [1, 8, 16])
@pytest.mark.parametrize("lens", [[131072], [40, 70000], [70000, 3, 66000, 1]])
def test_segments_cut_into_many_pieces(gpu, lens, Hq):
    """One kv-head, so that a request spans more workgroups than the merge's waves have lanes; in
    front of it, short ones that start in the middle of a share."""
    bs = 256
    q, cache, table, scale = ordinary_inputs(Hq, lens, Hq, 1, bs)
    # Shares of 16 units (of 32 tokens) at least: the longest takes that many workgroups.
    units = [-(-n // 32) for n in lens]
    assert max(units) / (sum(units) / min(256, -(-sum(units) // 16))) > 65
    want, _, _, _ = ref.mxfp4_attention(q, cache, table, lens, scale)
    got = run(gpu, q, cache, table, lens, scale, num_workgroups=256)
    assert off(got, want) < NORM
    assert np.array_equal(got, run(gpu, q, cache, table, lens, scale, num_workgroups=256))
    assert off(run(gpu, q, cache, table, lens, scale), want) < NORM
