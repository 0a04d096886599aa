"""GPU tests of the prompt attention (prefill.py) on keys and values at the ends of their range,
over rows and paged caches, whole and split. Tolerances: tests/test_prefill.py.
"""

import numpy as np
import pytest
import torch

import prefill
from test_prefill import D, check, f64, normal, packed_want, paged_want, pages, sums, tensor

pytestmark = pytest.mark.gpu

INF = float("inf")

def check_all(out, lse, want, label=""):
    """check, and NaN log-sum-exps in their places."""
    check(out, lse, want, label)
    assert np.array_equal(np.isnan(f64(lse)), np.isnan(want[1])), f"{label}: NaN in other lse"


def forms(gpu, q, k, v, news, lens, scale, causal=True, splits=(1, 3), sizes=(16, 8, 12)):
    """Results over rows and over paged caches of several block sizes, whole and split. A block
    size of None: rows. The caches hold NaN wherever no request's keys lie."""
    cu_q, cu_k = sums(news), sums(lens)
    for ns in splits:
        yield (f"rows, splits {ns}", prefill.gqa_prefill_packed(
            q.to(gpu), k.to(gpu), v.to(gpu), tensor(cu_q, gpu), tensor(cu_k, gpu), scale,
            causal=causal, num_splits=ns, return_lse=True))
        for bs in sizes:
            table, num = pages(lens, bs, torch.Generator().manual_seed(bs))
            kc = torch.full((num, bs) + tuple(k.shape[1:]), float("nan"), dtype=torch.bfloat16)
            vc = kc.clone()
            for b, n in enumerate(lens):
                at = table[b].long()[torch.arange(n) // bs], torch.arange(n) % bs
                kc[at], vc[at] = k[cu_k[b]:cu_k[b + 1]], v[cu_k[b]:cu_k[b + 1]]
            yield (f"blocks of {bs}, splits {ns}", prefill.gqa_prefill(
                q.to(gpu), kc.to(gpu), vc.to(gpu), table.to(gpu), tensor(lens, gpu), scale,
                cu_seqlens=tensor(cu_q, gpu), causal=causal, num_splits=ns, return_lse=True))


def with_reach(want, of_finite):
    """`want`, its tolerance being that of the keys with finite scores (those whose scores are
    -infinity weigh nothing)."""
    return want[:3] + (of_finite[3],) + want[4:]


# Few rows behind many keys, prompts of some tiles of rows, and enough rows for eight waves.
SHAPES = {
    "drafts": ([3, 1], [400, 90], 8, 2),
    "prompts": ([300, 70], [300, 200], 8, 2),
    "long": ([1100], [1100], 64, 8),
}


def rows(shape, seed):
    news, lens, Hq, Hkv = SHAPES[shape]
    gen = torch.Generator().manual_seed(seed)
    q = normal(gen, sum(news), Hq, D)
    return q, normal(gen, sum(lens), Hkv, D), normal(gen, sum(lens), Hkv, D), news, lens


@pytest.mark.parametrize("shape", SHAPES)
def test_largest_values(gpu, shape):
    """Sums of many values next to bf16's largest: their means are numbers."""
    q, k, v, news, lens = rows(shape, 2)
    most = torch.finfo(torch.bfloat16).max
    v.copy_(torch.where(v > 0, most, -most))
    v[:, :, :40], v[:, :, 40:80] = most, -most
    want = packed_want(q, k, v, sums(news), sums(lens), 0.1, True)
    assert (np.abs(want[0]) <= most * (1 + 2.0 ** -20)).all()
    for label, got in forms(gpu, q, k, v, news, lens, 0.1):
        check_all(*got, want, label)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_infinite_values(gpu, shape, causal):
    """A value that is not finite gives NaN in its dim to every row that sees it, whether the row
    sees its tile whole (the first keys) or in part (near the end)."""
    q, k, v, news, lens = rows(shape, 1)
    v[3, 0, 5], v[7, 1, 9], v[70, 0, 77] = INF, -INF, INF
    v[71, 0, 77] = -INF
    v[lens[0] - 2, 1, 30] = -INF
    cu_q, cu_k = sums(news), sums(lens)
    want = packed_want(q, k, v, cu_q, cu_k, 0.1, causal)
    for label, got in forms(gpu, q, k, v, news, lens, 0.1, causal):
        check_all(*got, want, label)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale", [0.1, -0.1])
def test_infinite_keys(gpu, shape, scale):
    """A key with an infinite score has no weight or gives NaN; a row whose keys' scores are all
    -infinity gives NaN, in one split or all of them, and a row without keys zeros as ever."""
    q, k, v, news, lens = rows(shape, 3)
    news, at = news + [2, 1, 3, 2], sum(news)
    Hq, Hkv, end = q.shape[1], k.shape[1], sum(lens)
    gen = torch.Generator().manual_seed(4)
    lens = lens + [2, 0, 200, 130]  # all infinite; no key; all infinite; the first 100 of 130
    q = torch.cat([q, normal(gen, 8, Hq, D)])
    k = torch.cat([k, normal(gen, 332, Hkv, D)])
    v = torch.cat([v, normal(gen, 332, Hkv, D)])
    q[:, :, 11] = q[:, :, 11].abs() + 1.0
    k[5, 0, 11] = k[80, 1, 11] = k[end:end + 302, 0, 11] = -INF if scale > 0 else INF
    k[20, 1, 11] = INF if scale > 0 else -INF  # (a score of +infinity: NaN)
    cu_q, cu_k = sums(news), sums(lens)
    for causal in (True, False):
        finite = torch.where(torch.isfinite(k), k, 0.0)
        want = with_reach(packed_want(q, k, v, cu_q, cu_k, scale, causal),
                          packed_want(q, finite, v, cu_q, cu_k, scale, causal))
        nan = np.isnan(want[0]).all(axis=2)
        G = Hq // Hkv
        assert nan[at:at + 2, :G].all() and not nan[at:at + 2, G:].any()
        assert not want[0][at + 2].any() and nan[at + 3:at + 6, :G].all()
        assert not nan[at + 6:, :].any()
        for label, got in forms(gpu, q, k, v, news, lens, scale, causal, splits=(1, 2, 7)):
            check_all(*got, want, label)


def test_infinite_keys_and_ids_outside(gpu):
    """Keys in blocks outside the cache are not seen: only the others' scores count."""
    gen = torch.Generator().manual_seed(5)
    Hq, Hkv, bs, lens, news = 4, 1, 16, [160, 160, 160], [3, 3, 3]
    q, cu = normal(gen, 9, Hq, D), sums(news)
    q[:, :, 0] = 1.0
    table, num = pages(lens, bs, gen)
    kc, vc = normal(gen, num, bs, Hkv, D), normal(gen, num, bs, Hkv, D)
    kc[table[0].long()] = kc[table[1, :5].long()] = kc[table[2, 5:].long()] = 1.0
    for ids in (table[0], table[1, :5], table[2, 5:]):
        kc[ids.long(), :, :, 0] = -INF
    table[0, 2:8] = -1   # what is left has scores of -infinity: NaN
    table[1, 5:] = num   # as well
    table[2, 5:] = -3    # finite ones are left
    table[0, 0] = num + 5
    finite = torch.where(torch.isfinite(kc), kc, 0.0)
    want = with_reach(paged_want(q, kc, vc, table, lens, cu, 0.1, True),
                      paged_want(q, finite, vc, table, lens, cu, 0.1, True))
    assert np.isnan(want[0][:6]).all() and np.isfinite(want[0][6:]).all()
    table4 = torch.cat([table, torch.full((1, 10), -1, dtype=torch.int32)])  # no key at all: zeros
    cu4, q4 = sums(news + [2]), torch.cat([q, q[:2]])
    want4 = with_reach(paged_want(q4, kc, vc, table4, lens + [100], cu4, 0.1, True),
                       paged_want(q4, finite, vc, table4, lens + [100], cu4, 0.1, True))
    for ns in (1, 2, 5):
        check_all(*prefill.gqa_prefill(q.to(gpu), kc.to(gpu), vc.to(gpu), table.to(gpu),
                                       tensor(lens, gpu), 0.1, cu_seqlens=tensor(cu, gpu),
                                       num_splits=ns, return_lse=True), want, f"splits {ns}")
        got = prefill.gqa_prefill(q4.to(gpu), kc.to(gpu), vc.to(gpu), table4.to(gpu),
                                  tensor(lens + [100], gpu), 0.1, cu_seqlens=tensor(cu4, gpu),
                                  num_splits=ns, return_lse=True)
        check_all(*got, want4, f"splits {ns}, a request without keys")
        assert not got[0][9:].any() and torch.isneginf(got[1][9:]).all()


@pytest.mark.parametrize("shape", SHAPES)
def test_log_sums_are_of_fp32_weights(gpu, shape):
    """The log-sum-exps of few large weights, which bf16 would move by up to 2^-8. Of 4 dims: their
    raw scores are off by 4 * 2^-24 of the sum of |q k|, 3 roundings more until the exponent,
    which the tolerance doubles; the exponential 2^-22, twice for a sum that is rescaled; sums
    of 64 keys in a row, one of them to the next; the logarithm and its sum with the
    reference, 4 steps of fp32 of the result and 2^-20."""
    q, k, v, news, lens = rows(shape, 6)
    q[:, :, 4:], k[:, :, 4:] = 0.0, 0.0
    scale = 2.0
    cu_q, cu_k = sums(news), sums(lens)
    for causal in (True, False):
        want = packed_want(q, k, v, cu_q, cu_k, scale, causal)
        _, want_lse, _, reach, count = want
        tol = (16 * 2.0 ** -24 * reach + 2.0 ** -21 + (count / 64 + 64) * 2.0 ** -24
               + 4 * 2.0 ** -23 * np.abs(want_lse) + 2.0 ** -20)
        plain = {}
        for label, (out, lse) in forms(gpu, q, k, v, news, lens, scale, causal):
            check_all(out, lse, want, label)
            off = np.abs(f64(lse) - want_lse) / tol
            assert (off <= 1).all(), f"{label}: lse off by {off.max()} of the tolerance"
            plain[label] = out
        for ns in (1, 3):  # and the results are the same without them
            got = prefill.gqa_prefill_packed(q.to(gpu), k.to(gpu), v.to(gpu), tensor(cu_q, gpu),
                                             tensor(cu_k, gpu), scale, causal=causal, num_splits=ns)
            assert torch.equal(got, plain[f"rows, splits {ns}"])
