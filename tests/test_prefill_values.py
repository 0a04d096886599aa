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
