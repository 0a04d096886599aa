"""GPU tests of the prompt attention (prefill.py): ragged requests that workgroups of eight waves
take in the order of their keys, and tables far wider than any request. Tolerances:
tests/test_prefill.py."""

import pytest
import torch

import prefill
from test_prefill import D, normal, packed_want, paged_want, pages, sums, tensor
from test_prefill_values import check_all

pytestmark = pytest.mark.gpu


def splits_of(run, want):
    for ns in (0, 1, 3):
        check_all(*run(num_splits=ns), want, f"splits {ns}")


@pytest.mark.parametrize("news,lens,behind", [
    ([300, 0, 210, 190], [400, 50, 700, 190], 7), ([150, 150], [600, 600], 0),
    ([1, 400, 6], [64, 400, 3], 70)])
@pytest.mark.parametrize("Hq,Hkv,bs", [(8, 2, 8), (16, 1, 24)])
@pytest.mark.parametrize("causal", [True, False])
def test_eight_waves_over_pages(gpu, news, lens, behind, Hq, Hkv, bs, causal):
    """Blocks of 8 tokens modulo 16 take eight waves; more rows than a workgroup a request."""
    gen = torch.Generator().manual_seed(bs)
    cu = sums(news)
    assert sum(news) * Hq // Hkv > 256 * len(news)
    table, num = pages(lens, bs, gen)
    q = normal(gen, sum(news) + behind, Hq, D)
    kc, vc = normal(gen, num, bs, Hkv, D), normal(gen, num, bs, Hkv, D)
    splits_of(lambda **kw: prefill.gqa_prefill(
        q.to(gpu), kc.to(gpu), vc.to(gpu), table.to(gpu), tensor(lens, gpu), 0.1,
        cu_seqlens=tensor(cu, gpu), causal=causal, return_lse=True, **kw),
        paged_want(q, kc, vc, table, lens, cu, 0.1, causal))


@pytest.mark.parametrize("news,lens,behind", [
    ([700, 0, 500, 600], [1500, 0, 1100, 1700], 9), ([620, 620], [1100, 1100], 0)])
def test_eight_waves_over_rows(gpu, news, lens, behind):
    """1024 keys a request and more, 2048 rows a request, more workgroups than CUs."""
    Hq, Hkv, B = 64, 8, len(news)
    assert sum(lens) >= 1024 * B and sum(news) * 8 >= 2048 * B and sum(news) * 8 // 256 * 8 > 256
    gen = torch.Generator().manual_seed(B)
    cu_q, cu_k = sums(news), sums(lens)
    q = normal(gen, sum(news) + behind, Hq, D)
    k, v = normal(gen, sum(lens), Hkv, D), normal(gen, sum(lens), Hkv, D)
    splits_of(lambda **kw: prefill.gqa_prefill_packed(
        q.to(gpu), k.to(gpu), v.to(gpu), tensor(cu_q, gpu), tensor(cu_k, gpu), 0.1,
        return_lse=True, **kw), packed_want(q, k, v, cu_q, cu_k, 0.1, True))


@pytest.mark.parametrize("news,lens", [([100], [100]), ([3, 5, 1], [900, 3000, 70]),
                                       ([256], [1256]), ([130, 7], [130, 400])])
@pytest.mark.parametrize("bs", [16, 64, 20])
def test_wide_tables(gpu, news, lens, bs):
    """Tables for 131072 tokens, whatever the requests have of them."""
    Hq, Hkv, cu = 8, 2, sums(news)
    gen = torch.Generator().manual_seed(bs)
    table, num = pages(lens, bs, gen, width_extra=131072 // bs)
    q = normal(gen, sum(news), Hq, D)
    kc, vc = normal(gen, num, bs, Hkv, D), normal(gen, num, bs, Hkv, D)
    want = paged_want(q, kc, vc, table, lens, cu, 0.1, True)
    for ns in (0, 1, 128):
        check_all(*prefill.gqa_prefill(q.to(gpu), kc.to(gpu), vc.to(gpu), table.to(gpu),
                                       tensor(lens, gpu), 0.1, cu_seqlens=tensor(cu, gpu),
                                       num_splits=ns, return_lse=True), want, f"splits {ns}")
