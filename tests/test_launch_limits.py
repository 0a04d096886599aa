"""CPU tests of sizes whose launches would have 2^32 threads or more, which HIP refuses: the
prompt attention and the 8-bit append refuse them before any launch."""

import pytest

import capi
from test_prefill_abi import INVALID, SOME, append_args, packed, paged


@pytest.mark.parametrize("make", [paged, packed])
@pytest.mark.parametrize("over", [
    dict(T=1 << 20, B=1 << 20, Hq=16, Hkv=16), dict(T=100, B=1 << 20, Hq=64, Hkv=16),
    dict(T=1 << 20, B=1 << 20, Hq=32, Hkv=32, cu_seqlens_q=SOME)])
def test_more_workgroups_than_a_launch_has(make, over):
    assert capi.prefill_gqa_launch(make(**over), 1, None, 0, None) == INVALID


def test_more_workgroups_of_eight_waves():
    """(Blocks of 8 tokens take them: half as many workgroups are too many.)"""
    a = paged(T=1 << 20, B=1 << 20, Hq=8, Hkv=8, block_size=8)
    assert capi.prefill_gqa_launch(a, 1, None, 0, None) == INVALID


@pytest.mark.parametrize("make", [paged, packed])
def test_more_rows_than_the_second_launch_joins(make):
    a = make(T=1 << 23, Hq=8, Hkv=8)
    need = capi.prefill_gqa_workspace_bytes(a, 2)
    assert need == (1 << 26) * 2 * 520
    assert capi.prefill_gqa_launch(a, 2, SOME, need, None) == INVALID


@pytest.mark.parametrize("over", [
    dict(T=1 << 20, B=1 << 20, Hkv=16), dict(T=1 << 23, B=1 << 20, Hkv=8, cu_seqlens=SOME)])
def test_more_tiles_than_an_append_has(over):
    assert capi.kv8_append_launch(append_args(**over), SOME, SOME, None) == INVALID
