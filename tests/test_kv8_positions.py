"""GPU tests of kv_cache.kv_append_fp8's positions: they turn the rows, whose places in the cache
stay; a position outside the rotation table turns a row to NaN. Codes, scales and queries
against oracle/kv8_reference.py and oracle/kv_reference.py, as in tests/test_kv8.py."""

import numpy as np
import pytest
import torch

import kv_cache
from oracle import kv8_reference as ref
from oracle import kv_reference as kv
from test_kv8 import check_bytes, random_cache
from test_kv_cache import STEPS, check_bf16, f64, make_step, normal, tensor, turned

pytestmark = pytest.mark.gpu

D = 128


@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("rot,interleaved", [(128, False), (64, True), (96, False)])
def test_positions(gpu, step, rot, interleaved):
    Hq, Hkv, bs, table_rows = 6, 2, 32, 500
    news, lens = STEPS[step]
    cu, T, table, num_blocks = make_step(news, lens, bs, seed=rot,
                                         pad_rows=3 if news is not None else 0)
    gen = torch.Generator().manual_seed(rot + T)
    q, k, v = normal(gen, T, Hq, D), normal(gen, T, Hkv, D, std=3.0), normal(gen, T, Hkv, D)
    cos_sin = kv_cache.rotary_table(table_rows, rot, device="cpu")
    pos = torch.randint(0, table_rows, (T,), generator=gen).int()
    pos[::5], pos[3::7] = table_rows, -1  # outside, on both sides
    want, want_scales = random_cache(num_blocks, Hkv, bs, T)
    cache, scales = (torch.from_numpy(x.copy()).to(gpu) for x in (want, want_scales))
    got = kv_cache.kv_append_fp8(q.to(gpu), k.to(gpu), v.to(gpu), cache, scales, table.to(gpu),
                                 tensor(lens, gpu), cos_sin.to(gpu), cu_seqlens=tensor(cu, gpu),
                                 positions=pos.to(gpu), interleaved=interleaved)
    where = kv.places(T, lens, cu)
    rows = kv.turn_rows(cos_sin.numpy(), pos.tolist())
    ref.append(want, want_scales, where, table.numpy(), turned(k, None, 0.0, rows, interleaved)[0],
               f64(v))
    check_bytes(cache, scales, want, want_scales)
    y, mag = turned(q, None, 0.0, rows, interleaved)
    live = np.array([p is not None for p in where])
    live = live[:, None, None]
    check_bf16(got, np.where(live, y, 0.0), np.where(live, mag, 0.0), "q")
