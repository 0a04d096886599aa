"""GPU tests of the cache operators' appends at the edges of what their documentation
allows, against oracle/kv_reference.py in 64 bits (tolerances: tests/test_kv_cache.py)."""

import numpy as np
import pytest
import torch

import kv_cache
from oracle import kv_reference as ref

pytestmark = pytest.mark.gpu

D = 128


def f64(t):
    return t.double().cpu().numpy()


def check_rows(got, want, mag):
    """Half a bf16 step (of the smallest normal one below those) and 32 steps of fp32."""
    tol = np.maximum(2.0 ** -8 * np.abs(want), 2.0 ** -134) + 32 * 2.0 ** -24 * mag
    got = f64(got)
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size}"


def far_rows(gen, *shape):
    """Rows of very different magnitudes: token t's values around 2^far[t]."""
    x = torch.randn(*shape, generator=gen).clamp(-3.9, 3.9).double()
    far = [125, 100, 64, 63, 62, 30, 0, -30, -50, -60, -62, -64, -80, -100, -118]
    for t in range(shape[0]):
        x[t] *= 2.0 ** far[t % len(far)]
    return x.float().bfloat16()


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6, 2.0])
@pytest.mark.parametrize("T,Hq,Hkv,rot", [(15, 8, 2, 128), (15, 5, 3, 64), (1020, 32, 8, 0)])
def test_norm_of_very_large_and_small_rows(gpu, T, Hq, Hkv, rot, eps):
    """Squares past fp32's range on either side."""
    gen = torch.Generator().manual_seed(T + Hq)
    q, k, v = (far_rows(gen, T, h, D) for h in (Hq, Hkv, Hkv))
    w = 1 + 0.2 * torch.randn(D, generator=gen)
    nb = -(-T // 16)
    table = torch.arange(nb, dtype=torch.int32)[None]
    lens, cu = torch.tensor([T], dtype=torch.int32), torch.tensor([0, T], dtype=torch.int32)
    cs = kv_cache.rotary_table(T, rot, device="cpu") if rot else None
    dv = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    kc, vc = (torch.zeros(nb, 16, Hkv, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    mx = kv_cache.new_mxfp4_cache(nb, 16, Hkv)
    how = dict(cu_seqlens=dv(cu), q_weight=dv(w), k_weight=dv(w), eps=eps)
    got = kv_cache.kv_append(dv(q), dv(k), dv(v), kc, vc, dv(table), dv(lens), dv(cs), **how)
    got4 = kv_cache.kv_append_mxfp4(dv(q), dv(k), dv(v), mx, dv(table), dv(lens), dv(cs), **how)
    eps32 = float(np.float32(eps))
    for rows, out in ((q, got), (q, got4), (k, kc.view(-1, Hkv, D)[:T])):
        y = ref.norm(f64(rows), w.numpy(), eps32)
        mag = np.abs(y)
        if rot:
            y = ref.rotate(y, cs.numpy(), False)
            mag = mag.max(axis=-1, keepdims=True) * 2
        check_rows(out, y, mag)


@pytest.mark.parametrize("eps", [0.0, 1e-6, 2.0])
def test_mla_norm_of_very_large_and_small_rows(gpu, eps):
    gen = torch.Generator().manual_seed(4)
    T = 30
    c = far_rows(gen, T, 512)
    q, k = (torch.zeros(T, *s, dtype=torch.bfloat16, device=gpu) for s in ((3, 64), (64,)))
    w = 1 + 0.2 * torch.randn(512, generator=gen)
    cache = torch.zeros(2, 16, 1, 576, dtype=torch.bfloat16, device=gpu)
    index = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    kv_cache.mla_append(q, c.to(gpu), k, cache, index([[0, 1]]), index([T]),
                        kv_cache.rotary_table(T, 64), cu_seqlens=index([0, T]),
                        c_weight=w.to(gpu), eps=eps)
    want = ref.norm(f64(c), w.numpy(), float(np.float32(eps)))
    check_rows(cache.view(-1, 576)[:T, :512], want, np.abs(want))


def step(gpu, T, Hq=8, Hkv=2):
    gen = torch.Generator().manual_seed(T)
    return [torch.randn(T, h, D, generator=gen).bfloat16().to(gpu) for h in (Hq, Hkv, Hkv)]


def test_rows_without_any_request(gpu):
    """No request (index tensors made empty, without memory) but rows: all of them padding."""
    q, k, v = step(gpu, 5)
    table = torch.empty(0, 3, dtype=torch.int32, device=gpu)
    lens = torch.empty(0, dtype=torch.int32, device=gpu)
    cu = torch.zeros(1, dtype=torch.int32, device=gpu)
    assert table.data_ptr() == 0 and lens.data_ptr() == 0
    kc, vc = (torch.ones(3, 16, 2, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    mx = torch.ones(3, 2, 1, 2176, dtype=torch.uint8, device=gpu)
    mla = torch.ones(3, 16, 1, 576, dtype=torch.bfloat16, device=gpu)
    cs, cs64 = kv_cache.rotary_table(4, 128), kv_cache.rotary_table(4, 64)
    outs = [kv_cache.kv_append(q, k, v, kc, vc, table, lens, cs, cu),
            kv_cache.kv_append_mxfp4(q, k, v, mx, table, lens, cs, cu),
            kv_cache.mla_append(q[..., :64], q.view(5, -1)[:, :512], k[:, 0, :64], mla, table, lens,
                                cs64, cu),
            *kv_cache.kv_read_mxfp4(mx, table, lens, cu, 5)]
    for out in outs:
        assert out.shape[0] == 5 and not out.any()
    for cache in (kc, vc, mx, mla):
        assert (cache == 1).all()


def test_strides_of_single_tokens_and_heads_do_not_matter(gpu):
    """q itself as q_out through another view of the same rows: a dimension of size 1 may have any
    stride."""
    table = torch.zeros(1, 1, dtype=torch.int32, device=gpu)
    one = torch.ones(1, dtype=torch.int32, device=gpu)
    cs, cs64 = kv_cache.rotary_table(4, 128), kv_cache.rotary_table(4, 64)
    kc, vc = (torch.zeros(1, 16, 2, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    q, k, v = step(gpu, 1)
    want = kv_cache.kv_append(q, k, v, kc, vc, table, one, cs)
    qkv = torch.cat([q, k, v], dim=1)
    view = qkv[:, :8]
    same = view.as_strided((1, 8, D), (8 * D, D, 1))
    assert view.stride() != same.stride()
    kv_cache.kv_append(view, qkv[:, 8:10], qkv[:, 10:], kc, vc, table, one, cs, q_out=same)
    assert torch.equal(view, want) and torch.equal(qkv[:, 8:10], k)
    # One head: its stride may be anything as well.
    T = 3
    tables = torch.arange(T, dtype=torch.int32, device=gpu)[:, None]
    lens = torch.ones(T, dtype=torch.int32, device=gpu)
    row = torch.randn(T, 640, generator=torch.Generator().manual_seed(0)).bfloat16().to(gpu)
    cache = torch.zeros(T, 16, 1, 576, dtype=torch.bfloat16, device=gpu)
    q1 = row[:, 576:].as_strided((T, 1, 64), (640, 64, 1), 576)
    q2 = row[:, 576:].as_strided((T, 1, 64), (640, 1, 1), 576)
    args = (row[:, :512], row[:, 512:576], cache, tables, lens, cs64)
    want = kv_cache.mla_append(q1, *args)
    kv_cache.mla_append(q1, *args, q_out=q2)
    assert torch.equal(q1, want)
    # Rows that do overlap are still refused.
    with pytest.raises(RuntimeError, match="overlap"):
        kv_cache.kv_append(view, k, v, kc, vc, table, one, cs,
                           q_out=qkv.as_strided((1, 8, D), (8 * D, D, 1), D))
