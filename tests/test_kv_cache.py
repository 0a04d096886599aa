"""GPU tests of the cache operators (kv_cache.py) against oracle/kv_reference.py
in 64 bits.

Tolerances, derived from the arithmetic:
  bf16 results of norm and rotation: half a bf16 step (2^-8 of the value) and
    the fp32 steps before it, for M = |a cos| + |b sin| (or |x|): a rounding
    for each product and the fma (2), and with a norm 12 for the sum of
    squares (halved by the root), 4 for mean, eps, root and quotient, 2 for the
    two factors: under 32 * 2^-24 M.
  codes of the 4-bit cache: none, they are the formula's (fp64 before the rounding).
  attention over it: half a bf16 step; the weights, each off by 2^-15 (their two
    bf16 parts are truncated), by 2^-22 (exponential) and by twice the score's
    error d, which is at most 256 * 2^-24 (sums of 128 products and 2 parts) +
    2^-21 (the queries' two e4m3 parts) of the sum of |q k scale|; numerator and
    denominator: twice that, of the sum of weight times |value|; and the fp32
    sums over n keys, n / 16 + 64 steps of 2^-23. A weight is relative to the
    largest, so one below fp32's smallest normal, 2^-126, may count as 0 (the
    exponential's result, the second bf16 part, its product): at most
    4 * 2^-126 of the largest |value| for each key, whatever the formula's own
    result (where one key takes all and holds a 0, that is what is left).
"""

import math

import numpy as np
import pytest
import torch

import binding
import kv_cache
import mla
from oracle import kv_reference as ref
from oracle import mla_reference
from oracle import reference as gqa_ref

pytestmark = pytest.mark.gpu

D = 128


def f64(t):
    return t.double().cpu().numpy()


def normal(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).bfloat16()


def make_step(news, lens, bs, *, pool_extra=3, width_extra=0, seed=0, pad_rows=0):
    """(cu_seqlens or None, T, block_table, num_blocks) of a step; table entries past a request
    are -1."""
    gen = torch.Generator().manual_seed(seed)
    blocks = [(max(n, 0) + bs - 1) // bs for n in lens]
    num_blocks = sum(blocks) + pool_extra
    ids = torch.randperm(num_blocks, generator=gen).int()
    table = torch.full((len(lens), max(1, max(blocks)) + width_extra), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = ids[at:at + n]
        at += n
    if news is None:
        return None, len(lens), table, num_blocks
    cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    return cu, int(cu[-1]) + pad_rows, table, num_blocks


def tensor(x, dev):
    return None if x is None else torch.as_tensor(np.asarray(x), dtype=torch.int32).to(dev)


def turned(x, weight, eps, rows, interleaved):
    """(value, M) of norm and rotation in 64 bits; rows None: no rotation."""
    y = ref.norm(f64(x), None if weight is None else f64(weight), eps)
    if rows is None:
        return y, np.abs(y)
    half = rows.shape[1] // 2
    plus = np.concatenate([np.abs(rows[:, :half]), -np.abs(rows[:, half:])], axis=1)
    # |a cos| + |b sin| of both: rotate the magnitudes with signs that add (second pair's too).
    m1 = ref.rotate(np.abs(y), plus, interleaved)
    m2 = ref.rotate(np.abs(y), np.abs(rows), interleaved)
    return ref.rotate(y, rows, interleaved), np.maximum(m1, m2)


def check_bf16(got, want, mag, label):
    got = f64(got)
    assert np.array_equal(np.isnan(got), np.isnan(want)), label
    tol = 2.0 ** -8 * np.abs(want) + 32 * 2.0 ** -24 * mag
    bad = ~(np.abs(got - want) <= tol) & ~np.isnan(want)
    assert not bad.any(), f"{label}: {bad.sum()} of {bad.size}, worst {np.nanmax(np.abs(got - want) / tol)}"


STEPS = {
    # new tokens a request (None: one each, without cu_seqlens), lengths after them
    "one": (None, [1]),
    "decode": (None, [1, 17, 16, 0, 300, 33]),
    "ragged": ([1, 5, 0, 37, 2, 16], [1, 5, 9, 100, 33, 16]),
    "prefill": ([131], [131]),
    "chunk": ([64, 3], [200, 67]),
    # A request shorter than its rows, one whose length is 0, one of negative length.
    "short": ([6, 4, 2], [4, 0, -3]),
}


@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("Hq,Hkv,bs,rot,interleaved,norm", [
    (32, 8, 16, 128, False, False), (8, 8, 64, 64, True, True), (5, 1, 48, 32, False, True),
    (6, 3, 16, 96, True, False), (2, 2, 32, 16, False, "q"), (7, 7, 16, 0, False, "k"),
    (12, 4, 16, 112, False, True)])
def test_append(gpu, step, mx, Hq, Hkv, bs, rot, interleaved, norm):
    news, lens = STEPS[step]
    pad_rows = 5 if news is not None else 0
    cu, T, table, num_blocks = make_step(news, lens, bs, seed=Hq, pad_rows=pad_rows)
    gen = torch.Generator().manual_seed(Hq * 100 + T)
    q, k, v = normal(gen, T, Hq, D), normal(gen, T, Hkv, D, std=3.0), normal(gen, T, Hkv, D)
    qw = (1 + 0.2 * torch.randn(D, generator=gen)).bfloat16() if norm in (True, "q") else None
    kw = 1 + 0.2 * torch.randn(D, generator=gen) if norm in (True, "k") else None  # fp32
    cos_sin = kv_cache.rotary_table(400, rot, device="cpu") if rot else None
    eps = 1e-5

    dv = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    args = [dv(q), dv(k), dv(v)]
    if mx:
        gen_bytes = np.random.default_rng(T).integers(0, 256, (num_blocks, Hkv, bs // 16, 2176))
        before = gen_bytes.astype(np.uint8)
        cache = torch.from_numpy(before.copy()).to(gpu)
        args += [cache]
    else:
        kc, vc = normal(gen, num_blocks, bs, Hkv, D), normal(gen, num_blocks, bs, Hkv, D)
        k_cache, v_cache = dv(kc), dv(vc)
        args += [k_cache, v_cache]
    fn = kv_cache.kv_append_mxfp4 if mx else kv_cache.kv_append
    got = fn(*args, dv(table), tensor(lens, gpu), dv(cos_sin), cu_seqlens=tensor(cu, gpu),
             q_weight=dv(qw), k_weight=dv(kw), eps=eps, interleaved=interleaved)

    where = ref.places(T, lens, cu)
    spots = ref.slots(where, table.numpy(), num_blocks, bs)
    rows = None
    if rot:
        rows = ref.turn_rows(cos_sin.numpy(), [0 if p is None else p[1] for p in where])
    eps32 = float(np.float32(eps))
    want_q, mag_q = turned(q, qw, eps32, rows, interleaved)
    want_k, mag_k = turned(k, kw, eps32, rows, interleaved)
    pad = np.array([p is None for p in where])
    want_q[pad], mag_q[pad] = 0.0, 0.0
    check_bf16(got, want_q, mag_q, "q")
    assert torch.equal(dv(q), args[0])  # the input stays
    live = [t for t in range(T) if spots[t] is not None]
    if mx:
        want = before
        for t in live:
            for h in range(Hkv):
                ref.mxfp4_store(want, *spots[t], h, want_k[t, h], f64(v[t, h]))
        assert np.array_equal(cache.cpu().numpy(), want)
        rk, rv = kv_cache.kv_read_mxfp4(cache, dv(table), tensor(lens, gpu), tensor(cu, gpu), T)
        for t in range(T):
            for h in range(Hkv):
                wk, wv = ((np.zeros(D), np.zeros(D)) if spots[t] is None
                          else ref.mxfp4_load(want, *spots[t], h))
                assert np.array_equal(f64(rk[t, h]), wk) and np.array_equal(f64(rv[t, h]), wv)
        return
    touched = torch.zeros(num_blocks, bs, dtype=torch.bool)
    for t in live:
        touched[spots[t]] = True
        check_bf16(k_cache[spots[t]], want_k[t], mag_k[t], "k")
        assert torch.equal(v_cache[spots[t]].cpu(), v[t])
    assert int(touched.sum()) == len(live)
    assert torch.equal(k_cache.cpu()[~touched], kc[~touched])
    assert torch.equal(v_cache.cpu()[~touched], vc[~touched])


def decode_inputs(gpu, T=9, Hq=8, Hkv=2, bs=16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    _, _, table, nb = make_step(None, [40] * T, bs, seed=seed)
    q, k, v = normal(gen, T, Hq, D), normal(gen, T, Hkv, D), normal(gen, T, Hkv, D)
    kc, vc = normal(gen, nb, bs, Hkv, D), normal(gen, nb, bs, Hkv, D)
    lens = torch.randint(1, 41, (T,), generator=gen, dtype=torch.int32)
    table_f = kv_cache.rotary_table(64, 128, device="cpu")
    return [t.to(gpu) for t in (q, k, v, kc, vc, table, lens, table_f)]


def test_append_strided_views_and_in_place(gpu):
    q, k, v, kc, vc, table, lens, cs = decode_inputs(gpu)
    T, Hq, Hkv = 9, 8, 2
    want_kc, want_vc = kc.clone(), vc.clone()
    want = kv_cache.kv_append(q, k, v, want_kc, want_vc, table, lens, cs)
    # Views of one projection, dims at odd offsets (2-byte aligned), heads before tokens.
    for layout in ("fused", "odd", "heads_first"):
        if layout == "heads_first":
            buf = torch.zeros(Hq + 2 * Hkv, T, D, dtype=torch.bfloat16, device=gpu).transpose(0, 1)
        else:
            w, off = (D, 0) if layout == "fused" else (D + 3, 1)
            buf = torch.zeros(T, Hq + 2 * Hkv, w, dtype=torch.bfloat16, device=gpu)[..., off:off + D]
        buf[:, :Hq], buf[:, Hq:Hq + Hkv], buf[:, Hq + Hkv:] = q, k, v
        views = [buf[:, :Hq], buf[:, Hq:Hq + Hkv], buf[:, Hq + Hkv:]]
        a, b = kc.clone(), vc.clone()
        got = kv_cache.kv_append(*views, a, b, table, lens, cs)
        assert torch.equal(got, want) and torch.equal(a, want_kc) and torch.equal(b, want_vc)
        a, b = kc.clone(), vc.clone()
        got = kv_cache.kv_append(*views, a, b, table, lens, cs, q_out=views[0])
        assert got.data_ptr() == views[0].data_ptr()
        assert torch.equal(views[0], want) and torch.equal(a, want_kc)
        assert torch.equal(views[1], k) and torch.equal(views[2], v)  # neighbours stay


def test_append_refuses_on_device(gpu):
    q, k, v, kc, vc, table, lens, cs = decode_inputs(gpu)
    good = dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, block_table=table, seq_lens=lens,
                cos_sin=cs)
    kv_cache.kv_append(**good)
    cu = torch.arange(10, dtype=torch.int32, device=gpu)
    qkv = torch.zeros(9, 12, D, dtype=torch.bfloat16, device=gpu)
    for over, match in [
            (dict(q=q.float()), "q must be bf16"), (dict(k=k[:-1], v=v[:-1]), "number of tokens"),
            (dict(v=v[:, :1]), "same shape"), (dict(q=q[..., :64]), "head dim 128"),
            (dict(q=q.transpose(1, 2)), "contiguous dims|head dim"),
            (dict(k_cache=kc[:, :, :1]), "contiguous"), (dict(v_cache=vc[1:]), "same shape"),
            (dict(k_cache=kc.float()), "must be bf16"),
            (dict(block_table=table.long()), "int32"), (dict(block_table=table[:3]), "batch dim"),
            (dict(seq_lens=lens[:3]), "batch dim"), (dict(seq_lens=lens[:3], block_table=table[:3]),
                                                     "one new token a request"),
            (dict(cu_seqlens=cu[:-1]), "B . 1"), (dict(cu_seqlens=cu.long()), "int32"),
            (dict(positions=lens[:-1]), "positions must be"),
            (dict(cos_sin=cs.bfloat16()), "fp32"), (dict(cos_sin=cs[:, :24].contiguous()), "multiple of 16"),
            (dict(cos_sin=cs[:0]), "at least one position"), (dict(cos_sin=cs[:, :64]), "contiguous"),
            (dict(q_weight=torch.ones(64, device=gpu)), "q_weight"),
            (dict(k_weight=torch.ones(128, device=gpu, dtype=torch.float16)), "bf16 or fp32"),
            (dict(q_out=torch.empty_like(q)[:, :4]), "q's shape"),
            (dict(k=kc.view(-1, 2, D)[:9]), "k and k_cache must not overlap"),
            (dict(q_out=kc.view(-1, 8, D)[:9]), "overlap"),
            (dict(q_out=q[:1].expand(9, -1, -1)), "overlap"),
            (dict(q=qkv[:, :8], k=qkv[:, 8:10], v=qkv[:, 10:], q_out=qkv[:, 4:]), "overlap"),
            (dict(v_cache=kc), "overlap")]:
        with pytest.raises(RuntimeError, match=match):
            kv_cache.kv_append(**{**good, **over})
    # The same token rows, heads apart: no overlap.
    wide = torch.zeros(9, 20, D, dtype=torch.bfloat16, device=gpu)
    kv_cache.kv_append(wide[:, :8], wide[:, 16:18], wide[:, 18:], kc, vc, table, lens, cs,
                       q_out=wide[:, 8:16])
    mx = kv_cache.new_mxfp4_cache(4, 16, 3)
    with pytest.raises(RuntimeError, match="number of heads"):
        kv_cache.kv_append_mxfp4(q, k, v, mx, table, lens, cs)
    with pytest.raises(RuntimeError, match="2176"):
        kv_cache.kv_read_mxfp4(mx[..., :2048].contiguous(), table, lens)
    with pytest.raises(RuntimeError, match="needs num_tokens"):
        kv_cache.kv_read_mxfp4(mx, table, lens, cu)
    with pytest.raises(RuntimeError, match="divisible"):
        kv_cache.gqa_decode_mxfp4(q, mx, table, lens, 0.1)
    with pytest.raises(RuntimeError, match="finite"):
        kv_cache.gqa_decode_mxfp4(q[:, :6].contiguous(), mx, table, lens, math.nan)


def test_append_positions(gpu):
    """positions turn rows, the cache's places stay; outside the table gives NaN."""
    q, k, v, kc, vc, table, lens, cs = decode_inputs(gpu)
    pos = torch.tensor([0, 63, 5, 64, -1, 2**31 - 1, 7, 63, 1], dtype=torch.int32, device=gpu)
    got = kv_cache.kv_append(q, k, v, kc, vc, table, lens, cs[:, :].contiguous(), positions=pos)
    rows = ref.turn_rows(cs.cpu().numpy(), pos.tolist())
    want, mag = turned(q.cpu(), None, 0, rows, False)
    check_bf16(got, want, mag, "q")
    want_k, mag_k = turned(k.cpu(), None, 0, rows, False)
    for t, n in enumerate(lens.tolist()):
        spot = (int(table[t, (n - 1) // 16]), (n - 1) % 16)
        check_bf16(kc[spot], want_k[t], mag_k[t], "k")
        assert torch.equal(vc[spot], v[t])


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mxfp4"])
def test_append_bad_pages_write_nothing(gpu, mx):
    """Ids outside the cache and positions past the table: nothing written, q turned all the
    same."""
    q, k, v, kc, vc, table, lens, cs = decode_inputs(gpu)
    good = kv_cache.kv_append(q, k, v, kc.clone(), vc.clone(), table, lens, cs)
    table = torch.tensor([-1, 10**6, 2**31 - 1, -2**31, kc.shape[0]], dtype=torch.int32,
                         device=gpu)[torch.arange(9, device=gpu) % 5][:, None].expand(-1, 3)
    lens2 = lens.clone()
    lens2[8] = 49  # past three blocks of 16
    cs2 = cs
    if mx:
        cache = torch.randint(0, 256, (4, 2, 1, 2176), device=gpu).to(torch.uint8)
        was = cache.clone()
        got = kv_cache.kv_append_mxfp4(q, k, v, cache, table.contiguous(), lens2, cs2)
        assert torch.equal(cache, was)
        rk, rv = kv_cache.kv_read_mxfp4(cache, table.contiguous(), lens2)
        assert not rk.any() and not rv.any()
    else:
        a, b = kc.clone(), vc.clone()
        got = kv_cache.kv_append(q, k, v, a, b, table.contiguous(), lens2, cs2)
        assert torch.equal(a, kc) and torch.equal(b, vc)
    assert torch.equal(got[:8], good[:8])


def test_append_special_values(gpu):
    """Infinities, NaN, the largest and the smallest values, zeros of both signs."""
    T, H = 8, 2
    x = torch.zeros(T, H, D, dtype=torch.bfloat16)
    big, small = torch.finfo(torch.bfloat16).max, 2.0 ** -133
    x[0, 0, 3], x[0, 1, 100] = math.inf, -math.inf
    x[1, 0, 40] = math.nan
    x[2, 0], x[2, 1] = big, -big
    x[3, 0], x[3, 1] = small, 2.0 ** -126
    x[4] = -0.0
    x[5, 0, ::2] = 7.0
    x[5, 1, ::2] = 7.0625  # the next bf16 value
    x[6, 0, 5] = 2.0 ** -124
    x[7] = torch.arange(D) * 0.25 - 16
    table = torch.arange(T, dtype=torch.int32)[:, None]
    lens = torch.full((T,), 4, dtype=torch.int32)
    cache = kv_cache.new_mxfp4_cache(T, 16, H)
    kv_cache.kv_append_mxfp4(x.to(gpu), x.to(gpu), x.flip(1).contiguous().to(gpu), cache,
                             table.to(gpu), lens.to(gpu))
    want = np.zeros((T, H, 1, 2176), dtype=np.uint8)
    for t in range(T):
        for h in range(H):
            ref.mxfp4_store(want, t, 3, h, f64(x[t, h]), f64(x[t, 1 - h]))
    assert np.array_equal(cache.cpu().numpy(), want)
    # The bf16 caches take all of them as they are.
    kc, vc = (torch.zeros(T, 16, H, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    q = kv_cache.kv_append(x.to(gpu), x.to(gpu), x.to(gpu), kc, vc, table.to(gpu), lens.to(gpu))
    for got in (q.cpu(), kc[:, 3].cpu(), vc[:, 3].cpu()):
        assert np.array_equal(got.float().numpy(), x.float().numpy(), equal_nan=True)


@pytest.mark.parametrize("Hq,Hkv,interleaved,rot", [(32, 8, False, 128), (7, 7, True, 64),
                                                    (64, 4, False, 96)])
def test_append_large_steps(gpu, Hq, Hkv, interleaved, rot):
    """A prefill large enough for waves that take several heads (and several passes, MLA) gives the
    bits of the same rows appended a few at a time, and what the oracle gives."""
    news, past, bs = [1, 1700, 0, 333, 967], [5, 0, 9, 40, 1], 16
    lens = [n + m for n, m in zip(news, past)]
    cu, T, table, nb = make_step(news, lens, bs, seed=3, pad_rows=9)
    gen = torch.Generator().manual_seed(Hq)
    q, k, v = (normal(gen, T, h, D).to(gpu) for h in (Hq, Hkv, Hkv))
    q_pe, c, k_pe = (normal(gen, T, *n).to(gpu) for n in ((20, 64), (512,), (64,)))
    w, wc = (torch.rand(n, generator=gen).to(gpu) + 0.5 for n in (D, 512))
    cs, cs64 = kv_cache.rotary_table(2000, rot), kv_cache.rotary_table(2000, 64)
    table_d = table.to(gpu)

    def caches():
        return (torch.zeros(nb, bs, Hkv, D, dtype=torch.bfloat16, device=gpu),
                torch.zeros(nb, bs, Hkv, D, dtype=torch.bfloat16, device=gpu),
                kv_cache.new_mxfp4_cache(nb, bs, Hkv),
                torch.zeros(nb, bs, 1, 576, dtype=torch.bfloat16, device=gpu))

    def step(t0, t1, cu_step, lens_step, to):
        how = dict(cu_seqlens=tensor(cu_step, gpu), interleaved=interleaved)
        L = tensor(lens_step, gpu)
        rows = [x[t0:t1] for x in (q, k, v)]
        norms = dict(q_weight=w, k_weight=w)
        return (kv_cache.kv_append(*rows, to[0], to[1], table_d, L, cs, **how, **norms),
                kv_cache.kv_append_mxfp4(*rows, to[2], table_d, L, cs, **how, **norms),
                kv_cache.mla_append(q_pe[t0:t1], c[t0:t1], k_pe[t0:t1], to[3], table_d, L, cs64,
                                    c_weight=wc, **how))

    one, few = caches(), caches()
    whole = step(0, T, cu, lens, one)
    parts = []
    for t0 in range(0, T, 100):
        t1 = min(t0 + 100, T)
        inside = [max(0, min(t1, cu[b + 1]) - max(t0, cu[b])) for b in range(5)]
        upto = [past[b] + max(0, min(t1, cu[b + 1]) - cu[b]) for b in range(5)]
        parts.append(step(t0, t1, np.concatenate([[0], np.cumsum(inside)]), upto, few))
    for a, b in zip(whole, zip(*parts)):
        assert torch.equal(a, torch.cat(b))
    for a, b in zip(one, few):
        assert torch.equal(a, b)
    where = ref.places(T, lens, cu)
    some = [0, 1, 1000, 1700, 1701, 2033, 2034, 3000, T - 9, T - 1]
    pos = [0 if where[t] is None else where[t][1] for t in some]
    want, mag = turned(q[some].cpu(), w.cpu(), float(np.float32(1e-6)),
                       ref.turn_rows(cs.cpu().numpy(), pos), interleaved)
    pad = np.array([where[t] is None for t in some])
    want[pad] = 0.0
    assert pad.tolist() == [False] * 8 + [True] * 2
    check_bf16(whole[0][some], want, mag, "q")
    assert torch.equal(whole[0], whole[1])


MLA_STEPS = ["one", "decode", "ragged", "prefill", "short"]


@pytest.mark.parametrize("step", MLA_STEPS)
@pytest.mark.parametrize("h_q,bs,interleaved,weight", [
    (16, 64, True, torch.bfloat16), (1, 16, False, None), (7, 1, True, torch.float32),
    (128, 64, False, torch.bfloat16), (8, 20, True, None)])
def test_mla_append(gpu, step, h_q, bs, interleaved, weight):
    news, lens = STEPS[step]
    cu, T, table, num_blocks = make_step(news, lens, bs, seed=h_q, pad_rows=3 if news else 0)
    gen = torch.Generator().manual_seed(h_q + T)
    q_full = normal(gen, T, h_q, 192).to(gpu)
    row = normal(gen, T, 576, std=2.0).to(gpu)
    absorbed = normal(gen, T, h_q, 576).to(gpu)
    cache = normal(gen, num_blocks, bs, 1, 576)
    w = None if weight is None else (1 + 0.2 * torch.randn(512, generator=gen)).to(weight)
    cs = kv_cache.rotary_table(400, 64, device="cpu")
    kept, before = absorbed.clone(), cache.clone()
    cache_d = cache.to(gpu)
    got = kv_cache.mla_append(q_full[..., 128:], row[:, :512], row[:, 512:], cache_d,
                              table.to(gpu), tensor(lens, gpu), cs.to(gpu),
                              cu_seqlens=tensor(cu, gpu),
                              c_weight=None if w is None else w.to(gpu), eps=1e-6,
                              interleaved=interleaved, q_out=absorbed[..., 512:])
    assert got.data_ptr() == absorbed[..., 512:].data_ptr()
    assert torch.equal(absorbed[..., :512], kept[..., :512])
    where = ref.places(T, lens, cu)
    spots = ref.slots(where, table.numpy(), num_blocks, bs)
    rows = ref.turn_rows(cs.numpy(), [0 if p is None else p[1] for p in where])
    want, mag = turned(q_full[..., 128:].cpu(), None, 0, rows, interleaved)
    pad = np.array([p is None for p in where])
    want[pad], mag[pad] = 0.0, 0.0
    check_bf16(got, want, mag, "q_pe")
    want_k, mag_k = turned(row[:, None, 512:].cpu(), None, 0, rows, interleaved)
    c = ref.norm(f64(row[:, :512]), None if w is None else f64(w), float(np.float32(1e-6)))
    touched = torch.zeros(num_blocks, bs, dtype=torch.bool)
    for t in range(T):
        if spots[t] is None:
            continue
        touched[spots[t]] = True
        check_bf16(cache_d[spots[t]][0, :512], c[t], np.abs(c[t]), "c")
        check_bf16(cache_d[spots[t]][0, 512:], want_k[t, 0], mag_k[t, 0], "k_pe")
    assert torch.equal(cache_d.cpu()[~touched], before[~touched])


def test_mla_append_new_and_in_place(gpu):
    gen = torch.Generator().manual_seed(0)
    q, c, k = (normal(gen, 4, *s).to(gpu) for s in ((16, 64), (512,), (64,)))
    table = torch.arange(4, dtype=torch.int32, device=gpu)[:, None]
    lens = torch.tensor([1, 2, 64, 0], dtype=torch.int32, device=gpu)
    cs = kv_cache.rotary_table(64, 64)
    caches = [torch.zeros(4, 64, 1, 576, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    fresh = kv_cache.mla_append(q, c, k, caches[0], table, lens, cs)
    assert fresh.shape == q.shape and not fresh[3].any()
    buf = q.clone()
    assert torch.equal(kv_cache.mla_append(buf, c, k, caches[1], table, lens, cs, q_out=buf), fresh)
    assert torch.equal(caches[0], caches[1])
    for over, match in [(dict(q_pe=q[..., :32]), "h_q, 64"), (dict(c_kv=c[:, :256]), "512"),
                        (dict(k_pe=k[:2]), "number of tokens"),
                        (dict(kv_cache=caches[0][..., :512].contiguous()), "576"),
                        (dict(cos_sin=cs[:, :32].contiguous()), "positions, 64"),
                        (dict(c_weight=torch.ones(64, device=gpu)), "c_weight")]:
        args = dict(q_pe=q, c_kv=c, k_pe=k, kv_cache=caches[0], block_table=table, seq_lens=lens,
                    cos_sin=cs)
        with pytest.raises(RuntimeError, match=match):
            kv_cache.mla_append(**{**args, **over})


# ------------------------------------------------ attention over the 4-bit cache


def filled_cache(gen, num_blocks, Hkv, bs, *, scales=(122, 130)):
    """Random codes, scales of magnitudes around 1."""
    rng = np.random.default_rng(int(torch.randint(1 << 30, (1,), generator=gen)))
    cache = rng.integers(0, 256, (num_blocks, Hkv, bs // 16, 2176), dtype=np.uint8)
    cache[..., 2048:] = rng.integers(*scales, (num_blocks, Hkv, bs // 16, 128), dtype=np.uint8)
    return cache


def poison(cache, table, lens, bs):
    """NaN scales in every slot that must not be read: blocks no request holds, slots behind
    each request's last token."""
    out = cache.copy()
    free = set(range(cache.shape[0])) - {int(i) for i in table.flatten().tolist()}
    for b in free:
        out[b, ..., 2048:] = 255
    for b, n in enumerate(lens):
        for t in range(max(n, 0), -(-max(n, 0) // bs) * bs):
            tile = out[int(table[b, t // bs]), :, t % bs // 16]
            r = t % 16
            tile[:, [2048 + g * 16 + r for g in range(4)]] = 255
            tile[:, [2112 + r // 4 * 16 + g * 4 + r % 4 for g in range(4)]] = 255
    return out


def largest_value(cache):
    """The largest magnitude of a value (scale 255, NaN, is never read)."""
    scales = cache[..., 2112:].astype(np.float64)
    return 6.0 * 2.0 ** (np.where(scales < 255, scales, 0).max() - 127.0)


def check_attention(got, q, cache, table, lens, scale, label=""):
    want, mass, reach, count = ref.mxfp4_attention(f64(q), cache, np.asarray(table), lens, scale)
    got = f64(got)
    assert np.isfinite(got).all(), label
    d = reach * (256 * 2.0 ** -24 + 2.0 ** -21)
    weights = 2 * (2.0 ** -15 + 2.0 ** -22 + 2 * d) + (count / 16 + 64) * 2.0 ** -23
    under = 4 * 2.0 ** -126 * count * largest_value(cache)
    tol = 2.0 ** -8 * np.abs(want) + weights[..., None] * mass + under[..., None]
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{label}: {bad.sum()} of {bad.size}, worst {np.nanmax(np.abs(got - want) / tol)}"


LENGTHS = {
    "one": [1], "edge": [16, 17, 31, 32, 33, 15], "empty": [0, 5, 0, 0, 64, -3],
    "short": [777, 100, 1], "ragged": [2500, 3, 1100, 0, 640, 65, 1, 1999], "long": [9001],
}


@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("Hq,Hkv,bs", [(32, 8, 16), (8, 2, 64), (2, 2, 32), (5, 1, 48), (12, 1, 16),
                                       (20, 1, 16), (32, 2, 64), (6, 3, 16), (40, 1, 16)])
def test_decode(gpu, lens, Hq, Hkv, bs):
    S = LENGTHS[lens]
    if lens in ("ragged", "long") and Hq * Hkv > 100:
        S = [min(n, 1200) for n in S]
    gen = torch.Generator().manual_seed(Hq + len(S))
    _, B, table, nb = make_step(None, S, bs, seed=1)
    cache = poison(filled_cache(gen, nb, Hkv, bs), table, S, bs)
    q = normal(gen, B, Hq, D)
    args = (q.to(gpu), torch.from_numpy(cache).to(gpu), table.to(gpu), tensor(S, gpu), D ** -0.5)
    auto = kv_cache.gqa_decode_mxfp4(*args)
    check_attention(auto, q, cache, table, S, D ** -0.5, "automatic")
    for nwg in (1, 3, 61, 256):
        got = kv_cache.gqa_decode_mxfp4(*args, num_workgroups=nwg)
        check_attention(got, q, cache, table, S, D ** -0.5, f"{nwg} workgroups")
        assert torch.equal(got, kv_cache.gqa_decode_mxfp4(*args, num_workgroups=nwg))


@pytest.mark.parametrize("B,longest,Hq,Hkv", [(70, 900, 32, 8), (1100, 40, 8, 2), (300, 200, 20, 1),
                                              (65, 1500, 4, 4), (513, 33, 1, 1), (250, 200, 8, 2)])
def test_decode_many_requests(gpu, B, longest, Hq, Hkv):
    """More requests than a wave has lanes, more than a workgroup has threads, more segments than
    there are CUs: whole segments dealt out, and balanced shares; every seventh request empty."""
    gen = torch.Generator().manual_seed(B)
    S = torch.randint(1, longest + 1, (B,), generator=gen)
    S[::7] = 0
    S[-1], S[5] = longest, -1
    S = S.tolist()
    _, _, table, nb = make_step(None, S, 16, seed=B)
    cache = poison(filled_cache(gen, nb, Hkv, 16), table, S, 16)
    q = normal(gen, B, Hq, D)
    args = (q.to(gpu), torch.from_numpy(cache).to(gpu), table.to(gpu), tensor(S, gpu), 0.1)
    for nwg in (0, 256, 5):
        got = kv_cache.gqa_decode_mxfp4(*args, num_workgroups=nwg)
        check_attention(got, q, cache, table, S, 0.1, f"{nwg} workgroups")
        assert torch.equal(got, kv_cache.gqa_decode_mxfp4(*args, num_workgroups=nwg))


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0, 1e-30, 25.0])
def test_decode_scales(gpu, scale):
    """No softmax at all (0), the smallest key first (negative), one key taking all (large)."""
    S, Hkv, bs = [200, 33], 2, 16
    gen = torch.Generator().manual_seed(3)
    _, B, table, nb = make_step(None, S, bs)
    cache = filled_cache(gen, nb, Hkv, bs)
    q = normal(gen, B, 8, D)
    q[0, 1] = 0.0
    q[0, 2] *= 2.0 ** -60
    q[1, 3, ::2] *= 2.0 ** -20
    got = kv_cache.gqa_decode_mxfp4(q.to(gpu), torch.from_numpy(cache).to(gpu), table.to(gpu),
                                    tensor(S, gpu), scale)
    check_attention(got, q, cache, table, S, scale)


def test_decode_bad_pages_are_left_out(gpu):
    """Blocks outside the cache, in front, between and behind, and requests of nothing else."""
    S, Hkv, bs = [100, 64, 33, 200, 16], 2, 16
    gen = torch.Generator().manual_seed(4)
    _, B, table, nb = make_step(None, S, bs, seed=2)
    table[0, 0], table[0, 3] = -1, nb
    table[1, :] = 2**31 - 1
    table[2, 2] = -2**31
    table[3, 1:9] = -7
    cache = filled_cache(gen, nb, Hkv, bs)
    q = normal(gen, B, 8, D)
    for nwg in (0, 1, 40):
        got = kv_cache.gqa_decode_mxfp4(q.to(gpu), torch.from_numpy(cache).to(gpu), table.to(gpu),
                                        tensor(S, gpu), 0.1, num_workgroups=nwg)
        check_attention(got, q, cache, table, S, 0.1, nwg)
        assert not got[1].any()
    # No cache at all, and lengths past the table (cut to it).
    none = kv_cache.gqa_decode_mxfp4(q.to(gpu), kv_cache.new_mxfp4_cache(0, bs, Hkv),
                                     table.to(gpu), tensor(S, gpu), 0.1)
    assert not none.any()
    good = kv_cache.gqa_decode_mxfp4(q.to(gpu), torch.from_numpy(cache).to(gpu), table.to(gpu),
                                     tensor([10**6] * B, gpu), 0.1)
    check_attention(good, q, cache, table, [10**6] * B, 0.1)


def test_decode_nan_and_infinite_keys_stay_in_their_head(gpu):
    S, Hkv, bs = [40, 40], 2, 16
    gen = torch.Generator().manual_seed(5)
    _, B, table, nb = make_step(None, S, bs, seed=2)
    cache = filled_cache(gen, nb, Hkv, bs)
    cache[int(table[0, 1]), 1, 0, 2048 + 5] = 255  # a key of request 0, kv-head 1
    q = normal(gen, B, 8, D)
    got = kv_cache.gqa_decode_mxfp4(q.to(gpu), torch.from_numpy(cache).to(gpu), table.to(gpu),
                                    tensor(S, gpu), 0.1)
    assert torch.isnan(got[0, 4:]).all()
    got[0, 4:] = 0
    assert torch.isfinite(got).all()


def test_decode_queries_that_are_not_finite(gpu):
    """An infinity or NaN in a query gives its head NaN, and no other head."""
    S, Hkv, bs = [40, 70], 2, 16
    gen = torch.Generator().manual_seed(11)
    _, B, table, nb = make_step(None, S, bs, seed=2)
    cache = filled_cache(gen, nb, Hkv, bs)
    for Hq in (8, 24):
        q = normal(gen, B, Hq, D)
        q[0, 1, 77], q[1, 0, 3], q[1, Hq - 1, 127] = math.nan, math.inf, -math.inf
        got = kv_cache.gqa_decode_mxfp4(q.to(gpu), torch.from_numpy(cache).to(gpu), table.to(gpu),
                                        tensor(S, gpu), 0.1)
        bad = torch.zeros(B, Hq, dtype=torch.bool, device=gpu)
        bad[0, 1] = bad[1, 0] = bad[1, Hq - 1] = True
        assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()


def test_read_every_code_and_scale(gpu):
    """All 16 codes under all 256 scale bytes: the nearest bf16 (the value itself but for the
    overflow of the two largest scales), NaN under 255."""
    rng = np.random.default_rng(12)
    cache = rng.integers(0, 256, (32, 1, 1, 2176), dtype=np.uint8)
    cache[..., 2048:] = rng.permutation(np.tile(np.arange(256, dtype=np.uint8), 16)).reshape(32, 1, 1,
                                                                                         128)
    k, v = kv_cache.kv_read_mxfp4(torch.from_numpy(cache).to(gpu),
                                  torch.arange(32, dtype=torch.int32, device=gpu)[None],
                                  tensor([512], gpu), tensor([0, 512], gpu), 512)
    want = ref.mxfp4_rows(cache, np.arange(32), 512, 0)
    for got, w in zip((k, v), want):
        w = torch.from_numpy(w).float().bfloat16().float().numpy()
        assert np.array_equal(got[:, 0].float().cpu().numpy(), w, equal_nan=True)


def test_nothing_to_do(gpu):
    """No tokens, no requests, no blocks: every call returns, and what it returns is empty or
    zeros."""
    q, k, v, kc, vc, table, lens, cs = decode_inputs(gpu)
    mx = kv_cache.new_mxfp4_cache(3, 16, 2)
    none = [t[:0] for t in (q, k, v)]
    cu = torch.zeros(10, dtype=torch.int32, device=gpu)
    was = kc.clone()
    for args in ((table[:0], lens[:0], cs), (table, lens, cs, cu)):
        assert kv_cache.kv_append(*none, kc, vc, *args).shape == (0, 8, D)
        assert kv_cache.kv_append_mxfp4(*none, mx, *args).shape == (0, 8, D)
    assert torch.equal(kc, was) and not mx.any()
    # Rows with no request at all are padding.
    assert not kv_cache.kv_append(q, k, v, kc, vc, table[:0], lens[:0], cs, cu[:1]).any()
    assert torch.equal(kc, was)
    # Caches without blocks take nothing; the queries turn all the same.
    want = kv_cache.kv_append(q, k, v, kc, vc, table, lens, cs)
    assert torch.equal(kv_cache.kv_append(q, k, v, kc[:0], vc[:0], table, lens, cs), want)
    assert torch.equal(kv_cache.kv_append_mxfp4(q, k, v, mx[:0], table, lens, cs), want)
    rows = kv_cache.kv_read_mxfp4(mx[:0], table, lens)
    assert rows[0].shape == (9, 2, D) and not rows[0].any() and not rows[1].any()
    assert kv_cache.kv_read_mxfp4(mx, table[:0], lens[:0])[0].shape == (0, 2, D)
    assert kv_cache.kv_read_mxfp4(mx, table, lens, cu, 0)[1].shape == (0, 2, D)
    pe, c = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=gpu), q.new_zeros(0, 512)
    cache = torch.zeros(2, 64, 1, 576, dtype=torch.bfloat16, device=gpu)
    assert kv_cache.mla_append(pe, c, q.new_zeros(0, 64), cache, table[:0], lens[:0],
                               cs[:, :64].contiguous()).shape == (0, 4, 64)


def test_misaligned_caches_are_refused(gpu):
    q, k, v, kc, vc, table, lens, cs = decode_inputs(gpu)
    odd = torch.zeros(kc.numel() + 1, dtype=torch.bfloat16, device=gpu)[1:].view(kc.shape)
    with pytest.raises(RuntimeError, match="k_cache must be 16-byte aligned"):
        kv_cache.kv_append(q, k, v, odd, vc, table, lens, cs)
    mx = torch.zeros(4 * 2 * 2176 + 4, dtype=torch.uint8, device=gpu)[4:].view(4, 2, 1, 2176)
    for call in (lambda: kv_cache.kv_append_mxfp4(q, k, v, mx, table, lens, cs),
                 lambda: kv_cache.kv_read_mxfp4(mx, table, lens),
                 lambda: kv_cache.gqa_decode_mxfp4(q, mx, table, lens, 0.1)):
        with pytest.raises(RuntimeError, match="kv_cache must be 16-byte aligned"):
            call()


def test_decode_empty_batch_and_unaligned_q(gpu):
    cache = kv_cache.new_mxfp4_cache(4, 16, 2)
    out = kv_cache.gqa_decode_mxfp4(torch.zeros(0, 8, D, dtype=torch.bfloat16, device=gpu), cache,
                                    torch.zeros(0, 3, dtype=torch.int32, device=gpu),
                                    torch.zeros(0, dtype=torch.int32, device=gpu), 0.1)
    assert out.shape == (0, 8, D)
    gen = torch.Generator().manual_seed(6)
    c = torch.from_numpy(filled_cache(gen, 4, 2, 16)).to(gpu)
    table = torch.tensor([[2, 1]], dtype=torch.int32, device=gpu)
    lens = torch.tensor([30], dtype=torch.int32, device=gpu)
    flat = normal(gen, 8 * D + 1).to(gpu)
    q = flat[1:].view(1, 8, D)
    assert torch.equal(kv_cache.gqa_decode_mxfp4(q, c, table, lens, 0.1),
                       kv_cache.gqa_decode_mxfp4(q.clone(), c, table, lens, 0.1))


def test_offsets_past_32_bits(gpu):
    """Blocks at the far end of caches of more than 4 GiB give what small caches give."""
    Hkv, bs, far = 8, 16, 300000
    q, k, v, kc, vc, table, lens, cs = decode_inputs(gpu, Hq=32, Hkv=Hkv, bs=bs)
    nb = kc.shape[0]
    small = torch.zeros(nb, Hkv, 1, 2176, dtype=torch.uint8, device=gpu)
    big = torch.empty(far + nb, Hkv, 1, 2176, dtype=torch.uint8, device=gpu)
    big[far:] = 0
    assert big.numel() > 2**32
    tokens = [40] * 9
    cu = tensor(np.arange(10) * 40, gpu)
    gen = torch.Generator().manual_seed(7)
    rows = [normal(gen, 360, h, D).to(gpu) for h in (32, Hkv, Hkv)]
    outs = []
    for cache, shift in ((small, 0), (big, far)):
        t = torch.where(table >= 0, table + shift, table)
        qo = kv_cache.kv_append_mxfp4(*rows, cache, t, tensor(tokens, gpu), cs, cu_seqlens=cu)
        out = kv_cache.gqa_decode_mxfp4(q, cache, t, tensor(tokens, gpu), 0.1)
        outs.append((qo, out, *kv_cache.kv_read_mxfp4(cache, t, tensor(tokens, gpu), cu, 360)))
    assert torch.equal(small, big[far:])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    del big
    far = 140000
    big_k = torch.empty(far + nb, bs, Hkv, D, dtype=torch.bfloat16, device=gpu)
    big_v = torch.empty(far + nb, bs, Hkv, D, dtype=torch.bfloat16, device=gpu)
    assert big_k.numel() * 2 > 2**32
    big_k[far:], big_v[far:] = kc, vc
    kv_cache.kv_append(q, k, v, big_k, big_v, table + far, lens, cs)
    kv_cache.kv_append(q, k, v, kc, vc, table, lens, cs)
    assert torch.equal(big_k[far:], kc) and torch.equal(big_v[far:], vc)


# ---------------------------------------------------------- used together


def test_decode_steps_together(gpu):
    """A prompt, then ten steps of a ragged batch with an unused entry: append and attend, over
    the bf16 caches (the framework's attention) and the 4-bit cache, each against attention in
    64 bits on rows kept beside them."""
    Hq, Hkv, bs, cap = 16, 4, 16, 6
    prompts = [30, 1, 0, 77]
    B, gen = len(prompts), torch.Generator().manual_seed(8)
    nb = B * cap
    table = torch.randperm(nb, generator=gen).int().view(B, cap).to(gpu)
    cs = kv_cache.rotary_table(bs * cap, 128, base=5e5,
                               scaling={"type": "yarn", "factor": 4.0, "original_max_position": 32})
    qw, kw = (normal(gen, D).abs().to(gpu) for _ in range(2))
    kc, vc = (torch.full((nb, bs, Hkv, D), math.nan, dtype=torch.bfloat16, device=gpu)
              for _ in range(2))
    cache = torch.full((nb, Hkv, bs // 16, 2176), 255, dtype=torch.uint8, device=gpu)
    lens = list(prompts)
    for step in range(11):
        news = prompts if step == 0 else [1 if n else 0 for n in prompts]
        if step > 0:
            lens = [n + m for n, m in zip(lens, news)]
        T = sum(news) if step == 0 else B
        cu = np.concatenate([[0], np.cumsum(news)]) if step == 0 else None
        q, k, v = (normal(gen, T, h, D).to(gpu) for h in (Hq, Hkv, Hkv))
        L = tensor(lens, gpu)
        how = dict(cu_seqlens=tensor(cu, gpu), q_weight=qw, k_weight=kw)
        q1 = kv_cache.kv_append(q, k, v, kc, vc, table, L, cs, **how)
        q2 = kv_cache.kv_append_mxfp4(q, k, v, cache, table, L, cs, **how)
        assert torch.equal(q1, q2)
        if step == 0:
            continue
        live = [b for b in range(B) if lens[b]]
        out1 = binding.gqa_decode_v2(q1, kc, vc, table, L, D ** -0.5, 0)
        out2 = kv_cache.gqa_decode_mxfp4(q1, cache, table, L, D ** -0.5)
        host = [t.float().cpu().numpy() for t in (q1, kc, vc)]
        want = gqa_ref.attention_ref(*host, table.cpu().numpy(), lens, D ** -0.5, batches=live)
        assert np.allclose(out1.float().cpu().numpy()[live], want[live], atol=1e-2, rtol=1e-2)
        check_attention(out2, q1, cache.cpu().numpy(), table.cpu(), lens, D ** -0.5)
        assert not out2[2].any() and not q1[2].any()
    # The 4-bit rows are the 4-bit form of the bf16 ones (turned in 64 bits): near them.
    rk, rv = kv_cache.kv_read_mxfp4(cache, table, tensor(lens, gpu),
                                    tensor(np.concatenate([[0], np.cumsum(lens)]), gpu), sum(lens))
    ids = torch.cat([table[b, torch.arange(n, device=gpu) // bs].long() for b, n in enumerate(lens)])
    at = torch.cat([torch.arange(n, device=gpu) % bs for n in lens])
    for got, rows in ((rk, kc[ids, at]), (rv, vc[ids, at])):
        x = f64(rows).reshape(-1, Hkv, 4, 32)
        top = np.abs(x).max(-1, keepdims=True)
        # Half the widest step (2, of magnitudes up to 7 times the scale, over 3.5), and a bf16
        # step that moves a value over a border.
        err = np.abs(f64(got).reshape(x.shape) - x)
        assert (err <= top * (1 / 3.5 + 2.0 ** -7)).all()


def test_mla_steps_together(gpu):
    """Prompts and steps through mla_append and the framework's MLA attention."""
    h_q, bs, cap, prompts = 16, 64, 2, [70, 3]
    gen = torch.Generator().manual_seed(9)
    B = len(prompts)
    table = torch.randperm(B * cap, generator=gen).int().view(B, cap).to(gpu)
    cache = torch.full((B * cap, bs, 1, 576), math.nan, dtype=torch.bfloat16, device=gpu)
    cs = kv_cache.rotary_table(bs * cap, 64)
    w = (1 + 0.1 * torch.randn(512, generator=gen)).bfloat16().to(gpu)
    lens = list(prompts)
    for step in range(4):
        T = sum(prompts) if step == 0 else B
        cu = tensor([0, prompts[0], T], gpu) if step == 0 else None
        lens = lens if step == 0 else [n + 1 for n in lens]
        q = normal(gen, T, h_q, 576).to(gpu)
        row = normal(gen, T, 576).to(gpu)
        q_pe = normal(gen, T, h_q, 64).to(gpu)
        kv_cache.mla_append(q_pe, row[:, :512], row[:, 512:], cache, table, tensor(lens, gpu), cs,
                            cu_seqlens=cu, c_weight=w, q_out=q[..., 512:])
        if step == 0:
            continue
        out, lse = mla.flash_mla_with_kvcache(q[:, None], cache, table, tensor(lens, gpu), 512)
        bits = lambda t: t.contiguous().cpu().view(torch.int16).numpy().view(np.uint16)  # noqa: E731
        want, want_l = mla_reference.mla_decode_ref(bits(q[:, None]), bits(cache),
                                                    table.cpu().numpy(), lens, 576 ** -0.5)
        assert np.allclose(out.float().cpu().numpy(), want, atol=2e-2, rtol=2e-2)
        assert np.allclose(lse.cpu().numpy(), want_l, atol=5e-3)


def test_graph_replays(gpu):
    """append, read and both launches of the attention in one captured graph, replayed over
    changed inputs and lengths with eager work between, each replay against the eager result."""
    Hq, Hkv, bs, cap, B = 16, 2, 16, 100, 6
    gen = torch.Generator().manual_seed(10)
    table = torch.randperm(B * cap, generator=gen).int().view(B, cap).to(gpu)
    cs = kv_cache.rotary_table(bs * cap, 128)
    filled = torch.from_numpy(filled_cache(gen, B * cap, Hkv, bs)).to(gpu)
    cache = filled.clone()
    q, k, v = (torch.zeros(B, h, D, dtype=torch.bfloat16, device=gpu) for h in (Hq, Hkv, Hkv))
    lens = torch.ones(B, dtype=torch.int32, device=gpu)

    def step(c, nwg):
        qo = kv_cache.kv_append_mxfp4(q, k, v, c, table, lens, cs)
        rows = kv_cache.kv_read_mxfp4(c, table, lens)
        return (qo, *rows, kv_cache.gqa_decode_mxfp4(qo, c, table, lens, 0.1, nwg))

    side = torch.cuda.Stream()
    for nwg in (0, 50):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(filled.clone(), nwg)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(cache, nwg)
        for i in range(4):
            for t in (q, k, v):
                t.copy_(normal(gen, *t.shape))
            lens.copy_(torch.randint(0, bs * cap + 1, (B,), generator=gen, dtype=torch.int32))
            cache.copy_(filled)
            eager = filled.clone()
            want = step(eager, nwg)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(cache, eager)
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_another_stream(gpu):
    """Operators run on the current stream: after work queued there, beside another stream's."""
    q, k, v, kc, vc, table, lens, cs = decode_inputs(gpu, T=9)
    mx = kv_cache.new_mxfp4_cache(kc.shape[0], 16, 2)
    want = kv_cache.kv_append_mxfp4(q, k, v, mx, table, lens, cs)
    want_out = kv_cache.gqa_decode_mxfp4(want, mx, table, lens, 0.1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            c = torch.zeros_like(mx)
            late = torch.zeros_like(q)
            torch.cuda._sleep(2000000)
            late.copy_(q)
            for _ in range(20):
                a = kv_cache.kv_append_mxfp4(late, k, v, c, table, lens, cs)
                o = kv_cache.gqa_decode_mxfp4(a, c, table, lens, 0.1, num_workgroups=7)
            results.append((a, o, c))
    torch.cuda.synchronize()
    seven = kv_cache.gqa_decode_mxfp4(want, mx, table, lens, 0.1, num_workgroups=7)
    for a, o, c in results:
        assert torch.equal(a, want) and torch.equal(c, mx) and torch.equal(o, seven)
    check_attention(want_out, want, mx.cpu().numpy(), table.cpu(), lens.tolist(), 0.1)
