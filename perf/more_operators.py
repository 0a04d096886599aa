"""Performance cases of prompt attention and of the 8-bit cache, one call (or the
two or three calls that go together) per layer.

  prefill   prefill.gqa_prefill: causal attention of a step's new tokens (whole
            prompts, chunks of them, drafted tokens) over the paged bf16 cache;
  packed    prefill.gqa_prefill_packed: the same over rows [T, kv_heads, 128],
            as one projection gives them, without a cache;
  chunk8    kv_cache.kv_read_fp8 and prefill.gqa_prefill_packed: a chunk of each
            prompt over all that the 8-bit cache holds of it;
  append8   kv_cache.kv_append_fp8: norm, position rotation and the append of a
            step to the 8-bit cache, followed by kv_cache.kv_read_fp8, which hands
            back as bf16 the rows of the 16-token blocks that the step wrote to;
  decode8   kv_cache.gqa_decode_fp8: single-token attention over the 8-bit cache.

The 8-bit cache holds e4m3 codes, bytes [num_blocks, kv_heads, block_size / 16,
4096], tiles of 16 tokens of one head: 2048 bytes of keys (by 16-dim half of each
32-dim group, then group, then token, 16 dims), 2048 of values (by 4-dim half of
each 8 dims, then group of 4 tokens, then 8 dims, then 4 dims of 4 tokens each).
scales [num_blocks, kv_heads, block_size / 16, 2] has a byte e, standing for
2^(e - 127), for a tile's keys and one for its values: the least from 10 to 246
under which the largest magnitude is at most 448, and no less than before if the
tile has older tokens; those are rounded again if it grows.
"""

import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda"
D = 128
TILE, TILE_BYTES = 16, 4096  # tokens and bytes of a tile of the 8-bit cache
EPS = 1e-6


def _ops():
    """The framework's operators."""
    path = os.path.join(os.getcwd(), "mla-decode-kernels_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kv_cache
    import prefill
    return kv_cache, prefill


# ---------------------------------------------------------------- the cases


def _step(name, op, B, new, past, Hq, Hkv, block, lens="ragged"):
    """B requests with up to `past` cached tokens take up to `new` tokens each."""
    return {"name": name, "op": op, "B": B, "new": new, "past": past, "Hq": Hq, "Hkv": Hkv,
            "block": block, "lens": lens}


def _append(name, B, new, past, Hq, Hkv, block, rot=D, interleaved=False, norm=False):
    return {**_step(name, "append8", B, new, past, Hq, Hkv, block), "rot": rot,
            "interleaved": interleaved, "norm": norm}


def _decode(name, B, S, Hq, Hkv, block, lens="uniform"):
    return _step(name, "decode8", B, 1, S - 1, Hq, Hkv, block, lens)


def listed():
    return [
        # One user's short prompt: latency counts.
        _step("prefill_b1_s100", "prefill", 1, 100, 0, 32, 8, 16, "uniform"),
        # Drafted tokens of a batch, verified over long contexts: few rows, a long axis.
        _step("prefill_drafts_h64", "prefill", 16, 5, 16000, 64, 8, 64),
        # A step of continuous batching: prompts and chunks of all lengths behind cached prefixes.
        _step("prefill_ragged", "prefill", 13, 2000, 3001, 32, 8, 16),
        # One long document.
        _step("prefill_b1_s16384", "prefill", 1, 16384, 0, 32, 8, 64, "uniform"),
        # A batch of prompts straight from the projection (scoring, embedding: nothing is cached).
        _step("packed_b32_h64", "packed", 32, 1000, 0, 64, 8, 16),
        # A chunk of each of a few long prompts over what the 8-bit cache holds.
        _step("chunk8_b4", "chunk8", 4, 1024, 7001, 32, 8, 16),
        # A decode batch into the 8-bit cache: tiles that are partly filled.
        _append("append8_b128", 128, 1, 8191, 32, 8, 16),
        # A prefill step into the 8-bit cache, norms and all.
        _append("append8_prefill", 7, 1500, 2000, 32, 8, 64, norm=True),
        # One user, a short prompt: the smallest attention call.
        _decode("decode8_b1_s512", 1, 512, 32, 8, 16),
        # A large batch of short chats of an odd length.
        _decode("decode8_b128_s777", 128, 777, 32, 8, 16),
        # The representative batch.
        _decode("decode8_b32_s8192", 32, 8192, 32, 8, 16),
        # Continuous batching over the whole range of lengths, wide groups.
        _decode("decode8_b64_ragged_h64", 64, 32768, 64, 8, 64, "ragged"),
    ]


# Drawn cases stay under the largest listed ones (decode: tokens; append: new tokens; the
# others: rows times visible keys), in the units of _size.
_MOST = {"prefill": 4.3e9, "packed": 4.3e9, "chunk8": 4.3e9, "append8": 6500, "decode8": 1000000}
_HEADS = [(32, 8), (64, 8), (32, 8), (16, 8), (40, 8), (8, 8), (128, 8), (16, 4), (64, 16)]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["prefill", "prefill", "packed", "chunk8", "append8", "decode8", "decode8"])
        Hq, Hkv = rng.choice(_HEADS)
        block = rng.choice([16, 16, 32, 64])
        lens = rng.choice(["uniform", "ragged"])
        if op == "decode8":
            case = _decode("", _log_int(rng, 1, 64), _log_int(rng, 100, 32768), Hq, Hkv, block, lens)
        elif op == "append8":
            case = _append("", _log_int(rng, 1, 200), rng.choice([1, _log_int(rng, 2, 2000)]),
                           _log_int(rng, 1, 16384), Hq, Hkv, block, rng.choice([128, 128, 64, 32]),
                           rng.random() < 0.4, rng.random() < 0.5)
        else:
            B, new = _log_int(rng, 1, 64), _log_int(rng, 1, 12000)
            past = 0 if op == "packed" else rng.choice([0, _log_int(rng, 1, 16384)])
            if op == "packed":
                new = max(new, 40)
            case = _step("", op, B, new, past, Hq, Hkv, block, lens)
        del case["name"]
        if _size(case) <= _MOST[op] and sum(_lengths(case)[0]) * Hkv <= 8 * 1100000:
            return case


def _size(case):
    lens, news = _lengths(case)
    if case["op"] == "decode8":
        return sum(lens) * case["Hkv"] / 8 * max(1.0, case["Hq"] / case["Hkv"] / 8)
    if case["op"] == "append8":
        return sum(news) * (case["Hq"] + 2 * case["Hkv"]) / 48
    return _pairs(lens, news) * case["Hq"]


def _pairs(lens, news):
    """The (row, visible key) pairs of a head."""
    return float(sum(n * (L - n) + n * (n + 1) // 2 for L, n in zip(lens, news)))


def _lengths(case):
    """Each request's length with its new tokens, and the number of those: the same for every
    seed."""
    B, new, past = case["B"], case["new"], case["past"]
    r = random.Random(B * 1000003 + new * 1009 + past)
    if case["lens"] == "uniform":
        return [past + new] * B, [new] * B
    news = [1 if new == 1 else r.randint(1, new) for _ in range(B)]
    return [n + r.randint(0, past) for n in news], news


def _tile_rows(lens, news):
    """For each request the rows from the start of the first tile that its new tokens touch."""
    return [L - (L - n) // TILE * TILE for L, n in zip(lens, news)]


def work(case):
    lens, news = _lengths(case)
    B, T, total = case["B"], float(sum(news)), float(sum(lens))
    Hq, Hkv = case["Hq"], case["Hkv"]
    blocks = sum((n + case["block"] - 1) // case["block"] for n in lens)
    row, row8 = 2.0 * D, D + 1.0 / TILE  # bytes of a key or value
    if case["op"] == "append8":
        back = float(sum(_tile_rows(lens, news)))
        moved = T * ((2 * Hq + 2 * Hkv) * row + case["rot"] * 4.0) + 4.0 * (2 * B + 1 + T)
        moved += 2 * Hkv * (T * row8 + back * (row8 + row))
        turned = T * (Hq + Hkv)
        return {"bytes": moved + (4.0 * D if case["norm"] else 0.0),
                "flops": turned * (3.0 * case["rot"] + (4.0 * D if case["norm"] else 0.0))}
    rows = T * Hq * 2 * row + 4.0 * (2 * B + 2)
    if case["op"] == "decode8":
        return {"bytes": rows + total * Hkv * 2 * row8 + 4.0 * blocks, "flops": 4.0 * D * Hq * total}
    held = total * Hkv * 2 * (row8 if case["op"] == "chunk8" else row)
    return {"bytes": rows + held + (0.0 if case["op"] == "packed" else 4.0 * blocks),
            "flops": 4.0 * D * Hq * _pairs(lens, news)}


# ---------------------------------------------------------------- the inputs


def _pages(case, lens, cpu):
    """A shuffled block table over a pool of 1.25 times the blocks in use; -1 past each request."""
    blocks = [(n + case["block"] - 1) // case["block"] for n in lens]
    pool = sum(blocks) + (sum(blocks) + 3) // 4
    ids = torch.randperm(pool, generator=cpu).to(torch.int32)
    table = torch.full((case["B"], max(blocks)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, pool


def _angles(positions, rot):
    """The rotation table [positions, rot]: cosines, then sines, base 10000; computed in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEVICE) / rot)
    a = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * inv
    return torch.cat([torch.cos(a), torch.sin(a)], dim=1).float()


def _filled8(pool, case, gen):
    """An 8-bit cache whose every tile holds 16 keys and values: N(0, 1), with a few key channels
    many times as large, as trained models have them, and tiles of different magnitudes."""
    Hkv, bs = case["Hkv"], case["block"]
    tiles = bs // TILE
    cache = torch.empty(pool, Hkv, tiles, TILE_BYTES, dtype=torch.uint8, device=DEVICE)
    scales = torch.empty(pool, Hkv, tiles, 2, dtype=torch.uint8, device=DEVICE)
    loud = 1.0 + 7.0 * (torch.rand(Hkv, 1, 1, D, device=DEVICE, generator=gen) < 0.03)
    step = max(1, (1 << 16) // bs)
    for at in range(0, pool, step):
        n = min(step, pool - at)
        x = torch.empty(2, n, Hkv, tiles, TILE, D, device=DEVICE).normal_(generator=gen)
        x[0] *= loud
        x *= 0.5 + torch.rand(2, n, Hkv, tiles, 1, 1, device=DEVICE, generator=gen)
        for i in (0, 1):
            e = _scale8(x[i].abs().amax((-1, -2)))
            code = _to_codes(x[i], e[..., None, None])
            cache[at:at + n, ..., 2048 * i:2048 * (i + 1)] = _tile_bytes(code, i)
            scales[at:at + n, ..., i] = e
    return cache, scales


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    lens, news = _lengths(case)
    order = torch.randperm(case["B"], generator=cpu).tolist()
    lens, news = [lens[i] for i in order], [news[i] for i in order]
    table, pool = _pages(case, lens, cpu)
    bs, T, op = case["block"], sum(news), case["op"]
    Hq, Hkv = case["Hq"], case["Hkv"]

    def normal(*shape):
        return torch.empty(*shape, dtype=torch.bfloat16, device=DEVICE).normal_(generator=gen)

    def index(x):
        return torch.tensor(x, dtype=torch.int32, device=DEVICE)

    def sums(counts):
        at = [0]
        for n in counts:
            at.append(at[-1] + n)
        return index(at)

    s = {"case": case, "lens_list": lens, "news_list": news, "table": table.to(DEVICE),
         "lens": index(lens), "first": sums(news)}
    if op == "append8" and case["new"] == 1:
        s["first"] = None
    # One projection's output, cut into views.
    if op in ("packed", "append8"):
        qkv = normal(T, Hq + 2 * Hkv, D)
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    else:
        s["q"] = normal(T, Hq, D)
    if op == "prefill":
        s["k_cache"], s["v_cache"] = normal(pool, bs, Hkv, D), normal(pool, bs, Hkv, D)
    if op in ("chunk8", "decode8", "append8"):
        s["cache"], s["scales"] = _filled8(pool, case, gen)
    if op == "chunk8":
        s["whole"] = sums(lens)
    if op == "append8":
        s["back"] = sums(_tile_rows(lens, news))
        s["cos_sin"] = _angles(max(lens), case["rot"])
        s["q_weight"] = (1.0 + 0.1 * normal(D)).bfloat16() if case["norm"] else None
        s["k_weight"] = (1.0 + 0.1 * normal(D)).bfloat16() if case["norm"] else None
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ---------------------------------------------------------- the plain forms


def _times2(x, e):
    """x 2^e, the power made from its bits (pow's may be off by a last place)."""
    return x * ((e.long() + 1023) << 52).view(torch.float64).to(x.dtype)


def _scale8(top):
    """The scale byte for a largest magnitude."""
    m, e = torch.frexp(top)  # top = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0, e - 9 + (m > 0.875), torch.full_like(e, -117)).clamp(-117, 119)
    return (e + 127).to(torch.uint8)


def _to_codes(x, scale):
    """x -> the nearest e4m3 codes of x / 2^(scale - 127), ties to the even code."""
    y = _times2(x, 127 - scale.int()).abs().clamp(max=448.0)
    # y's last place: 3 bits behind the first, 2^-9 at least; n of them, 0 .. 16.
    step = torch.where(y < 2.0 ** -6, -9, torch.frexp(y)[1] - 4)
    n = torch.round(_times2(y, -step)).int()
    # Exponent field and mantissa in one number: from n = 8 on, n 2^step is (step + 10, n - 8).
    code = ((step + 9) * 8 + n).to(torch.uint8)
    return code | (torch.signbit(x).to(torch.uint8) << 7)


def _values8(codes, scale):
    """The values that codes and scale bytes stand for, fp32."""
    c = codes.int() & 127
    e, m = c >> 3, (c & 7).float()
    y = torch.where(e > 0, _times2(8.0 + m, e - 10), m * 2.0 ** -9)
    y = torch.where(codes > 127, -y, y)
    return _times2(y, scale.int() - 127)


def _tile_bytes(code, values):
    """Codes [.., 16 tokens, 128] as a tile's 2048 bytes, keys or values."""
    if values:
        # token 4g + t, dim 8c + 4j + d -> [j, g, c, d, t]
        c = code.unflatten(-1, (16, 2, 4)).unflatten(-4, (4, 4))  # [.., g, t, c, j, d]
        return c.movedim(-2, -5).movedim(-3, -1).flatten(-5)
    c = code.unflatten(-1, (4, 2, 16))                            # [.., token, g, j, d]
    return c.movedim(-4, -2).movedim(-3, -4).flatten(-4)


def _tile_codes(data, values):
    """A tile's 2048 bytes as codes [.., 16 tokens, 128]."""
    if values:
        c = data.unflatten(-1, (2, 4, 16, 4, 4))  # [.., j, g, c, d, t]
        return c.movedim(-1, -3).movedim(-5, -2).flatten(-5, -4).flatten(-3)
    c = data.unflatten(-1, (2, 4, 16, 16))        # [.., j, g, token, d]
    return c.movedim(-2, -4).movedim(-3, -2).flatten(-3)


def _places(s):
    """Each new token's request and position."""
    lens = s["lens"].long()
    if s["first"] is None:
        return torch.arange(lens.numel(), device=lens.device), lens - 1
    first = s["first"].long()
    t = torch.arange(s["q"].shape[0], device=lens.device)
    b = (t[:, None] >= first[1:]).sum(1)
    return b, lens[b] - first[b + 1] + t


def _normed(x, weight):
    if weight is None:
        return x
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(x.dtype)


def _rotated(x, cos_sin, interleaved):
    """x [T, heads, dims] with its first dims turned by the tokens' angles [T, rot]."""
    rot = cos_sin.shape[1]
    h = rot // 2
    cos, sin = cos_sin[:, None, :h].to(x.dtype), cos_sin[:, None, h:].to(x.dtype)
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([y, x[..., rot:]], dim=-1)


def _plain_append(s):
    case, bs = s["case"], s["case"]["block"]
    inter = case["interleaved"]
    b, pos = _places(s)
    turn = s["cos_sin"][pos]
    q = _rotated(_normed(s["q"].float(), s["q_weight"]), turn, inter).bfloat16()
    # In 64 bits: a key next to a border between two codes takes the nearer.
    k = _rotated(_normed(s["k"].double(), s["k_weight"]), turn, inter)
    # The tiles that the step touches, in order: rows of tokens of a tile each, in fp64.
    width = s["table"].shape[1] * (bs // TILE)
    tiles, row = torch.unique(b * width + pos // TILE, return_inverse=True)
    rb, rt = tiles // width, tiles % width
    block, tile = s["table"][rb, rt // (bs // TILE)].long(), rt % (bs // TILE)
    start = torch.full_like(tiles, TILE).scatter_reduce(0, row, pos % TILE, "amin")
    for i, x in ((0, k), (1, s["v"].double())):
        new = x.new_zeros(tiles.numel(), TILE, case["Hkv"], D)
        new[row, pos % TILE] = x
        new = new.transpose(1, 2)                                # [tiles, Hkv, 16, 128]
        here = torch.zeros(tiles.numel(), TILE, dtype=torch.bool, device=x.device)
        here[row, pos % TILE] = True
        old_e = s["scales"][block, :, tile, i]                   # [tiles, Hkv]
        need = _scale8(new.abs().amax((-1, -2)))
        e = torch.where(start[:, None] > 0, torch.maximum(need, old_e), need)
        data = s["cache"][block, :, tile, 2048 * i:2048 * (i + 1)]
        codes = _tile_codes(data, i)
        again = _to_codes(_values8(codes, old_e[..., None, None]), e[..., None, None])
        older = torch.arange(TILE, device=x.device)[None, :] < start[:, None]
        codes = torch.where(older[:, None, :, None], again, codes)
        codes = torch.where(here[:, None, :, None], _to_codes(new, e[..., None, None]), codes)
        s["cache"][block, :, tile, 2048 * i:2048 * (i + 1)] = _tile_bytes(codes, i)
        s["scales"][block, :, tile, i] = e
    return (q, *_plain_read(s, _tile_rows(s["lens_list"], s["news_list"])))


def _plain_read(s, rows):
    """The last rows[b] keys and values of each request, bf16 [sum(rows), Hkv, 128]."""
    bs, dev = s["case"]["block"], s["table"].device
    n = torch.tensor(rows, device=dev)
    b = torch.arange(len(rows), device=dev).repeat_interleave(n)
    pos = s["lens"].long()[b] - n.cumsum(0)[b] + torch.arange(sum(rows), device=dev)
    block, slot = s["table"][b, pos // bs].long(), pos % bs
    out = []
    for i in (0, 1):
        t = slot % TILE
        if i:
            d = torch.arange(D, device=dev)
            at = d // 4 % 2 * 1024 + (t // 4)[:, None] * 256 + d // 8 * 16 + d % 4 * 4 + t[:, None] % 4
        else:
            d = torch.arange(D, device=dev)
            at = d // 16 % 2 * 1024 + d // 32 * 256 + t[:, None] * 16 + d % 16
        heads = torch.arange(s["case"]["Hkv"], device=dev)[None, :, None]
        where = (block[:, None, None], heads, (slot // TILE)[:, None, None])
        codes = s["cache"][(*where, 2048 * i + at[:, None])]
        out.append(_values8(codes, s["scales"][(*where, torch.full_like(where[0], i))]).bfloat16())
    return out


def _plain_attend(q, k, v, n):
    """One request: q [n, Hq, 128] at its end, k and v [L, Hkv, 128] -> fp32 [n, Hq, 128]."""
    L, Hkv, Hq = k.shape[0], k.shape[1], q.shape[1]
    kt = k.float().permute(1, 2, 0).contiguous()                 # [Hkv, 128, L]
    vt = v.float().transpose(0, 1).contiguous()                  # [Hkv, L, 128]
    out = []
    step = max(1, (1 << 28) // (Hq * L))
    for at in range(0, n, step):
        m = min(step, n - at)
        seen = L - n + at + m                                    # keys that the last row sees
        x = q[at:at + m].float().unflatten(1, (Hkv, -1)).permute(1, 0, 2, 3).flatten(1, 2)
        sc = torch.matmul(x, kt[..., :seen]) * D ** -0.5         # [Hkv, m * group, seen]
        sc = sc.unflatten(1, (m, -1))
        row = torch.arange(m, device=q.device)[:, None]
        dead = torch.arange(seen, device=q.device)[None, :] > L - n + at + row
        sc = sc.masked_fill(dead[None, :, None, :], -math.inf)
        p = torch.exp(sc - sc.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = torch.matmul(p.flatten(1, 2), vt[:, :seen])          # [Hkv, m * group, 128]
        out.append(o.unflatten(1, (m, -1)).permute(1, 0, 2, 3).flatten(1, 2))
    return torch.cat(out)


def _requests(s):
    """Each request's number, first row, new tokens and length."""
    at = 0
    for b, (L, n) in enumerate(zip(s["lens_list"], s["news_list"])):
        yield b, at, n, L
        at += n


def _plain_attention(s):
    case, out = s["case"], []
    if case["op"] == "chunk8":
        rows = _plain_read(s, s["lens_list"])
        ends = [0]
        for n in s["lens_list"]:
            ends.append(ends[-1] + n)
    for b, at, n, L in _requests(s):
        if case["op"] == "packed":
            k, v = s["k"][at:at + n], s["v"][at:at + n]
        elif case["op"] == "chunk8":
            k, v = (x[ends[b]:ends[b + 1]] for x in rows)
        else:
            ids = s["table"][b, :(L + case["block"] - 1) // case["block"]].long()
            k, v = (c[ids].flatten(0, 1)[:L] for c in (s["k_cache"], s["v_cache"]))
        out.append(_plain_attend(s["q"][at:at + n], k, v, n).bfloat16())
    return torch.cat(out)


def _plain_decode(s):
    case, q, lens = s["case"], s["q"], s["lens"].long()
    ids = s["table"].clamp(min=0).long()
    tiles = s["cache"][ids].transpose(1, 2).flatten(2, 3)        # [B, Hkv, all tiles, bytes]
    e = s["scales"][ids].transpose(1, 2).flatten(2, 3)
    S = tiles.shape[2] * TILE
    dead = torch.arange(S, device=q.device)[None, :] >= lens[:, None]
    qt = q.float().unflatten(1, (case["Hkv"], -1)).transpose(2, 3).contiguous()
    k = _values8(_tile_codes(tiles[..., :2048], 0), e[..., 0, None, None]).flatten(2, 3)
    sc = torch.matmul(k, qt) * D ** -0.5                         # [B, Hkv, S, group]
    del k
    sc = sc.masked_fill(dead[:, None, :, None], -math.inf)
    p = torch.exp(sc - sc.amax(2, keepdim=True))
    p = (p / p.sum(2, keepdim=True)).transpose(2, 3).contiguous()
    v = _values8(_tile_codes(tiles[..., 2048:], 1), e[..., 1, None, None]).flatten(2, 3)
    v = v.masked_fill(dead[:, None, :, None], 0.0)
    return torch.matmul(p, v).flatten(1, 2).bfloat16()


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        if op == "decode8":
            return _plain_decode(s)
        return _plain_append(s) if op == "append8" else _plain_attention(s)
    kv, prefill = _ops()
    if op == "decode8":
        return kv.gqa_decode_fp8(s["q"], s["cache"], s["scales"], s["table"], s["lens"], D ** -0.5)
    if op == "prefill":
        return prefill.gqa_prefill(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                   D ** -0.5, cu_seqlens=s["first"])
    if op == "packed":
        return prefill.gqa_prefill_packed(s["q"], s["k"], s["v"], s["first"], s["first"], D ** -0.5)
    if op == "chunk8":
        k, v = kv.kv_read_fp8(s["cache"], s["scales"], s["table"], s["lens"],
                              cu_seqlens=s["whole"], num_tokens=sum(s["lens_list"]))
        return prefill.gqa_prefill_packed(s["q"], k, v, s["first"], s["whole"], D ** -0.5)
    q = kv.kv_append_fp8(s["q"], s["k"], s["v"], s["cache"], s["scales"], s["table"], s["lens"],
                         s["cos_sin"], cu_seqlens=s["first"], q_weight=s["q_weight"],
                         k_weight=s["k_weight"], eps=EPS, interleaved=s["case"]["interleaved"])
    k, v = kv.kv_read_fp8(s["cache"], s["scales"], s["table"], s["lens"], cu_seqlens=s["back"],
                          num_tokens=sum(_tile_rows(s["lens_list"], s["news_list"])))
    return q, k, v


# ------------------------------------------------------------ in 64 bits


def _grid8():
    """The values of the codes 0 .. 126: the e4m3 numbers up to 448."""
    low = [m * 2.0 ** -9 for m in range(8)]
    return torch.tensor(low + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:119],
                        dtype=torch.float64, device=DEVICE)


def _power(e):
    """2^e for whole numbers e, from a table."""
    table = torch.tensor([2.0 ** i for i in range(-150, 151)], dtype=torch.float64, device=DEVICE)
    return table[e.long() + 150]


def _round8(x, scale):
    """x rounded to scale times the e4m3 numbers: the nearer of the two around it."""
    grid = _grid8()
    y = (x / scale).abs().clamp(max=448.0).contiguous()
    hi = torch.searchsorted(grid, y).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    d = (y - grid[lo]) - (grid[hi] - y)
    up = (d > 0) | ((d == 0) & (hi % 2 == 0))
    return torch.copysign(torch.where(up, grid[hi], grid[lo]), x) * scale


def _least8(top):
    """The least power of two under which `top` is at most 448."""
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -120) / 448.0))
    e = torch.where(top > 448.0 * _power(e), e + 1, e)  # (log2 next to a whole number)
    e = torch.where(top <= 224.0 * _power(e), e - 1, e)
    return _power(e.clamp(-117, 119))


def _held8(s, b, L):
    """The values that the cache holds of a request's first L tokens: [2, Hkv, L, 128], and the
    scales [2, Hkv, tiles]; picked out byte by byte."""
    grid = torch.cat([_grid8(), torch.full((1,), math.nan, dtype=torch.float64, device=DEVICE)])
    ids = s["table"][b, :(L + s["case"]["block"] - 1) // s["case"]["block"]].long()
    tiles = s["cache"][ids].transpose(0, 1).flatten(1, 2)        # [Hkv, tiles, bytes]
    e = _power(s["scales"][ids].transpose(0, 1).flatten(1, 2).int() - 127)
    t, d = torch.arange(TILE, device=DEVICE)[:, None], torch.arange(D, device=DEVICE)
    at = (d // 16 % 2 * 1024 + d // 32 * 256 + t * 16 + d % 16,
          2048 + d // 4 % 2 * 1024 + t // 4 * 256 + d // 8 * 16 + d % 4 * 4 + t % 4)
    out = []
    for i in (0, 1):
        c = tiles[..., at[i]].long()                             # [Hkv, tiles, 16, 128]
        x = torch.where(c > 127, -grid[c & 127], grid[c & 127]) * e[..., i, None, None]
        out.append(x.flatten(1, 2)[:, :L])
    return torch.stack(out), e.movedim(-1, 0)


def _attend64(q, k, v, n):
    """q [n, Hq, 128] at the end of k, v [Hkv, L, 128], head by head and in pieces of rows."""
    Hkv, L = k.shape[:2]
    G = q.shape[1] // Hkv
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    pos = torch.arange(L - n, L, device=q.device)
    key = torch.arange(L, device=q.device)
    for h in range(Hkv):
        kt = k[h].double().t().contiguous()
        for at in range(0, n, 2048):
            p = pos[at:at + 2048]
            x = q[at:at + 2048, h * G:(h + 1) * G].double().transpose(0, 1)   # [G, m, 128]
            sc = torch.matmul(x, kt) * D ** -0.5
            sc = torch.where(key[None, :] <= p[:, None], sc, -math.inf)
            o = torch.matmul(torch.softmax(sc, dim=-1), v[h].double())
            out[at:at + 2048, h * G:(h + 1) * G] = o.transpose(0, 1)
    return out


def _turn64(x, cos_sin, interleaved):
    """The rotation as a product of complex numbers."""
    x = x.double()
    rot = cos_sin.shape[-1]
    w = torch.complex(cos_sin[:, :rot // 2].double(), cos_sin[:, rot // 2:].double())[:, None]
    head, tail = x[..., :rot], x[..., rot:]
    pair = (head.unflatten(-1, (rot // 2, 2)) if interleaved
            else torch.stack([head[..., :rot // 2], head[..., rot // 2:]], dim=-1))
    y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * w)
    y = y.flatten(-2) if interleaved else torch.cat([y[..., 0], y[..., 1]], dim=-1)
    return torch.cat([y, tail], dim=-1)


def _norm64(x, weight):
    x = x.double()
    if weight is None:
        return x
    return x * torch.rsqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()


def _append64(s):
    """Request by request, tile by tile: what the cache holds afterwards of the touched tiles."""
    case = s["case"]
    qs, rows = [], []
    for b, at, n, L in _requests(s):
        turn = s["cos_sin"][L - n:L]
        qs.append(_turn64(_norm64(s["q"][at:at + n], s["q_weight"]), turn, case["interleaved"]))
        k = _turn64(_norm64(s["k"][at:at + n], s["k_weight"]), turn, case["interleaved"])
        first = (L - n) // TILE
        old, e = _held8(s, b, L)
        got = torch.stack([k, s["v"][at:at + n].double()]).transpose(1, 2)     # [2, Hkv, n, 128]
        for t in range(first, (L - 1) // TILE + 1):
            lo, hi = max(t * TILE, L - n), min((t + 1) * TILE, L)
            x = got[:, :, lo - (L - n):hi - (L - n)]
            scale = _least8(x.abs().amax((-1, -2)))                            # [2, Hkv]
            if lo > t * TILE:
                scale = torch.maximum(scale, e[..., t])
                x = torch.cat([old[:, :, t * TILE:lo], x], dim=2)
            rows.append(_round8(x, scale[..., None, None]).transpose(1, 2))    # [2, rows, Hkv, 128]
    rows = torch.cat(rows, dim=1)
    return torch.cat(qs), rows[0], rows[1]


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "append8":
        return _append64(s)
    out = []
    for b, at, n, L in _requests(s):
        if op == "packed":
            k, v = s["k"][at:at + n].transpose(0, 1), s["v"][at:at + n].transpose(0, 1)
        elif op == "prefill":
            ids = s["table"][b].long()[torch.arange(L, device=DEVICE) // case["block"]]
            slot = torch.arange(L, device=DEVICE) % case["block"]
            k, v = (c[ids, slot].transpose(0, 1) for c in (s["k_cache"], s["v_cache"]))
        else:
            k, v = _held8(s, b, L)[0]
        out.append(_attend64(s["q"][at:at + n], k, v, n))
    return torch.cat(out)
