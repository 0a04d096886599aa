"""The paged caches around the decode attention: filling them, and holding them
in 4 bits.

A decode or prefill step hands its new rows to one call a layer, which norms
and turns them and puts the keys and values where the attention finds them:

    cos_sin = rotary_table(max_position, 128, base=1e6)          # once
    q = kv_append(q, k, v, k_cache, v_cache, block_table, seq_lens, cos_sin,
                  q_weight=q_norm, k_weight=k_norm)
    out = binding.gqa_decode_v2(q, k_cache, v_cache, block_table, seq_lens, scale, 0)

with a cache of 4-bit elements (136 bytes a token and kv-head for the bf16
caches' 512):

    cache = new_mxfp4_cache(num_blocks, block_size, Hkv)
    q = kv_append_mxfp4(q, k, v, cache, block_table, seq_lens, cos_sin)
    out = gqa_decode_mxfp4(q, cache, block_table, seq_lens, scale)

and for MLA (q_nope absorbed into the first 512 dims of q by the caller):

    mla_append(q_pe, c_kv, k_pe, kv_cache, block_table, seq_lens, cos_sin,
               c_weight=kv_norm, q_out=q[..., 512:])
    out, lse = mla.flash_mla_with_kvcache(q[:, None], kv_cache, block_table, seq_lens, 512)

Tokens. q, k, v hold T new rows in request order, and seq_lens counts them
already. Without cu_seqlens every request has one (T = B); with it (int32
[B + 1]) request b has rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1, the last of
them at position seq_lens[b] - 1. A row without a place -- at or past
cu_seqlens[B], or of a request with seq_lens[b] below its number of rows, as 0
for an unused entry of a fixed-size batch -- is padding: it writes nothing to a
cache and its row of the result is zeros. A position past the block table, or
a block id outside the cache, writes nothing either. A block that the call writes
to must stand once in its table rows: no other request's, and not twice in one.

Norm and rotation. q_weight / k_weight (bf16 or fp32 [128]) ask for
x / sqrt(mean(x^2) + eps) * weight over each head; cos_sin (rotary_table) turns the
first rotary_dim dims by the token's position, or by positions[t] (int32 [T])
where the rotation does not follow the cache; None leaves them as they are.
Pairs are dims (i, i + rotary_dim / 2), or (2i, 2i + 1) with interleaved=True.
A position outside the table gives NaN. Everything is rounded once.

q, k and v may be strided views (of one projection's output) with contiguous
dims. q_out takes the turned queries; it may be q itself. The operators run on
the current stream, allocate their result (and the attention its workspace)
from torch's allocator and can be captured into graphs. Rejected arguments
raise RuntimeError. There is no fallback: a missing build raises ImportError.
"""

import glob
import importlib.util
import math
import os

import torch

_LIB_DIR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lib")


def _load_extension():
    paths = sorted(glob.glob(os.path.join(_LIB_DIR, "kv_cache_ext*.so")))
    if not paths:
        raise ImportError(
            f"kv_cache_ext not built in {_LIB_DIR}; run "
            "`python mla-decode-kernels_amd/build.py` (or __graft_entry__.build())"
        )
    spec = importlib.util.spec_from_file_location("kv_cache_ext", paths[0])
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


_ext = _load_extension()
EXTENSION_PATH = _ext.__file__

# kv_append(q, k, v, k_cache, v_cache, block_table, seq_lens, cos_sin=None,
#           cu_seqlens=None, positions=None, q_weight=None, k_weight=None,
#           eps=1e-6, interleaved=False, q_out=None) -> q_out [T, Hq, 128]
kv_append = _ext.kv_append
# kv_append_mxfp4(q, k, v, kv_cache, block_table, seq_lens, ...the same)
kv_append_mxfp4 = _ext.kv_append_mxfp4
# kv_read_mxfp4(kv_cache, block_table, seq_lens, cu_seqlens=None, num_tokens=None)
#   -> (k, v) bf16 [num_tokens, Hkv, 128]: the rows an append with these
#   arguments writes. num_tokens (cu_seqlens' last entry, known on the host) goes
#   with cu_seqlens.
kv_read_mxfp4 = _ext.kv_read_mxfp4
# mla_append(q_pe [T, h_q, 64], c_kv [T, 512], k_pe [T, 64], kv_cache,
#            block_table, seq_lens, cos_sin, cu_seqlens=None, positions=None,
#            c_weight=None, eps=1e-6, interleaved=True, q_out=None) -> q_out
mla_append = _ext.mla_append
# gqa_decode_mxfp4(q [B, Hq, 128], kv_cache, block_table, seq_lens, scale,
#                  num_workgroups=0) -> out [B, Hq, 128]; a request of length 0
#   gets zeros. num_workgroups > 0 sets the token-balanced launch's grid; 0 chooses
#   launch and grid from the sizes, block_table's width among them, and the device.
gqa_decode_mxfp4 = _ext.gqa_decode_mxfp4

MXFP4_TILE_TOKENS = 16
MXFP4_TILE_BYTES = 2176


def new_mxfp4_cache(num_blocks, block_size, num_kv_heads, device="cuda"):
    """A 4-bit cache of zeros: uint8 [num_blocks, num_kv_heads, block_size / 16, 2176], whose
    bytes include/kv_cache.h lays out. block_size is a multiple of 16."""
    if block_size < 1 or block_size % MXFP4_TILE_TOKENS:
        raise ValueError("block_size must be a multiple of 16")
    if num_blocks < 0 or num_kv_heads < 1:
        raise ValueError("num_blocks must not be negative, num_kv_heads must be positive")
    return torch.zeros(num_blocks, num_kv_heads, block_size // MXFP4_TILE_TOKENS,
                       MXFP4_TILE_BYTES, dtype=torch.uint8, device=device)


def rotary_table(max_position, rotary_dim, base=10000.0, scaling=None, device="cuda"):
    """The rotation table of kv_append and mla_append: fp32 [max_position, rotary_dim], the
    cosines of position * frequency_i, then the sines, frequency_i = base^(-2i / rotary_dim).
    Computed in 64 bits and rounded once, so far positions keep their angles.

    scaling stretches it for contexts longer than the model was trained on; a dict with "type":
      "linear"  positions divided by "factor".
      "ntk"     base times factor^(rotary_dim / (rotary_dim - 2)): the slowest frequency is
                divided by "factor", the fastest kept.
      "llama3"  frequencies with a wavelength over original / low_freq_factor divided by
                "factor", those under original / high_freq_factor kept, a straight line in
                original / wavelength between ("original_max_position", "low_freq_factor" = 1,
                "high_freq_factor" = 4).
      "yarn"    frequencies that turn less than "beta_slow" (1) times in
                "original_max_position" divided by "factor", those that turn more than
                "beta_fast" (32) times kept, a line over the column between; cosines and
                sines times "attention_factor", 0.1 ln(factor) + 1 by default.
    """
    if max_position < 1:
        raise ValueError("max_position must be positive")
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    half = rotary_dim // 2
    col = torch.arange(half, dtype=torch.float64, device=device)
    inv = float(base) ** (-2.0 * col / rotary_dim)
    pos = torch.arange(max_position, dtype=torch.float64, device=device)
    gain = 1.0
    if scaling is not None:
        kind, factor = scaling["type"], float(scaling["factor"])
        if factor <= 0:
            raise ValueError("scaling factor must be positive")
        if kind == "linear":
            inv = inv / factor
        elif kind == "ntk":
            if rotary_dim == 2:
                raise ValueError("ntk scaling needs a rotary_dim over 2")
            stretched = float(base) * factor ** (rotary_dim / (rotary_dim - 2))
            inv = stretched ** (-2.0 * col / rotary_dim)
        elif kind == "llama3":
            original = float(scaling["original_max_position"])
            low = float(scaling.get("low_freq_factor", 1.0))
            high = float(scaling.get("high_freq_factor", 4.0))
            if high <= low:
                raise ValueError("high_freq_factor must be over low_freq_factor")
            turns = original * inv / (2.0 * math.pi)  # original / wavelength
            keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
            inv = inv * keep + inv / factor * (1.0 - keep)
        elif kind == "yarn":
            original = float(scaling["original_max_position"])
            fast = float(scaling.get("beta_fast", 32.0))
            slow = float(scaling.get("beta_slow", 1.0))

            def column(turns):  # the column that turns so often over the original length
                return (rotary_dim * math.log(original / (turns * 2.0 * math.pi))
                        / (2.0 * math.log(base)))

            first = max(math.floor(column(fast)), 0)
            last = min(math.ceil(column(slow)), rotary_dim - 1)
            drop = ((col - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
            inv = inv * (1.0 - drop) + inv / factor * drop
            gain = scaling.get("attention_factor")
            if gain is None:
                gain = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
        else:
            raise ValueError(f"unknown scaling type {kind!r}")
    angle = pos[:, None] * inv
    return torch.cat([torch.cos(angle) * gain, torch.sin(angle) * gain], dim=1).float()
