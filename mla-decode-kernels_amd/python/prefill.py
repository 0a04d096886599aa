"""Attention of many new tokens a request: whole prompts, chunks of them behind a
cached prefix, drafted tokens. (Single tokens: binding.py.)

A prefill step appends its rows and attends over the cache they went to:

    q = kv_cache.kv_append(q, k, v, k_cache, v_cache, block_table, seq_lens, cos_sin,
                           cu_seqlens=cu_seqlens)
    out = gqa_prefill(q, k_cache, v_cache, block_table, seq_lens, scale,
                      cu_seqlens=cu_seqlens)

or, where nothing is cached, over the step's own rows; or over rows that a
compressed cache hands back (seq_lens' running sum in cu_seqlens_k):

    out = gqa_prefill_packed(q, k, v, cu_seqlens, cu_seqlens, scale)

    k, v = kv_cache.kv_read_fp8(cache, scales, block_table, seq_lens,
                                cu_seqlens=cu_seqlens_k, num_tokens=total)
    out = gqa_prefill_packed(q, k, v, cu_seqlens, cu_seqlens_k, scale)

Request b's rows are cu_seqlens[b] .. cu_seqlens[b + 1] - 1 of q [T, Hq, 128] (bf16, a
strided view if need be), the last of them at its last key (seq_lens counts the
new tokens); without cu_seqlens every request has one row. Row i of n sees the keys
up to its own position, causal=False: all of them. kv_head = q_head // (Hq // Hkv).

The result is [T, Hq, 128]; with return_lse=True a pair of it and the natural
logarithms of the softmax sums, fp32 [T, Hq], from which results over parts of the keys
can be joined. Rows without a place (of no request, or at a negative position) and
rows that see no key get zeros and -infinity. Block ids outside the cache are left out.

The softmax weights are rounded to bf16 (by 2^-8 of each at most) for the product with the
values and divided by the sum of the rounded ones; log-sum-exps are of the fp32 weights.
Values, queries and scores that are not finite give NaN to the rows that see them (a value
in its dim alone), but for scores of -infinity beside finite ones, which weigh nothing.

num_splits > 0 cuts every request's keys into so many pieces and joins them in a
second launch; 0 chooses from the sizes. Over paged caches the pieces are of what
block_table's width holds: a table much wider than the longest request leaves most of
them empty and few workgroups with the work (pass the columns in use, or more pieces). The
operators run on the current stream, allocate their results (and a workspace)
from torch's allocator and can be captured into graphs. Rejected arguments raise
RuntimeError. There is no fallback: a missing build raises ImportError.
"""

import glob
import importlib.util
import os

_LIB_DIR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lib")


def _load_extension():
    paths = sorted(glob.glob(os.path.join(_LIB_DIR, "prefill_ext*.so")))
    if not paths:
        raise ImportError(
            f"prefill_ext not built in {_LIB_DIR}; run "
            "`python mla-decode-kernels_amd/build.py` (or __graft_entry__.build())"
        )
    spec = importlib.util.spec_from_file_location("prefill_ext", paths[0])
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


_ext = _load_extension()
EXTENSION_PATH = _ext.__file__


def gqa_prefill(q, k_cache, v_cache, block_table, seq_lens, scale, cu_seqlens=None, causal=True,
                num_splits=0, return_lse=False):
    """Attention of q [T, Hq, 128] over the paged caches [num_blocks, block_size, Hkv, 128]."""
    out, lse = _ext.gqa_prefill(q, k_cache, v_cache, block_table, seq_lens, scale, cu_seqlens,
                                causal, num_splits, return_lse)
    return (out, lse) if return_lse else out


def gqa_prefill_packed(q, k, v, cu_seqlens_q, cu_seqlens_k, scale, causal=True, num_splits=0,
                       return_lse=False):
    """Attention of q [T, Hq, 128] over rows k and v [Tk, Hkv, 128], request b's keys being rows
    cu_seqlens_k[b] .. cu_seqlens_k[b + 1] - 1. (k and v are strided views at will; unless they
    start at 16 bytes and have strides of multiples of 8 elements, they are copied.)"""
    out, lse = _ext.gqa_prefill_packed(q, k, v, cu_seqlens_q, cu_seqlens_k, scale, causal,
                                       num_splits, return_lse)
    return (out, lse) if return_lse else out
