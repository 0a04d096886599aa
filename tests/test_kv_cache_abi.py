"""CPU tests of the cache operators' boundary, without launching anything: what
the library exports, what the launchers and the torch operators refuse, the
rules for where tokens go (csrc/kv_places.hpp compiled for the host), and the
rotation table."""

import ctypes
import math
import os
import random
import re
import subprocess

import numpy as np
import pytest
import torch

import capi
import kv_cache
from oracle import kv_reference as ref

INVALID = capi.HIP_ERROR_INVALID_VALUE
CSRC = os.path.join(os.path.dirname(capi.LIB_PATH), "..", "csrc")


def test_exports():
    declared = capi.declared_kv_functions()
    assert declared == ["kv_append_launch", "kv_append_mla_launch", "kv_append_mxfp4_launch",
                        "kv_decode_mxfp4_launch", "kv_decode_mxfp4_workspace_bytes",
                        "kv_read_mxfp4_launch"]
    out = subprocess.run(["nm", "-D", "--defined-only", capi.LIB_PATH], capture_output=True,
                         text=True, check=True).stdout
    names = {ln.split()[-1] for ln in out.splitlines() if ln.strip()}
    assert {n for n in names if n.startswith("kv_")} == set(declared)


@pytest.mark.parametrize("struct,name", [(capi.KvAppendArgs, "kv_append_args"),
                                         (capi.KvAppendMlaArgs, "kv_append_mla_args")])
def test_struct_fields_follow_the_header(struct, name):
    with open(capi.KV_HEADER_PATH) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    body = re.search(r"typedef struct " + name + r" \{(.*?)\} " + name, text, re.S).group(1)
    fields = []
    for decl in body.split(";"):
        if not decl.strip():
            continue
        parts = decl.replace("*", " * ").replace("const ", "").split(None, 1)
        for item in parts[1].split(","):
            pointer = "*" in item
            kind = ctypes.c_void_p if pointer else {"int64_t": ctypes.c_int64, "int": ctypes.c_int,
                                                    "float": ctypes.c_float}[parts[0]]
            fields.append((item.replace("*", "").strip(), kind))
    assert fields == struct._fields_


# A pointer that is never read: every call below is refused first, or empty.
SOME = 4096


def append_args(**over):
    a = capi.KvAppendArgs()
    for n in ("q", "k", "v", "q_out", "k_cache", "v_cache", "mxfp4_cache", "block_table",
              "seq_lens"):
        setattr(a, n, SOME)
    a.T = a.B = 4
    a.Hq, a.Hkv, a.num_blocks, a.block_size, a.max_blocks = 8, 2, 10, 16, 3
    for n, v in over.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("over", [
    dict(T=-1), dict(T=3), dict(T=(1 << 23) + 1, B=(1 << 23) + 1), dict(B=-1), dict(Hq=0),
    dict(Hkv=0), dict(Hq=5000), dict(num_blocks=-1), dict(block_size=0), dict(max_blocks=0),
    dict(rotary_dim=64), dict(cos_sin=SOME), dict(cos_sin=SOME, rotary_dim=24, table_rows=9),
    dict(cos_sin=SOME, rotary_dim=144, table_rows=9), dict(cos_sin=SOME, rotary_dim=-16),
    dict(cos_sin=SOME, rotary_dim=16, table_rows=-1), dict(q_weight=SOME, q_weight_type=2),
    dict(k_weight=SOME, k_weight_type=-1), dict(q=None), dict(k=None), dict(v=None),
    dict(q_out=None), dict(block_table=None), dict(seq_lens=None)])
def test_append_refuses(over):
    assert capi.kv_append_launch(append_args(**over), None) == INVALID
    assert capi.kv_append_mxfp4_launch(append_args(**over), None) == INVALID


def test_more_requests_than_the_search_counts():
    over = dict(T=4, B=(1 << 30) + 1, cu_seqlens=SOME)
    assert capi.kv_append_launch(append_args(**over), None) == INVALID
    assert capi.kv_append_mxfp4_launch(append_args(**over), None) == INVALID
    a = capi.KvAppendMlaArgs()
    for n in ("q_pe", "c", "k_pe", "q_out", "kv_cache", "block_table", "seq_lens", "cos_sin"):
        setattr(a, n, SOME)
    a.h_q, a.num_blocks, a.block_size, a.max_blocks, a.table_rows = 16, 10, 64, 3, 100
    a.T, a.B, a.cu_seqlens = 4, (1 << 30) + 1, SOME
    assert capi.kv_append_mla_launch(a, None) == INVALID
    args = [SOME, SOME, SOME, SOME, SOME, SOME, 4, (1 << 30) + 1, 2, 10, 16, 3, None]
    assert capi.kv_read_mxfp4_launch(*args) == INVALID


def test_append_refuses_caches():
    for over in (dict(k_cache=None), dict(v_cache=None), dict(k_cache=SOME + 8),
                 dict(v_cache=SOME + 2)):
        assert capi.kv_append_launch(append_args(**over), None) == INVALID
    for over in (dict(mxfp4_cache=None), dict(mxfp4_cache=SOME + 2), dict(block_size=24)):
        assert capi.kv_append_mxfp4_launch(append_args(**over), None) == INVALID
    assert capi.lib().kv_append_launch(None, None) == INVALID
    assert capi.lib().kv_append_mla_launch(None, None) == INVALID


def test_empty_steps_launch_nothing():
    assert capi.kv_append_launch(append_args(T=0, B=0), None) == 0
    assert capi.kv_append_mxfp4_launch(append_args(T=0, B=3, cu_seqlens=SOME), None) == 0
    assert capi.kv_read_mxfp4_launch(SOME, SOME, SOME, SOME, SOME, SOME, 0, 2, 8, 4, 16, 2,
                                     None) == 0
    assert capi.kv_decode_mxfp4_launch(SOME, SOME, SOME, SOME, SOME, 0, 8, 2, 4, 16, 2, 0.1, 0,
                                       None, 0, None) == 0


@pytest.mark.parametrize("over", [
    dict(T=-1), dict(T=3), dict(B=-1), dict(h_q=0), dict(h_q=5000), dict(num_blocks=-1),
    dict(block_size=0), dict(max_blocks=0), dict(table_rows=-1),
    dict(c_weight=SOME, c_weight_type=3), dict(q_pe=None), dict(c=None), dict(k_pe=None),
    dict(q_out=None), dict(block_table=None), dict(seq_lens=None), dict(cos_sin=None),
    dict(kv_cache=None), dict(kv_cache=SOME + 4)])
def test_mla_append_refuses(over):
    a = capi.KvAppendMlaArgs()
    for n in ("q_pe", "c", "k_pe", "q_out", "kv_cache", "block_table", "seq_lens", "cos_sin"):
        setattr(a, n, SOME)
    a.T = a.B = 4
    a.h_q, a.num_blocks, a.block_size, a.max_blocks, a.table_rows = 16, 10, 64, 3, 100
    for n, v in over.items():
        setattr(a, n, v)
    assert capi.kv_append_mla_launch(a, None) == INVALID


@pytest.mark.parametrize("at,value", [(1, None), (2, None), (4, None), (5, None), (6, -1),
                                      (7, -1), (8, 0), (9, -1), (10, 24), (10, 0), (11, 0),
                                      (0, None), (4, SOME + 8), (0, SOME + 2), (6, 5)])
def test_read_refuses(at, value):
    args = [SOME, SOME, SOME, None, SOME, SOME, 4, 4, 2, 10, 16, 3, None]
    args[at] = value
    assert capi.kv_read_mxfp4_launch(*args) == INVALID


@pytest.mark.parametrize("at,value", [
    (0, None), (0, SOME + 8), (1, None), (1, SOME + 4), (2, None), (3, None), (4, None),
    (4, SOME + 2), (5, -1), (5, (1 << 20) + 1), (6, 0), (6, 7), (7, 0), (8, -1), (9, 24), (9, 0),
    (10, 0), (10, 1 << 28), (11, math.nan), (11, math.inf), (12, 1 << 23), (13, None),
    (13, SOME + 8), (14, 100)])
def test_decode_refuses(at, value):
    ws = capi.kv_decode_mxfp4_workspace_bytes(4, 8, 2, 16, 100, 64)
    args = [SOME, SOME, SOME, SOME, SOME, 4, 8, 2, 10, 16, 100, 0.1, 64, SOME, ws, None]
    args[at] = value
    assert capi.kv_decode_mxfp4_launch(*args) == INVALID


def test_decode_workspace_bytes():
    f = capi.kv_decode_mxfp4_workspace_bytes
    # A record of 16 bytes and two states of min(16, group) heads of 132 floats a workgroup.
    assert f(4, 32, 8, 16, 100, 64) == 64 * (16 + 2 * 4 * 132 * 4)
    assert f(4, 160, 8, 16, 100, 64) == 64 * (16 + 2 * 16 * 132 * 4)
    assert f(4, 32, 8, 16, 1, 0) == 0  # short sequences need none
    assert f(4, 30, 8, 16, 100, 64) == 0 and f(-1, 32, 8, 16, 100, 64) == 0
    assert f(4, 32, 8, 24, 100, 64) == 0


# ------------------------------------------------------ where tokens go


@pytest.fixture(scope="module")
def places_lib(tmp_path_factory):
    """csrc/kv_places.hpp on the host: the search as the lanes run it, with every access to the
    arrays checked."""
    tmp = tmp_path_factory.mktemp("places")
    src = tmp / "places.cpp"
    src.write_text(r"""
#include "kv_places.hpp"
extern "C" int place(int t, int T, int B, const int* lens, const int* cu, int group, int* out) {
  int b = t, first = t, next = t + 1, len = 0, probes = 0;
  if (cu) {
    kv::Search s = kv::Search::begin(B);
    first = cu[0];
    while (!s.done()) {
      if (++probes > 64) return -1;  // does not end
      const int step = s.step(group), lo = s.lo, hi = s.hi;
      int count = 0;
      for (int sub = 0; sub < group; ++sub) {
        const int at = lo + sub * step;
        if (at >= hi) continue;
        if (at < 1 || at > B) return -2;  // outside cu_seqlens
        count += cu[at] <= t;
      }
      // What the lanes hand over, with the lanes that have it checked.
      const int last = lo + (count - 1) * step, behind = lo + count * step;
      if (count > 0) {
        if (last >= hi) return -4;
        first = cu[last];
      }
      if (s.narrow(step, count)) {
        if (behind >= hi || count >= group) return -5;
        next = cu[behind], len = lens[behind - 1];
      }
    }
    b = s.request();
    if (b < 0 || b > B) return -3;
  } else if (t < B) {
    len = lens[t];
  }
  if (b >= B || t >= T) { out[2] = 0; return probes; }
  const kv::Place p = kv::place_in(t, b, first, next, len);
  out[0] = p.b, out[1] = p.pos, out[2] = p.live;
  return probes;
}
""")
    so = tmp / "places.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-fwrapv", f"-I{CSRC}",
                    str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    ip = ctypes.POINTER(ctypes.c_int)
    lib.place.argtypes = [ctypes.c_int] * 3 + [ip, ip, ctypes.c_int, ip]

    def place(t, T, lens, cu, group):
        lens = (ctypes.c_int * max(1, len(lens)))(*lens)
        n = len(cu) - 1 if cu is not None else len(lens)
        cu = None if cu is None else (ctypes.c_int * len(cu))(*cu)
        out = (ctypes.c_int * 3)()
        probes = lib.place(t, T, n, lens, cu, group, out)
        assert probes >= 0, (t, probes)
        return ((out[0], out[1]) if out[2] else None), probes

    return place


@pytest.mark.parametrize("group", [16, 64])
@pytest.mark.parametrize("B", [1, 2, 15, 16, 17, 63, 64, 65, 300, 4097])
def test_places(places_lib, B, group):
    rng = random.Random(B)
    news = [rng.choice([0, 0, 1, 1, 2, 7]) for _ in range(B)]
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    T = cu[-1] + 5  # rows behind the last sequence
    lens = [max(0, n + rng.randint(-2, 40)) for n in news]
    want = ref.places(T, lens, cu)
    rows = range(T) if T < 400 else sorted(rng.sample(range(T), 400))
    for t in rows:
        got, probes = places_lib(t, T, lens, cu, group)
        assert got == want[t], t
        assert probes <= (1 if B <= group else 2 if B <= group * group else 4)


def test_places_without_cu_seqlens(places_lib):
    lens = [3, 0, 1, -5]
    assert [places_lib(t, 4, lens, None, 16)[0] for t in range(4)] == [(0, 2), None, (2, 0), None]


@pytest.mark.parametrize("group", [16, 64])
def test_places_survive_bad_cu_seqlens(places_lib, group):
    """Entries out of order, negative or past T: a place that is one, no access outside."""
    rng = random.Random(5)
    for _ in range(300):
        B = rng.choice([1, 3, 20, 70, 300])
        cu = [rng.randint(-2**31, 2**31 - 1) if rng.random() < 0.3 else rng.randint(-5, 50)
              for _ in range(B + 1)]
        lens = [rng.randint(-3, 60) for _ in range(B)]
        for t in (0, 1, 7, 49, 1000):
            got, _ = places_lib(t, 50, lens, cu, group)
            assert got is None or (0 <= got[0] < B and 0 <= got[1] < lens[got[0]])


# ------------------------------------------------- the torch operators


def cpu_inputs(T=2, Hq=4, Hkv=2, bs=16):
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t)  # noqa: E731
    return dict(q=z(T, Hq, 128), k=z(T, Hkv, 128), v=z(T, Hkv, 128),
                k_cache=z(3, bs, Hkv, 128), v_cache=z(3, bs, Hkv, 128),
                block_table=z(T, 2, t=torch.int32), seq_lens=z(T, t=torch.int32))


def test_operators_refuse_host_tensors():
    a = cpu_inputs()
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        kv_cache.kv_append(**a)
    mx = kv_cache.new_mxfp4_cache(3, 16, 2, device="cpu")
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        kv_cache.kv_append_mxfp4(a["q"], a["k"], a["v"], mx, a["block_table"], a["seq_lens"])
    with pytest.raises(RuntimeError, match="kv_cache must be a CUDA tensor"):
        kv_cache.kv_read_mxfp4(mx, a["block_table"], a["seq_lens"])
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        kv_cache.gqa_decode_mxfp4(a["q"], mx, a["block_table"], a["seq_lens"], 0.1)
    with pytest.raises(RuntimeError, match="q_pe must be a CUDA tensor"):
        kv_cache.mla_append(torch.zeros(2, 4, 64), torch.zeros(2, 512), torch.zeros(2, 64), mx,
                            a["block_table"], a["seq_lens"], torch.zeros(4, 64))
    with pytest.raises(TypeError):
        kv_cache.kv_append(a["q"])


def test_new_mxfp4_cache():
    c = kv_cache.new_mxfp4_cache(5, 48, 3, device="cpu")
    assert c.shape == (5, 3, 3, 2176) and c.dtype == torch.uint8 and not c.any()
    for bad in ((5, 24, 3), (5, 0, 3), (-1, 16, 3), (5, 16, 0)):
        with pytest.raises(ValueError):
            kv_cache.new_mxfp4_cache(*bad, device="cpu")


# ------------------------------------------------------ rotation tables


def angles(table):
    half = table.shape[1] // 2
    return table[:, :half].double(), table[:, half:].double()


def test_rotary_table_plain():
    t = kv_cache.rotary_table(70000, 64, base=10000.0, device="cpu")
    assert t.shape == (70000, 64) and t.dtype == torch.float32
    pos, i = 69999, 5
    a = pos * 10000.0 ** (-2 * i / 64)
    # Rounded once from 64 bits: half a step of fp32 at most 1, and the angle's own 2^-52.
    assert abs(float(t[pos, i]) - math.cos(a)) < 2 ** -24
    assert abs(float(t[pos, 32 + i]) - math.sin(a)) < 2 ** -24


def freqs(scaling, dim=128, base=10000.0):
    """The frequencies a table was made of, from its row 1 (angles below pi)."""
    c, s = angles(kv_cache.rotary_table(2, dim, base=base, scaling=scaling, device="cpu"))
    return torch.atan2(s[1], c[1]).numpy(), float(torch.hypot(s[1], c[1]).mean())


def test_rotary_scalings():
    plain, gain = freqs(None)
    assert np.allclose(plain, 10000.0 ** (-np.arange(64) / 64.0), rtol=1e-5) and \
        abs(gain - 1) < 1e-6
    linear, _ = freqs({"type": "linear", "factor": 4.0})
    assert np.allclose(linear, plain / 4, rtol=1e-5)
    ntk, _ = freqs({"type": "ntk", "factor": 8.0})
    assert abs(ntk[0] - 1) < 1e-6 and abs(ntk[-1] * 8 / plain[-1] - 1) < 1e-4
    assert (ntk <= plain * (1 + 1e-6)).all()
    llama, _ = freqs({"type": "llama3", "factor": 8.0, "original_max_position": 8192},
                     base=500000.0)
    base5, _ = freqs(None, base=500000.0)
    wave = 2 * np.pi / base5
    assert np.allclose(llama[wave < 8192 / 4], base5[wave < 8192 / 4], rtol=1e-5)
    assert np.allclose(llama[wave > 8192], base5[wave > 8192] / 8, rtol=1e-4)
    mid = (wave >= 8192 / 4) & (wave <= 8192)
    w = (8192 / wave[mid] - 1) / 3
    assert mid.any() and np.allclose(llama[mid], base5[mid] * (w + (1 - w) / 8), rtol=1e-4)
    yarn, gain = freqs({"type": "yarn", "factor": 16.0, "original_max_position": 4096})
    turns = 4096 * plain / (2 * np.pi)
    assert abs(gain - (0.1 * math.log(16) + 1)) < 1e-6
    assert np.allclose(yarn[turns > 40], plain[turns > 40], rtol=1e-5)
    assert np.allclose(yarn[turns < 0.8], plain[turns < 0.8] / 16, rtol=1e-4)
    assert (np.diff(yarn) <= 0).all()
    _, gain = freqs({"type": "yarn", "factor": 16.0, "original_max_position": 4096,
                     "attention_factor": 1.0})
    assert abs(gain - 1) < 1e-6


@pytest.mark.parametrize("args", [(0, 64), (10, 63), (10, 0)])
def test_rotary_table_refuses(args):
    with pytest.raises(ValueError):
        kv_cache.rotary_table(*args, device="cpu")


@pytest.mark.parametrize("scaling", [
    {"type": "other", "factor": 2.0}, {"type": "linear", "factor": 0.0},
    {"type": "llama3", "factor": 2.0, "original_max_position": 64, "low_freq_factor": 4.0}])
def test_rotary_scaling_refuses(scaling):
    with pytest.raises(ValueError):
        kv_cache.rotary_table(8, 64, scaling=scaling, device="cpu")
