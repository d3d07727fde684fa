"""The decoding step's C ABI and Python entry points without a GPU: struct layouts, refusals, and the
float64 oracle the kernels are checked against (``oracle/decode.py``)."""
from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from dsalt_amd import _lib, ops
from oracle import decode as OD

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dsalt_amd.h")
FAKE = 1 << 20  # never dereferenced: validation fails before any launch
STRUCTS = {"dsalt_cache": _lib.Cache, "dsalt_cache_rows_args": _lib.CacheRowsArgs, "dsalt_cache_write_args": _lib.CacheWriteArgs,
           "dsalt_cache_read_args": _lib.CacheReadArgs, "dsalt_cache_attn_args": _lib.CacheAttnArgs,
           "dsalt_sample_args": _lib.SampleArgs}


def test_struct_layouts_match_c(tmp_path):
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"%s\"\nint main(void){" % HEADER
    for c, cls in STRUCTS.items():
        src += 'printf("%%zu\\n",sizeof(%s));' % c
        src += "".join('printf("%%zu\\n",offsetof(%s,%s));' % (c, f) for f, _ in cls._fields_)
    (tmp_path / "l.c").write_text(src + "return 0;}")
    subprocess.run(["gcc", "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in STRUCTS.values():
        want += [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def _cache(**kw):
    f = dict(n_blocks=8, n_kv_heads=2, block_tokens=64, head_dim=64, k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE)
    f.update(kw)
    return _lib.Cache(*f.values())


def _refused(name, a, code, msg=None):
    lib = _lib.load()
    assert getattr(lib, name)(ctypes.byref(a) if a is not None else None, None) == code
    assert lib.dsalt_last_error()
    if msg:
        assert msg in lib.dsalt_last_error()


BAD_CACHE = [("n_blocks", 0, 1), ("n_kv_heads", 0, 1), ("n_kv_heads", 65536, 1), ("block_tokens", 48, 1), ("block_tokens", 256, 1),
             ("head_dim", 96, 2), ("k", None, 1), ("v", FAKE + 8, 1), ("k_scale", None, 1)]


def _rows_args():
    a = _lib.CacheRowsArgs(4, 16, 64, 256, 12, 64)
    for f in ("seq_len", "new_len", "table", "free_blocks", "span", "granted", "cu", "req", "pos", "slot", "pieces"):
        setattr(a, f, FAKE)
    a.seq_out, a.span_out, a.table_stride = 2 * FAKE, 2 * FAKE, 16
    a.workspace, a.workspace_bytes = FAKE, _lib.load().dsalt_cache_rows_workspace_bytes(ctypes.byref(a))
    return a


@pytest.mark.parametrize("field,value,code", [
    ("n_reqs", 0, 1), ("table_cols", 0, 1), ("table_cols", 1 << 26, 1), ("table_stride", 15, 1), ("block_tokens", 8, 1),
    ("n_rows", -1, 1), ("n_pieces", 11, 1), ("n_pieces", 257, 1), ("n_free", 0, 1), ("seq_len", None, 1), ("pieces", None, 1),
    ("pieces", FAKE + 4, 1), ("span", None, 1), ("cu", None, 1), ("seq_out", FAKE, 1), ("span_out", FAKE, 1), ("workspace", None, 3),
    ("workspace_bytes", 300, 3)])
def test_rows_refusals(field, value, code):
    a = _rows_args()
    if code == 3:  # only many requests need a workspace
        a.n_reqs, a.n_pieces = 5000, 256
        assert _lib.load().dsalt_cache_rows_workspace_bytes(ctypes.byref(a)) > 300
    setattr(a, field, value)
    _refused("dsalt_cache_rows", a, code)


@pytest.mark.parametrize("field,value", [("n_rows", (1 << 30) + 1), ("n_rows", 0x7fffffff), ("n_reqs", (1 << 24) + 1)])
def test_rows_past_the_largest_sizes(field, value):
    a = _rows_args()
    a.n_pieces = 1 << 27
    setattr(a, field, value)
    _refused("dsalt_cache_rows", a, 1, b"at most 2^24")


def _write_args(c=None):
    return _lib.CacheWriteArgs(c or _cache(), 32, 4, 1, FAKE, 128, 64, FAKE, 128, 64, FAKE)


def _read_args(c=None):
    return _lib.CacheReadArgs(c or _cache(), 4, 16, 32, 1, FAKE, 16, FAKE, None, FAKE, FAKE)


def _attn_args(c=None):
    return _lib.CacheAttnArgs(c or _cache(), 4, 8, 4, 16, 8, 1, 512, FAKE, 16, FAKE, 512, 64, FAKE, FAKE, FAKE, FAKE, None, FAKE,
                              512, 64, FAKE, 0.125)


@pytest.mark.parametrize("field,value,code", BAD_CACHE)
def test_bad_caches_are_refused(field, value, code):
    for name, make in (("dsalt_cache_write", _write_args), ("dsalt_cache_read", _read_args), ("dsalt_cache_attn", _attn_args)):
        _refused(name, make(_cache(**{field: value})), code)


@pytest.mark.parametrize("name,make,field,value", [
    ("dsalt_cache_write", _write_args, f, v) for f, v in
    (("n_rows", -1), ("n_pieces", -1), ("dtype", 3), ("k", None), ("v", FAKE + 2), ("k_stride_t", 100), ("v_stride_t", 0),
     ("pieces", None), ("pieces", FAKE + 8))] + [
    ("dsalt_cache_read", _read_args, f, v) for f, v in
    (("n_reqs", 0), ("table_cols", 0), ("n_rows", -1), ("dtype", 5), ("table", None), ("table_stride", 3), ("cu_seqlens", None),
     ("k", None), ("v", FAKE + 4))] + [
    ("dsalt_cache_attn", _attn_args, f, v) for f, v in
    (("n_rows", -1), ("n_heads", 7), ("n_heads", 0), ("n_reqs", 0), ("table_cols", 0), ("table_stride", 15), ("k_lmk", 2049),
     ("k_lmk", -1), ("dtype", 3), ("w_max", -1), ("q", FAKE + 2), ("q_stride_t", 63), ("out", None), ("req", None), ("pos", None),
     ("w", None), ("lse", None), ("lmk_idx", None), ("scale", 0.0), ("scale", float("nan")))])
def test_refusals(name, make, field, value):
    a = make()
    setattr(a, field, value)
    _refused(name, a, 1)


@pytest.mark.parametrize("field,value", [("rows", -1), ("n_cols", 0), ("n_cols", (1 << 20) + 1), ("dtype", 3), ("u_bytes", 2),
                                         ("logits", None), ("logits", FAKE + 1), ("logits_stride", -1), ("u", None), ("token", None),
                                         ("logp", None)])
def test_sample_refusals(field, value):
    a = _lib.SampleArgs(4, 100, 1, 4, FAKE, 100, FAKE)
    a.token = a.logp = FAKE
    setattr(a, field, value)
    _refused("dsalt_sample_rows", a, 1)


def test_null_structs_and_empty_calls():
    lib = _lib.load()
    for name in ("dsalt_cache_rows", "dsalt_cache_write", "dsalt_cache_read", "dsalt_cache_attn", "dsalt_sample_rows"):
        _refused(name, None, 1)
    for name, make in (("dsalt_cache_write", _write_args), ("dsalt_cache_read", _read_args), ("dsalt_cache_attn", _attn_args)):
        a = make()
        a.n_rows = 0
        assert getattr(lib, name)(ctypes.byref(a), None) == 0
    a = _lib.SampleArgs(0, 100, 1, 4)
    assert lib.dsalt_sample_rows(ctypes.byref(a), None) == 0


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("n_heads", [2, 8])
def test_calls_without_rows_need_no_workspace(head_dim, n_heads):
    """A step without query tokens, whatever its tables and windows would hold: the query that precedes each call gives
    zero, and the call does nothing."""
    lib = _lib.load()
    for cols in (1, 16, 64, 1 << 20 >> 6, 1 << 30 >> 6):
        for w_max in (0, 1, 512, 1 << 20, 0x7fffffff):
            for k_lmk in (0, 8, 2048):
                a = _attn_args(_cache(head_dim=head_dim))
                a.n_rows, a.n_heads, a.table_cols, a.table_stride, a.w_max, a.k_lmk = 0, n_heads, cols, cols, w_max, k_lmk
                assert lib.dsalt_cache_attn_workspace_bytes(ctypes.byref(a)) == 0
                assert lib.dsalt_cache_attn(ctypes.byref(a), None) == 0


def test_python_refuses_cpu_tensors():
    c = ops.new_cache(2, 1, 64, device="cpu")
    i = torch.zeros(1, dtype=torch.int32)
    t = torch.zeros((1, 2), dtype=torch.int32)
    x = torch.zeros((1, 1, 64))
    for call in (lambda: ops.cache_rows_(i, i, t, i, torch.zeros(2, dtype=torch.int64), 1),
                 lambda: ops.cache_write_(x, x, c, torch.zeros((1, 4), dtype=torch.int32)),
                 lambda: ops.cache_read(c, t, torch.zeros(2, dtype=torch.int32), n_rows=1),
                 lambda: ops.cache_attention(x, c, t, i, i, i, torch.zeros((1, 1, 1, 0), dtype=torch.int32)),
                 lambda: ops.sample_rows(torch.zeros(1, 4), torch.zeros(1))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for kw in (dict(block_tokens=48), dict(head_dim=96)):
        with pytest.raises(ValueError, match="block_tokens"):
            ops.new_cache(**{**dict(n_blocks=1, n_kv_heads=1, head_dim=64, device="cpu"), **kw})


@pytest.mark.parametrize("dt", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int32, torch.uint32, torch.int64, torch.uint64,
                                torch.float16, torch.bfloat16, torch.float32, torch.float64, torch.bool])
def test_counts_of_every_type(dt):
    """A row's top_k from tensors of any type: small counts as they are, negative ones negative, what passes the largest
    vocabulary as all of it (as that size, or negative)."""
    signed = not (dt == torch.bool or dt.is_floating_point is False and torch.iinfo(dt).min == 0)
    top = 1 if dt == torch.bool else (min(torch.finfo(dt).max, 2.0 ** 40) if dt.is_floating_point else torch.iinfo(dt).max)
    values = [0, 1] + ([7, 100] if dt != torch.bool else []) + ([-1, -5] if signed else []) + [top]
    t = torch.tensor([int(v) for v in values], dtype=torch.int64 if dt != torch.uint64 else dt).to(dt)
    if dt != torch.uint64:
        t = torch.stack([t, t], 1)[:, 0]  # strided
    got = ops._counts(t)
    assert got.dtype == torch.int32 and got.is_contiguous() and got.shape == t.shape
    for v, k in zip(values, got.tolist()):
        if v < 0:
            assert k < 0, (v, k)
        elif v > ops.MAX_VOCAB:
            assert k < 0 or k >= ops.MAX_VOCAB, (v, k)
        else:
            assert k == int(v), (v, k)


def test_windows_past_32_bits():
    """A window longer than int32 names stays longer than any cache."""
    w = [1, 0, -3, 512, (1 << 31) - 1, 1 << 31, (1 << 32) + 5, 1 << 40, (1 << 63) - 1, -(1 << 40) + 9]
    got = ops._i32(ops._windows(torch.tensor(w))).tolist()
    assert [max(x, 1) for x in got] == [max(min(x, (1 << 31) - 1), 1) for x in w]
    narrow = torch.tensor([1, 5], dtype=torch.int32)
    assert ops._windows(narrow) is narrow


@pytest.mark.parametrize("heads", [(0, 2), (0, 0), (3, 2)])
def test_attention_refuses_head_counts(monkeypatch, heads):
    """A cache without heads, or query heads that do not share its heads evenly, is an argument error like any other."""
    monkeypatch.setattr(ops, "_on", lambda *ts: 0)  # (the checks come before anything runs)
    n_kv, n = heads
    i = torch.zeros(1, dtype=torch.int32)
    c = ops.new_cache(2, n_kv, 64, device="cpu")
    with pytest.raises(ValueError, match="H a multiple"):
        ops.cache_attention(torch.zeros(1, n, 64), c, torch.zeros((1, 2), dtype=torch.int32), i, i, i,
                            torch.zeros((n, 1, 1, 0), dtype=torch.int32))


# ------------------------------------------------------------------------ the oracle itself
def test_oracle_rounds_as_torch_does():
    """Every finite bf16 within 448: the oracle's e4m3 is torch's conversion."""
    x = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    x = x[torch.isfinite(x) & (x.abs() <= 448)]
    assert np.array_equal(OD.e4m3(x.double().numpy()), x.to(torch.float8_e4m3fn).double().numpy())
    assert OD.e4m3(np.array([500.0, -1e30]))[0] == 448 and np.isnan(OD.e4m3(np.array([np.inf, np.nan]))).all()


def test_oracle_scale_is_the_least():
    for x in (448.0, 448.0000001, 1.0, 3.3e38, 1e-45, 0.0, 447.9, 2.0 ** -117):
        s = OD.scale_of(np.array([x, np.inf]))
        assert x <= 448 * s or s == 2.0 ** 119
        assert s == 2.0 ** -126 or x > 448 * s / 2


def test_oracle_rows_serve_in_order():
    """Two pages are free: the first request takes one, the second wants two and is refused, the third needs
    none and is granted, the fourth would fit but comes after the second."""
    table = np.full((5, 4), -1)
    table[2, 0] = table[4, 0] = 9
    table[4, 1] = 8
    ring = [5, 6, 0, 0]
    s = OD.rows([0, 0, 3, 0, 20], [16, 20, 1, 16, -1], table, ring, (0, 2), 60, 16)
    assert s["granted"] == [1, 0, 1, 0, 1] and s["seq_len"] == [16, 0, 4, 0, 0] and s["span"] == [1, 4]
    assert ring == [5, 6, 9, 8] and table[0, 0] == 5 and s["pos"][36] == 3 and s["slot"][36] == 9 * 16 + 3
    assert s["pieces"][:3].tolist() == [[0, 16, 5, 0], [36, 1, 9, 3], [0, 0, 0, 0]]


def test_oracle_sampling_counts():
    """Tokens drawn over an even grid of u fall in the proportions of the kept weights."""
    x = np.log(np.array([0.4, 0.1, 0.3, 0.2]))
    n = 4000
    draw = [OD.sample(x, (i + 0.5) / n, 1.0, 3, 0.95, 0.0)[0] for i in range(n)]
    got = np.bincount(draw, minlength=4) / n
    assert np.allclose(got, [4 / 9, 0, 3 / 9, 2 / 9], atol=2 / n)
    assert OD.sample(x, 0.99, 1.0, 0, 0.6, 0.0)[0] == 2 and OD.sample(x, 0.99, 1.0, 0, 1.0, 0.6)[0] == 2
