"""The 4-bit cache, verification and query/key norms without a GPU: struct layouts, refusals, and the float64 oracles the
kernels are checked against (``oracle/decode4.py``, ``oracle/qk_norm.py``)."""
from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad as fwAD

from dsalt_amd import _lib, ops
from dsalt_amd.kernels import qk_norm_rope
from dsalt_amd.model import DSALTConfig, DSALTLMHeadModel
from dsalt_amd.modules import DSALTAttention
from oracle import decode4 as O4
from oracle import qk_norm as OQ

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dsalt_amd.h")
FAKE = 1 << 20  # never dereferenced: validation fails before any launch
STRUCTS = {"dsalt_cache4": _lib.Cache4, "dsalt_cache4_write_args": _lib.Cache4WriteArgs, "dsalt_cache4_read_args": _lib.Cache4ReadArgs,
           "dsalt_cache4_attn_args": _lib.Cache4AttnArgs, "dsalt_verify_args": _lib.VerifyArgs,
           "dsalt_qk_norm_rope_args": _lib.QkNormRopeArgs, "dsalt_qk_norm_rope_bwd_args": _lib.QkNormRopeBwdArgs}


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


def _refused(name, a, code):
    lib = _lib.load()
    assert getattr(lib, name)(ctypes.byref(a) if a is not None else None, None) == code
    assert lib.dsalt_last_error()


def _cache(**kw):
    f = dict(n_blocks=8, n_kv_heads=2, block_tokens=64, head_dim=64, kv=FAKE, scale=FAKE)
    f.update(kw)
    return _lib.Cache4(*f.values())


def _write_args(c=None):
    return _lib.Cache4WriteArgs(c or _cache(), 32, 4, 1, FAKE, 128, 64, FAKE, 128, 64, FAKE)


def _read_args(c=None):
    return _lib.Cache4ReadArgs(c or _cache(), 4, 16, 32, 1, FAKE, 16, FAKE, None, FAKE, FAKE)


def _attn_args(c=None):
    return _lib.Cache4AttnArgs(c or _cache(), 4, 8, 4, 16, 8, 1, 512, 1, FAKE, 16, FAKE, 512, 64, FAKE, FAKE, FAKE, FAKE, None, FAKE,
                               512, 64, FAKE, 0.125)


def _verify_args():
    a = _lib.VerifyArgs(2, 6, 100, 1, 4, FAKE, 100, FAKE, 100, FAKE, FAKE, FAKE, FAKE, None, None, 1.0, 1.0, FAKE, FAKE)
    a.workspace, a.workspace_bytes = FAKE, _lib.load().dsalt_verify_workspace_bytes(ctypes.byref(a))
    return a


def _qk_args():
    a = _lib.QkNormRopeArgs(10, 2, 4, 2, 64, 1, 0, 100, 1e-6)
    for f in ("q", "k", "q_weight", "k_weight", "cu_seqlens", "cos", "sin"):
        setattr(a, f, FAKE)
    for f, n in (("q", 4), ("k", 2), ("qo", 4), ("ko", 2)):
        setattr(a, f + "_stride_t", 64 * n)
        setattr(a, f + "_stride_h", 64)
    a.q_out = a.k_out = 2 * FAKE
    return a


def _qk_bwd_args():
    a = _lib.QkNormRopeBwdArgs(_qk_args(), FAKE, 256, 64, FAKE, 128, 64, FAKE, FAKE)
    a.workspace, a.workspace_bytes = FAKE, _lib.load().dsalt_qk_norm_rope_bwd_workspace_bytes(ctypes.byref(a))
    return a


@pytest.mark.parametrize("field,value,code", [
    ("n_blocks", 0, 1), ("n_kv_heads", 0, 1), ("n_kv_heads", 65536, 1), ("block_tokens", 48, 1), ("block_tokens", 256, 1),
    ("n_blocks", 1 << 26, 1), ("head_dim", 96, 2), ("kv", None, 1), ("kv", FAKE + 8, 1), ("scale", None, 1), ("scale", FAKE + 4, 1)])
def test_bad_caches_are_refused(field, value, code):
    for name, make in (("dsalt_cache4_write", _write_args), ("dsalt_cache4_read", _read_args), ("dsalt_cache4_attn", _attn_args)):
        _refused(name, make(_cache(**{field: value})), code)


@pytest.mark.parametrize("name,make,field,value,code", [
    ("dsalt_cache4_write", _write_args, f, v, 1) for f, v in
    (("n_rows", -1), ("n_pieces", -1), ("dtype", 3), ("k", None), ("v", FAKE + 2), ("k_stride_t", 100), ("v_stride_t", 0),
     ("pieces", None), ("pieces", FAKE + 8))] + [
    ("dsalt_cache4_read", _read_args, f, v, 1) for f, v in
    (("n_reqs", 0), ("table_cols", 0), ("n_rows", -1), ("dtype", 5), ("table", None), ("table_stride", 3), ("cu_seqlens", None),
     ("k", None), ("v", FAKE + 4))] + [
    ("dsalt_cache4_attn", _attn_args, f, v, 1) for f, v in
    (("n_rows", -1), ("n_heads", 7), ("n_heads", 0), ("n_reqs", 0), ("table_cols", 0), ("table_stride", 15), ("k_lmk", 2049),
     ("k_lmk", -1), ("dtype", 3), ("w_max", -1), ("rows_per_req", 0), ("q", FAKE + 2), ("q_stride_t", 63), ("out", None),
     ("req", None), ("pos", None), ("w", None), ("lse", None), ("lmk_idx", None), ("scale", 0.0), ("scale", float("nan")))] + [
    ("dsalt_verify_rows", _verify_args, f, v, 1) for f, v in
    (("n_reqs", -1), ("n_reqs", (1 << 22) + 1), ("n_rows", -1), ("n_rows", (1 << 22) + 1), ("n_cols", 0), ("n_cols", (1 << 20) + 1),
     ("dtype", 3), ("u_bytes", 2), ("logits", None), ("logits", FAKE + 1), ("logits_stride", -1), ("draft_logits", FAKE + 1),
     ("draft_stride", -1), ("tokens", None), ("cu", None), ("u", None), ("v", None), ("accepted", None), ("out", None))] + [
    ("dsalt_verify_rows", _verify_args, "workspace", None, 3), ("dsalt_verify_rows", _verify_args, "workspace_bytes", 8, 3)])
def test_refusals(name, make, field, value, code):
    a = make()
    setattr(a, field, value)
    _refused(name, a, code)


@pytest.mark.parametrize("field,value", [
    ("total_len", -1), ("n_q_heads", -1), ("n_k_heads", 65536), ("head_dim", 8), ("head_dim", 72), ("head_dim", 272), ("dtype", 3),
    ("weight_dtype", 3), ("eps", -1.0), ("eps", float("nan")), ("cu_seqlens", None), ("pos", FAKE), ("num_seqs", 0), ("max_pos", 0),
    ("cos", None), ("sin", FAKE + 4), ("q_weight", None), ("k_weight", FAKE + 4), ("q", None), ("k", FAKE + 2), ("q_out", None),
    ("ko_stride_t", 100), ("q_stride_h", 4)])
def test_qk_refusals(field, value):
    a = _qk_args()
    setattr(a, field, value)
    _refused("dsalt_qk_norm_rope", a, 1)
    b = _qk_bwd_args()
    setattr(b.base, field, value)
    _refused("dsalt_qk_norm_rope_bwd", b, 1)


def test_qk_outputs_over_one_input_alone_are_refused():
    a = _qk_args()
    a.q_out = a.q
    _refused("dsalt_qk_norm_rope", a, 1)
    a.k_out, a.ko_stride_h = a.k, 128
    _refused("dsalt_qk_norm_rope", a, 1)


@pytest.mark.parametrize("field,value,code", [("dq", None, 1), ("dk", FAKE + 2, 1), ("dk_stride_t", 0, 1), ("dq_weight", None, 1),
                                              ("dk_weight", None, 1), ("workspace", None, 3), ("workspace_bytes", 8, 3)])
def test_qk_backward_refusals(field, value, code):
    b = _qk_bwd_args()
    setattr(b, field, value)
    _refused("dsalt_qk_norm_rope_bwd", b, code)


def _elements(at, st, sh, heads, T, D):
    return [at + t * st + h * sh + d for t in range(T) for h in range(heads) for d in range(D)]


def _layouts():
    """Random sides of few rows and heads, and those that a user meets: (T, (place, strides, heads) of two sides, exact)."""
    r, D = np.random.RandomState(0), 16
    for _ in range(2000):
        T, H, G = (int(x) for x in r.randint(1, 5, 3))
        a, b = ((int(r.randint(0, 12) * 8), int(r.randint(1, 14) * 8), int(r.randint(0, 8) * 8), n) for n in (H, G))
        if r.rand() < 0.6:
            b = (b[0], a[1], *b[2:])
        yield T, a, b
    for T in (1, 2, 5):
        for H, G in ((4, 2), (1, 1), (2, 4), (3, 1)):
            row = (H + 2 * G) * D
            yield T, (0, row, D, H), (H * D, row, D, G)                         # columns of one projection
            yield T, (0, row, D, H), (H * D - 8, row, D, G)                     # and half a head too near
            yield T, (0, D, T * D, H), (H * T * D, D, T * D, G)                 # heads first
            yield T, (0, 2 * H * D, 2 * D, H), (D, 2 * H * D, 2 * D, min(H, G))  # query and key heads in turn
            yield T, (0, D, D, H), (T * H * D + D, D, D, G)                     # a row's second head is the next row's first
            yield T, (0, row, D, H), (0, row, D, H)                             # the same memory


def test_heads_that_share_elements_are_found():
    """Against the sets of elements themselves, through Python and the C entry points (which then launch nothing); only two sides that
    cross at different token strides may be taken to share what they do not."""
    D, lib = 16, _lib.load()
    ref = lambda at, st, sh, n: _elements(at, st, sh, n, T, D)  # noqa: E731
    found = [0, 0, 0]
    for T, a, b in _layouts():
        x = torch.empty(T, 1, D, dtype=torch.bfloat16)
        where = [(FAKE + 2 * at, st, sh) for at, st, sh, _ in (a, b)]
        own = [len(set(ref(*s))) < len(ref(*s)) for s in (a, b)]
        for w, s, want in zip(where, (a, b), own):
            assert ops._share(w, w, s[3], s[3], x) == want
        cross, got = bool(set(ref(*a)) & set(ref(*b))), ops._share(*where, a[3], b[3], x)
        apart = min(ref(*a)) > max(ref(*b)) or min(ref(*b)) > max(ref(*a))
        assert got == cross or (got and T > 1 and a[1] != b[1] and not apart)
        found[0 if any(own) else 1 if got else 2] += 1
        if any(own) or got:
            c = _qk_args()
            c.total_len, c.head_dim, c.n_q_heads, c.n_k_heads = T, D, a[3], b[3]
            for n, w in zip("qk", where):
                setattr(c, n, w[0])
                setattr(c, n + "_out", w[0])
                for f in (n, n + "o"):
                    setattr(c, f + "_stride_t", w[1])
                    setattr(c, f + "_stride_h", w[2])
            _refused("dsalt_qk_norm_rope", c, 1)
            g = _lib.QkNormRopeBwdArgs(c, FAKE << 8, 4096, 64, FAKE << 8, 4096, 64, FAKE, FAKE)
            g.base.q = g.base.k = FAKE << 9
            g.workspace, g.workspace_bytes = FAKE, 1 << 30
            _refused("dsalt_qk_norm_rope_bwd", g, 1)
    assert min(found) > 100, found


def test_qk_outputs_over_what_is_read_are_refused():
    for field, at, stride in (("q_out", FAKE + 128, 256), ("k_out", FAKE + 10 * 4 * 64 * 2 - 16, 128), ("q_out", FAKE - 16, 512)):
        a = _qk_args()
        a.k, a.q_out, a.k_out = 2 * FAKE, 4 * FAKE, 8 * FAKE
        setattr(a, field, at)
        setattr(a, field[0] + "o_stride_t", stride)
        _refused("dsalt_qk_norm_rope", a, 1)
        b = _qk_bwd_args()
        b.base = a
        b.base.q = b.base.k = 16 * FAKE
        b.workspace_bytes = 1 << 30
        _refused("dsalt_qk_norm_rope_bwd", b, 1)  # over dq, dk


def test_heads_that_share_elements_are_not_written_in_place(monkeypatch):
    """Refused before anything is launched, whichever way they share; what lies apart in one buffer is taken."""
    launched = []
    monkeypatch.setattr(ops, "_on", lambda *ts: 0)
    monkeypatch.setattr(ops, "_call", lambda name, a, at, *more: launched.append(name))
    w, tab = torch.ones(64), torch.zeros(8, 64)
    x = torch.zeros(8192)
    where = dict(pos=torch.zeros(6, dtype=torch.int32), inplace=True)
    chain, rows = x.as_strided((6, 2, 64), (64, 64, 1)), x[:6 * 256].view(6, 4, 64)
    for q, k in ((chain, None), (None, chain), (rows, rows), (rows[:, :3], rows[:, 2:]), (rows[:, :2], x[64:64 + 6 * 256].view(6, 4, 64)[:, :2]),
                 (rows, x[6 * 256 - 64:6 * 512 - 64].view(6, 4, 64)), (rows[:, :1].expand(6, 2, 64), None)):
        with pytest.raises(ValueError, match="share"):
            ops.qk_norm_rope(q, k, w if q is not None else None, w if k is not None else None, tab, tab, **where)
    assert not launched
    for q, k in ((rows[:, :2], rows[:, 2:]), (rows[:, ::2], rows[:, 1::2]), (rows[:, 3:], rows[:, :3]), (rows, x[6 * 256:6 * 512].view(6, 4, 64)),
                 (x[:6 * 256].view(4, 6, 64).transpose(0, 1), x[6 * 256:6 * 512].view(4, 6, 64).transpose(0, 1))):
        assert ops.qk_norm_rope(q, k, w, w, tab, tab, **where) == (q, k)
    assert len(launched) == 5


def test_qk_without_heads(monkeypatch):
    """No heads on either side: nothing to do, no workspace, and gradients of the weights that are zeros (as beside a side that
    has heads)."""
    lib = _lib.load()
    for n_rows in (0, 1, 10):
        b = _lib.QkNormRopeBwdArgs(_qk_args())
        b.base.total_len, b.base.n_q_heads, b.base.n_k_heads = n_rows, 0, 0
        assert lib.dsalt_qk_norm_rope_bwd_workspace_bytes(ctypes.byref(b)) == 0
        assert lib.dsalt_qk_norm_rope_bwd(ctypes.byref(b), None) == 0 and lib.dsalt_qk_norm_rope(ctypes.byref(b.base), None) == 0
    for q_heads, k_heads in ((0, 3), (3, 0)):
        b = _qk_bwd_args()
        b.base.n_q_heads, b.base.n_k_heads = q_heads, k_heads
        assert lib.dsalt_qk_norm_rope_bwd_workspace_bytes(ctypes.byref(b)) > 0
    monkeypatch.setattr(ops, "_on", lambda *ts: 0)
    monkeypatch.setattr(ops, "_set_workspace", lambda a, need, at: None)
    monkeypatch.setattr(ops, "_call", lambda name, a, at, *more: None)
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *s, **kw: empty(*s, **kw).fill_(9))  # (as memory that is not written)
    q, w, tab = torch.zeros(10, 0, 64), torch.ones(64), torch.zeros(8, 64)
    where = dict(pos=torch.zeros(10, dtype=torch.int32))
    dq, dk, dqw, dkw = ops.qk_norm_rope_backward(q, None, q, None, w, None, tab, tab, **where)
    assert dq.shape == q.shape and dk is None and dkw is None and not dqw.any()
    k = torch.zeros(10, 2, 64)
    assert not ops.qk_norm_rope_backward(q, k, q, k, w, w, tab, tab, **where)[2].any()
    assert not ops.qk_norm_rope_backward(k, q, k, q, w, w, tab, tab, **where)[3].any()


def test_null_structs_and_empty_calls():
    lib = _lib.load()
    for name in ("dsalt_cache4_write", "dsalt_cache4_read", "dsalt_cache4_attn", "dsalt_verify_rows", "dsalt_qk_norm_rope",
                 "dsalt_qk_norm_rope_bwd"):
        _refused(name, None, 1)
    assert lib.dsalt_cache_rows_held(None, None, None) == 1
    for name, make in (("dsalt_cache4_write", _write_args), ("dsalt_cache4_read", _read_args), ("dsalt_cache4_attn", _attn_args)):
        a = make()
        a.n_rows = 0
        assert getattr(lib, name)(ctypes.byref(a), None) == 0
    a = _qk_args()
    a.total_len = 0
    assert lib.dsalt_qk_norm_rope(ctypes.byref(a), None) == 0
    a = _verify_args()
    a.n_reqs = a.n_rows = 0
    assert lib.dsalt_verify_rows(ctypes.byref(a), None) == 0


@pytest.mark.parametrize("head_dim", [64, 128])
def test_attention_without_rows_needs_no_workspace(head_dim):
    lib = _lib.load()
    for cols in (1, 16, 64, 1 << 30 >> 6):
        for w_max in (0, 1, 512, 1 << 20, 0x7fffffff):
            for per in (1, 5, 0x7fffffff):
                a = _attn_args(_cache(head_dim=head_dim))
                a.n_rows, a.table_cols, a.table_stride, a.w_max, a.rows_per_req = 0, cols, cols, w_max, per
                assert lib.dsalt_cache4_attn_workspace_bytes(ctypes.byref(a)) == 0
                assert lib.dsalt_cache4_attn(ctypes.byref(a), None) == 0


def test_python_refuses_cpu_tensors_and_bad_arguments():
    c = ops.new_cache(2, 1, 64, device="cpu", bits=4)
    assert c.kv.shape == (2, 1, 64, 2, 32) and c.scale.shape == (2, 1, 64, 2, 2)
    i = torch.zeros(1, dtype=torch.int32)
    t, x, cu = torch.zeros((1, 2), dtype=torch.int32), torch.zeros((1, 1, 64)), torch.zeros(2, dtype=torch.int32)
    w, tab = torch.ones(64), torch.zeros((4, 64))
    for call in (lambda: ops.cache_write_(x, x, c, torch.zeros((1, 4), dtype=torch.int32)),
                 lambda: ops.cache_read(c, t, cu, n_rows=1),
                 lambda: ops.cache_attention(x, c, t, i, i, i, torch.zeros((1, 1, 1, 0), dtype=torch.int32)),
                 lambda: ops.cache_rows_(i, i, t, i, torch.zeros(2, dtype=torch.int64), 1, held=i),
                 lambda: ops.qk_norm_rope(x, x, w, w, tab, tab, pos=i),
                 lambda: ops.qk_norm_rope_backward(x, x, x, x, w, w, tab, tab, pos=i),
                 lambda: qk_norm_rope(x, x, w, w, tab, tab, pos=i),
                 lambda: ops.verify_rows(x[0], i.long(), cu, torch.zeros(1), torch.zeros(1))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="bits"):
        ops.new_cache(2, 1, 64, device="cpu", bits=2)


def test_argument_checks(monkeypatch):
    """Shapes and types that do not fit are argument errors (the checks come before anything runs)."""
    monkeypatch.setattr(ops, "_on", lambda *ts: 0)
    c = ops.new_cache(4, 2, 64, block_tokens=16, device="cpu", bits=4)
    i, lmk = torch.zeros(3, dtype=torch.int32), torch.zeros((4, 3, 1, 2), dtype=torch.int32)
    good = dict(q=torch.zeros(3, 4, 64), cache=c, table=torch.zeros((3, 2), dtype=torch.int32), req=i, pos=i, w=i, lmk_idx=lmk)
    for bad in (dict(q=torch.zeros(3, 4, 128)), dict(q=torch.zeros(3, 3, 64)), dict(rows_per_req=0), dict(lmk_idx=lmk[:2]),
                dict(cache=c._replace(kv=c.kv[..., :16])), dict(cache=c._replace(kv=c.kv.view(torch.int8))),
                dict(cache=c._replace(scale=c.scale[:2])), dict(cache=c._replace(scale=c.scale.float())),
                dict(cache=c._replace(kv=c.kv.transpose(0, 1)))):
        with pytest.raises(ValueError):
            ops.cache_attention(**{**good, **bad})
    q, k, w, tab = torch.zeros(5, 4, 64), torch.zeros(5, 2, 64), torch.ones(64), torch.zeros((8, 64))
    qk = dict(q=q, k=k, q_weight=w, k_weight=w, cos=tab, sin=tab, pos=torch.zeros(5, dtype=torch.int32))
    for bad in (dict(q=None, k=None), dict(k=k[:4]), dict(k=k[..., :32]), dict(q_weight=None), dict(k_weight=w[:32]),
                dict(cos=tab.half()), dict(sin=tab[:4]), dict(cos=tab[:, :32], sin=tab[:, :32]), dict(pos=None),
                dict(cu_seqlens=torch.tensor([0, 5])), dict(pos=torch.zeros(4, dtype=torch.int32)),
                dict(pos=None, cu_seqlens=torch.tensor([0])), dict(pos=None, cu_seqlens=torch.tensor([0, 5]), max_seqlen=9),
                dict(q=q.transpose(1, 2).contiguous().transpose(1, 2), inplace=True), dict(q=torch.zeros(5, 4, 65)[..., 1:], inplace=True)):
        with pytest.raises(ValueError):
            ops.qk_norm_rope(**{**qk, **bad})
    for bad in (dict(q=q.double(), k=k.double()), dict(q_weight=w.half())):
        with pytest.raises(TypeError):
            ops.qk_norm_rope(**{**qk, **bad})
    for bad in (dict(dq=None), dict(dk=k[:4])):
        with pytest.raises(ValueError):
            ops.qk_norm_rope_backward(**{**dict(dq=q, dk=k), **qk, **bad})
    x, tok, u, v = torch.zeros(6, 10), torch.zeros(6, dtype=torch.int64), torch.zeros(6), torch.zeros(2)
    ver = dict(logits=x, tokens=tok, cu=torch.tensor([0, 3, 6]), u=u, v=v)
    for bad in (dict(logits=x[0]), dict(logits=torch.zeros(6, 0)), dict(draft_logits=x[:5]), dict(draft_logits=x.half()), dict(tokens=tok[:5]),
                dict(u=u[:5]), dict(v=u), dict(temperature=torch.ones(6)), dict(draft_temperature=torch.ones(2, 1)),
                dict(cu=torch.zeros((2, 2))), dict(logits=torch.zeros(1, 4).expand((1 << 22) + 1, 4))):
        with pytest.raises(ValueError):
            ops.verify_rows(**{**ver, **bad})
    for bad in (dict(tokens=tok.float()), dict(u=u.half()), dict(v=v.double())):
        with pytest.raises(TypeError):
            ops.verify_rows(**{**ver, **bad})


@pytest.fixture
def norm_calls(monkeypatch):
    """A layer of two heads of 64 whose norm-and-rotation calls are noted in place of running."""
    calls = []
    monkeypatch.setattr(ops, "_on", lambda *ts: 0)
    monkeypatch.setattr(ops, "_call", lambda name, a, at, *more: calls.append(a))
    layer = DSALTAttention(128, 2, 2, 8, 4, 32, n_kv_heads=1, qk_norm=True)
    layer.run = lambda q, k: layer._norm_rope(q, k, *layer._rope_tables32(), torch.tensor([0, len(q)], dtype=torch.int32), len(q))
    return layer, calls


@pytest.mark.parametrize("training,grad", [(True, True), (True, False), (False, True), (False, False)])
def test_layer_writes_over_its_own_projection_alone(norm_calls, training, grad):
    layer, calls = norm_calls
    layer.train(training)
    x = torch.randn(5, 3, 64)
    with torch.set_grad_enabled(grad):
        q, k = layer.run(x[:, :2], x[:, 2:])
    a, = calls
    over = not training and not grad  # the branch whose queries and keys are columns of a buffer that it made
    assert (a.q_out == a.q == x.data_ptr()) == over and (a.k_out == a.k) == over
    assert (q.data_ptr() == x.data_ptr()) == over


@pytest.mark.parametrize("grad", [True, False])
def test_layer_takes_each_norms_own_eps(norm_calls, grad):
    layer, calls = norm_calls
    layer.eval()
    layer.k_norm.eps = 0.5
    x = torch.randn(5, 3, 64)
    with torch.set_grad_enabled(grad):
        layer.run(x[:, :2], x[:, 2:])
        assert [(a.n_q_heads, a.n_k_heads, a.eps) for a in calls] == [(2, 0, pytest.approx(1e-6)), (0, 1, 0.5)]
        del calls[:]
        layer.q_norm.eps = 0.5
        layer.run(x[:, :2], x[:, 2:])
        assert [(a.n_q_heads, a.n_k_heads, a.eps) for a in calls] == [(2, 1, 0.5)]
        del calls[:]
        layer.k_norm.to(torch.bfloat16)  # weights of two types are two calls as well
        layer.run(x[:, :2], x[:, 2:])
        assert [(a.n_q_heads, a.n_k_heads, a.weight_dtype) for a in calls] == [(2, 0, 0), (0, 1, 1)]


class _Double(torch.nn.Module):
    def forward(self, x):
        return (2 * x).double()


def _rotated(x, tab, pos):
    half = x.shape[-1] // 2
    return x * tab[0][pos][:, None] + torch.cat([-x[..., half:], x[..., :half]], -1) * tab[1][pos][:, None]


@pytest.mark.parametrize("training,grad", [(True, True), (True, False), (False, True), (False, False)])
def test_layer_calls_a_norm_in_the_place_of_its_own(norm_calls, training, grad):
    """Another module, a replaced ``forward``, hooks of each kind: the norm is called and its side rotated; the other stays with the
    kernel."""
    layer, calls = norm_calls
    layer.train(training)
    x = torch.randn(5, 3, 64)
    tab, pos, seen = layer._rope_tables32(), torch.tensor([0, 1, 2, 0, 1]), []
    before = x.clone()

    def run():
        del calls[:]
        with torch.set_grad_enabled(grad):
            return layer._norm_rope(x[:, :2], x[:, 2:], *tab, torch.tensor([0, 3, 5], dtype=torch.int32), 3)

    own = layer.q_norm
    layer.q_norm = _Double()
    q, _ = run()
    assert q.dtype == x.dtype and torch.equal(q, _rotated(2 * x[:, :2], tab, pos)) and [(a.n_q_heads, a.n_k_heads) for a in calls] == [(0, 1)]
    layer.q_norm, layer.k_norm = layer.k_norm, _Double()
    _, k = run()
    assert torch.equal(k, _rotated(2 * x[:, 2:], tab, pos)) and [(a.n_q_heads, a.n_k_heads) for a in calls] == [(2, 0)]
    layer.q_norm, layer.k_norm = own, type(own)(64)
    want = _rotated(own.forward(x[:, :2]).detach(), tab, pos)
    for add in (lambda: own.register_forward_hook(lambda m, i, o: seen.append(1)), lambda: own.register_forward_pre_hook(lambda m, i: seen.append(1)),
                lambda: own.register_full_backward_hook(lambda m, i, o: None), lambda: own.register_full_backward_pre_hook(lambda m, o: None)):
        handle = add()
        q, _ = run()
        assert torch.allclose(q, want, atol=1e-6) and [(a.n_q_heads, a.n_k_heads) for a in calls] == [(0, 1)]
        handle.remove()
        run()
        assert [(a.n_q_heads, a.n_k_heads) for a in calls] == [(2, 1)]
        x.copy_(before)
    assert len(seen) == 2
    own.forward = lambda t: 0 * t
    assert not run()[0].any() and len(calls) == 1
    with pytest.raises(ValueError, match="positions"):
        layer._norm_rope(x[:, :2], x[:, 2:], *(t[:4] for t in tab), torch.tensor([0, 5], dtype=torch.int32), 5)
    del own.forward
    own.eps = None  # the type's own, which the module knows
    run()
    assert [(a.n_q_heads, a.n_k_heads) for a in calls] == [(0, 1)]


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("which", ["heads", "weight"])
def test_layer_drops_no_forward_mode_tangents(norm_calls, training, which):
    """Without autograd as with it: the norm and rotation has no forward-mode derivative, and says so."""
    layer, calls = norm_calls
    layer.train(training)
    x = torch.randn(5, 3, 64)
    with fwAD.dual_level():
        if which == "heads":
            x = fwAD.make_dual(x, torch.ones_like(x))
        else:
            w = layer.k_norm.weight
            del layer.k_norm.weight
            layer.k_norm.weight = fwAD.make_dual(w.detach(), torch.ones_like(w))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                layer.run(x[:, :2], x[:, 2:])


def test_head_sizes_that_the_norm_does_not_take_are_refused_when_built():
    size = dict(n_heads=2, n_min=2, n_max=8, k_lmk=4, max_seq_len=32)
    for d in (72, 8, 24, 272):
        with pytest.raises(ValueError, match="head_dim"):
            DSALTAttention(2 * d, **size, qk_norm=True)
        with pytest.raises(ValueError, match="head_dim"):
            DSALTLMHeadModel.from_config(DSALTConfig(vocab_size=16, d_model=2 * d, n_layers=1, **size, qk_norm=True))
        assert DSALTAttention(2 * d, **size).head_dim == d  # (as without the norm)
    for d in (16, 48, 128, 256):
        assert DSALTAttention(2 * d, **size, qk_norm=True).k_norm.weight.shape == (d,)


def test_config_carries_qk_norm(tmp_path):
    c = DSALTConfig(vocab_size=64, d_model=64, n_layers=1, n_heads=2, n_min=2, n_max=8, k_lmk=4, max_seq_len=32, qk_norm=True)
    c.save(tmp_path / "c.json")
    assert DSALTConfig.load(tmp_path / "c.json").qk_norm and not DSALTConfig.from_dict({**c.to_dict(), "qk_norm": False}).qk_norm


# ------------------------------------------------------------------------ the oracles themselves
def test_oracle_rounds_to_the_nearest_code():
    x = np.linspace(-8, 8, 20001)
    y = O4.e2m1(x)
    assert set(np.abs(y)) == set(O4.GRID)
    for v, r in zip(x, y):
        assert abs(r - np.clip(v, -6, 6)) <= np.abs(np.sign(v or 1) * O4.GRID - np.clip(v, -6, 6)).min()
    ties = {0.25: 0, 0.75: 1, 1.25: 1, 1.75: 2, 2.5: 2, 3.5: 4, 5: 4, 7: 6}
    assert O4.e2m1(np.array(list(ties))).tolist() == list(ties.values())


def test_oracle_scale_is_the_least_and_bounds_the_error():
    r = np.random.RandomState(0)
    for top in (7.0, 7.0000001, 1.0, 3.4e38, 1e-45, 0.0, 6.9, 2.0 ** -124, 3.5):
        x = r.uniform(-1, 1, 32) * top
        x[0] = top
        e = O4.exponent_of(x)
        assert top <= 7 * 2.0 ** e or e == 125
        assert e == -126 or top > 7 * 2.0 ** (e - 1)
        assert (np.abs(O4.block(x)[0] - x) <= 2.0 ** e).all() or e == 125
    assert np.isnan(O4.block(np.array([1.0] * 31 + [np.inf]))[0]).all()


def test_oracle_verification_draws_from_the_target():
    """Over even grids of u and v and draws of the draft in proportion to q, the first token of a request falls in the target's
    proportions, whatever the draft's."""
    p, q = np.array([0.4, 0.1, 0.3, 0.2]), np.array([0.1, 0.5, 0.15, 0.25])
    n, count = 60, np.zeros(4)
    for x in range(4):
        for i in range(n):
            for j in range(n):
                a, out = O4.verify(np.log(np.stack([p, p])), [9, x], [0, 2], [(i + 0.5) / n] * 2, [(j + 0.5) / n], np.log(np.stack([q, q])),
                                   [1.0], [1.0])
                count[out[0]] += q[x] / n ** 2
                assert a[0] == (out[1] >= 0) and (a[0] == 0 or out[0] == x)
    assert np.allclose(count, p, atol=2 / n)
    # without the draft's logits
    count[:] = 0
    for x in range(4):
        for i in range(n):
            for j in range(n):
                out = O4.verify(np.log(np.stack([p, p])), [9, x], [0, 2], [(i + 0.5) / n] * 2, [(j + 0.5) / n], None, [1.0], [1.0])[1]
                count[out[0]] += 0.25 / n ** 2
    assert np.allclose(count, p, atol=2 / n)


def test_oracle_gradients_are_the_differences():
    r = np.random.RandomState(1)
    T, H, D, eps = 5, 3, 32, 1e-3
    x, w, d = r.randn(T, H, D), 1 + 0.2 * r.randn(D), r.randn(T, H, D)
    cos, sin = r.randn(4, D), r.randn(4, D)
    pos = np.array([0, 3, -1, 4, 2])  # two rows without a position
    dx, dw, _, _ = OQ.backward(d, x, w, pos, cos, sin, eps)
    assert not dx[2].any() and not dx[3].any()
    h = 1e-5
    for _ in range(10):
        vx, vw = r.randn(*x.shape), r.randn(D)
        f = [(OQ.forward(x + s * h * vx, w + s * h * vw, pos, cos, sin, eps)[0] * d).sum() for s in (1, -1)]
        assert abs((f[0] - f[1]) / (2 * h) - (dx * vx).sum() - (dw * vw).sum()) < 1e-6
