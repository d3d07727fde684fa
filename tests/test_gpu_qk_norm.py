"""Norms of query and key heads with the rotation, and their gradients, on the GPU against the float64 oracle, and the layer
that uses them.

Tolerances, from the arithmetic (u = 2^-24, D terms a head).  The sum of squares and its root are off by (D + 8) u / 2 of
themselves in any order of the sum, an output then by (D / 2 + 12) u of |n1 cos| + |n2 sin| (``reach``), and by half a step of its type.  A
gradient of an input: (2 D + 24) u of the sizes it is summed from.  A weight's gradient over N rows and heads, in any
order: (N + D / 2 + 16) u of the sum of sizes."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from dsalt_amd import ops
from dsalt_amd.kernels import qk_norm_rope
from dsalt_amd.model import DSALTConfig, DSALTLMHeadModel
from dsalt_amd.modules import DSALTAttention
from oracle import qk_norm as OQ

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
E = 2.0 ** -24


def f64(t):
    return t.detach().cpu().double().numpy()


def _case(T, H, G, D, dt, seed, max_pos=64, wt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, H + 2 * G, D, generator=g) * torch.exp2(2 * torch.randn(T, 1, 1, generator=g))).to(dt)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(wt) for _ in range(2)]
    tab = [torch.randn(max_pos, D, generator=g) for _ in range(2)]  # (any tables, both halves their own)
    d = [torch.randn(T, n, D, generator=g).to(dt) for n in (H, G)]
    return x, w, tab, d


def _check(x, H, G, w, tab, d, where, pos, eps=1e-6, inplace=True):
    """Forward (new outputs and in place) and backward of q = x[:, :H], k = x[:, H:H + G], views of one buffer."""
    dt, D, T = x.dtype, x.shape[2], x.shape[0]
    dev = x.to(DEV)
    a = (*(t.to(DEV) for t in w), *(t.to(DEV) for t in tab))
    q, k = dev[:, :H], dev[:, H:H + G]
    out = ops.qk_norm_rope(q, k, *a, eps=eps, **where)
    grads = ops.qk_norm_rope_backward(d[0].to(DEV), d[1].to(DEV), q, k, *a, eps=eps, **where)
    again = ops.qk_norm_rope_backward(d[0].to(DEV), d[1].to(DEV), q, k, *a, eps=eps, **where)
    assert all(torch.equal(p, r) for p, r in zip(grads, again))
    assert torch.equal(dev.cpu(), x)  # the inputs stay
    cos, sin = (f64(t) for t in tab)
    tiny = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -126
    for i, (lo, hi) in enumerate(((0, H), (H, H + G))):
        xf, wf = f64(x[:, lo:hi]), f64(w[i])
        ref, reach = OQ.forward(xf, wf, pos, cos, sin, eps)
        tol = (D / 2 + 12) * E * reach + U[dt] * np.abs(ref) + tiny
        assert out[i].dtype == dt and (np.abs(f64(out[i]) - ref) <= tol).all()
        dx, dw, ax, aw = OQ.backward(f64(d[i]), xf, wf, pos, cos, sin, eps)
        assert grads[i].dtype == dt and (np.abs(f64(grads[i]) - dx) <= (2 * D + 24) * E * ax + U[dt] * np.abs(dx) + tiny).all()
        N = T * (hi - lo)
        assert grads[2 + i].dtype == torch.float32 and (np.abs(f64(grads[2 + i]) - dw) <= (N + D / 2 + 16) * E * aw + 1e-30).all()
    if inplace:
        got = ops.qk_norm_rope(q, k, *a, eps=eps, inplace=True, **where)
        assert got[0] is q and got[1] is k and torch.equal(dev[:, H + G:].cpu(), x[:, H + G:])
        on = torch.from_numpy((pos >= 0) & (pos < len(cos)))
        for i, (lo, hi) in enumerate(((0, H), (H, H + G))):
            assert torch.equal(dev[:, lo:hi].cpu(), torch.where(on[:, None, None], out[i].cpu(), x[:, lo:hi]))
    return out, grads


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,G,D", [(1, 1, 1, 64), (1, 16, 2, 128), (37, 4, 4, 64), (64, 3, 1, 32), (50, 5, 2, 16), (33, 4, 2, 96), (20, 2, 2, 80),
                                     (9, 2, 1, 256), (130, 8, 2, 48)])
def test_follows_the_oracle(dt, T, H, G, D):
    """By sequence, with an empty one, and by position, rows outside the tables among them."""
    x, w, tab, d = _case(T, H, G, D, dt, T + D, max_pos=max(T, 3))
    cut = [0, T // 3, T // 3, T - T // 4, T]
    _check(x, H, G, w, tab, d, dict(cu_seqlens=torch.tensor(cut, device=DEV)), OQ.positions(T, cut))
    r = np.random.RandomState(T)
    pos = r.randint(-2, len(tab[0]) + 2, T)
    _check(x, H, G, w, tab, d, dict(pos=torch.tensor(pos, device=DEV)), pos)


@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float16])
def test_weights_of_16_bits(wt):
    x, w, tab, d = _case(21, 4, 2, 64, torch.bfloat16, 3, wt=wt)
    _check(x, 4, 2, w, tab, d, dict(cu_seqlens=torch.tensor([0, 21], device=DEV)), np.arange(21))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_many_rows(dt):
    """Rows past what a pass of the blocks takes, several heads a wave, and rows of no sequence at both ends."""
    T = 9001
    x, w, tab, d = _case(T, 6, 2, 64, dt, 1, max_pos=5000)
    cut = [3, 4000, 4001, 8999]
    out, grads = _check(x, 6, 2, w, tab, d, dict(cu_seqlens=torch.tensor(cut, device=DEV), max_seqlen=4998), OQ.positions(T, cut))
    assert not out[0][:3].any() and not out[1][8999:].any() and not grads[0][:3].any()


def test_positions_past_32_bits_and_other_types():
    x, w, tab, d = _case(5, 2, 1, 64, torch.float32, 2)
    big = [3, (1 << 32) + 3, 1 << 31, -(1 << 40), 63]
    _check(x, 2, 1, w, tab, d, dict(pos=torch.tensor(big, device=DEV)), np.array([3, -1, -1, -1, 63]))
    a = (x.to(DEV)[:, :2], x.to(DEV)[:, 2:3], *(t.to(DEV) for t in w + tab))
    p = torch.tensor([3, 9, 1, 0, 63], device=DEV)
    ref = ops.qk_norm_rope(*a, pos=p)
    for other in (p.int(), p.short(), torch.stack([p, p], 1)[:, 0]):
        assert all(torch.equal(s, t) for s, t in zip(ops.qk_norm_rope(*a, pos=other), ref))


def test_zeros_infinities_and_eps():
    """Rows of zeros (eps alone holds the root; without it the formula has no value), infinities and NaN stay in their head."""
    x, w, tab, d = _case(6, 3, 1, 64, torch.float32, 4)
    x[1] = 0
    pos = np.array([0, 1, 2, 3, 4, -1])
    _check(x, 3, 1, w, tab, d, dict(pos=torch.tensor(pos, device=DEV)), pos)
    a = (*(t.to(DEV) for t in w + tab),)
    y = x.clone()
    y[2, 1, 5], y[3, 0, 63], y[5] = float("inf"), float("nan"), float("nan")
    where = dict(pos=torch.tensor(pos, device=DEV), eps=0.0)
    q, k = ops.qk_norm_rope(y.to(DEV)[:, :3], y.to(DEV)[:, 3:4], *a, **where)
    bad = torch.zeros(6, 3, dtype=torch.bool)
    bad[1] = bad[2, 1] = bad[3, 0] = True
    assert torch.equal(q.isfinite().all(-1).cpu(), ~bad) and not q[5].any() and not k[5].any()
    dq, dk, dqw, _ = ops.qk_norm_rope_backward(d[0].to(DEV), d[1].to(DEV), y.to(DEV)[:, :3], y.to(DEV)[:, 3:4], *a, **where)
    assert torch.equal(dq.isfinite().all(-1).cpu(), ~bad) and not dq[5].any()
    fine = torch.tensor([0, 4, 5], device=DEV)  # a row without a position adds nothing, whatever it holds and eps is
    part = ops.qk_norm_rope_backward(d[0].to(DEV)[fine], d[1].to(DEV)[fine], y.to(DEV)[fine][:, :3], y.to(DEV)[fine][:, 3:4], *a,
                                     pos=where["pos"][fine], eps=0.0)
    assert all(t.isfinite().all() for t in part)
    large = x * 1e10  # squares stay within float32 (1e10^2 64)
    _check(large, 3, 1, w, tab, d, dict(pos=torch.tensor(pos, device=DEV)), pos)


def test_one_side_alone_and_layouts():
    x, w, tab, d = _case(30, 4, 2, 64, torch.bfloat16, 5)
    a = [t.to(DEV) for t in tab]
    where = dict(cu_seqlens=torch.tensor([0, 11, 30], device=DEV))
    q, k = x.to(DEV)[:, :4], x.to(DEV)[:, 4:6]
    wq, wk = (t.to(DEV) for t in w)
    ref = ops.qk_norm_rope(q, k, wq, wk, *a, **where)
    g = ops.qk_norm_rope_backward(d[0].to(DEV), d[1].to(DEV), q, k, wq, wk, *a, **where)
    one, none = ops.qk_norm_rope(q, None, wq, None, *a, **where)
    assert none is None and torch.equal(one, ref[0])
    none, one = ops.qk_norm_rope(None, k, None, wk, *a, **where)
    assert none is None and torch.equal(one, ref[1])
    got = ops.qk_norm_rope_backward(None, d[1].to(DEV), None, k, None, wk, *a, **where)
    assert got[0] is None and got[2] is None and torch.equal(got[1], g[1])
    # the heads of one side alone are cut over the waves otherwise: the same terms in another order, each sum within the bound
    # of any order, (N + D / 2 + 16) u of the sum of sizes, of the exact one, and so twice that of each other
    aw = OQ.backward(f64(d[1]), f64(k), f64(wk), OQ.positions(30, [0, 11, 30]), *(f64(t) for t in tab), 1e-6)[3]
    assert (np.abs(f64(got[3]) - f64(g[3])) <= 2 * (60 + 32 + 16) * E * aw).all()
    odd = torch.zeros(30 * 4 * 64 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(30, 4, 64)
    odd.copy_(q)
    wide = torch.cat([wq, wq])[1::2].new_zeros(129)[1:65].copy_(wq)  # off 16 bytes
    for y in (odd, q.transpose(0, 1).contiguous().transpose(0, 1), q.transpose(1, 2).contiguous().transpose(1, 2)):
        for ww in (wq, wide):
            assert torch.equal(ops.qk_norm_rope(y, k, ww, wk, *(t.T.contiguous().T for t in a), **where)[0], ref[0])
        assert torch.equal(ops.qk_norm_rope_backward(d[0].to(DEV).float(), d[1].to(DEV), y, k, wq, wk, *a, **where)[0], g[0])
    for T in (0,):
        e = ops.qk_norm_rope(q[:0], k[:0], wq, wk, *a, cu_seqlens=torch.tensor([0, 0], device=DEV))
        assert e[0].shape == (0, 4, 64)
        e = ops.qk_norm_rope_backward(q[:0], k[:0], q[:0], k[:0], wq, wk, *a, cu_seqlens=torch.tensor([0, 0], device=DEV))
        assert not e[2].any() and not e[3].any()


def test_gradients_are_the_differences():
    """Directional differences of the float32 forward at two steps: their own distance bounds what the curve leaves, the rounding of
    the outputs the rest."""
    T, H, G, D = 12, 3, 2, 64
    x, w, tab, d = _case(T, H, G, D, torch.float32, 7)
    x = x / x.abs().amax((1, 2), keepdim=True)
    pos = np.arange(T) - 1
    where = dict(pos=torch.tensor(pos, device=DEV))
    a = [t.to(DEV) for t in tab]
    wd = [t.to(DEV) for t in w]
    grads = ops.qk_norm_rope_backward(d[0].to(DEV), d[1].to(DEV), x.to(DEV)[:, :H], x.to(DEV)[:, H:H + G], *wd, *a, **where)
    g = torch.Generator().manual_seed(1)
    vx, vw = torch.randn(x.shape, generator=g), [torch.randn(D, generator=g) for _ in range(2)]

    def value(s):
        y = (x + s * vx).to(DEV)
        out = ops.qk_norm_rope(y[:, :H], y[:, H:H + G], *(p + s * q.to(DEV) for p, q in zip(wd, vw)), *a, **where)
        return sum((f64(o) * f64(e)).sum() for o, e in zip(out, d))

    def diff(h):
        return (value(h) - value(-h)) / (2 * h)
    h = 2.0 ** -8
    noise = sum((np.abs(f64(d[i])) * OQ.forward(f64(x[:, lo:hi]), f64(w[i]), pos, *(f64(t) for t in tab), 1e-6)[1]).sum() * (D / 2 + 16) * E
                for i, (lo, hi) in enumerate(((0, H), (H, H + G)))) / h
    want = (f64(grads[0]) * f64(vx[:, :H])).sum() + (f64(grads[1]) * f64(vx[:, H:H + G])).sum() + sum(
        (f64(grads[2 + i]) * f64(vw[i])).sum() for i in range(2))
    near, far = diff(h), diff(2 * h)
    assert abs(near - want) <= abs(near - far) + noise and abs(near - far) < 0.1 * abs(want)


# ------------------------------------------------------------------------ autograd, the layer and the model
def _torch_norm_rope(q, k, wq, wk, cos, sin, pos, eps):
    out = []
    for x, w in ((q, wq), (k, wk)):
        n = (x.double() / (x.double().pow(2).mean(-1, keepdim=True) + eps).sqrt()) * w.double()
        half = n.shape[-1] // 2
        rot = torch.cat([-n[..., half:], n[..., :half]], -1)
        out.append((n * cos.double()[pos][:, None] + rot * sin.double()[pos][:, None]).to(x.dtype))
    return out


def test_autograd():
    T, H, G, D = 40, 4, 2, 64
    x, w, tab, d = _case(T, H, G, D, torch.float32, 8)
    cu, pos = torch.tensor([0, 15, T], device=DEV), torch.cat([torch.arange(15), torch.arange(T - 15)]).to(DEV)
    res = []
    for own in (True, False):
        y = x.to(DEV).requires_grad_()
        ws = [t.to(DEV).requires_grad_() for t in w]
        t = [t.to(DEV) for t in tab]
        q, k = (qk_norm_rope(y[:, :H], y[:, H:H + G], *ws, *t, cu_seqlens=cu) if own else
                _torch_norm_rope(y[:, :H], y[:, H:H + G], *ws, *t, pos, 1e-6))
        ((q * d[0].to(DEV)).sum() + (k * d[1].to(DEV)).sum()).backward()
        res.append([y.grad, *(p.grad for p in ws)])
    for a, b in zip(*res):
        # both round sums of up to T H terms in float32 on the way
        assert (a - b).abs().max() <= (T * H + 2 * D + 40) * E * b.abs().max()
    y = x.to(DEV).requires_grad_()
    q, k = qk_norm_rope(y[:, :H], y[:, H:H + G], *(t.to(DEV) for t in w), *(t.to(DEV) for t in tab), pos=pos)
    g, = torch.autograd.grad(q.sum(), y, create_graph=True)  # one output unused; the weights without gradient
    assert not g[:, H:].any()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), y)


def test_autograd_of_one_side():
    """Queries or keys alone, forward and backward: the results that they have beside the others."""
    T, H, G, D = 20, 4, 2, 64
    x, w, tab, d = _case(T, H, G, D, torch.bfloat16, 12)
    cu, t = torch.tensor([0, T], device=DEV), [a.to(DEV) for a in tab]

    def run(q_on, k_on):
        y = x.to(DEV).requires_grad_()
        ws = [a.to(DEV).requires_grad_() for a in w]
        q, k = qk_norm_rope(y[:, :H] if q_on else None, y[:, H:H + G] if k_on else None, ws[0] if q_on else None, ws[1] if k_on else None,
                            *t, cu_seqlens=cu)
        sum((o * g.to(DEV)).sum() for o, g in ((q, d[0]), (k, d[1])) if o is not None).backward()
        return q, k, y.grad[:, :H], y.grad[:, H:H + G], *(a.grad for a in ws)

    both = run(True, True)
    q, none, gq, _, gw, nw = run(True, False)
    assert none is None and nw is None and torch.equal(q, both[0]) and torch.equal(gq, both[2])
    # (the weights' sums are cut by the heads that are there: up to T H products in another order, float32)
    assert (gw - both[4]).abs().max() <= 2 * (T * H + D) * E * T * H * 8
    none, k, _, gk, nw, gw = run(False, True)
    assert none is None and nw is None and torch.equal(k, both[1]) and torch.equal(gk, both[3])


def test_heads_that_share_elements_are_not_written():
    x = torch.randn(6, 1, 64, device=DEV)
    w, tab = torch.ones(64, device=DEV), [torch.ones(6, 64, device=DEV)] * 2
    cu = torch.tensor([0, 6], device=DEV)
    for q in (x.expand(6, 3, 64), x[:1].expand(6, 1, 64)):
        with pytest.raises(ValueError):
            ops.qk_norm_rope(q, None, w, None, *tab, cu_seqlens=cu, inplace=True)
        assert torch.equal(ops.qk_norm_rope(q, None, w, None, *tab, cu_seqlens=cu)[0],
                           ops.qk_norm_rope(q.contiguous(), None, w, None, *tab, cu_seqlens=cu)[0])


@pytest.mark.parametrize("D", [64, 96])
@pytest.mark.parametrize("mode", ["train", "eval with autograd", "inference"])
def test_layer(monkeypatch, mode, D):
    """DSALTAttention(qk_norm=True) with the norm and rotation replaced by torch operations: outputs and gradients agree to the
    layer's float32 tolerance (1e-4 of the largest; both sides then run the same kernels on inputs 2^-22 apart)."""
    torch.manual_seed(0)
    H, G = 4, 2
    layer = DSALTAttention(H * D, H, 8, 40, 6, 256, n_kv_heads=G, qkv_bias=True, qk_norm=True).to(DEV)
    with torch.no_grad():
        for n in (layer.q_norm, layer.k_norm):
            n.weight.add_(0.3 * torch.randn_like(n.weight))
    layer.train(mode == "train")
    cu = torch.tensor([0, 70, 150], dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(70), torch.arange(80)]).to(DEV)
    x = torch.randn(150, H * D, device=DEV)
    rope_cs = (layer.rope_cos[pos], layer.rope_sin[pos])

    def run(**kw):
        layer.zero_grad()
        y = x.clone().requires_grad_(mode != "inference")
        with torch.set_grad_enabled(mode != "inference"):
            out, _ = layer(y, cu, **kw)
        if mode == "inference":
            return [out]
        (out * torch.linspace(-1, 1, out.numel(), device=DEV).view_as(out)).sum().backward()
        return [out.detach(), y.grad, *(p.grad.clone() for p in layer.parameters() if p.grad is not None)]
    own, rows = run(), run(rope_cs=rope_cs)
    norm = lambda q, k, cos, sin, c, m: tuple(_torch_norm_rope(q, k, layer.q_norm.weight, layer.k_norm.weight, layer.rope_cos, layer.rope_sin,  # noqa: E731
                                                               pos, 1e-6))
    monkeypatch.setattr(layer, "_norm_rope", norm)
    ref = run()
    assert len(own) == len(ref) and (mode == "inference" or layer.q_norm.weight.grad is not None)
    for a, b, c in zip(own, rows, ref):
        assert torch.equal(a, b)
        assert (a - c).abs().max() <= 1e-4 * c.abs().max().clamp(min=1e-3)


def test_model_with_qk_norm():
    """The model runs, trains and answers with it; its weights travel in the state; without it nothing changes."""
    cfg = DSALTConfig(vocab_size=97, d_model=128, n_layers=2, n_heads=2, n_min=4, n_max=16, k_lmk=4, max_seq_len=64, n_kv_heads=1,
                      loss_fn="liger", qk_norm=True)
    torch.manual_seed(1)
    m = DSALTLMHeadModel.from_config(cfg).to(DEV)
    assert {k for k in m.state_dict() if "q_norm" in k} == {f"layers.{i}.attn.q_norm.weight" for i in range(2)}
    plain = DSALTLMHeadModel.from_config(DSALTConfig.from_dict({**cfg.to_dict(), "qk_norm": False}))
    assert not [k for k in plain.state_dict() if "_norm" in k and "attn." in k and ("q_norm" in k or "k_norm" in k)]
    ids = torch.randint(0, 97, (50,), device=DEV)
    cu = torch.tensor([0, 20, 50], dtype=torch.int32, device=DEV)
    m.train()
    for ckpt in (False, True):
        m.zero_grad()
        m(ids, cu, labels=ids, gradient_checkpointing=ckpt)["loss"].backward()
        assert all(l.attn.q_norm.weight.grad.isfinite().all() and l.attn.k_norm.weight.grad.any() for l in m.layers)
    m.eval()
    with torch.no_grad():
        a = m(ids, cu)["logits"]
        m.bfloat16()
        b = m(ids, cu)["logits"]
    assert a.isfinite().all() and (a - b.float()).abs().max() < 0.1 * a.abs().max()


def test_two_streams_and_captured():
    """Forward and backward on two streams at once, and captured and replayed on inputs of the moment."""
    cases = [_case(2000 + i, 8, 2, 128, torch.bfloat16, i, max_pos=2048) for i in range(2)]
    cases = [(x.to(DEV), [t.to(DEV) for t in w], [t.to(DEV) for t in tab], [t.to(DEV) for t in d], torch.tensor([0, 700, len(x)], device=DEV,
              dtype=torch.int32)) for x, w, tab, d in cases]

    def work(i):
        x, w, tab, d, cu = cases[i]
        a = (x[:, :8], x[:, 8:10], *w, *tab)
        return [*ops.qk_norm_rope(*a, cu_seqlens=cu, max_seqlen=2001), *ops.qk_norm_rope_backward(*d, *a, cu_seqlens=cu, max_seqlen=2001)]
    ref = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    res = [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                res[i].append(work(i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for got in res[i] for a, b in zip(got, ref[i]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(0)
    for rep in range(4):
        cases[0][0].copy_(torch.randn_like(cases[0][0]))
        ref = work(0)
        for t in outs:
            t.fill_(-9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, ref)), rep


def test_sides_without_heads():
    x, w, tab, d = _case(10, 2, 2, 64, torch.bfloat16, 6)
    a = [t.to(DEV) for t in w + tab]
    cu = torch.tensor([0, 10], device=DEV)
    q, k, dk = x.to(DEV)[:, :0], x.to(DEV)[:, 2:4], d[1].to(DEV)
    ref = ops.qk_norm_rope_backward(None, dk, None, k, None, *a[1:], cu_seqlens=cu)
    dq, dkey, dqw, dkw = ops.qk_norm_rope_backward(q, dk, q, k, *a, cu_seqlens=cu)
    assert dq.shape == q.shape and not dqw.any() and torch.equal(dkey, ref[1]) and torch.equal(dkw, ref[3])
    dq, dkey, dqw, dkw = ops.qk_norm_rope_backward(q, q, q, q, *a, cu_seqlens=cu)
    assert dq.shape == dkey.shape == q.shape and not dqw.any() and not dkw.any()
    assert ops.qk_norm_rope(q, q, *a, cu_seqlens=cu)[0].shape == q.shape


def test_written_in_place_beside_each_other():
    """Heads that lie apart in one buffer, in the layouts that are taken: the results of new outputs."""
    T, D = 300, 64
    x, w, tab, _ = _case(T, 4, 0, D, torch.bfloat16, 9, max_pos=T)
    a, cu = [t.to(DEV) for t in w + tab], torch.tensor([0, 100, T], device=DEV)
    heads_first = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    for split in (lambda t: (t[:, :3], t[:, 3:]), lambda t: (t[:, ::2], t[:, 1::2]), lambda t: (t[:, 2:], t[:, :1]),
                  lambda t: (heads_first(t)[:, :2], heads_first(t)[:, 2:])):
        q, k = split(x.to(DEV))
        ref = ops.qk_norm_rope(q, k, *a, cu_seqlens=cu)
        got = ops.qk_norm_rope(q, k, *a, cu_seqlens=cu, inplace=True)
        assert got[0] is q and got[1] is k and torch.equal(q, ref[0]) and torch.equal(k, ref[1])
    y = torch.zeros((T + 1) * D, device=DEV, dtype=torch.bfloat16)
    for q, k in ((y.as_strided((T, 2, D), (D, D, 1)), None), (y[:T * D].view(T, 1, D),) * 2):
        with pytest.raises(ValueError):
            ops.qk_norm_rope(q, k, a[0], a[1] if k is not None else None, *a[2:], cu_seqlens=cu, inplace=True)
    assert not y.any()


@pytest.mark.parametrize("grad", [False, True])
def test_layer_in_training_leaves_what_projections_return(grad):
    """With and without autograd: an output that a hook keeps, and the layer's input where a projection returns it."""
    torch.manual_seed(2)
    layer = DSALTAttention(128, 2, 4, 16, 4, 64, qk_norm=True).to(DEV).train()
    x, cu = torch.randn(40, 128, device=DEV), torch.tensor([0, 15, 40], dtype=torch.int32, device=DEV)
    kept = []
    layer.k_proj.register_forward_hook(lambda m, i, o: kept.append((o, o.detach().clone())))
    layer.q_proj = torch.nn.Identity()
    before = x.clone()
    with torch.set_grad_enabled(grad):
        out, _ = layer(x, cu)
    assert torch.equal(x, before) and all(torch.equal(o, c) for o, c in kept) and len(kept) == 1
    with torch.set_grad_enabled(not grad):
        assert torch.equal(layer(x, cu)[0], out)


@pytest.mark.parametrize("mode", ["train", "eval with autograd", "inference"])
def test_layer_with_two_eps(mode):
    """Each side by its own norm: the results of torch operations, to the layer's float32 tolerance (as test_layer)."""
    torch.manual_seed(3)
    H, G, D, T = 4, 2, 64, 90
    layer = DSALTAttention(H * D, H, 8, 40, 6, 256, n_kv_heads=G, qk_norm=True).to(DEV).train(mode == "train")
    layer.q_norm.eps, layer.k_norm.eps = 1e-6, 0.3
    x = torch.randn(T, H * D, device=DEV)
    cu, pos = torch.tensor([0, T], dtype=torch.int32, device=DEV), torch.arange(T, device=DEV)

    def run():
        layer.zero_grad()
        y = x.clone().requires_grad_(mode != "inference")
        with torch.set_grad_enabled(mode != "inference"):
            out, _ = layer(y, cu)
        if mode == "inference":
            return [out]
        (out * torch.linspace(-1, 1, out.numel(), device=DEV).view_as(out)).sum().backward()
        return [out.detach(), y.grad, layer.q_norm.weight.grad.clone(), layer.k_norm.weight.grad.clone()]

    own = run()

    def plain(q, k, cos, sin, c, m):
        a = (layer.q_norm.weight, layer.k_norm.weight, layer.rope_cos, layer.rope_sin, pos)
        return _torch_norm_rope(q, k, *a, 1e-6)[0], _torch_norm_rope(q, k, *a, 0.3)[1]
    layer._norm_rope = plain
    for a, b in zip(own, run()):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max().clamp(min=1e-3)


@pytest.mark.parametrize("mode", ["train", "eval with autograd", "inference"])
def test_layer_with_a_hooked_norm(mode):
    """A hook on a norm is called and does not move the results past the layer's float32 tolerance (as test_layer); a norm that is
    replaced is used."""
    torch.manual_seed(4)
    layer = DSALTAttention(256, 4, 8, 40, 6, 256, n_kv_heads=2, qk_norm=True).to(DEV).train(mode == "train")
    x, cu = torch.randn(90, 256, device=DEV), torch.tensor([0, 33, 90], dtype=torch.int32, device=DEV)

    def run():
        layer.zero_grad()
        y = x.clone().requires_grad_(mode != "inference")
        with torch.set_grad_enabled(mode != "inference"):
            out, _ = layer(y, cu)
        if mode == "inference":
            return [out]
        (out * torch.linspace(-1, 1, out.numel(), device=DEV).view_as(out)).sum().backward()
        return [out.detach(), y.grad, *(n.weight.grad.clone() for n in (layer.q_norm, layer.k_norm) if hasattr(n, "weight"))]

    own, seen = run(), []
    for n in (layer.q_norm, layer.k_norm):
        n.register_forward_hook(lambda m, i, o: seen.append((o, o.detach().clone())))
    for a, b in zip(own, run()):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max().clamp(min=1e-3)
    assert len(seen) == 2 and all(torch.equal(o, c) for o, c in seen)
    layer.q_norm = torch.nn.Identity()
    other = run()
    assert not torch.allclose(other[0], own[0], rtol=1e-2)
