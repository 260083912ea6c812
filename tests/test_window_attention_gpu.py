"""GPU tests of window_attention / window_attention_backward against the definition in 64 bits.

Tolerances, per element, u = eps / 2 of the storage type, E = 2^-24, w = |scale| * sum_d |q_d k_d| of a pair:
  a score's fp32 dot product is off by at most hd E w, its scaling, the running maximum and exp2 by a few E of it: relative error of a
  probability  t = (hd + 8) E w + 8 E (|s| + |lse|) + 8 E;
  o:  P is rounded once for the product (u), sums in fp32 over the keys (n E), one rounding of the result;
      fp16: P below the normal numbers is off by 2^-25 where the row's largest is at least 1;
  dV: the same over the queries, P carried times 2^14 in fp16;
  dS = P (dP - delta): dP and delta off by (hd + 8) E of their magnitudes, dS rounded once (u; fp16: to 2^-25 of a scale that is at least
      2^14 / (2 |do|_2 |v|_2), norms over the batch entry), then summed against k or q; for dK a bf16 P of 112 and 128 columns is fp16
      times 2^14 on its way (2^-11 relative, 2^-25 * 2^-14 below the normal numbers);
  fp32 and bf16 results below the smallest normal number, 2^-126, count as 0 (v_exp_f32 and the MFMA operands flush them): a probability is
  off by up to TINY = 2^-126 on top, and so is a bf16 result -- a key whose probabilities are all below it has gradients of 0."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TINY = 2.0 ** -126
F16, BF16 = torch.float16, torch.bfloat16


def _mask(B, Lq, Lk, left, right, sinks, ql, kl):
    i = torch.arange(Lq, device="cuda").view(1, -1, 1)
    j = torch.arange(Lk, device="cuda").view(1, 1, -1)
    ql, kl = ql.view(-1, 1, 1), kl.view(-1, 1, 1)
    p = kl - ql + i
    ok = (i < ql) & (j < kl)
    if right >= 0:
        ok = ok & (j <= p + right)
    if left >= 0:
        ok = ok & ((j >= p - left) | (j < sinks))
    return ok


class Ref:
    """Forward (and backward) in 64 bits with the bounds above; tensors [B, heads, L, hd]."""

    def __init__(self, q, k, v, H, Hkv, left, right, sinks, ql=None, kl=None, scale=None):
        B, Lq, hd = q.shape[0], q.shape[1], q.reshape(q.shape[0], q.shape[1], -1).shape[2] // H
        Lk = k.shape[1]
        self.dt, self.hd, self.G, self.scale = q.dtype, hd, H // Hkv, hd ** -0.5 if scale is None else scale
        full = lambda n: torch.full((B,), n, device="cuda")
        self.ql = full(Lq) if ql is None else ql.long().clamp(0, Lq)
        self.kl = full(Lk) if kl is None else kl.long().clamp(0, Lk)
        f = lambda t, n: t.double().reshape(B, t.shape[1], n, hd).transpose(1, 2)
        rep = lambda t: t.repeat_interleave(self.G, 1)
        self.ok = _mask(B, Lq, Lk, left, right, sinks, self.ql, self.kl).unsqueeze(1)
        used = self.ok.any(2)                                                   # [B, 1, Lk]
        hidden = ~used.unsqueeze(-1)
        self.q = f(q, H).masked_fill((torch.arange(Lq, device="cuda").view(1, 1, -1, 1) >= self.ql.view(-1, 1, 1, 1)), 0.0)
        self.k = rep(f(k, Hkv).masked_fill(hidden, 0.0))
        self.v = rep(f(v, Hkv).masked_fill(hidden, 0.0))
        s = (self.q @ self.k.transpose(2, 3)) * self.scale
        w = (self.q.abs() @ self.k.abs().transpose(2, 3)) * self.scale
        s = s.masked_fill(~self.ok, -torch.inf)
        self.lse = torch.logsumexp(s, 3, keepdim=True)
        lse0 = self.lse.masked_fill(self.lse == -torch.inf, 0.0)
        self.p = torch.exp(s - lse0)
        self.t = ((hd + 8) * E * w + 8 * E * (s.masked_fill(~self.ok, 0.0).abs() + lse0.abs()) + 8 * E).masked_fill(~self.ok, 0.0)
        self.o = self.p @ self.v
        u = torch.finfo(self.dt).eps / 2
        n = self.ok.sum(3, keepdim=True)
        self.u = u
        self.o_tol = u * self.o.abs() + (1 + u) * ((self.p * (u + 2 * self.t + n * E)) @ self.v.abs()
                                                   + self.o.abs() * ((self.p * self.t).sum(3, keepdim=True) + n * E))
        if self.dt == F16:
            # relative to the largest probability of the row, which is carried as 1 at least
            self.o_tol = self.o_tol + 2.0 ** -25 * self.p.amax(3, keepdim=True) * (self.ok.double() @ self.v.abs()) + 2.0 ** -25
        else:
            self.o_tol = self.o_tol + TINY * (self.ok.double() @ self.v.abs()) + TINY
        self.lse_tol = ((self.p * self.t).sum(3) + 4 * n.squeeze(3) * E + 4 * E * lse0.squeeze(3).abs())

    def check(self, o, lse=None):
        B, Lq, H = o.shape[0], o.shape[1], self.q.shape[1]
        got = o.double().reshape(B, Lq, H, self.hd).transpose(1, 2)
        assert torch.isfinite(got).all()
        bad = (got - self.o).abs() > self.o_tol
        assert not bad.any(), (bad.nonzero()[0].tolist(), ((got - self.o).abs() / (self.o_tol + 1e-300)).max().item())
        empty = ~self.ok.any(3).expand(B, H, Lq)
        assert (got[empty] == 0).all()
        if lse is not None:
            assert lse.dtype == torch.float32 and (lse[empty] == -torch.inf).all()
            d = (lse.double() - self.lse.squeeze(3))[~empty]
            assert (d.abs() <= self.lse_tol[~empty]).all()

    def check_grads(self, do, o, lse, dq, dk, dv):
        B, Lq, H, hd, u, c = self.q.shape[0], self.q.shape[2], self.q.shape[1], self.hd, self.u, self.scale
        Lk, Hkv = self.k.shape[2], H // self.G
        pad = torch.arange(Lq, device="cuda").view(1, 1, -1, 1) >= self.ql.view(-1, 1, 1, 1)
        f = lambda t: t.double().reshape(B, Lq, H, hd).transpose(1, 2).masked_fill(pad, 0.0)
        g, o = f(do), f(o)
        ls = lse.double().unsqueeze(3)
        s = (self.q @ self.k.transpose(2, 3)) * c
        p = torch.exp((s - ls.masked_fill(ls == -torch.inf, 0.0)).masked_fill(~self.ok, -torch.inf))
        t = self.t + 4 * E * ls.masked_fill(ls == -torch.inf, 0.0).abs()
        delta = (g * o).sum(3, keepdim=True)
        dp = g @ self.v.transpose(2, 3)
        ds = p * (dp - delta)
        e_dp = (hd + 8) * E * (g.abs() @ self.v.abs().transpose(2, 3) + (g * o).abs().sum(3, keepdim=True))
        e_ds = (u + 2 * t) * ds.abs() + p * e_dp * (1 + u)
        e_p = (u + 2 * t) * p
        if self.dt == F16:
            norm = 2 * g.norm(dim=3).amax((1, 2)).view(-1, 1, 1, 1) * self.v.norm(dim=3).amax((1, 2)).view(-1, 1, 1, 1)
            e_ds = e_ds + (2.0 ** -25 * 2.0 ** -14) * norm * self.ok
            e_p = e_p + 2.0 ** -39 * self.ok
        else:
            e_ds = e_ds + TINY * (1 + (dp - delta).abs()) * self.ok            # P and dS
            if 96 < hd <= 128:
                e_ds = e_ds + 2.0 ** -11 * ds.abs() + 2.0 ** -39 * (dp - delta).abs() * self.ok
            e_p = e_p + TINY * self.ok
        nk, nq = self.ok.sum(3, keepdim=True), (self.ok.sum(2).unsqueeze(3) * self.G)
        shared = lambda x: x.reshape(B, Hkv, self.G, Lk, hd).sum(2)
        tr = lambda x: x.transpose(2, 3)
        floor = 2.0 ** -25 if self.dt == F16 else TINY
        out = {}
        out["dq"] = (dq, H, c * (ds @ self.k), c * ((e_ds + nk * E * ds.abs()) @ self.k.abs()))
        out["dk"] = (dk, Hkv, c * shared(tr(ds) @ self.q), c * shared(tr(e_ds) @ self.q.abs() + nq * E * (tr(ds.abs()) @ self.q.abs())))
        out["dv"] = (dv, Hkv, shared(tr(p) @ g), shared(tr(e_p) @ g.abs() + nq * E * (tr(p) @ g.abs())))
        for name, (got, heads, ref, slack) in out.items():
            got = got.double().reshape(B, got.shape[1], heads, hd).transpose(1, 2)
            assert torch.isfinite(got).all(), name
            tol = u * ref.abs() + (1 + u) * slack + floor
            bad = (got - ref).abs() > tol
            assert not bad.any(), (name, bad.nonzero()[0].tolist(), ((got - ref).abs() / (tol + 1e-300)).max().item())
        unseen = ~self.ok.any(2).expand(B, 1, Lk).reshape(B, Lk)
        assert (dk.reshape(B, Lk, -1)[unseen] == 0).all() and (dv.reshape(B, Lk, -1)[unseen] == 0).all()


def _qkv(B, Lq, Lk, H, Hkv, hd, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 101 + Lq * 7 + Lk * 3 + H + hd)
    r = lambda L, n: torch.randn(B, L, n * hd, generator=g, device="cuda").to(dtype)
    return r(Lq, H), r(Lk, Hkv), r(Lk, Hkv), (0.1 * torch.randn(B, Lq, H * hd, generator=g, device="cuda")).to(dtype)


def _lens(*n):
    return torch.tensor(n, device="cuda", dtype=torch.int32)


def _both(B, Lq, Lk, H, Hkv, hd, dtype, left, right, sinks, ql=None, kl=None, seed=0, grads=True, scale=None):
    from hallo_amd import ops
    q, k, v, do = _qkv(B, Lq, Lk, H, Hkv, hd, dtype, seed)
    kw = dict(kv_heads=Hkv, left=left, right=right, sinks=sinks, q_len=ql, kv_len=kl, scale=scale)
    o, lse = ops.window_attention(q, k, v, H, return_lse=True, **kw)
    ref = Ref(q, k, v, H, Hkv, left, right, sinks, ql, kl, scale)
    ref.check(o, lse)
    if grads:
        a = ops.window_attention_backward(do, q, k, v, o, lse, H, **kw)
        ref.check_grads(do, o, lse, *a)
        b = ops.window_attention_backward(do, q, k, v, o, lse, H, **kw)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    return o


HEAD_DIMS = [8, 16, 24, 32, 40, 48, 64, 72, 80, 96, 104, 112, 128, 136, 144, 160]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", HEAD_DIMS)
def test_head_dims(dtype, hd):
    _both(2, 150, 150, 4, 2, hd, dtype, 40, 0, 5)          # few blocks: keys split over workgroups
    _both(16, 140, 140, 8, 4, hd, dtype, 33, 20, 3)        # 128-query blocks


WINDOWS = [(-1, 0, 0), (-1, -1, 0), (0, 0, 0), (0, 0, 1), (7, 0, 2), (63, 64, 0), (100, 0, 130), (31, -1, 4), (5, 5, 300), (-1, 9, 7), (1 << 40, 0, 1 << 40)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
def test_windows(dtype, left, right, sinks):
    _both(1, 333, 333, 2, 1, 64, dtype, left, right, sinks)
    _both(20, 200, 290, 4, 2, 40, dtype, left, right, sinks, _lens(*range(181, 201)), _lens(*range(270, 290)))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 2), (2, 1), (31, 33), (32, 32), (33, 31), (64, 65), (127, 129), (128, 128), (129, 127), (1, 1000), (257, 64),
                                   (16, 4000), (40, 3000), (700, 20)])
def test_lengths(dtype, Lq, Lk):
    for H, Hkv, left, right, sinks in ((3, 3, -1, 0, 0), (6, 2, 50, 0, 4), (5, 1, 20, 20, 0)):
        _both(2, Lq, Lk, H, Hkv, 64, dtype, left, right, sinks)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_ragged_and_empty(dtype):
    """Entries without keys, without queries, with more queries than keys (rows before the first key see nothing), lengths past the
    tensors, and padding that holds NaN and infinities."""
    from hallo_amd import ops
    B, Lq, Lk, H, Hkv, hd = 7, 150, 170, 4, 2, 64
    ql, kl = _lens(150, 0, 100, 150, 3, 149, 9999), _lens(170, 50, 0, 20, 170, 1, 9999)
    for left, right, sinks in ((-1, 0, 0), (30, 0, 4), (20, 10, 0), (-1, -1, 0)):
        q, k, v, do = _qkv(B, Lq, Lk, H, Hkv, hd, dtype, 3)
        ref = Ref(q, k, v, H, Hkv, left, right, sinks, ql, kl)
        bad = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0], device="cuda").to(dtype)
        for b in range(B):
            n, m = min(int(ql[b]), Lq), min(int(kl[b]), Lk)
            for t, e in ((q, n), (do, n), (k, m), (v, m)):
                t[b, e:] = bad[torch.arange(t[b, e:].numel(), device="cuda") % 4].view_as(t[b, e:])
        kw = dict(kv_heads=Hkv, left=left, right=right, sinks=sinks, q_len=ql, kv_len=kl)
        out = torch.full_like(q, 5.0)
        o, lse = ops.window_attention(q, k, v, H, return_lse=True, out=out, **kw)
        assert o is out
        ref.check(o, lse)
        oo, ll = o.clone(), lse.clone()
        for b in range(B):                       # what the backward pass must not read
            n = min(int(ql[b]), Lq)
            oo[b, n:] = float("nan")
            ll[b, :, n:] = float("nan")
        ref.check_grads(do, o, lse, *ops.window_attention_backward(do, q, k, v, oo, ll, H, **kw))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_hidden_keys_between(dtype):
    """One token at a time with a window: cache places between the sinks and the window hold garbage."""
    from hallo_amd import ops
    for n in (1, 5, 40, 300, 1111):
        q, k, v, _ = _qkv(3, 1, 1200, 8, 2, 128, dtype, n)
        kl = _lens(n, max(1, n - 7), n)
        ref = Ref(q, k, v, 8, 2, 63, 0, 3, None, kl)
        gone = ~ref.ok.any(2).reshape(3, 1200)
        k[gone] = float("nan")
        v[gone] = float("inf")
        ref.check(*ops.window_attention(q, k, v, 8, kv_heads=2, left=63, sinks=3, kv_len=kl, return_lse=True))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_hidden_keys_in_the_backward_pass(dtype):
    """Queries at the end of the keys with a window: keys that no query sees hold garbage; their gradients are zeros and the others do
    not know of them (large finite values would take the fp16 scale down, infinities take it away)."""
    from hallo_amd import ops
    for Lq, left, sinks in ((5, 63, 3), (100, 20, 0), (1, 0, 1)):
        q, k, v, do = _qkv(2, Lq, 400, 4, 2, 64, dtype, Lq)
        ql, kl = _lens(Lq, max(1, Lq - 2)), _lens(400, 333)
        kw = dict(kv_heads=2, left=left, sinks=sinks, q_len=ql, kv_len=kl)
        ref = Ref(q, k, v, 4, 2, left, 0, sinks, ql, kl)
        o, lse = ops.window_attention(q, k, v, 4, return_lse=True, **kw)
        clean = ops.window_attention_backward(do, q, k, v, o, lse, 4, **kw)
        ref.check_grads(do, o, lse, *clean)
        gone = ~ref.ok.any(2).reshape(2, 400)
        for bad in (float("nan"), float("inf"), 30000.0):
            k[gone], v[gone] = bad, -bad
            got = ops.window_attention_backward(do, q, k, v, o, lse, 4, **kw)
            assert all(torch.equal(a, b) for a, b in zip(got, clean))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("small", [0.0, 2.0 ** -10, 2.0 ** -5])
def test_small_values_under_large_probabilities(dtype, small):
    """First keys that every query looks at and whose values are next to nothing: dS = P (dP - delta) is as large as the other keys'
    values make delta, not as their own values make dP."""
    from hallo_amd import ops
    for B, L, H, Hkv, hd in ((1, 200, 4, 2, 64), (2, 300, 2, 2, 80), (16, 140, 8, 4, 40)):
        q, k, v, do = _qkv(B, L, L, H, Hkv, hd, dtype, 5)
        k[:, :2] = q[:, L // 2:L // 2 + 2].view(B, 2, Hkv, H // Hkv, hd)[:, :, :, 0].reshape(B, 2, Hkv * hd)
        v[:, :2] *= small
        v[:, 2:] *= 8.0
        kw = dict(kv_heads=Hkv, left=50, sinks=4)
        ref = Ref(q, k, v, H, Hkv, 50, 0, 4)
        o, lse = ops.window_attention(q, k, v, H, return_lse=True, **kw)
        ref.check(o, lse)
        ref.check_grads(do, o, lse, *ops.window_attention_backward(do, q, k, v, o, lse, H, **kw))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (7, 1), (8, 8), (12, 4), (32, 2)])
def test_single_tokens_follow_the_prompt(dtype, H, Hkv):
    """A cache filled token by token answers as the whole sequence does."""
    from hallo_amd import ops
    L, hd = 70, 80
    q, k, v, _ = _qkv(2, L, L, H, Hkv, hd, dtype, 8)
    kw = dict(kv_heads=Hkv, left=20, sinks=2)
    ref = Ref(q, k, v, H, Hkv, 20, 0, 2)
    whole = ops.window_attention(q, k, v, H, **kw)
    steps = torch.cat([ops.window_attention(q[:, t:t + 1], k, v, H, kv_len=_lens(t + 1, t + 1), **kw) for t in range(L)], 1)
    ref.check(whole)
    ref.check(steps)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_layouts(dtype):
    """Column slices of a fused buffer, head-major caches, 4-D views, outputs in place of strided memory."""
    from hallo_amd import ops
    B, L, H, Hkv, hd = 2, 200, 6, 2, 40
    q, k, v, do = _qkv(B, L, L, H, Hkv, hd, dtype, 2)
    kw = dict(kv_heads=Hkv, left=50, right=3, sinks=2)
    want, lse = ops.window_attention(q, k, v, H, return_lse=True, **kw)
    grads = ops.window_attention_backward(do, q, k, v, want, lse, H, **kw)
    fused = torch.cat([q, k, v], 2)
    parts = fused.split([H * hd, Hkv * hd, Hkv * hd], 2)
    wide = torch.full((B, L, H * hd + 16), 9.0, device="cuda", dtype=dtype)
    o = ops.window_attention(*parts, H, out=wide[..., 8:8 + H * hd], **kw)
    assert torch.equal(o, want) and (wide[..., :8] == 9).all() and (wide[..., 8 + H * hd:] == 9).all()
    km, vm = (t.view(B, L, Hkv, hd).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (k, v))
    qm = q.view(B, L, H, hd).permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    assert torch.equal(ops.window_attention(qm, km, vm, H, **kw).reshape(B, L, -1), want)
    dfused = torch.full_like(fused, 4.0)
    dparts = dfused.split([H * hd, Hkv * hd, Hkv * hd], 2)
    got = ops.window_attention_backward(do, *parts, want, lse, H, dq=dparts[0], dk=dparts[1], dv=dparts[2], **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, grads))
    got = ops.window_attention_backward(do.view(B, L, H, hd), qm, km, vm, want.view(B, L, H, hd), lse, H, **kw)
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, grads))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_broadcast_keys(dtype):
    """One key sequence for the whole batch (batch stride 0), as a shared prompt."""
    from hallo_amd import ops
    q, k, v, _ = _qkv(3, 5, 500, 4, 4, 64, dtype, 6)
    k1, v1 = k[:1].expand(3, -1, -1), v[:1].expand(3, -1, -1)
    Ref(q, k1.contiguous(), v1.contiguous(), 4, 4, -1, 0, 0).check(ops.window_attention(q, k1, v1, 4))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size", [0.01, 8.0])
def test_score_range(dtype, size):
    """Near-uniform rows, and rows that one key takes with scores in the hundreds (the running maximum moves far)."""
    from hallo_amd import ops
    B, L, H, hd = 2, 260, 4, 64
    q, k, v, do = _qkv(B, L, L, H, H, hd, dtype, 4)
    q, k = (q.float() * size).to(dtype), (k.float() * size).to(dtype)
    o, lse = ops.window_attention(q, k, v, H, left=99, sinks=1, return_lse=True)
    ref = Ref(q, k, v, H, H, 99, 0, 1)
    ref.check(o, lse)
    ref.check_grads(do, o, lse, *ops.window_attention_backward(do, q, k, v, o, lse, H, left=99, sinks=1))


def test_small_gradients_in_fp16():
    """Gradients of a few 1e-4 over long rows: P and dS are far below fp16's normal numbers, dq / dk / dv are not lost."""
    from hallo_amd import ops
    q, k, v, do = _qkv(1, 2000, 2000, 2, 2, 64, F16, 5)
    do = (do.float() * torch.logspace(-3, 0, 2000, device="cuda").view(1, -1, 1)).half()
    o, lse = ops.window_attention(q, k, v, 2, right=-1, return_lse=True)
    g = ops.window_attention_backward(do, q, k, v, o, lse, 2, right=-1)
    Ref(q, k, v, 2, 2, -1, -1, 0).check_grads(do, o, lse, *g)


def test_gradient_against_differences():
    from hallo_amd import ops
    B, L, H, Hkv, hd, kw = 1, 12, 2, 1, 8, dict(kv_heads=1, left=3, right=1, sinks=1)
    q, k, v, do = _qkv(B, L, L, H, Hkv, hd, F16, 11)
    o, lse = ops.window_attention(q, k, v, H, return_lse=True, **kw)
    got = dict(zip("qkv", ops.window_attention_backward(do, q, k, v, o, lse, H, **kw)))
    ok = _mask(1, L, L, 3, 1, 1, _lens(L), _lens(L)).unsqueeze(1)
    heads = lambda t, n: t.view(B, L, n, hd).transpose(1, 2)

    def loss(a):
        s = heads(a["q"], H) @ heads(a["k"], 1).transpose(2, 3) * hd ** -0.5
        return (torch.softmax(s.masked_fill(~ok, -torch.inf), 3) @ heads(a["v"], 1) * heads(do.double(), H)).sum()
    base = {"q": q.double(), "k": k.double(), "v": v.double()}
    for name in "qkv":
        n = base[name].numel()
        for i in range(0, n, 5):
            e = torch.zeros(n, device="cuda", dtype=torch.float64)
            e[i] = 1e-4
            e = e.view_as(base[name])
            num = ((loss(dict(base, **{name: base[name] + e})) - loss(dict(base, **{name: base[name] - e}))) / 2e-4).item()
            # P, dS, o rounded to fp16 (2^-11 of terms of at most |do| |v| ~ 2, up to 24 of them) and the result
            assert abs(num - got[name].view(-1)[i].item()) <= 2.0 ** -11 * (abs(num) + 24 * 0.2), (name, i)


def test_long_cache_past_32_bits():
    """A cache of more than 2^32 elements: the last entry and the last keys are found."""
    from hallo_amd import ops
    B, Lk, Hkv, hd = 3, 720000, 16, 128                                        # 4.4e9 elements, 8.8 GB each
    k = torch.zeros(B, Lk, Hkv * hd, device="cuda", dtype=BF16)
    v = torch.zeros(B, Lk, Hkv * hd, device="cuda", dtype=BF16)
    q, kt, vt, _ = _qkv(B, 2, 300, Hkv, Hkv, hd, BF16, 1)
    k[:, -300:], v[:, -300:] = kt, vt
    o = ops.window_attention(q, k, v, Hkv, left=298)
    Ref(q, kt, vt, Hkv, Hkv, 298, 0, 0).check(o)


def test_nothing_to_do():
    from hallo_amd import ops
    z = lambda B, L, dt=F16: torch.zeros(B, L, 64, device="cuda", dtype=dt)
    for B, Lq, Lk in ((0, 3, 3), (2, 0, 5), (2, 3, 0)):
        o, lse = ops.window_attention(z(B, Lq), z(B, Lk), z(B, Lk), 2, return_lse=True)
        assert o.shape == (B, Lq, 64) and (o == 0).all() and (lse == -torch.inf).all()
        g = ops.window_attention_backward(z(B, Lq), z(B, Lq), z(B, Lk), z(B, Lk), o, lse, 2)
        assert [t.shape for t in g] == [(B, Lq, 64), (B, Lk, 64), (B, Lk, 64)] and all((t == 0).all() for t in g)


def test_random_shapes():
    """Shapes over the whole range, many small."""
    import random
    rng = random.Random(7)
    for n in range(40):
        Hkv, G, hd = rng.choice([1, 2, 3]), rng.choice([1, 2, 5]), 8 * rng.randint(1, 20)
        Lk = rng.choice([rng.randint(1, 40), rng.randint(1, 700)])
        Lq = Lk if rng.random() < 0.5 else rng.randint(1, 300)
        B = rng.randint(1, 12)
        left, right = rng.choice([-1, rng.randint(0, 300)]), rng.choice([0, -1, rng.randint(0, 100)])
        ql = kl = None
        if rng.random() < 0.6:
            ql, kl = (_lens(*[rng.randint(0, L) for _ in range(B)]) for L in (Lq, Lk))
        _both(B, Lq, Lk, Hkv * G, Hkv, hd, rng.choice([F16, BF16]), left, right, rng.choice([0, 1, 17, 200]), ql, kl, n)


def test_other_stream():
    """Launched on the current stream, whichever it is, with results ordered on it."""
    from hallo_amd import ops
    q, k, v, do = _qkv(2, 300, 300, 4, 2, 64, BF16, 9)
    kw = dict(kv_heads=2, left=60, sinks=2)
    want, lse = ops.window_attention(q, k, v, 4, return_lse=True, **kw)
    grads = ops.window_attention_backward(do, q, k, v, want, lse, 4, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o, l2 = ops.window_attention(q, k, v, 4, return_lse=True, **kw)
        g = ops.window_attention_backward(do, q, k, v, o, l2, 4, **kw)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(o, want) and torch.equal(l2, lse) and all(torch.equal(a, b) for a, b in zip(g, grads))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,hd,left,right,sinks", [
    (6, 2100, 2100, 2, 2, 64, -1, 0, 0),         # row blocks of 32 queries under a long causal mask, more of them than run at once
    (1, 1100, 1100, 8, 2, 128, -1, 0, 0),        # dK / dV in parts, keys of a triangle
    (2, 1100, 1100, 4, 2, 80, 40, -1, 200),      # no right edge: the last keys have the most queries; sinks and the rest in parts
    (1, 90, 2500, 14, 2, 40, -1, 3, 0),          # heads of 90 queries packed to 96 rows, keys of dq split
    (3, 70, 1300, 4, 1, 160, 1000, 0, 5),
])
def test_plans(dtype, B, Lq, Lk, H, Hkv, hd, left, right, sinks):
    """Sizes that take each way of dividing the work."""
    _both(B, Lq, Lk, H, Hkv, hd, dtype, left, right, sinks, _lens(*[Lq - 5 * b for b in range(B)]), _lens(*[Lk - 7 * b for b in range(B)]))
