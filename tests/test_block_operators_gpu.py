"""The training operators together, as a transformer block over video tokens uses them: LayerNorm -> q | k | v -> rotary positions ->
window attention -> projection, forward and backward; the same block for single tokens against a cache; and both as captured graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

B, T, Hh, W, H, Hkv, hd = 2, 4, 6, 8, 6, 2, 40
L, Cd = T * Hh * W, H * hd
QKV = (H + 2 * Hkv) * hd
LEFT, SINKS = 3 * Hh * W, Hh * W


def _weights(dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return {"x": r(B, L, Cd).to(dtype), "gamma": (1 + 0.1 * r(Cd)).to(dtype), "beta": (0.1 * r(Cd)).to(dtype),
            "wqkv": (r(QKV, Cd) * Cd ** -0.5).to(dtype), "wo": (r(Cd, Cd) * Cd ** -0.5).to(dtype), "dy": (0.1 * r(B, L, Cd)).to(dtype)}


def _block(w, axes):
    """Forward and backward of x + attention(LayerNorm(x)); matrix products by ops.gemm."""
    from hallo_amd import ops
    kw = dict(kv_heads=Hkv, left=LEFT, right=0, sinks=SINKS)
    n, stats = ops.layernorm_train(w["x"], w["gamma"], w["beta"])
    qkv = ops.gemm(n.view(B * L, Cd), w["wqkv"]).view(B, L, QKV)
    rot = qkv[..., :(H + Hkv) * hd]
    ops.rope(rot, axes, grid=(T, Hh, W), out=rot)
    q, k, v = qkv.split([H * hd, Hkv * hd, Hkv * hd], 2)
    o, lse = ops.window_attention(q, k, v, H, return_lse=True, **kw)
    y = ops.gemm(o.view(B * L, Cd), w["wo"], residual=w["x"].view(B * L, Cd)).view(B, L, Cd)
    do = ops.gemm(w["dy"].view(B * L, Cd), w["wo"].t().contiguous()).view(B, L, Cd)
    dqkv = torch.empty_like(qkv)
    dq, dk, dv = dqkv.split([H * hd, Hkv * hd, Hkv * hd], 2)
    ops.window_attention_backward(do, q, k, v, o, lse, H, dq=dq, dk=dk, dv=dv, **kw)
    drot = dqkv[..., :(H + Hkv) * hd]
    ops.rope(drot, axes, grid=(T, Hh, W), inverse=True, out=drot)
    dn = ops.gemm(dqkv.view(B * L, QKV), w["wqkv"].t().contiguous()).view(B, L, Cd)
    dx, dgamma, dbeta = ops.layernorm_backward(dn, w["x"], stats, w["gamma"])
    return {"y": y, "k": k, "v": v, "dx": dx, "dgamma": dgamma, "dbeta": dbeta, "dqkv": dqkv}


def _reference(w):
    """The block in 64 bits with torch's own differentiation."""
    p = {n: t.double().requires_grad_(n != "dy") for n, t in w.items()}
    x = p["x"]
    d = x - x.mean(-1, keepdim=True)
    n = d * (d.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * p["gamma"] + p["beta"]
    qkv = n @ p["wqkv"].t()
    pos = torch.stack(torch.meshgrid(torch.arange(T), torch.arange(Hh), torch.arange(W), indexing="ij"), -1).view(1, L, 3).double().cuda()
    parts, at = [], 0
    heads = qkv.view(B, L, H + 2 * Hkv, hd)
    for a, width in enumerate((8, 16, 16)):
        ang = pos[..., a:a + 1] * 10000.0 ** (-torch.arange(0, width, 2, device="cuda").double() / width)
        c, s = ang.cos().unsqueeze(2), ang.sin().unsqueeze(2)
        m, o2 = heads[..., at:at + width // 2], heads[..., at + width // 2:at + width]
        parts += [m * c - o2 * s, o2 * c + m * s]
        at += width
    rot = torch.cat(parts, -1)
    q, k, v = rot[:, :, :H], rot[:, :, H:H + Hkv], heads[:, :, H + Hkv:]
    rep = lambda t: t.repeat_interleave(H // Hkv, 2).transpose(1, 2)
    s = q.transpose(1, 2) @ rep(k).transpose(2, 3) * hd ** -0.5
    i, j = torch.arange(L, device="cuda").view(-1, 1), torch.arange(L, device="cuda").view(1, -1)
    s = s.masked_fill(~((j <= i) & ((j >= i - LEFT) | (j < SINKS))), -torch.inf)
    o = (torch.softmax(s, -1) @ rep(v)).transpose(1, 2).reshape(B, L, Cd)
    y = x.detach() + o @ p["wo"].t()
    y.backward(p["dy"])
    return {"y": y, "dx": x.grad, "dgamma": p["gamma"].grad, "dbeta": p["beta"].grad}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_block(dtype):
    from hallo_amd import ops
    w = _weights(dtype)
    got, want = _block(w, ops.RopeAxes((8, 16, 16), hd)), _reference(w)
    # a chain of at most eight roundings to the storage type per value (x - products - rotation - P - o, and back), each half a step
    # relative and independent of the next product's terms: relative error of the whole tensor (2-norm) below 8 u
    for n in ("y", "dx", "dgamma", "dbeta"):
        e = (got[n].double() - want[n]).norm() / want[n].norm()
        assert e <= 8 * torch.finfo(dtype).eps / 2, (n, e.item())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_single_tokens(dtype):
    """The block's attention token by token: rotary at explicit positions into the cache, window over it."""
    from hallo_amd import ops
    w = _weights(dtype, 1)
    axes = ops.RopeAxes((8, 16, 16), hd)
    n = ops.layernorm_train(w["x"], w["gamma"], w["beta"])[0]
    qkv = ops.gemm(n.view(B * L, Cd), w["wqkv"]).view(B, L, QKV)
    pos = torch.stack(torch.meshgrid(torch.arange(T), torch.arange(Hh), torch.arange(W), indexing="ij"), -1).view(L, 3).int().cuda()
    cut = H * hd, Hkv * hd, Hkv * hd
    rot = qkv.clone()
    ops.rope(rot[..., :(H + Hkv) * hd], axes, grid=(T, Hh, W), out=rot[..., :(H + Hkv) * hd])
    q, k, v = rot.split(cut, 2)
    whole = ops.window_attention(q, k, v, H, kv_heads=Hkv, left=LEFT, sinks=SINKS)
    kc, vc = (torch.full((B, L + 9, Hkv * hd), float("nan"), device="cuda", dtype=dtype) for _ in range(2))
    for t in range(L):
        x1 = w["x"][:, t].contiguous()
        one = ops.gemm(ops.layernorm_train(x1, w["gamma"], w["beta"])[0], w["wqkv"]).view(B, 1, QKV)
        r = ops.rope(one[..., :(H + Hkv) * hd], axes, pos=pos[t:t + 1])
        kc[:, t], vc[:, t] = r[:, 0, H * hd:], one[:, 0, (H + Hkv) * hd:]
        o = ops.window_attention(r[..., :H * hd], kc, vc, H, kv_heads=Hkv, left=LEFT, sinks=SINKS,
                                 kv_len=torch.full((B,), t + 1, device="cuda", dtype=torch.int32))
        # the two ways differ by the order of fp32 sums and by P's rounding: u per term of a mean of |v| (below 4), and the result's
        assert ((o[:, 0].double() - whole[:, t].double()).abs() <= torch.finfo(dtype).eps * 4).all(), t


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_graphs(dtype):
    """Two captured blocks (forward and backward) replayed in turn and at the same time, each against its eager results, with eager
    work between the replays: captured graphs share no workspace."""
    from hallo_amd import ops
    axes = ops.RopeAxes((8, 16, 16), hd)
    ws = [_weights(dtype, 2), _weights(dtype, 3)]
    want = [{n: t.clone() for n, t in _block(w, axes).items()} for w in ws]
    torch.cuda.synchronize()
    graphs, outs, scratch = [], [], [ops.Scratch("cuda") for _ in ws]      # the matrix products' scratch, one for each graph
    for w, own in zip(ws, scratch):
        with ops.scratch_scope(own):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(_block(w, axes))
            graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for o in outs:
            for t in o.values():
                t.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            if turn % 2:
                with torch.cuda.stream(s):
                    g.replay()
            else:
                g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, want):
            for n in e:
                assert torch.equal(o[n], e[n]), (turn, n)
        again = _block(ws[turn % 2], axes)
        assert all(torch.equal(again[n], want[turn % 2][n]) for n in again)
