"""GPU tests of window_attention / window_attention_backward where 16-bit operands of the second products could lose what the row sums
and the results still hold: probabilities below half of fp16's smallest number, gradients and values that are small where a window looks
and large elsewhere.  E = 2^-24, u = eps / 2 of the storage type, as in test_window_attention_gpu.py."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Lq,H,N", [(1, 1, 2, 1000), (1, 1, 2, 6000), (1, 9, 4, 6000), (9, 500, 8, 1000)])
def test_many_small_weights_beside_a_large_one(dtype, B, Lq, H, N):
    """One key scores S = 18.25, the other N - 1 score 0: each of these weighs 2^-26.3 of the first, all of them together decide o, since
    the first key's value is 0.  In one piece, in parts, and (last row) in blocks of 128 queries.

    fp16 carries P times 2^9 at least, so a weight is off by at most 2^-25 * 2^-9 of the largest; bf16 rounds it (u).  The row sum and
    the product add N terms in fp32; the exponential and the division are good to a few E."""
    from hallo_amd import ops
    hd, S = 64, 18.25
    g = torch.Generator(device="cuda").manual_seed(N + Lq)
    q = torch.zeros(B, Lq, H, hd, device="cuda", dtype=dtype)
    k = torch.zeros(B, N, H, hd, device="cuda", dtype=dtype)
    q[..., 0] = 1.0
    k[:, 0, :, 0] = S
    col = (512 + 512 * torch.rand(B, 1, H, hd, generator=g, device="cuda")).to(dtype)
    v = col.repeat(1, N, 1, 1)
    v[:, 0] = 0.0
    o, lse = ops.window_attention(q, k, v, H, right=-1, scale=1.0, return_lse=True)
    w = math.exp(-S)
    ref = (N - 1) * w / (1 + (N - 1) * w) * col.double()
    u = torch.finfo(dtype).eps / 2
    tol = ref * (2 * u + 4 * N * E + 64 * E)
    if dtype == F16:
        tol = tol + (N - 1) * 2.0 ** -34 * col.double()
    assert ((o.double() - ref).abs() <= tol).all(), (o[0, 0, 0, :4].tolist(), ref[0, 0, 0, :4].tolist())
    assert ((lse.double() - (S + math.log1p((N - 1) * w))).abs() <= 64 * E * S + 4 * N * E).all()


def _near(x, reach):
    """Largest value of x [L] within `reach` places."""
    return torch.nn.functional.max_pool1d(x.view(1, 1, -1), 2 * reach + 1, 1, reach).view(-1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [64, 160])
@pytest.mark.parametrize("which", ["do", "v"])
def test_small_far_from_large(dtype, hd, which):
    """Gradients (values) of the first 700 tokens are 2^22 times those of the rest, the window is 400 tokens: dq, dk and dv behind it
    know nothing of the large ones and keep their accuracy.

    fp16: dS is carried times a power of two that 2 |do|_2 |v|_2 bounds, norms over what a workgroup of 128 keys or queries meets:
    queries within 400 + 128 tokens (and up to 63 to the end of a block of norms), keys within another 400 + 64 of those; so dS is off by
    2^-25 * 2^-14 of that product.  The other terms as in test_window_attention_gpu.py."""
    from hallo_amd import ops
    L, H, left, cut = 2600, 2, 400, 700
    g = torch.Generator(device="cuda").manual_seed(hd)
    r = lambda: torch.randn(1, L, H * hd, generator=g, device="cuda")
    size = torch.where(torch.arange(L, device="cuda") < cut, 2.0 ** 7, 2.0 ** -15).view(1, -1, 1)
    flat = torch.full((1, 1, 1), 2.0 ** 10, device="cuda")
    q, k = r().to(dtype), r().to(dtype)
    v, do = (r() * (size if which == "v" else flat)).to(dtype), (r() * (size if which == "do" else flat)).to(dtype)
    o, lse = ops.window_attention(q, k, v, H, left=left, return_lse=True)
    got = ops.window_attention_backward(do, q, k, v, o, lse, H, left=left)

    u, c = torch.finfo(dtype).eps / 2, hd ** -0.5
    f = lambda t: t.double().view(L, H, hd).transpose(0, 1)
    Q, K, V, G, O = (f(t) for t in (q, k, v, do, o))
    i, j = torch.arange(L, device="cuda").view(-1, 1), torch.arange(L, device="cuda").view(1, -1)
    ok = (j <= i) & (j >= i - left)
    s = (Q @ K.transpose(1, 2)) * c
    ls = lse.double().view(H, L, 1)
    p = torch.exp((s - ls).masked_fill(~ok, -torch.inf))
    t = ((hd + 8) * E * c * (Q.abs() @ K.abs().transpose(1, 2)) + 12 * E * (s.abs() + ls.abs()) + 8 * E) * ok
    dp, delta = G @ V.transpose(1, 2), (G * O).sum(2, keepdim=True)
    ds = p * (dp - delta)
    e_ds = (u + 2 * t) * ds.abs() + p * (1 + u) * (hd + 8) * E * (G.abs() @ V.abs().transpose(1, 2) + (G * O).abs().sum(2, keepdim=True))
    e_p = (u + 2 * t) * p
    if dtype == F16:
        meets = _near(G.norm(dim=2).amax(0), left + 128 + 63) * _near(V.norm(dim=2).amax(0), 2 * left + 128 + 128)
        scale = torch.maximum(meets.view(-1, 1), meets.view(1, -1))       # the workgroup of the query (dq) or of the key (dk)
        e_ds = e_ds + 2.0 ** -38 * scale * ok
        e_p = e_p + 2.0 ** -39 * ok
    else:
        e_ds = e_ds + 2.0 ** -126 * (1 + (dp - delta).abs()) * ok
        e_p = e_p + 2.0 ** -126 * ok
    n = left + 1
    tr = lambda x: x.transpose(1, 2)
    want = {"dq": (c * (ds @ K), c * ((e_ds + n * E * ds.abs()) @ K.abs())),
            "dk": (c * (tr(ds) @ Q), c * ((tr(e_ds) + n * E * tr(ds).abs()) @ Q.abs())),
            "dv": (tr(p) @ G, (tr(e_p) + n * E * tr(p)) @ G.abs())}
    floor = 2.0 ** -25 if dtype == F16 else 2.0 ** -126
    for (name, (ref, slack)), x in zip(want.items(), got):
        x = f(x)
        tol = u * ref.abs() + (1 + u) * slack + floor
        # the first rows' probabilities are near 1, so some of the large results pass the type's largest number: those round to infinity
        fits = ref.abs() + tol < torch.finfo(dtype).max
        assert fits[:, cut + 1200:].all() and torch.isfinite(x[fits]).all(), name
        bad = fits & ~((x - ref).abs() <= tol)
        assert not bad.any(), (name, bad.sum().item(), bad.nonzero()[0].tolist(), ((x - ref).abs() / tol)[bad].max().item())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Lq,H,N", [(1, 1, 2, 1000), (1, 3, 4, 6000), (9, 500, 8, 1000)])
def test_equal_scores_of_any_size(dtype, B, Lq, H, N):
    """All keys score the same, up to 6 10^7, where a rounding of the score in log2 units is several units: the weights are all alike and o
    is the mean of v.  (All P of a row have one value: half a step of the storage type, the result's half a step, sums in fp32.)"""
    from hallo_amd import ops
    hd = 64
    g = torch.Generator(device="cuda").manual_seed(N)
    v = torch.randn(B, N, H, hd, generator=g, device="cuda").to(dtype)
    mean = v.double().mean(1, keepdim=True)
    u = torch.finfo(dtype).eps / 2
    tol = (u * mean.abs() + (u + 4 * N * E) * v.double().abs().mean(1, keepdim=True)) * (1 + u)
    for size in (16.0, 512.0, 768.0, 896.0):
        q = torch.full((B, Lq, H, hd), size, device="cuda", dtype=dtype)
        k = torch.full((B, N, H, hd), size, device="cuda", dtype=dtype)
        for scale in (1.0, 0.9, 1.1, 1.17, -1.0):
            k2 = -k if scale < 0 else k
            o, lse = ops.window_attention(q, k2, v, H, right=-1, scale=abs(scale), return_lse=True)
            s = scale * size * size * hd
            assert ((o.double() - mean).abs() <= tol).all(), (size, scale, o[0, 0, 0, :4].tolist(), mean[0, 0, 0, :4].tolist())
            assert ((lse.double() - (s + math.log(N))).abs() <= 16 * E * abs(s) + 1e-4).all(), (size, scale)
