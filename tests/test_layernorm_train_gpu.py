"""GPU tests of layernorm_train / layernorm_backward against the formulas in 64 bits.

Tolerances: one rounding to the storage type (u = eps / 2, relative) plus the fp32 arithmetic in front of it.  A row sum of C terms in
fp32 through a tree of at most 40 sequential and 8 exchanged additions is off by at most 48 * 2^-24 of the sum of magnitudes; the
remaining operations add a few 2^-24 of the terms they join."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
DTYPES = [torch.float16, torch.bfloat16]


def _data(rows, C, dtype, seed=0, offset=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows * 31 + C)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = (r(rows, C) * 1.3 + offset * r(rows, 1)).to(dtype)
    return x, (1 + 0.2 * r(C)).to(dtype), (0.3 * r(C)).to(dtype), (0.1 * r(rows, C)).to(dtype)


def _fwd_ref(x, gamma, beta, eps):
    x = x.double()
    C = x.shape[1]
    g = gamma.double() if gamma is not None else torch.ones(C, device=x.device, dtype=torch.float64)
    b = beta.double() if beta is not None else torch.zeros(C, device=x.device, dtype=torch.float64)
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = (d.square().mean(1, keepdim=True) + eps).rsqrt()
    y = d * rstd * g + b
    # fp32: mean off by 48 E mean|x|; d by that and one rounding; rstd by half the relative error of the variance
    dm = 49 * E * x.abs().mean(1, keepdim=True) + E * d.abs()
    drstd = 52 * E + (dm * 2 * d.abs()).mean(1, keepdim=True) * rstd.square()      # relative
    slack = ((dm + d.abs() * (drstd + 3 * E)) * rstd * g.abs()) + E * (y.abs() + b.abs())
    return y, torch.cat([mean, rstd], 1), slack, torch.cat([dm.amax(1, keepdim=True), rstd * drstd], 1)


def _check_fwd(x, gamma, beta, eps, y, stats):
    u = torch.finfo(x.dtype).eps / 2
    ref, st, slack, st_slack = _fwd_ref(x, gamma, beta, eps)
    assert ((y.double() - ref).abs() <= u * ref.abs() + slack * (1 + u) + 2.0 ** -25).all()
    assert ((stats.double() - st).abs() <= st_slack + E * st.abs()).all()


def _bwd_ref(dy, x, stats, gamma):
    dy, x, st = dy.double(), x.double(), stats.double()
    C = x.shape[1]
    g = gamma.double() if gamma is not None else torch.ones(C, device=x.device, dtype=torch.float64)
    xh = (x - st[:, :1]) * st[:, 1:]
    t = dy * g
    c1, c2 = t.mean(1, keepdim=True), (t * xh).mean(1, keepdim=True)
    dx = st[:, 1:] * (t - c1 - xh * c2)
    xe = E * (xh.abs() + 2 * x.abs() * st[:, 1:])                                  # error of xh
    e1 = 52 * E * t.abs().mean(1, keepdim=True)
    e2 = (52 * E * t.abs() * xh.abs() + t.abs() * xe).mean(1, keepdim=True)
    slack = st[:, 1:] * (4 * E * (t.abs() + c1.abs() + (xh * c2).abs()) + e1 + xh.abs() * e2 + xe * c2.abs())
    return dx, (dy * xh).sum(0), dy.sum(0), slack, (dy.abs() * (xe + E * xh.abs())).sum(0), (dy * xh).abs().sum(0), dy.abs().sum(0)


def _check_bwd(dy, x, stats, gamma, dx, dgamma, dbeta):
    u = torch.finfo(x.dtype).eps / 2
    rdx, rg, rb, slack, ge, ga, ba = _bwd_ref(dy, x, stats, gamma)
    assert ((dx.double() - rdx).abs() <= u * rdx.abs() + slack * (1 + u) + 2.0 ** -25).all()
    if dgamma is not None:
        # a column passes through at most rows / 1024 + 1 additions per lane, 6 + 2 in the workgroup, 64 + 16 in the join
        n = (x.shape[0] / 1024 + 90) * E
        assert ((dgamma.double() - rg).abs() <= ge + n * ga + E * rg.abs()).all()
        assert ((dbeta.double() - rb).abs() <= n * ba + E * rb.abs()).all()


# every lane count (8, 16, 32, 64, 256), each vector count, odd and unaligned widths, one row to many
SHAPES = [(1, 1), (3, 7), (5, 8), (2, 64), (9, 99), (33, 200), (257, 320), (40, 333), (65, 640), (31, 768), (130, 1000), (17, 1280), (8, 2049),
          (6, 2560), (7, 2568), (5, 4096), (3, 8192), (2, 8199), (2, 16384), (5000, 320), (2100, 768), (1100, 2600), (3001, 48)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,C", SHAPES)
def test_forward_and_backward(dtype, rows, C):
    from hallo_amd import ops
    x, gamma, beta, dy = _data(rows, C, dtype)
    y, stats = ops.layernorm_train(x, gamma, beta, 1e-5)
    _check_fwd(x, gamma, beta, 1e-5, y, stats)
    dx, dg, db = ops.layernorm_backward(dy, x, stats, gamma)
    _check_bwd(dy, x, stats, gamma, dx, dg, db)
    again = ops.layernorm_backward(dy, x, stats, gamma)
    assert all(torch.equal(a, b) for a, b in zip((dx, dg, db), again))
    only = ops.layernorm_backward(dy, x, stats, gamma, weight_grads=False)
    assert torch.equal(only[0], dx) and only[1] is None and only[2] is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["f32", "none", "gamma_only"])
def test_weight_forms(dtype, kind):
    from hallo_amd import ops
    for C in (320, 333):
        x, gamma, beta, dy = _data(70, C, dtype, 3)
        g, b = {"f32": (gamma.float() + 1e-4, beta.float()), "none": (None, None), "gamma_only": (gamma, None)}[kind]
        y, stats = ops.layernorm_train(x, g, b, 1e-6)
        _check_fwd(x, g, b, 1e-6, y, stats)
        _check_bwd(dy, x, stats, g, *ops.layernorm_backward(dy, x, stats, g))


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_in_place_and_surroundings(dtype):
    """Column slices at odd offsets and pitches; in place; nothing beside the rows is written."""
    from hallo_amd import ops
    for C, pitch, off in ((320, 400, 8), (320, 401, 3), (77, 90, 5)):
        x, gamma, beta, dy = _data(50, C, dtype, 5)
        bx, bd, bo = (torch.full((52, pitch), 7.0, device="cuda", dtype=dtype) for _ in range(3))
        vx, vd, vo = (t[1:51, off:off + C] for t in (bx, bd, bo))
        vx.copy_(x), vd.copy_(dy)
        y, stats = ops.layernorm_train(vx, gamma, beta, out=vo)
        y2, stats2 = ops.layernorm_train(x, gamma, beta)
        _check_fwd(x, gamma, beta, 1e-5, y.contiguous(), stats)
        assert (bo.double().sum() - vo.double().sum() - 7.0 * (52 * pitch - 50 * C)).abs() < 1e-6
        dx, dg, db = ops.layernorm_backward(vd, vx, stats, gamma, out=vd)
        _check_bwd(dy, x, stats, gamma, dx.contiguous(), dg, db)
        assert torch.equal(bx[1:51, off:off + C], x)
        ops.layernorm_train(vx, gamma, beta, out=vx)
        _check_fwd(x, gamma, beta, 1e-5, vx.contiguous(), stats)
        del y2, stats2


@pytest.mark.parametrize("dtype", DTYPES)
def test_constant_rows_nan_and_no_rows(dtype):
    from hallo_amd import ops
    x, gamma, beta, dy = _data(6, 320, dtype, 9)
    x[1] = 3.0                                   # variance 0: y = beta, rstd = eps^-1/2
    x[4, 17] = float("nan")
    y, stats = ops.layernorm_train(x, gamma, beta, 1e-5)
    keep = [0, 1, 2, 3, 5]
    _check_fwd(x[keep], gamma, beta, 1e-5, y[keep], stats[keep])
    assert torch.isnan(y[4]).all() and not torch.isnan(y[keep]).any()
    dx, dg, db = ops.layernorm_backward(dy, x, stats, gamma)
    _check_bwd(dy[keep], x[keep], stats[keep], gamma, dx[keep], None, None)
    assert torch.isnan(dx[4]).all()
    e = x[:0]
    y, stats = ops.layernorm_train(e, gamma, beta)
    dx, dg, db = ops.layernorm_backward(e, e, stats, gamma)
    assert y.shape == (0, 320) and dx.shape == (0, 320) and (dg == 0).all() and (db == 0).all()


def test_gradient_against_differences():
    """The backward pass against central differences of the forward formula in 64 bits."""
    from hallo_amd import ops
    x, gamma, beta, dy = _data(4, 40, torch.float16, 13)
    _, stats = ops.layernorm_train(x, gamma, beta)
    dx, dg, db = ops.layernorm_backward(dy, x, stats, gamma)

    def loss(xx, gg, bb):
        d = xx - xx.mean(1, keepdim=True)
        return ((d * (d.square().mean(1, keepdim=True) + 1e-5).rsqrt() * gg + bb) * dy.double()).sum()
    h = 1e-5
    for name, t, got in (("x", x, dx), ("g", gamma, dg), ("b", beta, db)):
        t = t.double()
        for k in range(0, t.numel(), 7):
            step = torch.zeros_like(t).view(-1)
            step[k] = h
            step = step.view_as(t)
            a = {"x": x.double(), "g": gamma.double(), "b": beta.double()}
            hi, lo = dict(a, **{name: t + step}), dict(a, **{name: t - step})
            num = (loss(hi["x"], hi["g"], hi["b"]) - loss(lo["x"], lo["g"], lo["b"])) / (2 * h)
            # third-order term of the difference ~ h^2, its rounding ~ 1e-16 / h; one fp16 rounding of dx; stats in fp32
            assert abs(num.item() - got.view(-1)[k].item()) <= 2.0 ** -11 * abs(num.item()) + 1e-6


def test_same_as_inference_layernorm():
    """The training forward agrees with ops.layernorm to the last rounding."""
    from hallo_amd import ops
    for dtype in DTYPES:
        x, gamma, beta, _ = _data(300, 320, dtype, 21)
        a = ops.layernorm(x, gamma, beta, 1e-5).double()
        b = ops.layernorm_train(x, gamma, beta, 1e-5)[0].double()
        assert ((a - b).abs() <= torch.finfo(dtype).eps * a.abs() + 1e-6).all()
