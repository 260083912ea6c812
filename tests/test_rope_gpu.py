"""GPU tests of multi-axis rotary positions against the definition in 64 bits.

Tolerance per element of a pair (m, n): one rounding to the storage type, two products and a sum in fp32 (3 * 2^-24 of |m| + |n|), and
the angle: 2^-32 turns cut off, one fp32 rounding of a value below half a turn (pi * 2^-25), sincospi's own 2 ulp -- together under
2^-21 of |m| + |n|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def _ref(x, dims, hd, pos, theta, interleaved, inverse):
    """(y, |m| + |n| per element) in 64 bits; pos [B or 1, L, axes]."""
    B, L, W = x.shape
    x = x.double().reshape(B, L, W // hd, hd)
    y, mag = x.clone(), torch.zeros_like(x)
    at = 0
    for a, d in enumerate(dims):
        for i in range(d // 2):
            ang = pos[:, :, a].double() * theta ** (-2.0 * i / d)
            c, s = ang.cos()[..., None], ang.sin()[..., None] * (-1 if inverse else 1)
            m, n = (at + 2 * i, at + 2 * i + 1) if interleaved else (at + i, at + i + d // 2)
            y[..., m] = x[..., m] * c - x[..., n] * s
            y[..., n] = x[..., n] * c + x[..., m] * s
            mag[..., m] = mag[..., n] = x[..., m].abs() + x[..., n].abs()
        at += d
    return y.reshape(B, L, W), mag.reshape(B, L, W)


def _check(x, got, dims, hd, pos, theta, il, inverse):
    u = torch.finfo(x.dtype).eps / 2
    y, mag = _ref(x, dims, hd, pos, theta, il, inverse)
    tol = u * y.abs() + 2.0 ** -21 * (1 + u) * mag
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25                   # half a step of the subnormal numbers
    assert ((got.double() - y).abs() <= tol).all()


def _x(B, L, W, dtype, seed=0, pitch=0, off=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 13 * L + W)
    return torch.randn(B, L, W + pitch, generator=g, device="cuda").to(dtype)[..., off:off + W]


# piece widths 8 / 4 / 2 / 1, one to four axes, columns that pass through, one token to many, one head to many
CASES = [((16,), 16, 1, 1, 1), ((32, 48, 48), 128, 3, 5, 4), ((8, 16, 16), 40, 16, 2, 100), ((12, 26, 26), 80, 3, 2, 37), ((2, 4, 6, 50), 64, 2, 1, 23),
         ((22, 24, 28), 74, 5, 3, 19), ((2,), 256, 1, 1, 300), ((64, 64, 64, 64), 256, 2, 1, 70), ((10, 10), 22, 7, 1, 2000), ((160,), 160, 1, 2, 65),
         ((128,), 128, 40, 8, 1), ((4, 4, 4), 12, 1, 1, 5000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims,hd,heads,B,L", CASES)
def test_positions(dtype, interleaved, dims, hd, heads, B, L):
    from hallo_amd import ops
    axes = ops.RopeAxes(dims, hd, theta=10000.0, interleaved=interleaved)
    x = _x(B, L, heads * hd, dtype)
    g = torch.Generator(device="cuda").manual_seed(L)
    pos = torch.randint(-1000, 100000, (B, L, len(dims)), generator=g, device="cuda", dtype=torch.int32)
    y = ops.rope(x, axes, pos=pos)
    _check(x, y, dims, hd, pos, 10000.0, interleaved, False)
    _check(x, ops.rope(x, axes, pos=pos[0]), dims, hd, pos[:1], 10000.0, interleaved, False)
    back = ops.rope(x, axes, pos=pos, inverse=True)
    _check(x, back, dims, hd, pos, 10000.0, interleaved, True)
    z = x.clone()
    assert ops.rope(z, axes, pos=pos, out=z) is z and torch.equal(z, y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("grid,origin", [((5, 3, 7), None), ((1, 1, 1), (4, 5, 6)), ((16, 8, 9), (1000000, -3, 2)), ((2, 33, 65), (0, 0, 0))])
def test_grid(dtype, grid, origin):
    from hallo_amd import ops
    dims, hd, heads = (8, 16, 16), 40, 3
    L = math.prod(grid)
    axes = ops.RopeAxes(dims, hd, theta=500.0)
    x = _x(2, L, heads * hd, dtype)
    o = origin or (0, 0, 0)
    pos = torch.stack(torch.meshgrid(*[torch.arange(n, device="cuda") + s for n, s in zip(grid, o)], indexing="ij"), -1).view(1, L, 3)
    y = ops.rope(x, axes, grid=grid, origin=origin)
    _check(x, y, dims, hd, pos, 500.0, False, False)
    assert torch.equal(y, ops.rope(x, axes, pos=pos[0].int().contiguous()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_positions(dtype):
    """Positions over the whole 32-bit range: the angle keeps its place within the turn."""
    from hallo_amd import ops
    axes = ops.RopeAxes((64,), 64)
    vals = [0, 1, -1, 2 ** 24 + 1, 2 ** 30 + 7, 2 ** 31 - 1, -2 ** 31, -2 ** 31 + 5]
    pos = torch.tensor(vals, device="cuda", dtype=torch.int32).view(-1, 1)
    x = _x(1, len(vals), 2 * 64, dtype)
    # freq = 2^-53 relative and theta^x of the two sides as well: 2^31 * 2^-52 rad = 2^-21
    u = torch.finfo(dtype).eps / 2
    y, mag = _ref(x, (64,), 64, pos.view(1, -1, 1), 10000.0, False, False)
    got = ops.rope(x, axes, pos=pos)
    assert ((got.double() - y).abs() <= u * y.abs() + 2.0 ** -20 * mag + (2.0 ** -25 if dtype == torch.float16 else 0)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pitch,off", [(80, 0), (80, 8), (7, 3), (6, 2)])
def test_views(dtype, pitch, off):
    """q | k columns of a wider buffer (aligned and not), in place: the other columns stay."""
    from hallo_amd import ops
    dims, hd = (8, 16, 16), 40
    axes = ops.RopeAxes(dims, hd)
    x = _x(2, 60, 4 * hd, dtype, 5, pitch, off)
    base = x._base if x._base is not None else x
    buf = torch.full((2, 60, 4 * hd + pitch), 3.0, device="cuda", dtype=dtype)
    v = buf[..., off:off + 4 * hd]
    v.copy_(x)
    pos = torch.stack(torch.meshgrid(torch.arange(3), torch.arange(4), torch.arange(5), indexing="ij"), -1).view(1, 60, 3).cuda()
    ops.rope(v, axes, grid=(3, 4, 5), out=v)
    _check(x, v, dims, hd, pos, 10000.0, False, False)
    assert (buf[..., :off] == 3.0).all() and (buf[..., off + 4 * hd:] == 3.0).all()
    w = ops.rope(x.transpose(0, 1).contiguous().transpose(0, 1), axes, grid=(3, 4, 5))      # batch inside the rows
    assert torch.equal(w, v)
    del base


def test_gradient():
    """inverse=True is the transposed map: <rope(x), dy> = <x, rope(dy, inverse)>, against 64-bit differences too."""
    from hallo_amd import ops
    axes = ops.RopeAxes((6, 10), 20)
    x, dy = _x(1, 9, 40, torch.float16, 1), _x(1, 9, 40, torch.float16, 2)
    pos = torch.randint(0, 500, (9, 2), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(4))
    dx = ops.rope(dy, axes, pos=pos, inverse=True)
    for k in range(0, 360, 11):
        e = torch.zeros(360, device="cuda", dtype=torch.float64)
        e[k] = 1e-3
        e = e.view(1, 9, 40)
        f = lambda t: (_ref(t, (6, 10), 20, pos[None], 10000.0, False, False)[0] * dy.double()).sum()
        num = ((f(x.double() + e) - f(x.double() - e)) / 2e-3).item()
        assert abs(num - dx.view(-1)[k].item()) <= 2.0 ** -11 * abs(num) + 2.0 ** -19


def test_nothing_to_do():
    from hallo_amd import ops
    axes = ops.RopeAxes((8,), 8)
    assert ops.rope(torch.empty(2, 0, 8, device="cuda", dtype=torch.float16), axes, pos=torch.empty(0, 1, device="cuda", dtype=torch.int32)).shape == (2, 0, 8)
    assert ops.rope(torch.empty(0, 3, 8, device="cuda", dtype=torch.float16), axes, grid=(3,)).shape == (0, 3, 8)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims,hd", [((6, 10), 24), ((8, 16), 32), ((6, 8), 20)])
def test_no_number_stays_where_it_is(dims, hd, interleaved):
    """A NaN or an infinity reaches its pair, at every angle, and nothing else; columns that pass through keep theirs."""
    from hallo_amd import ops
    axes = ops.RopeAxes(dims, hd, interleaved=interleaved)
    pos = torch.tensor([[0, 0], [3, 0], [0, 5]], device="cuda", dtype=torch.int32)
    for bad in (float("nan"), float("inf")):
        for col in range(hd):
            x = torch.ones(1, 3, 2 * hd, device="cuda", dtype=torch.float16)
            x[..., hd + col] = bad
            got = torch.isfinite(ops.rope(x, axes, pos=pos))
            want = torch.isfinite(_ref(x, dims, hd, pos[None], 10000.0, interleaved, False)[0])
            assert torch.equal(got, want), (bad, col)
