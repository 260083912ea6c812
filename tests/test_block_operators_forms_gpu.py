"""GPU tests at sizes that take each form of the block operators: window attention in blocks of 128 queries and in packed rows (asked of
the library, so that a change of its rule cannot move a test to another form unseen), LayerNorm gradients over several row groups per
workgroup, rotary positions of rows wider than a staged tile.  Bounds as in the operators' own tests."""
import ctypes as C

import pytest
import torch

import test_layernorm_train_gpu as ln
import test_rope_gpu as rt
from test_window_attention_gpu import HEAD_DIMS, WINDOWS, Ref, _both, _lens, _qkv

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _splits(B, Lq, Lk, H, Hkv, hd, left, right, sinks):
    """0: blocks of 128 queries; n: packed rows, the keys in n parts."""
    from hallo_amd import lib, ops
    d = lib.WindowAttnDesc(batch=B, heads=H, kv_heads=Hkv, head_dim=hd, Lq=Lq, Lk=Lk, left=ops._edge(left), right=ops._edge(right), sinks=ops._edge(sinks),
                           scale=1.0)
    return lib.load().hallo_window_attention_splits(C.byref(d))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", HEAD_DIMS)
def test_query_blocks_of_every_width(dtype, hd):
    for left, right, sinks in ((40, 0, 5), (-1, -1, 0), (33, 20, 70)):
        assert _splits(20, 150, 170, 8, 4, hd, left, right, sinks) == 0
        _both(20, 150, 170, 8, 4, hd, dtype, left, right, sinks, grads=False)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
def test_query_blocks_of_every_window(dtype, left, right, sinks):
    ql, kl = _lens(*range(181, 201)), _lens(*range(271, 291))
    for hd in (40, 64, 128, 160):                # two, two, one and two stages per pass; tiles of 64 and of 32 keys
        assert _splits(20, 200, 290, 8, 2, hd, left, right, sinks) == 0
        _both(20, 200, 290, 8, 2, hd, dtype, left, right, sinks, ql, kl, grads=False)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [64, 128])
def test_query_blocks_under_a_long_causal_mask(dtype, hd):
    assert _splits(1, 2100, 2100, 16, 8, hd, -1, 0, 0) == 0
    _both(1, 2100, 2100, 16, 8, hd, dtype, -1, 0, 0, _lens(2001), _lens(2077))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [48, 64, 80, 128, 144])
def test_query_blocks_ragged_and_empty(dtype, hd):
    """Entries without keys or queries, more queries than keys, lengths past the tensors, padding that holds NaN and infinities."""
    from hallo_amd import ops
    B, Lq, Lk, H, Hkv = 21, 150, 170, 8, 4
    ql, kl = _lens(*[150, 0, 100, 150, 3, 149, 9999] * 3), _lens(*[170, 50, 0, 20, 170, 1, 9999] * 3)
    for left, right, sinks in ((-1, 0, 0), (30, 0, 4), (20, 10, 0), (-1, -1, 0)):
        assert _splits(B, Lq, Lk, H, Hkv, hd, left, right, sinks) == 0
        q, k, v, do = _qkv(B, Lq, Lk, H, Hkv, hd, dtype, 3)
        ref = Ref(q, k, v, H, Hkv, left, right, sinks, ql, kl)
        bad = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0], device="cuda").to(dtype)
        gone = ~ref.ok.any(2).reshape(B, Lk)
        late = torch.arange(Lq, device="cuda") >= ref.ql.view(-1, 1)
        for t, rows in ((q, late), (do, late), (k, gone), (v, gone)):
            t[rows] = bad.repeat(t.shape[2] // 4)
        kw = dict(kv_heads=Hkv, left=left, right=right, sinks=sinks, q_len=ql, kv_len=kl)
        o, lse = ops.window_attention(q, k, v, H, return_lse=True, out=torch.full_like(q, 5.0), **kw)
        ref.check(o, lse)
        ref.check_grads(do, o, lse, *ops.window_attention_backward(do, q, k, v, o, lse, H, **kw))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", HEAD_DIMS)
def test_keys_in_parts(dtype, hd):
    """Few queries against many keys: parts of every width, joined by the second launch."""
    Lk = max(4000, 120000 // hd)                 # keys times columns decide
    for Lq, left, sinks in ((1, -1, 0), (3, Lk * 3 // 4, 7), (40, -1, 0)):
        assert _splits(2, Lq, Lk, 4, 2, hd, left, 0, sinks) > 1
        _both(2, Lq, Lk, 4, 2, hd, dtype, left, 0, sinks, None, _lens(Lk, Lk // 3), grads=False)


# row counts that leave a last group of fewer rows, over 1024 groups each: 8, 16, 32 and 64 lanes a row, one to three vectors a lane
@pytest.mark.parametrize("dtype", ln.DTYPES)
@pytest.mark.parametrize("rows,C", [(40001, 50), (33003, 99), (33001, 160), (17003, 320), (9001, 640), (4503, 1000), (70001, 64)])
def test_layernorm_over_several_row_groups(dtype, rows, C):
    from hallo_amd import ops
    x, gamma, beta, dy = ln._data(rows, C, dtype, 31)
    y, stats = ops.layernorm_train(x, gamma, beta, 1e-5)
    ln._check_fwd(x, gamma, beta, 1e-5, y, stats)
    got = ops.layernorm_backward(dy, x, stats, gamma)
    ln._check_bwd(dy, x, stats, gamma, *got)
    assert all(torch.equal(a, b) for a, b in zip(got, ops.layernorm_backward(dy, x, stats, gamma)))
    # at an odd pitch and in place: dx takes dy's place, and x's
    for name in ("dy", "x"):
        wide = torch.full((rows, C + 3), 7.0, device="cuda", dtype=dtype)
        view = wide[:, 1:C + 1]
        view.copy_(dy if name == "dy" else x)
        a, b = (view, x) if name == "dy" else (dy, view)
        dx, dg, db = ops.layernorm_backward(a, b, stats, gamma, out=view)
        ln._check_bwd(dy, x, stats, gamma, dx.contiguous(), dg, db)
        assert (wide[:, 0] == 7).all() and (wide[:, C + 1:] == 7).all()


@pytest.mark.parametrize("dtype", ln.DTYPES)
@pytest.mark.parametrize("rows,C", [(700, 130), (700, 136), (2, 192), (300, 191)])
def test_layernorm_three_vectors_on_eight_lanes(dtype, rows, C):
    from hallo_amd import ops
    x, gamma, beta, dy = ln._data(rows, C, dtype, 32)
    y, stats = ops.layernorm_train(x, gamma, beta, 1e-5)
    ln._check_fwd(x, gamma, beta, 1e-5, y, stats)
    ln._check_bwd(dy, x, stats, gamma, *ops.layernorm_backward(dy, x, stats, gamma))


def _rope(dims, hd, heads, B, L, dtype, interleaved, pitch=0, off=0):
    from hallo_amd import ops
    axes = ops.RopeAxes(dims, hd, interleaved=interleaved)
    x = rt._x(B, L, heads * hd, dtype, 3, pitch, off)
    pos = torch.randint(-1000, 100000, (B, L, len(dims)), generator=torch.Generator(device="cuda").manual_seed(L), device="cuda", dtype=torch.int32)
    y = ops.rope(x, axes, pos=pos)
    rt._check(x, y, dims, hd, pos, 10000.0, interleaved, False)
    wide = torch.full((B, L, heads * hd + pitch + 8), 3.0, device="cuda", dtype=dtype)
    view = wide[..., off:off + heads * hd]
    view.copy_(x)
    ops.rope(view, axes, pos=pos, out=view)
    assert torch.equal(view, y) and (wide[..., :off] == 3).all() and (wide[..., off + heads * hd:] == 3).all()


@pytest.mark.parametrize("dtype", rt.DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims,hd,heads", [((12, 26, 26), 80, 120), ((12, 26, 26), 74, 130), ((6, 10), 16, 600), ((254,), 256, 33), ((2,), 2, 5000)])
def test_rope_rows_wider_than_a_staged_tile(dtype, interleaved, dims, hd, heads):
    for pitch, off in ((0, 0), (24, 8), (5, 3)):
        _rope(dims, hd, heads, 2, 7, dtype, interleaved, pitch, off)


@pytest.mark.parametrize("dtype", rt.DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims,hd", [((16, 16), 40), ((8, 8), 16), ((6, 10), 22), ((4,), 4)])
def test_rope_most_tokens_of_a_workgroup(dtype, interleaved, dims, hd):
    _rope(dims, hd, 1, 2, 40009, dtype, interleaved)
