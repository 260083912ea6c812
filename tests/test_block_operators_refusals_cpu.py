"""CPU tests of calls that the block operators refuse because their results could not be right: outputs whose parts lie on one another or
on an input, positions past 32 bits."""
import ctypes as C

import pytest
import torch

from hallo_amd import ops

from test_block_operators_cpu import Err, _mem, _rope_desc, host, lib  # noqa: F401  (fixtures)

H = torch.float16


def _strided(n, shape, strides, offset=0):
    return torch.zeros(n, dtype=H).as_strided(shape, strides, offset)


@pytest.mark.parametrize("shape,strides", [((2, 6, 32), (32, 32, 1)), ((2, 6, 32), (96, 32, 1)), ((2, 6, 32), (200, 40, 1)), ((3, 2, 32), (48, 100, 1)),
                                           ((2, 6, 32), (176, 64, 1))])
def test_rope_entries_on_one_another(host, shape, strides):  # noqa: F811
    axes = ops.RopeAxes((8, 8), 16, device="cpu")
    x, pos = torch.zeros(shape, dtype=H), torch.zeros(shape[1], 2, dtype=torch.int32)
    with pytest.raises(Err, match="overlap"):
        ops.rope(x, axes, pos=pos, out=_strided(4096, shape, strides))


@pytest.mark.parametrize("shape,strides", [((2, 6, 32), (192, 32, 1)), ((2, 6, 32), (32, 64, 1)), ((2, 6, 32), (40, 80, 1)), ((1, 6, 32), (0, 32, 1)),
                                           ((2, 1, 32), (32, 0, 1)), ((2, 6, 32), (500, 50, 1))])
def test_rope_entries_apart(host, shape, strides):  # noqa: F811
    """Batch outside or inside of the rows, with and without room between them: these reach the library."""
    axes = ops.RopeAxes((8, 8), 16, device="cpu")
    x, pos = torch.zeros(shape, dtype=H), torch.zeros(shape[1], 2, dtype=torch.int32)
    host.setattr(ops, "_call", lambda *a: None)
    out = _strided(4096, shape, strides)
    assert ops.rope(x, axes, pos=pos, out=out) is out


def test_rope_abi_entries_on_one_another(lib):  # noqa: F811
    keep, p = _mem(1 << 16)
    call = lambda **kw: lib.hallo_rope(C.byref(_rope_desc(p, **dict(dict(y=p + 8192, batch=2), **kw))), None)
    for kw in (dict(y_bs=0), dict(y_bs=40), dict(y_bs=200), dict(y_bs=-240), dict(y_bs=100, y_rs=80), dict(y_bs=39, y_rs=80)):
        assert call(**kw) == -22, kw
    del keep


def test_rope_abi_positions_past_32_bits(lib):  # noqa: F811
    keep, p = _mem(1 << 16)
    call = lambda **kw: lib.hallo_rope(C.byref(_rope_desc(p, **kw)), None)
    for origin in ((2 ** 31 - 1, 0), (0, 2 ** 31 - 2)):
        assert call(origin=origin) == -22, origin
    del keep


def _accepted(f, *a, **kw):
    f(*a, **kw)


def _refused(f, *a, match, **kw):
    with pytest.raises(Err, match=match):
        f(*a, **kw)


def test_layernorm_outputs_on_inputs(host):  # noqa: F811
    host.setattr(ops, "_call", lambda *a: None)
    buf = torch.zeros(4096, dtype=H)
    rows = lambda off, pitch=48, n=8: buf.as_strided((n, 32), (pitch, 1), off)
    x, gamma, stats = rows(0), buf[3000:3032], torch.zeros(8, 2)
    far = buf[2000:2256].view(8, 32)
    for out in (rows(8), rows(48), rows(0, 64), rows(0, 32), rows(24, 96)):
        _refused(ops.layernorm_train, x, out=out, match="overlaps x")
        _refused(ops.layernorm_backward, far, x, stats, out=out, weight_grads=False, match="overlaps x")
        _refused(ops.layernorm_backward, x, far, stats, out=out, weight_grads=False, match="overlaps dy")
    _refused(ops.layernorm_train, x, gamma, out=rows(2900), match="overlaps gamma")
    _refused(ops.layernorm_train, x, None, gamma, out=rows(2900), match="overlaps beta")
    wide = buf.as_strided((8, 32), (96, 1), 0)
    for out in (rows(0), far, rows(8 * 48)):     # the same rows, others, behind them
        _accepted(ops.layernorm_train, x, out=out)
        _accepted(ops.layernorm_backward, far, x, stats, out=out, weight_grads=False)
    for off in (32, 64):                         # column slices of one buffer
        _accepted(ops.layernorm_train, wide, out=buf.as_strided((8, 32), (96, 1), off))
    one = buf.as_strided((1, 32), (7, 1), 0)     # the stride of a single row does not count
    _accepted(ops.layernorm_train, buf.as_strided((1, 32), (32, 1), 0), out=one)


def test_layernorm_abi_in_place_at_another_pitch(lib):  # noqa: F811
    keep, p = _mem(1 << 16)
    q = p + 8192
    assert lib.hallo_layernorm_train(p, 32, p, 40, None, None, 0, q, 4, 32, 1e-5, 0, None) == -22
    for dy, x, lddy, ldx in ((p, q, 32, 40), (q, p, 40, 32)):
        assert lib.hallo_layernorm_backward(dy, lddy, x, ldx, q, None, 0, p, 40, None, None, None, 0, 4, 32, 0, None) == -22
    del keep


def test_rope_outputs_on_inputs(host):  # noqa: F811
    host.setattr(ops, "_call", lambda *a: None)
    axes = ops.RopeAxes((8, 8), 16, device="cpu")
    buf = torch.zeros(8192, dtype=H)
    at = lambda off, bs=600, rs=96: buf.as_strided((2, 6, 32), (bs, rs, 1), off)
    x, pos = at(0), torch.zeros(6, 2, dtype=torch.int32)
    for out in (at(8), at(96), at(0, 600, 64), at(0, 700), at(80)):
        _refused(ops.rope, x, axes, pos=pos, out=out, match="overlaps x")
    for out in (at(0), at(32), at(64), at(2000)):
        _accepted(ops.rope, x, axes, pos=pos, out=out)


def test_window_attention_outputs_on_inputs(host):  # noqa: F811
    host.setattr(ops, "_call", lambda *a: None)

    class Lib:
        hallo_window_attention_workspace = hallo_window_attention_backward_workspace = staticmethod(lambda d: 0)
    host.setattr(ops._l, "load", lambda *a: Lib)
    q, k, v = (torch.zeros(2, 5, 64, dtype=H) for _ in range(3))
    for name, t in (("q", q), ("k", k), ("v", v)):
        _refused(ops.window_attention, q, k, v, 4, out=t, match=f"overlaps {name}")
    fused = torch.zeros(2, 5, 256, dtype=H)
    parts = fused.split(64, 2)
    _accepted(ops.window_attention, *parts[:3], 4, out=parts[3])
    _refused(ops.window_attention, *parts[:3], 4, out=fused[..., 184:248], match="overlaps v")
    heads = torch.zeros(2, 8, 5, 16, dtype=H)    # head-major
    _accepted(ops.window_attention, q.view(2, 5, 4, 16), k, v, 4, out=heads[:, 4:].transpose(1, 2))
    _refused(ops.window_attention, heads[:, :4].transpose(1, 2), k, v, 4, out=heads[:, 3:7].transpose(1, 2), match="overlaps q")
    lse, do, o = torch.zeros(2, 4, 5), torch.zeros_like(q), torch.zeros_like(q)
    b = lambda **kw: ops.window_attention_backward(do, q, k, v, o, lse, 4, **kw)
    for name, t in (("do", do), ("q", q), ("k", k), ("v", v), ("o", o)):
        for out in ("dq", "dk", "dv"):
            _refused(b, **{out: t}, match=f"{out}: overlaps {name}")
    d = torch.zeros_like(q)
    for a, c in (("dq", "dk"), ("dq", "dv"), ("dk", "dv")):
        _refused(b, **{a: d, c: d}, match=f"{a}: overlaps {c}")
        _refused(b, **{a: fused[..., :64], c: fused[..., 32:96]}, match=f"{a}: overlaps {c}")
    _accepted(b, dq=parts[0], dk=parts[1], dv=parts[2])
    _accepted(b, dq=parts[0])


def test_inputs_that_need_a_gradient(host):  # noqa: F811
    """The forward calls record nothing for torch's differentiation: an input that waits for a gradient would silently get none."""
    host.setattr(ops, "_call", lambda *a: None)

    class Lib:
        hallo_window_attention_workspace = staticmethod(lambda d: 0)
    host.setattr(ops._l, "load", lambda *a: Lib)
    leaf = lambda *s: torch.zeros(*s, dtype=H, requires_grad=True)
    x, w, axes = torch.zeros(4, 32, dtype=H), torch.zeros(32, dtype=H), ops.RopeAxes((8, 8), 16, device="cpu")
    s, pos = torch.zeros(2, 6, 32, dtype=H), torch.zeros(6, 2, dtype=torch.int32)
    calls = [(ops.layernorm_train, (leaf(4, 32),), {}), (ops.layernorm_train, (x, leaf(32), w), {}), (ops.layernorm_train, (x, w, leaf(32)), {}),
             (ops.layernorm_train, (x, torch.ones(32, requires_grad=True)), {}), (ops.rope, (leaf(2, 6, 32), axes), dict(pos=pos)),
             (ops.window_attention, (leaf(2, 6, 32), s, s, 2), {}), (ops.window_attention, (s, leaf(2, 6, 32), s, 2), {}),
             (ops.window_attention, (s, s, leaf(2, 6, 32) * 1, 2), {}), (ops.layernorm_train, (x,), dict(out=leaf(4, 32))),
             (ops.rope, (s, axes), dict(pos=pos, out=leaf(2, 6, 32))), (ops.window_attention, (s, s, s, 2), dict(out=leaf(2, 6, 32)))]
    for f, a, kw in calls:
        _refused(f, *a, **kw, match="gradient")
        with torch.no_grad():
            _accepted(f, *a, **kw)
        with torch.inference_mode():
            _accepted(f, *a, **kw)
        cut = lambda t: t.detach() if torch.is_tensor(t) else t
        _accepted(f, *map(cut, a), **{n: cut(t) for n, t in kw.items()})


def test_inside_a_function_of_torch(host):  # noqa: F811
    """torch calls forward() of an autograd.Function without recording: the calls a user's own Function makes pass."""
    host.setattr(ops, "_call", lambda *a: None)

    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, gamma):
            y, stats = ops.layernorm_train(x, gamma)
            ctx.save_for_backward(x, gamma, stats)
            return y

        @staticmethod
        def backward(ctx, dy):
            x, gamma, stats = ctx.saved_tensors
            return ops.layernorm_backward(dy.contiguous(), x, stats, gamma, weight_grads=False)[0], None
    x = torch.zeros(4, 32, dtype=H, requires_grad=True)
    Norm.apply(x, torch.ones(32, dtype=H)).sum().backward()
    assert x.grad.shape == x.shape


def test_given_outputs_count_as_changed(host):  # noqa: F811
    """torch notices that a tensor which it keeps for a gradient was written: its version goes up with every call that is given it."""
    host.setattr(ops, "_call", lambda *a: None)

    class Lib:
        hallo_window_attention_workspace = hallo_window_attention_backward_workspace = staticmethod(lambda d: 0)
    host.setattr(ops._l, "load", lambda *a: Lib)
    x, stats, axes, pos = torch.zeros(2, 6, 32, dtype=H), torch.zeros(12, 2), ops.RopeAxes((8, 8), 16, device="cpu"), torch.zeros(6, 2, dtype=torch.int32)
    a = [torch.zeros_like(x) for _ in range(6)]
    lse, new = torch.zeros(2, 2, 6), lambda: torch.zeros_like(x)
    calls = [lambda t: ops.layernorm_train(x, out=t), lambda t: ops.layernorm_backward(x, x, stats, weight_grads=False, out=t),
             lambda t: ops.rope(x, axes, pos=pos, out=t), lambda t: ops.window_attention(*a[:3], 2, out=t)]
    calls += [lambda t, n=n: ops.window_attention_backward(*a[:5], lse, 2, **{n: t}) for n in ("dq", "dk", "dv")]
    for f in calls:
        t, w = new(), torch.zeros(2, 6, 32, dtype=H, requires_grad=True)
        kept = (w * t).sum()
        v = t._version
        f(t)
        assert t._version > v
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()
        with torch.inference_mode():
            f(new())


def test_tensors_of_one_dimension(host):  # noqa: F811
    q, one, lse = torch.zeros(2, 5, 64, dtype=H), torch.zeros(64, dtype=H), torch.zeros(2, 2, 5)
    for lse_too in (False, True):
        _refused(ops.window_attention, one, q, q, 2, return_lse=lse_too, match="q:")
    _refused(ops.window_attention_backward, one, one, q, q, one, lse, 2, match="q:")


def test_rope_frequencies_past_a_float():
    for theta in (1e-300, 5e-324):
        _refused(ops.RopeAxes, (64,), 64, theta=theta, device="cpu", match="theta")


def test_window_attention_splits(lib):  # noqa: F811
    """How a call is divided, from its descriptor alone: one form refuses what the call refuses, and needs no memory."""
    from test_block_operators_cpu import BAD_ATTN, _attn_desc
    ask = lambda **kw: lib.hallo_window_attention_splits(C.byref(_attn_desc(0, **kw)))
    assert lib.hallo_window_attention_splits(None) == -22
    for kw in BAD_ATTN:
        assert ask(**kw) == -22, kw
    assert ask(batch=0) == 0 and ask(Lq=0) == 0 and ask() == 1
    assert ask(Lq=1, Lk=100000, left=-1) > 1 and ask(batch=64, heads=32, kv_heads=32, Lq=1000, Lk=1000) == 0


def test_rope_batch_inside_of_the_rows_is_told_at_once():
    """Tokens first, batch second, as a sequence-first model lays x out: no walk over the batch."""
    import time
    t = time.perf_counter()
    assert not ops._entries_meet(1 << 30, 7, 64, 64 << 30, 64) and ops._entries_meet(1 << 30, 7, 64, (64 << 30) - 1, 65)
    assert time.perf_counter() - t < 1.0
