"""CPU tests of what the training operators refuse: the C ABI returns -22 before it touches the device, the Python entry points raise
HalloLibraryError before they call the library."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

from hallo_amd import lib as L
from hallo_amd import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
Err = L.HalloLibraryError


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(L.LIB_PATH):
        from hallo_amd import build
        build.build()
    return L.load()


@pytest.fixture
def host(monkeypatch, lib):
    """Host tensors pass the device check, and no call reaches the library."""
    class Closed:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")
    monkeypatch.setattr(ops, "_chk_dev", lambda *t: None)
    monkeypatch.setattr(ops._l, "load", lambda *a: Closed())
    return monkeypatch


def _mem(n=4096):
    buf = (C.c_char * (n + 16))()
    return buf, (C.addressof(buf) + 15) // 16 * 16


def test_struct_sizes(lib):
    src = '#include "hallo_amd.h"\n#include <stdio.h>\nint main(){printf("%zu %zu %zu\\n", sizeof(hallo_rope_desc),' \
          ' sizeof(hallo_window_attn_desc), sizeof(hallo_window_attn_bwd_desc));return 0;}\n'
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "s.c"), os.path.join(td, "s")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [C.sizeof(t) for t in (L.RopeDesc, L.WindowAttnDesc, L.WindowAttnBwdDesc)]


def test_layernorm_abi(lib):
    keep, p = _mem()
    good = dict(x=p, ldx=32, y=p, ldy=32, g=p, b=p, f32=0, st=p, rows=4, C=32, eps=1e-5, dt=0)

    def fwd(**kw):
        a = dict(good, **kw)
        return lib.hallo_layernorm_train(a["x"], a["ldx"], a["y"], a["ldy"], a["g"], a["b"], a["f32"], a["st"], a["rows"], a["C"], a["eps"], a["dt"], None)
    for kw in (dict(x=None), dict(y=None), dict(st=None), dict(ldx=31), dict(ldy=31), dict(rows=-1), dict(C=0), dict(C=16385, ldx=16385, ldy=16385),
               dict(eps=-1.0), dict(eps=float("nan")), dict(f32=2), dict(dt=2), dict(dt=-1)):
        assert fwd(**kw) == -22, kw
    assert fwd(rows=0) == 0
    good = dict(dy=p, ldd=32, x=p, ldx=32, st=p, g=p, f32=0, dx=p, ldo=32, dg=p, db=p, ws=p, wb=1 << 20, rows=4, C=32, dt=0)

    def bwd(**kw):
        a = dict(good, **kw)
        return lib.hallo_layernorm_backward(a["dy"], a["ldd"], a["x"], a["ldx"], a["st"], a["g"], a["f32"], a["dx"], a["ldo"], a["dg"], a["db"], a["ws"],
                                            a["wb"], a["rows"], a["C"], a["dt"], None)
    for kw in (dict(dy=None), dict(x=None), dict(st=None), dict(dx=None), dict(dg=None), dict(db=None), dict(ws=None), dict(wb=0), dict(ldd=8),
               dict(ldx=8), dict(ldo=8), dict(rows=-1), dict(C=0), dict(f32=3), dict(dt=7)):
        assert bwd(**kw) == -22, kw
    assert lib.hallo_layernorm_backward_workspace(-1, 32) == -22 and lib.hallo_layernorm_backward_workspace(4, 0) == -22
    assert lib.hallo_layernorm_backward_workspace(1 << 40, 16384) == 1024 * 2 * 16384 * 4
    del keep


def _rope_desc(p, **kw):
    d = L.RopeDesc()
    d.x = d.y = d.freq = p
    d.x_bs = d.y_bs = 6 * 40
    d.x_rs = d.y_rs = 40
    d.batch, d.L, d.heads, d.head_dim, d.n_axes = 1, 6, 2, 20, 2
    for i, (n, g) in enumerate(((8, 2), (10, 3))):
        d.dims[i], d.grid[i] = n, g
    for k, v in kw.items():
        if isinstance(v, tuple):
            for i, x in enumerate(v):
                getattr(d, k)[i] = x
        else:
            setattr(d, k, v)
    return d


def test_rope_abi(lib):
    keep, p = _mem()
    call = lambda **kw: lib.hallo_rope(C.byref(_rope_desc(p, **kw)), None)
    assert lib.hallo_rope(None, None) == -22
    for kw in (dict(x=None), dict(y=None), dict(freq=None), dict(dtype=2), dict(batch=-1), dict(L=-1), dict(heads=0), dict(head_dim=0), dict(head_dim=19),
               dict(head_dim=258), dict(n_axes=0), dict(n_axes=5), dict(dims=(7, 10)), dict(dims=(0, 10)), dict(dims=(12, 10)), dict(grid=(2, 4)),
               dict(grid=(0, 3)), dict(grid=(1 << 30, 1 << 30)), dict(x_rs=-40), dict(y_rs=39), dict(x_bs=480)):
        assert call(**kw) == -22, kw
    assert call(batch=0) == 0 and call(L=0) == 0
    del keep


def _attn_desc(p, **kw):
    d = L.WindowAttnDesc()
    d.q = d.k = d.v = d.o = p
    for n in "qkvo":
        setattr(d, n + "_bs", 4 * 32)
        setattr(d, n + "_rs", 32)
        setattr(d, n + "_hs", 16)
    d.Lq = d.Lk = 4
    d.batch, d.heads, d.kv_heads, d.head_dim, d.scale = 1, 2, 2, 16, 0.25
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD_ATTN = [dict(dtype=2), dict(batch=-1), dict(heads=0), dict(kv_heads=0), dict(heads=3), dict(head_dim=0), dict(head_dim=12), dict(head_dim=168),
            dict(Lq=-1), dict(Lk=-1), dict(Lq=(1 << 29) + 1), dict(Lk=(1 << 29) + 1), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0),
            dict(scale=float("nan")), dict(scale=float("inf")), dict(q_rs=12), dict(k_bs=-8), dict(v_rs=(1 << 24) + 8), dict(o_hs=4), dict(batch=1 << 30, heads=2)]


def test_window_attention_abi(lib):
    keep, p = _mem()
    call = lambda **kw: lib.hallo_window_attention(C.byref(_attn_desc(p, **kw)), None)
    assert lib.hallo_window_attention(None, None) == -22 and lib.hallo_window_attention_workspace(None) == -22
    for kw in BAD_ATTN + [dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(q=p + 2), dict(o=p + 8)]:
        assert call(**kw) == -22, kw
    for kw in BAD_ATTN:
        assert lib.hallo_window_attention_workspace(C.byref(_attn_desc(p, **kw))) == -22, kw
    assert call(batch=0) == 0 and call(Lq=0) == 0
    long = dict(Lq=1, Lk=100000, left=-1)
    assert lib.hallo_window_attention_workspace(C.byref(_attn_desc(p, **long))) > 0 and call(**long) == -22      # no workspace
    assert lib.hallo_window_attention_workspace(C.byref(_attn_desc(p, Lq=1, Lk=100000, left=5, sinks=1))) == 0


@pytest.mark.parametrize("kw", [dict(scale=1e-31), dict(heads=1 << 28, kv_heads=1 << 28, Lq=8)])
def test_window_attention_limits(lib, kw):
    """A scale whose rescaling threshold would overflow, query rows that pass 32 bits."""
    keep, p = _mem()
    assert lib.hallo_window_attention(C.byref(_attn_desc(p, **kw)), None) == -22
    assert lib.hallo_window_attention_workspace(C.byref(_attn_desc(p, **kw))) == -22


def test_window_attention_backward_abi(lib):
    keep, p = _mem()

    def desc(fwd=None, **kw):
        d = L.WindowAttnBwdDesc()
        d.fwd = _attn_desc(p, **dict(dict(lse=p, workspace=p, workspace_bytes=1 << 30), **(fwd or {})))
        d.dout = d.dq = d.dk = d.dv = p
        for n in ("do", "dq", "dk", "dv"):
            setattr(d, n + "_bs", 4 * 32)
            setattr(d, n + "_rs", 32)
            setattr(d, n + "_hs", 16)
        for k, v in kw.items():
            setattr(d, k, v)
        return d
    call = lambda **kw: lib.hallo_window_attention_backward(C.byref(desc(**kw)), None)
    assert lib.hallo_window_attention_backward(None, None) == -22 and lib.hallo_window_attention_backward_workspace(None) == -22
    for kw in BAD_ATTN + [dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(lse=None), dict(workspace=None), dict(workspace_bytes=64),
                          dict(workspace=p + 4)]:
        assert call(fwd=kw) == -22, kw
    for kw in (dict(dout=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(do_rs=4), dict(dq_bs=-8), dict(dk_rs=(1 << 24) + 8), dict(dv=p + 2)):
        assert call(**kw) == -22, kw
    assert call(fwd=dict(batch=0)) == 0
    del keep


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 32, dtype=torch.float16)
    for f in (lambda: ops.layernorm_train(x), lambda: ops.layernorm_backward(x, x, x), lambda: ops.window_attention(x, x, x, 2),
              lambda: ops.window_attention_backward(x, x, x, x, x, x, 2), lambda: ops.rope(x, ops.RopeAxes((8,), 16, device="cpu"), grid=(4,))):
        with pytest.raises(Err, match="device"):
            f()


def _refused(f, *a, match=None, **kw):
    with pytest.raises((Err, TypeError), match=match):
        f(*a, **kw)


def test_layernorm_arguments(host):
    h = torch.float16
    x, st, w = torch.zeros(4, 32, dtype=h), torch.zeros(4, 2), torch.zeros(32, dtype=h)
    r = lambda *a, **kw: _refused(ops.layernorm_train, *a, **kw)
    r(x.float())
    r(x.t(), match="contiguous")
    r(torch.zeros(2, 4, 64, dtype=h)[..., :32], match="contiguous")
    r(torch.zeros((), dtype=h))
    r(x, w[:31], match="gamma")
    r(x, w, w.double(), match="beta")
    r(x, w, w.float(), match="different types")
    r(x, torch.zeros(64, dtype=h)[::2], match="gamma")
    r(x, w, w, out=x.float(), match="out")
    r(x, w, w, out=x[:3], match="out")
    b = lambda *a, **kw: _refused(ops.layernorm_backward, *a, **kw)
    b(x[:3], x, st, match="dy")
    b(x.bfloat16(), x, st, match="dy")
    b(x, x, st[:3], match="stats")
    b(x, x, st.half(), match="stats")
    b(x, x, torch.zeros(2, 4).t(), match="stats")
    b(x, x, st, w[:5], match="gamma")
    b(x, x, st, w, out=x.float(), match="out")


def test_rope_arguments(host):
    h = torch.float16
    for bad in (((), 16), ((3,), 16), ((0, 4), 16), ((8, 8, 8), 16), ((2,) * 5, 16), ((8,), 17), ((8,), 258)):
        _refused(ops.RopeAxes, *bad, device="cpu")
    _refused(ops.RopeAxes, (8,), 16, theta=0.0, device="cpu")
    axes = ops.RopeAxes((8, 8), 16, device="cpu")
    x, pos = torch.zeros(2, 6, 32, dtype=h), torch.zeros(6, 2, dtype=torch.int32)
    r = lambda *a, **kw: _refused(ops.rope, *a, **kw)
    r(x.float(), axes, pos=pos)
    r(x[0], axes, pos=pos, match="x:")
    r(x[..., :24], axes, pos=pos, match="x:")
    r(x.transpose(1, 2), ops.RopeAxes((2,), 6, device="cpu"), pos=pos, match="x:")
    r(x, axes, match="either")
    r(x, axes, pos=pos, grid=(2, 3), match="either")
    r(x, axes, pos=pos.long(), match="pos")
    r(x, axes, pos=pos[:5], match="pos")
    r(x, axes, pos=torch.zeros(2, 6, dtype=torch.int32).t(), match="pos")
    r(x, axes, pos=pos, origin=(0, 0), match="origin")
    r(x, axes, grid=(2, 4), match="grid")
    r(x, axes, grid=(6,), match="grid")
    r(x, axes, grid=(2, 3), origin=(0,), match="grid")
    r(x, axes, grid=(2, 3), origin=(2 ** 31 - 1, 0), match="32 bits")
    r(x, axes, grid=(2, 3), out=x[:1].expand(2, -1, -1), match="overlap")
    r(x, axes, grid=(2, 3), out=x.bfloat16(), match="out")


def test_window_attention_arguments(host):
    h = torch.float16
    q, k = torch.zeros(2, 5, 64, dtype=h), torch.zeros(2, 7, 32, dtype=h)
    n = torch.zeros(2, dtype=torch.int32)

    def r(*a, match=None, **kw):
        _refused(ops.window_attention, *a, match=match, **dict(dict(kv_heads=2), **kw))
    r(q.float(), k, k, 4)
    r(q, k, k, 0)
    r(q, k, k, 4, kv_heads=3, match="share")
    r(q, k, k, 3, kv_heads=3, match="q:")
    r(q, k, k, 16, kv_heads=2, match="head_dim")
    r(q, k.bfloat16(), k, 4, match="k ")
    r(q, k, k[:, :6], 4, match="v:")
    r(q, k[:1], k, 4, match="k:")
    r(q, k[..., :16], k, 4, match="k:")
    r(q, k, k, 4, q_len=n.long(), match="q_len")
    r(q, k, k, 4, kv_len=n[:1], match="kv_len")
    r(q, k, k, 4, sinks=-1, match="sinks")
    for s in (0.0, -1.0, float("nan"), float("inf")):
        r(q, k, k, 4, scale=s, match="scale")
    r(torch.zeros(2, 5, 68, dtype=h)[..., 1:65], k, k, 4, match="aligned|multiples")
    r(torch.zeros(2, 5, 68, dtype=h)[..., :64], k, k, 4, match="multiples")
    r(q, torch.zeros(2, 32, 7, dtype=h).transpose(1, 2), k, 4, match="contiguous")
    r(q, k, k, 4, out=q[:, :4], match="out")
    r(q, k, k, 4, out=q[:1].expand(2, -1, -1), match="overlap")
    r(q, k, k, 4, out=torch.zeros(1000, dtype=h).as_strided((2, 5, 64), (320, 56, 1)), match="overlap")
    r(q.view(2, 5, 4, 16), k, k, 4, out=torch.zeros(1000, dtype=h).as_strided((2, 5, 4, 16), (320, 64, 8, 1)), match="overlap")
    lse = torch.zeros(2, 4, 5)

    def b(*a, match=None, **kw):
        _refused(ops.window_attention_backward, *a, match=match, **dict(dict(kv_heads=2), **kw))
    b(q[:, :4], q, k, k, q, lse, 4, match="do")
    b(q, q, k, k, q.bfloat16(), lse, 4, match="o is")
    b(q, q, k, k, q, lse[:, :3], 4, match="lse")
    b(q, q, k, k, q, lse.half(), 4, match="lse")
    b(q, q, k, k, q, lse.transpose(1, 2).contiguous().transpose(1, 2), 4, match="lse")
    b(q, q, k, k, q, lse, 4, dk=k[:, :6], match="dk")
    b(q, q, k, k, q, lse, 4, dv=k[:1].expand(2, -1, -1), match="overlap")
    b(q, q, k, k, q, lse, 4, dq=q.float(), match="dq")
