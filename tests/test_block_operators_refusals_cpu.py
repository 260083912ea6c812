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
