"""GPU tests of window_attention / window_attention_backward where 16-bit operands of the second products could lose what the row sums
and the results still hold: probabilities below half of fp16's smallest number.  E = 2^-24, u = eps / 2 of the storage type, as in test_window_attention_gpu.py."""
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
