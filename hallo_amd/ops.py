"""Thin Python wrappers over the C ABI of libhallo_amd.so.

PyTorch is used only for device memory (tensor allocation / data_ptr) and the current HIP
stream; every computation goes through the hand-written gfx950 kernels.  Activations are
token-major: [frames, H*W, C] with C contiguous.
"""
import ctypes as C
import math
import threading

import numpy as np
import torch

from . import lib as _l

F16, BF16 = _l.F16, _l.BF16
ACT_NONE, ACT_SILU, ACT_RELU = _l.ACT_NONE, _l.ACT_SILU, _l.ACT_RELU
ACT_GELU, ACT_GELU_PRE = _l.ACT_GELU, _l.ACT_GELU_PRE


def dtype_code(dtype):
    if dtype == torch.float16:
        return F16
    if dtype == torch.bfloat16:
        return BF16
    raise TypeError(f"hallo_amd kernels store activations/weights as fp16 or bf16, got {dtype}")


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _chk_dev(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise _l.HalloLibraryError("hallo_amd operators need device (HIP) tensors; there is no CPU path")


_option_epoch = 0


def set_option(name, value):
    """Kernel A/B switch, e.g. set_option('gemm_variant', 0|1|2).  Bumps `option_epoch()` when the value CHANGES: captured
    hipGraphs hold the kernels the options routed to at capture time, so FaceAnimatePipeline keys its graphs on the epoch.
    Returns the previous value (None for write-only options)."""
    global _option_epoch
    lib = _l.load()
    prev = lib.hallo_get_option(name.encode())
    if prev == int(value):
        return prev
    _l.check(lib.hallo_set_option(name.encode(), int(value)), f"hallo_set_option({name})")
    _option_epoch += 1
    return prev if prev >= 0 else None


def option_epoch():
    return _option_epoch


def routing_option_names():
    """Every settable option of the library, from the library itself (hallo_option_names, ABI v8): an option added to a kernel file
    is part of the graph key without anybody remembering a Python tuple ('xattn_cap' was missing from one)."""
    return tuple(n for n in _l.load().hallo_option_names().decode().split(",") if n)


def options_fingerprint():
    """Values of every option that decides which kernel a launch is routed to: what a captured graph is valid for (the epoch
    counts CHANGES, and a routing scope that sets and restores options changes it twice per clip without changing anything)."""
    lib = _l.load()
    return tuple(lib.hallo_get_option(n.encode()) for n in routing_option_names())


# Kernel routing for THROUGHPUT: several independent clips in flight on one GPU (bench.py --inflight).  The
# library's defaults are tuned for one clip at a time, where the lowest-latency kernel wins; with another clip's kernels ready to
# fill every idle CU the winners change -- measured on MI355X, alternating runs on one box (profiles/r4_throughput_options_ab.json):
#   gemm_rs = 0   the row-stationary K = 320 / 640 GEMMs (one 133 KB-LDS workgroup per CU, all CUs in the same phase) -> the tiled
#                 kernels + hallo_row_stats: two to four co-resident workgroups leave room for the other clips        +3.9 %
#   ff_fused = 1  the 320-wide feed-forward as one kernel (a third of the HBM bytes; 13 % slower in isolation)          +1.8 %
#   gn_fused = 0  single-launch GroupNorm of the small maps -> statistics + apply launches                               +3.4 %
#   gemm4 = 0     the exact-fit one-workgroup-per-CU GEMM -> split big tile                                              +2.5 %
# together 17.9 -> 19.3 frames/s at three clips in flight (one clip at a time the same set LOSES 4 %: 15.6 against 16.2).
#   split_k_max = 4  split-K factors capped at 4 (8-16 alone): half the slab traffic, fewer but longer workgroups             +0.6 %
THROUGHPUT_OPTIONS = {"gemm_rs": 0, "ff_fused": 1, "gn_fused": 0, "gemm4": 0, "split_k_max": 4}
LATENCY_OPTIONS = {"gemm_rs": 2, "ff_fused": 0, "gn_fused": 1, "gemm4": 1, "split_k_max": 16}          # the library defaults
# Kernel routing for a BATCH of independent clips through one evaluation (FaceAnimatePipeline.call_batch, bench.py --batch-clips; round
# 6): one in-order stream whose launches carry K x the rows, so the lowest-latency kernels win as they do for one clip (the row-
# stationary K = 320 / 640 GEMMs: +7 % over gemm_rs = 0 at K = 4) -- except that the fused 320-wide feed-forward now has the rows to
# fill the chip several times over and its third of the HBM bytes pays (+0.4 %); alternating runs on one box, profiles/r6_batch_sweep.json.
BATCHED_OPTIONS = dict(LATENCY_OPTIONS, ff_fused=1)
ROUTINGS = {"throughput": THROUGHPUT_OPTIONS, "latency": LATENCY_OPTIONS, "batched": BATCHED_OPTIONS}


class routing:
    """`with ops.routing("throughput" | "latency" | {option: value} | None):` -- kernel routing as a property of the CALLER
    (FaceAnimatePipeline(routing=...)) instead of process-global state: the options are read by the library at ENQUEUE time (and
    baked into a graph at capture time), so a scope around the enqueue calls is all a pipeline needs; the previous values come
    back on exit, and an option that already has the wanted value is not touched (no epoch bump, captured graphs stay valid).
    None = leave everything as it is.  The options live in the library (one set per process), so a scope HOLDS a process-wide
    re-entrant lock from entry to exit -- also a `None` scope, whose launches must not see another thread's routing either: a
    second host thread that enters a scope while the first is enqueueing a clip waits for it (enqueueing a clip is ~150 ms of
    host work; the GPU work it queued runs on regardless).  Nested scopes of one thread are fine."""

    _lock = threading.RLock()

    def __init__(self, options):
        self.options = ROUTINGS[options] if isinstance(options, str) else options
        self._prev = None

    def __enter__(self):
        routing._lock.acquire()
        try:
            if self.options:
                self._prev = {k: set_option(k, v) for k, v in self.options.items()}
        except BaseException:
            routing._lock.release()
            raise
        return self

    def __exit__(self, *exc):
        try:
            if self._prev:
                for k, v in self._prev.items():
                    if v is not None:
                        set_option(k, v)
            self._prev = None
        finally:
            routing._lock.release()
        return False


def set_mode(throughput):
    """Process-wide default routing (kept for tools / old command lines; pipelines carry their own `routing`): several clips in
    flight (True) or one clip at a time (False, the library defaults).  Returns the previous values: `restore_options(prev)`."""
    return {k: set_option(k, v) for k, v in (THROUGHPUT_OPTIONS if throughput else LATENCY_OPTIONS).items()}


def restore_options(prev):
    for k, v in (prev or {}).items():
        if v is not None:
            set_option(k, v)


def get_option(name):
    return _l.load().hallo_get_option(name.encode())


SPLITK_WS_BYTES = 128 << 20
GN_WS_FLOATS = 1 << 20
WS_ZEROED = 1       # hallo_gemm_desc.workspace_zeroed as gemm() passes it: Scratch zeroes the counter tail once (tests set 0 to check the refusal)


class Scratch:
    """The launch scratch of ONE in-order sequence of launches (a pipeline object, a captured graph): the fp32 split-K /
    stream-K slab of hallo_gemm / hallo_conv3x3_nhwc and the partial-statistics buffer of hallo_groupnorm_nhwc.  Both are
    written by one launch and read by the next one on the same stream, so two sequences that may overlap on the GPU must never
    share them.  Fixed addresses (a captured launch stays replayable).  The slab's last 64 KB hold the arrival counters of
    csrc/gemm4.hip's K-split tail: zero before the first launch, restored to zero by every launch."""

    def __init__(self, device):
        self.device = torch.device(device)
        self.splitk = torch.empty(SPLITK_WS_BYTES // 4, device=device, dtype=torch.float32)
        self.splitk[-(65536 // 4):].zero_()
        self.gn = torch.empty(GN_WS_FLOATS, device=device, dtype=torch.float32)

    def gn_ws(self, need):
        if self.gn.numel() < need:
            if torch.cuda.is_current_stream_capturing():
                raise _l.HalloLibraryError(f"GroupNorm scratch of {need} floats needed inside a graph capture, {self.gn.numel()} allocated")
            # a graph captured earlier under this scratch has the OLD address baked in and may still be replayed: the old buffer
            # stays alive (and private to this scratch) for as long as the scratch does
            self._retired = getattr(self, "_retired", []) + [self.gn]
            self.gn = torch.empty(need, device=self.device, dtype=torch.float32)
        return self.gn


class _ScratchTLS(threading.local):
    def __init__(self):
        self.stack = []


_scratch_tls = _ScratchTLS()      # per host thread: two threads driving two pipelines never see each other's scope
_stream_scratch = {}


class scratch_scope:
    """`with ops.scratch_scope(s):` every launch enqueued inside uses the Scratch `s` (FaceAnimatePipeline wraps its clip in one:
    eager step 0 and the captured graph of a pipeline share that pipeline's scratch, other pipelines have their own).  Outside any
    scope the scratch is keyed by (device, current stream) -- NOTE that inside `torch.cuda.graph(...)` the current stream is
    torch's capture stream, one per process unless the caller passes `stream=`: graphs captured without a scope on that default
    stream would all bake in the same buffers and must not be replayed concurrently."""

    def __init__(self, scratch):
        self.scratch = scratch

    def __enter__(self):
        _scratch_tls.stack.append(self.scratch)
        return self.scratch

    def __exit__(self, *exc):
        _scratch_tls.stack.pop()
        return False


def current_scratch(device):
    for s in reversed(_scratch_tls.stack):        # the innermost scope of THIS thread that names a scratch (a None scope changes nothing)
        if s is not None:
            return s
    device = torch.device(device)
    key = (device, torch.cuda.current_stream(device).cuda_stream)
    s = _stream_scratch.get(key)
    if s is None:
        s = _stream_scratch[key] = Scratch(device)
    return s


def _workspace(device):
    return current_scratch(device).splitk


def publish_constant():
    """Call after building a lazily created constant that lives on a shared module (weight images, positional-encoding bias
    rows): other pipelines read it from THEIR streams without any ordering against the stream that built it, so the build is
    made visible with a one-off host wait on the current stream.  Lazy constants are built during a clip's eager step 0; inside a
    graph capture a host wait is impossible and the constant would live in the graph's private pool -- refuse."""
    if torch.cuda.is_current_stream_capturing():
        raise _l.HalloLibraryError("a shared constant was first built inside a graph capture: run one eager evaluation first")
    torch.cuda.current_stream().synchronize()


class RowParts:
    """LayerNorm statistics of a tensor's rows, delivered by the kernel that PRODUCED the tensor (hallo_gemm_desc.row_parts):
    fp32 [rows, parts, 2] = (sum, sum of squares) of the rounded values of each 64-column block.  A LayerNorm-fused consumer
    (gemm(..., ln_stats=RowParts)) reduces them to mean / rstd in its prologue; no pass over the tensor (hallo_row_stats)."""
    __slots__ = ("sums", "parts", "rows", "cols")

    def __init__(self, sums, parts, rows, cols):
        self.sums, self.parts, self.rows, self.cols = sums, parts, rows, cols


def gemm(a, w, bias=None, *, out=None, residual=None, rowscale=None, alpha=1.0, act=ACT_NONE, geglu=False,
         bias2=None, bias2_rows_per_group=0, out_f32=False, bias_per_row=False, lead_cols=0, lead_alpha=1.0,
         ln_colsum=None, ln_eps=1e-5, ln_stats=None, row_parts=False, kv_split=None):
    """out[M,N] = act(alpha * rowscale * (a[M,K] @ w[N,K]^T + bias) + residual).

    kv_split = (col0, L) (only where kv_split_ok() says so): returns (out [M, col0], kv [2, M // L, 8, L, 40]) -- the columns from
    col0 on, K then V of 8 heads x 40, leave the GEMM head-major (hallo_gemm_desc.kv_out), the layout attention(kv1_head_major=True)
    reads.

    a may be a 2-D view with arbitrary row stride (last dim contiguous).  geglu: w is [2N,K].
    row_parts=True: returns (out, RowParts) -- the output rows' LayerNorm partial sums from the epilogue.
    ln_stats: fp32 [M, 2] (mean, rstd) from row_stats / face_xattn, or a RowParts of `a` from its producer."""
    _chk_dev(a, w)
    assert a.dim() == 2 and w.dim() == 2 and a.stride(1) == 1 and w.stride(1) == 1
    M, K = a.shape
    N = w.shape[0] // 2 if geglu else w.shape[0]
    assert w.shape[1] == K, (a.shape, w.shape)
    kv = None
    if kv_split is not None:
        col0, L = kv_split
        assert out is None and not geglu and not out_f32 and N - col0 == 640 and M % L == 0 and lead_cols <= col0
        out = torch.empty((M, max(col0, 8)), device=a.device, dtype=a.dtype)     # (col0 = 0, K | V alone: the library still wants a valid C)
        kv = torch.empty((2, M // L, 8, L, 40), device=a.device, dtype=a.dtype)
    elif out is None:
        out = torch.empty((M, N), device=a.device, dtype=torch.float32 if out_f32 else a.dtype)
    assert out.stride(1) == 1 and out.shape[0] == M and (out.shape[1] == N or kv is not None)
    d = _l.GemmDesc()
    d.A, d.B, d.C = a.data_ptr(), w.data_ptr(), out.data_ptr()
    if kv is not None:
        d.kv_out, d.kv_col0, d.kv_rows_per_image, d.kv_tensor_stride = kv.data_ptr(), col0, L, kv.stride(0)
    d.M, d.N, d.K = M, N, K
    d.lda, d.ldb, d.ldc = a.stride(0), w.stride(0), out.stride(0)
    d.batch = 1
    d.stride_a = d.stride_b = d.stride_c = d.stride_r = 0
    d.bias = bias.data_ptr() if bias is not None else None
    d.bias_per_row = 1 if bias_per_row else 0
    d.bias2 = bias2.data_ptr() if bias2 is not None else None
    d.bias2_rows_per_group = bias2_rows_per_group
    d.bias2_ld = bias2.stride(0) if bias2 is not None else 0
    d.rowscale = rowscale.data_ptr() if rowscale is not None else None
    if rowscale is not None:
        assert rowscale.dtype == torch.float32 and rowscale.numel() == M
    if residual is not None:
        assert residual.stride(1) == 1 and residual.shape == out.shape
        d.residual, d.ldr = residual.data_ptr(), residual.stride(0)
    else:
        d.residual, d.ldr = None, 0
    d.alpha, d.act, d.geglu, d.out_f32 = float(alpha), act, 1 if geglu else 0, 1 if out_f32 else 0
    d.lead_cols, d.lead_alpha = int(lead_cols), float(lead_alpha)
    if ln_colsum is not None:
        # fused LayerNorm: `a` is the un-normalised input, w / bias / ln_colsum come from fold_layernorm()
        assert ln_colsum.dtype == torch.float32 and ln_colsum.is_contiguous() and ln_colsum.numel() == w.shape[0]
        d.ln_colsum, d.ln_eps = ln_colsum.data_ptr(), float(ln_eps)
        d.ln_parts = 0
        if isinstance(ln_stats, RowParts):
            assert ln_stats.rows == M and ln_stats.cols == K, (ln_stats.rows, ln_stats.cols, M, K)
            d.ln_stats, d.ln_parts = ln_stats.sums.data_ptr(), ln_stats.parts
        else:
            if ln_stats is not None:
                assert ln_stats.dtype == torch.float32 and ln_stats.is_contiguous() and ln_stats.numel() == 2 * M
            d.ln_stats = ln_stats.data_ptr() if ln_stats is not None else None
    else:
        d.ln_colsum, d.ln_eps, d.ln_stats, d.ln_parts = None, 0.0, None, 0
    d.dtype = dtype_code(a.dtype)
    parts = None
    if row_parts:
        assert not geglu and not out_f32 and N % 8 == 0
        P = (N + 63) // 64
        parts = RowParts(torch.empty((M, P, 2), device=a.device, dtype=torch.float32), P, M, N)
        d.row_parts = parts.sums.data_ptr()
    else:
        d.row_parts = None
    ws = _workspace(a.device)
    d.workspace, d.workspace_bytes, d.workspace_zeroed = ws.data_ptr(), SPLITK_WS_BYTES, WS_ZEROED
    _l.check(_l.load().hallo_gemm(C.byref(d), _stream()), "hallo_gemm")
    if kv is not None:
        return out[:, :kv_split[0]], kv
    return (out, parts) if row_parts else out


KV_HEAD_MAJOR = True      # False (bench.py --no-kv-head-major, A/B): the spatial self-attentions keep K / V as column views of the fused q|k|v buffer


def kv_split_ok(M, N, K, col0):
    """True when gemm(..., ln_colsum=..., kv_split=(col0, L)) is available for this problem under the current routing options (the
    row-stationary K = 320 kernel takes it: hallo_gemm_kv_split_ok)."""
    return bool(_l.load().hallo_gemm_kv_split_ok(M, N, K, col0))


def gemm_batched(a, w, out, *, out_f32=False, alpha=1.0, bias=None, bias_per_row=False, bias_stride=None, act=ACT_NONE,
                 residual=None):
    """Strided-batched out[b] = act(alpha * (a[b] @ w[b]^T + bias) + residual[b]); a [B,M,K], w [B,N,K], out [B,M,N]
    (3-D views: any batch / row stride, last dim contiguous).  `bias` is shared by the batch entries; `residual` is a
    view shaped like `out`."""
    _chk_dev(a, w, out)
    assert bias_stride is None, "per-batch bias is not part of the C ABI"
    assert a.stride(2) == 1 and w.stride(2) == 1 and out.stride(2) == 1
    Bn, M, K = a.shape
    N = w.shape[1]
    d = _l.GemmDesc()
    d.A, d.B, d.C = a.data_ptr(), w.data_ptr(), out.data_ptr()
    d.M, d.N, d.K = M, N, K
    d.lda, d.ldb, d.ldc = a.stride(1), w.stride(1), out.stride(1)
    d.batch = Bn
    d.stride_a, d.stride_b, d.stride_c, d.stride_r = a.stride(0), w.stride(0), out.stride(0), 0
    d.bias = bias.data_ptr() if bias is not None else None
    d.bias_per_row = 1 if bias_per_row else 0
    d.bias2, d.bias2_rows_per_group, d.bias2_ld, d.rowscale, d.residual, d.ldr = None, 0, 0, None, None, 0
    if residual is not None:
        assert residual.shape == out.shape and residual.stride(2) == 1
        d.residual, d.ldr, d.stride_r = residual.data_ptr(), residual.stride(1), residual.stride(0)
    d.alpha, d.act, d.geglu, d.out_f32 = float(alpha), act, 0, 1 if out_f32 else 0
    d.lead_cols, d.lead_alpha = 0, 1.0
    d.ln_colsum, d.ln_eps, d.ln_stats, d.ln_parts, d.row_parts = None, 0.0, None, 0, None
    d.dtype = dtype_code(a.dtype)
    d.workspace, d.workspace_bytes, d.workspace_zeroed = None, 0, 0
    _l.check(_l.load().hallo_gemm(C.byref(d), _stream()), "hallo_gemm(batched)")
    return out


def conv3x3(x, w, bias, n_img, H, W, *, stride=1, pad_t=1, pad_l=1, out_hw=None, upsample=False, bias2=None,
            bias2_rows_per_group=0, residual=None, alpha=1.0, act=ACT_NONE, out=None):
    """x [n_img, H*W, Cin] -> [n_img, OH*OW, Cout]; w [Cout, 3, 3, Cin] (flattened [Cout, 9*Cin])."""
    _chk_dev(x, w)
    Cin = x.shape[-1]
    Cout = w.shape[0]
    assert x.is_contiguous() and w.is_contiguous() and w.numel() == Cout * 9 * Cin
    VH, VW = (2 * H, 2 * W) if upsample else (H, W)
    if out_hw is None:
        OH = (VH + 2 * pad_t - 3) // stride + 1
        OW = (VW + 2 * pad_l - 3) // stride + 1
    else:
        OH, OW = out_hw
    if out is None:
        out = torch.empty((n_img, OH * OW, Cout), device=x.device, dtype=x.dtype)
    d = _l.ConvDesc()
    d.x, d.w, d.y = x.data_ptr(), w.data_ptr(), out.data_ptr()
    d.n_img, d.H, d.W, d.Cin, d.Cout, d.OH, d.OW = n_img, H, W, Cin, Cout, OH, OW
    d.stride, d.pad_t, d.pad_l, d.upsample = stride, pad_t, pad_l, 1 if upsample else 0
    d.bias = bias.data_ptr() if bias is not None else None
    d.bias2 = bias2.data_ptr() if bias2 is not None else None
    d.bias2_rows_per_group = bias2_rows_per_group
    d.bias2_ld = bias2.stride(0) if bias2 is not None else 0
    if residual is not None:
        assert residual.is_contiguous()
        d.residual, d.ldr = residual.data_ptr(), residual.shape[-1]
    else:
        d.residual, d.ldr = None, 0
    d.ldy = out.stride(-2)
    d.alpha, d.act, d.dtype = float(alpha), act, dtype_code(x.dtype)
    ws = _workspace(x.device)
    d.workspace, d.workspace_bytes = ws.data_ptr(), SPLITK_WS_BYTES
    _l.check(_l.load().hallo_conv3x3_nhwc(C.byref(d), _stream()), "hallo_conv3x3_nhwc")
    return out


def attention(q, k1, v1, heads, *, k2=None, v2=None, kv2_batch_div=1, kv2_batch_mod=0, kv2_first_batch=0, out=None,
              scale=None, rowscale=None, rowscale_head_div=0, q_prescaled=False, kv1_head_major=False, kv2_head_major=False):
    """softmax(q k^T * scale) v over up to two key/value segments.

    q [B, Lq, C], k1/v1 [B, Lkv1, C], k2/v2 [B2, Lkv2, C] are views with contiguous last dim
    (e.g. column slices of a fused projection buffer); C = heads * head_dim.
    kvN_head_major: that segment's K / V are contiguous [B, heads, Lkv, head_dim] tensors (gemm(kv_split=...), head_major())."""
    _chk_dev(q, k1, v1)
    B, Lq, Cq = q.shape
    hd = Cq // heads
    if kv1_head_major or kv2_head_major:
        return _attention_head_major(q, k1, v1, heads, k2, v2, kv2_batch_div, kv2_batch_mod, kv2_first_batch, out, rowscale,
                                     rowscale_head_div, q_prescaled, kv1_head_major, kv2_head_major)
    if out is None:
        out = torch.empty((B, Lq, Cq), device=q.device, dtype=q.dtype)
    d = _l.AttnDesc()
    d.q, d.k1, d.v1, d.o = q.data_ptr(), k1.data_ptr(), v1.data_ptr(), out.data_ptr()
    d.k2 = k2.data_ptr() if k2 is not None else None
    d.v2 = v2.data_ptr() if v2 is not None else None
    d.batch, d.heads, d.head_dim, d.Lq, d.Lkv1 = B, heads, hd, Lq, k1.shape[1]
    d.Lkv2 = k2.shape[1] if k2 is not None else 0
    for t in (q, k1, v1, out):
        assert t.stride(2) == 1
    d.q_bs, d.q_rs = q.stride(0), q.stride(1)
    d.k1_bs, d.k1_rs = (k1.stride(0) if k1.shape[0] > 1 else 0), k1.stride(1)
    d.v1_bs, d.v1_rs = (v1.stride(0) if v1.shape[0] > 1 else 0), v1.stride(1)
    if k2 is not None:
        assert k2.stride(2) == 1 and v2.stride(2) == 1
        d.k2_bs, d.k2_rs = (k2.stride(0) if k2.shape[0] > 1 else 0), k2.stride(1)
        d.v2_bs, d.v2_rs = (v2.stride(0) if v2.shape[0] > 1 else 0), v2.stride(1)
    else:
        d.k2_bs = d.k2_rs = d.v2_bs = d.v2_rs = 0
    d.o_bs, d.o_rs = out.stride(0), out.stride(1)
    d.kv2_batch_div, d.kv2_batch_mod, d.kv2_first_batch = kv2_batch_div, kv2_batch_mod, kv2_first_batch
    d.scale = float(scale if scale is not None else hd ** -0.5)
    d.dtype = dtype_code(q.dtype)
    d.q_prescaled = 1 if q_prescaled else 0
    if rowscale is not None:
        # fp32 [G, B*Lq]: head h is scaled by row h // rowscale_head_div of it (G = heads // rowscale_head_div groups)
        assert rowscale.dtype == torch.float32 and rowscale.is_contiguous()
        groups = heads // rowscale_head_div if rowscale_head_div > 0 else 1
        assert rowscale.numel() == groups * B * Lq, (rowscale.shape, groups, B, Lq)
        d.o_rowscale, d.o_rowscale_head_div, d.o_rowscale_stride = rowscale.data_ptr(), rowscale_head_div, B * Lq
    else:
        d.o_rowscale, d.o_rowscale_head_div, d.o_rowscale_stride = None, 0, 0
    _l.check(_l.load().hallo_attention(C.byref(d), _stream()), "hallo_attention")
    return out


def _attention_head_major(q, k1, v1, heads, k2, v2, kv2_batch_div, kv2_batch_mod, kv2_first_batch, out, rowscale, rowscale_head_div,
                          q_prescaled, hm1, hm2):
    """attention() with head-major K / V in segment 1 and / or 2 (hallo_attn_desc.kv1_hs / kv2_hs: head dim 40, pre-scaled q)."""
    assert q_prescaled and rowscale is None
    B, Lq, Cq = q.shape
    hd = Cq // heads
    if out is None:
        out = torch.empty((B, Lq, Cq), device=q.device, dtype=q.dtype)
    d = _l.AttnDesc()
    d.q, d.k1, d.v1, d.o = q.data_ptr(), k1.data_ptr(), v1.data_ptr(), out.data_ptr()
    d.batch, d.heads, d.head_dim, d.Lq = B, heads, hd, Lq
    assert q.stride(2) == 1 and out.stride(2) == 1
    d.q_bs, d.q_rs, d.o_bs, d.o_rs = q.stride(0), q.stride(1), out.stride(0), out.stride(1)

    def seg(k, v, hm):
        if hm:
            assert k.dim() == 4 and k.shape[1] == heads and k.shape[3] == hd and k.is_contiguous() and v.is_contiguous() and v.shape == k.shape
            L = k.shape[2]
            bs = heads * L * hd if k.shape[0] > 1 else 0
            return L, bs, hd, bs, hd, L * hd
        assert k.stride(2) == 1 and v.stride(2) == 1
        return k.shape[1], (k.stride(0) if k.shape[0] > 1 else 0), k.stride(1), (v.stride(0) if v.shape[0] > 1 else 0), v.stride(1), 0
    d.Lkv1, d.k1_bs, d.k1_rs, d.v1_bs, d.v1_rs, d.kv1_hs = seg(k1, v1, hm1)
    if k2 is not None:
        d.k2, d.v2 = k2.data_ptr(), v2.data_ptr()
        d.Lkv2, d.k2_bs, d.k2_rs, d.v2_bs, d.v2_rs, d.kv2_hs = seg(k2, v2, hm2)
    else:
        d.k2 = d.v2 = None
        d.Lkv2 = 0
    d.kv2_batch_div, d.kv2_batch_mod, d.kv2_first_batch = kv2_batch_div, kv2_batch_mod, kv2_first_batch
    d.scale = float(hd ** -0.5)
    d.dtype = dtype_code(q.dtype)
    d.q_prescaled = 1
    d.o_rowscale, d.o_rowscale_head_div, d.o_rowscale_stride = None, 0, 0
    _l.check(_l.load().hallo_attention(C.byref(d), _stream()), "hallo_attention(head-major)")
    return out


def head_major(k, v, heads):
    """[B, L, C] K / V views -> contiguous [B, heads, L, C // heads] copies (per-clip constants: the reference bank's K / V)."""
    B, L, Cd = k.shape
    f = lambda t: t.reshape(B, L, heads, Cd // heads).permute(0, 2, 1, 3).contiguous()
    return f(k), f(v)


LOG2E = 1.4426950408889634


def q_scale(head_dim):
    """The factor a q projection must carry for hallo_attention(q_prescaled=True): head_dim^-0.5 * log2(e)."""
    return head_dim ** -0.5 * LOG2E


def temporal_attention(qkv, B, F, HW, Cdim, heads, *, out=None, scale=None, lead=0):
    """qkv [B*F, HW, 3C] -> out [B*F, HW, C]: per-pixel attention over the F axis.  lead > 0: the first `lead` temporal
    positions of all B entries are stored at the front ([B*lead] frame rows), each entry's other F - lead positions behind them
    (hallo_temporal_attention_lead)."""
    _chk_dev(qkv)
    assert qkv.is_contiguous() and qkv.shape[-1] == 3 * Cdim and 0 <= lead < F
    if out is None:
        out = torch.empty((B * F, HW, Cdim), device=qkv.device, dtype=qkv.dtype)
    hd = Cdim // heads
    sc = float(scale if scale is not None else hd ** -0.5)
    _l.check(_l.load().hallo_temporal_attention_lead(_p(qkv), _p(out), B, F, int(lead), HW, Cdim, heads, sc, dtype_code(qkv.dtype),
                                                     _stream()), "hallo_temporal_attention_lead")
    return out


def groupnorm(x, gamma, beta, n_img, HW, groups, eps, *, silu=False, out=None, x2=None):
    """Per-frame GroupNorm (+SiLU) on x [n_img, HW, C].  x2 [n_img, HW, C2]: the norm runs over the channel concatenation
    [x | x2] read in place (hallo_groupnorm_nhwc2: the skip concatenation of the up blocks is never materialised); out is
    [n_img, HW, C + C2]."""
    _chk_dev(x)
    C1 = x.shape[-1]
    Cdim = C1 + (x2.shape[-1] if x2 is not None else 0)
    assert x.is_contiguous() and (x2 is None or (x2.is_contiguous() and x2.shape[:-1] == x.shape[:-1] and x2.dtype == x.dtype and C1 % 8 == 0))
    if out is None:
        out = torch.empty(x.shape[:-1] + (Cdim,), device=x.device, dtype=x.dtype)
    lib = _l.load()
    ws = current_scratch(x.device).gn_ws(n_img * lib.hallo_groupnorm_chunks(HW) * groups * 2)
    _l.check(lib.hallo_groupnorm_nhwc2(_p(x), C1, _p(x2), _p(out), _p(gamma), _p(beta), _p(ws), n_img, HW, Cdim, groups, float(eps),
                                       1 if silu else 0, dtype_code(x.dtype), _stream()), "hallo_groupnorm_nhwc2")
    return out


def layernorm(x, gamma, beta, eps=1e-5, *, pe=None, pe_rows_per_pos=1, pe_len=1, out=None):
    """Row LayerNorm on x [..., C] (+ fp32 positional-encoding table pe [pe_len, C])."""
    _chk_dev(x)
    Cdim = x.shape[-1]
    assert x.is_contiguous()
    rows = x.numel() // Cdim
    if out is None:
        out = torch.empty_like(x)
    _l.check(_l.load().hallo_layernorm(_p(x), _p(out), _p(gamma), _p(beta), _p(pe), rows, Cdim, float(eps),
                                       pe_rows_per_pos, pe_len, dtype_code(x.dtype), _stream()), "hallo_layernorm")
    return out


def softmax_rows(x, out, scale):
    _chk_dev(x, out)
    rows, cols = x.shape[-2] * (x.numel() // (x.shape[-1] * x.shape[-2])), x.shape[-1]
    assert x.dtype == torch.float32 and x.is_contiguous() and out.is_contiguous()
    _l.check(_l.load().hallo_softmax_rows(_p(x), _p(out), rows, cols, float(scale), dtype_code(out.dtype), _stream()),
             "hallo_softmax_rows")
    return out


def copy2d(src, dst, rows, width):
    """dst[r, :width] = src[r, :width]; src/dst are 2-D views (row pitch = stride(0))."""
    _chk_dev(src, dst)
    _l.check(_l.load().hallo_copy2d(_p(src), src.stride(0), _p(dst), dst.stride(0), rows, width, dtype_code(dst.dtype),
                                    _stream()), "hallo_copy2d")
    return dst


def nchw_to_nhwc(x, n, Cdim, HW, Cpad, dtype):
    """x [n, C, HW] (fp32 or `dtype`) -> [n, HW, Cpad] in `dtype`, padded channels zero."""
    _chk_dev(x)
    assert x.is_contiguous()
    out = torch.empty((n, HW, Cpad), device=x.device, dtype=dtype)
    src_f32 = 1 if x.dtype == torch.float32 else 0
    if not src_f32:
        assert x.dtype == dtype
    _l.check(_l.load().hallo_nchw_to_nhwc(_p(x), _p(out), n, Cdim, HW, Cpad, src_f32, dtype_code(dtype), _stream()),
             "hallo_nchw_to_nhwc")
    return out


def nhwc_to_nchw_f32(x, n, Cdim, HW, *, mul=1.0, add=0.0, lo=-3.0e38, hi=3.0e38):
    _chk_dev(x)
    out = torch.empty((n, Cdim, HW), device=x.device, dtype=torch.float32)
    _l.check(_l.load().hallo_nhwc_to_nchw_f32(_p(x), _p(out), n, Cdim, HW, x.stride(-2), float(mul), float(add), float(lo),
                                              float(hi), dtype_code(x.dtype), _stream()), "hallo_nhwc_to_nchw_f32")
    return out


def timestep_embedding(t, dim, dtype):
    """t fp32 [B] -> [B, dim] = [cos | sin] (diffusers Timesteps with flip_sin_to_cos)."""
    _chk_dev(t)
    assert t.dtype == torch.float32
    out = torch.empty((t.numel(), dim), device=t.device, dtype=dtype)
    _l.check(_l.load().hallo_timestep_embedding(_p(t), _p(out), t.numel(), dim, dtype_code(dtype), _stream()),
             "hallo_timestep_embedding")
    return out


DDIM_PRED = {"v_prediction": 0, "epsilon": 2, "sample": 4}       # HALLO_DDIM_PRED_* of include/hallo_amd.h
DDIM_CLIP_SAMPLE = 8


def cfg_ddim_step(model_out, latents, next_in, rows, Cdim, cfg, guidance_scale, alpha_t, alpha_prev, mode=0):
    """In-place DDIM (eta=0) update of fp32 latents [rows, C] from model_out [(2)rows, ldm]; `mode` = DDIM_PRED[type]
    (| DDIM_CLIP_SAMPLE), default v-prediction without clipping."""
    _chk_dev(model_out, latents)
    assert latents.dtype == torch.float32 and latents.is_contiguous()
    _l.check(_l.load().hallo_cfg_ddim_step(_p(model_out), model_out.stride(-2), _p(latents), _p(next_in),
                                           next_in.stride(-2) if next_in is not None else 0, rows, Cdim,
                                           (1 if cfg else 0) | int(mode), float(guidance_scale), float(alpha_t), float(alpha_prev),
                                           dtype_code(model_out.dtype), _stream()), "hallo_cfg_ddim_step")
    return latents


def frames_to_uint8(x, out=None):
    """x fp32 [F, C, HW] (planar, values in [0, 1]) -> uint8 [F, HW, C] = np.clip(x * 255, 0, 255).astype(np.uint8)
    (hallo/utils/util.py:308-312), byte-exact."""
    _chk_dev(x)
    assert x.dtype == torch.float32 and x.is_contiguous() and x.dim() == 3
    Fr, Cc, HW = x.shape
    if out is None:
        out = torch.empty((Fr, HW, Cc), device=x.device, dtype=torch.uint8)
    _l.check(_l.load().hallo_frames_to_uint8(_p(x), _p(out), Fr, Cc, HW, _stream()), "hallo_frames_to_uint8")
    return out


def face_xattn(x, sg, g, b, owp, bo, rows_per_batch, eps, out=None, stats_eps=None):
    """y = x + to_out(SDPA(to_q(LN(x)), K, V)) over 32 (head, token) pairs with the projections / LayerNorm affine folded
    into per-clip constants (see include/hallo_amd.h: hallo_face_xattn).  x [rows, C]; out may be x.
    stats_eps: returns (y, stats) with stats fp32 [rows, 2] = (mean, rstd) of y's rows for a LayerNorm with that eps, from the
    kernel's own epilogue (hallo_face_xattn_stats)."""
    _chk_dev(x, sg, owp)
    rows, Cd = x.shape
    assert x.is_contiguous() and sg.shape[-2:] == (32, Cd) and owp.shape[-2:] == (Cd, 32)
    assert g.dtype == torch.float32 and b.dtype == torch.float32 and g.is_contiguous() and b.is_contiguous()
    assert sg.is_contiguous() and owp.is_contiguous() and sg.dtype == x.dtype and owp.dtype == x.dtype
    if out is None:
        out = torch.empty_like(x)
    if stats_eps is not None:
        st = torch.empty((rows, 2), device=x.device, dtype=torch.float32)
        _l.check(_l.load().hallo_face_xattn_stats(_p(x), _p(out), _p(sg), _p(g), _p(b), _p(owp), _p(bo), rows, Cd,
                                                   int(rows_per_batch), float(eps), _p(st), float(stats_eps), dtype_code(x.dtype),
                                                   _stream()), "hallo_face_xattn_stats")
        return out, st
    _l.check(_l.load().hallo_face_xattn(_p(x), _p(out), _p(sg), _p(g), _p(b), _p(owp), _p(bo), rows, Cd,
                                         int(rows_per_batch), float(eps), dtype_code(x.dtype), _stream()),
             "hallo_face_xattn")
    return out


def face_xattn_constants(wq, kf, vf, wo, gamma, beta, heads, dtype):
    """Per-clip constant folding for face_xattn (once per clip and block).  wq [C, C] (to_q.weight), wo [C, C]
    (to_out[0].weight), kf / vf [nb, T, C] projected face tokens (heads * T must be 32), gamma / beta [C] of norm2.
    The two contractions over the head dimension run on hallo_gemm (strided-batched over the heads, fp32 output: round 4 -- they
    were torch.einsum calls, i.e. rocBLAS / Tensile kernels on the timed path); what is left to torch is elementwise work on
    [nb, 32, C] fp32 matrices."""
    nb, T, Cd = kf.shape
    hd = Cd // heads
    assert T == 4 and heads <= 8, "the fused kernel covers 8 heads x 4 tokens (fewer heads are zero-padded)"
    f = lambda t: t.float()
    HT = heads * T

    def per_head(tok, w_rows):
        """out[b, h*T + t, c] = sum_d tok[b, t, h*hd + d] * w_rows[c, h*hd + d]: batch = heads, A [nb*T, hd] (row pitch C), W [C, hd]"""
        a = tok.reshape(nb * T, Cd).view(nb * T, heads, hd).permute(1, 0, 2)
        w = w_rows.view(Cd, heads, hd).permute(1, 0, 2)
        out = torch.empty((heads, nb * T, Cd), device=tok.device, dtype=torch.float32)
        gemm_batched(a, w, out, out_f32=True)
        return out.view(heads, nb, T, Cd).permute(1, 0, 2, 3).reshape(nb, HT, Cd)

    sw = torch.zeros((nb, 32, Cd), device=kf.device, dtype=torch.float32)
    sw[:, :HT] = per_head(kf.contiguous(), wq.t().contiguous())           # sum_d K[b,t,h,d] * Wq[(h d), c]
    sw = sw * q_scale(hd)
    sg = (sw * f(gamma)).to(dtype).contiguous()
    g = sg.float().sum(-1).contiguous()                                   # from the ROUNDED sg: the kernel multiplies x by it
    b = (sw * f(beta)).sum(-1).contiguous()
    ow = torch.zeros((nb, 32, Cd), device=kf.device, dtype=torch.float32)  # padded heads: uniform p times zero rows
    ow[:, :HT] = per_head(vf.contiguous(), wo.contiguous())               # sum_d V[b,t,h,d] * Wo[c, (h d)]
    # k-slot order of the second MFMA: slot (ks2, hi, e) <-> (h,t) = 8*(2*ks2 + (e >> 2)) + 4*hi + (e & 3)
    ks2, hi, e = torch.meshgrid(torch.arange(2), torch.arange(2), torch.arange(8), indexing="ij")
    j = (8 * (2 * ks2 + (e >> 2)) + 4 * hi + (e & 3)).reshape(-1).to(ow.device)
    owp = ow[:, j, :].permute(0, 2, 1).to(dtype).contiguous()            # [nb, C, 32]
    return sg, g, b, owp


def fold_layernorm(gamma, beta, w, bias=None):
    """Constants of the fused LayerNorm GEMM (hallo_gemm ln_colsum): LN(x) @ w^T + bias with LN's affine folded in.
    Returns (w_f [N, K] in w.dtype = w * gamma, colsum fp32 [N] of the ROUNDED w_f, bias_f [N] = bias + w @ beta)."""
    wf = (w.float() * gamma.float()[None, :]).to(w.dtype).contiguous()
    colsum = wf.float().sum(dim=1).contiguous()
    bf = w.float() @ beta.float()
    if bias is not None:
        bf = bf + bias.float()
    return wf, colsum, bf.to(w.dtype).contiguous()


GELU_U_SCALE = 0.84932180028801904272        # csrc/common.h
GELU_U_INV = 1.17741002251547469101
FF320_C, FF320_INNER, FF320_STEP, FF320_IMAGE = 320, 1280, 16, 32768


def ff320_pack(w1, b1, w2):
    """Weight image of hallo_ff320 (layout: include/hallo_amd.h) from w1 [2560, 320] / b1 [2560] (GEGLU projection, LayerNorm
    already folded in: fold_layernorm) and w2 [320, 1280] (net[2].weight).  Pure gathers on the device, once per module."""
    Cd, I, CH = FF320_C, FF320_INNER, FF320_STEP
    assert tuple(w1.shape) == (2 * I, Cd) and tuple(w2.shape) == (Cd, I) and b1.numel() == 2 * I and w1.dtype == w2.dtype
    dev, ns = w1.device, I // CH
    ar = lambda n: torch.arange(n, device=dev)
    img = torch.zeros((ns, FF320_IMAGE), device=dev, dtype=torch.uint8)
    # W1: [step][sub-tile t][row r][stored piece q][8]  <-  row src(step, r), k = 64 t + 8 (q ^ ((r >> 1) & 7)) + e
    s_, t_, r_, q_, e_ = torch.meshgrid(ar(ns), ar(5), ar(32), ar(8), ar(8), indexing="ij")
    src_row = torch.where(r_ < 16, CH * s_ + r_, I + CH * s_ + r_ - 16)
    k = 64 * t_ + 8 * (q_ ^ ((r_ >> 1) & 7)) + e_
    w1i = w1.contiguous()[src_row, k]                                            # [ns, 5, 32, 8, 8]
    img[:, :20480] = w1i.reshape(ns, -1).view(torch.uint8)
    # W2: [step][n][stored half p][e]  <-  column 16 s + (e & 3) + 8 (e >> 2) + 4 h, h = p ^ ((n >> 3) & 1)
    s_, n_, p_, e_ = torch.meshgrid(ar(ns), ar(Cd), ar(2), ar(8), indexing="ij")
    h_ = p_ ^ ((n_ >> 3) & 1)
    col = CH * s_ + (e_ & 3) + 8 * (e_ >> 2) + 4 * h_
    w2i = w2.contiguous()[n_, col]                                               # [ns, 320, 2, 8]
    img[:, 20480:30720] = w2i.reshape(ns, -1).view(torch.uint8)
    # b1: fp32 [step][h][value 8 | gate 8], gelu_u scales folded in
    s_, h_, e_ = torch.meshgrid(ar(ns), ar(2), ar(8), indexing="ij")
    col = CH * s_ + (e_ & 3) + 8 * (e_ >> 2) + 4 * h_
    bf = b1.float()
    bb = torch.cat([bf[col] * GELU_U_INV, bf[I + col] * GELU_U_SCALE], dim=2).contiguous()      # [ns, 2, 16]
    img[:, 30720:30720 + 128] = bb.reshape(ns, -1).view(torch.uint8)
    assert img.numel() == _l.load().hallo_ff320_pack_bytes()
    return img


FF320_MIN_ROWS = 24576      # 128 rows per workgroup, every workgroup streams all 2.6 MB of weights: below ~192 workgroups the two-GEMM path wins


def ff320_enabled(rows):
    """Routing rule of FeedForward.run_ln for 320-wide blocks: the fused kernel when enough rows fill the chip and
    hallo_set_option("ff_fused", 0) has not switched it off."""
    return rows >= FF320_MIN_ROWS and get_option("ff_fused") > 0


def ff320(x2d, wpack, b2, *, residual=None, layernorm=True, eps=1e-5, out=None):
    """out = residual + net2(GEGLU(net0(LayerNorm(x2d)))) for 320-wide rows in one kernel (hallo_ff320); residual defaults
    to x2d, out may be x2d."""
    _chk_dev(x2d, wpack, b2)
    M, Cd = x2d.shape
    assert Cd == FF320_C and x2d.stride(1) == 1 and wpack.dtype == torch.uint8 and wpack.is_contiguous() and b2.dtype == x2d.dtype
    res = x2d if residual is None else residual
    assert res.shape == x2d.shape and res.stride(1) == 1 and res.dtype == x2d.dtype
    if out is None:
        out = torch.empty((M, Cd), device=x2d.device, dtype=x2d.dtype)
    assert out.shape == x2d.shape and out.stride(1) == 1 and out.dtype == x2d.dtype
    _l.check(_l.load().hallo_ff320(_p(x2d), x2d.stride(0), _p(res), res.stride(0), _p(out), out.stride(0), _p(wpack), _p(b2), M,
                                   1 if layernorm else 0, float(eps), dtype_code(x2d.dtype), _stream()), "hallo_ff320")
    return out


def row_stats(x2d, eps=1e-5):
    """(mean, rstd) per row of x2d [rows, C] as fp32 [rows, 2]: LayerNorm's statistics for hallo_gemm(ln_stats=...)."""
    _chk_dev(x2d)
    assert x2d.dim() == 2 and x2d.is_contiguous()
    rows, Cd = x2d.shape
    st = torch.empty((rows, 2), device=x2d.device, dtype=torch.float32)
    _l.check(_l.load().hallo_row_stats(_p(x2d), _p(st), rows, Cd, float(eps), dtype_code(x2d.dtype), _stream()), "hallo_row_stats")
    return st


def quant_rows_fp8(x2d, gamma=None, beta=None, eps=1e-5):
    """x2d [rows, C] (fp16 / bf16, any row stride) -> (q uint8 [rows, C] of e4m3 bytes, scale fp32 [rows]); with gamma / beta
    the rows go through LayerNorm first (hallo_quant_rows_fp8)."""
    _chk_dev(x2d)
    assert x2d.dim() == 2 and x2d.stride(1) == 1
    rows, Cd = x2d.shape
    q = torch.empty((rows, Cd), device=x2d.device, dtype=torch.uint8)
    sc = torch.empty((rows,), device=x2d.device, dtype=torch.float32)
    _l.check(_l.load().hallo_quant_rows_fp8(_p(x2d), x2d.stride(0), _p(q), _p(sc), rows, Cd, _p(gamma), _p(beta), float(eps),
                                            dtype_code(x2d.dtype), _stream()), "hallo_quant_rows_fp8")
    return q, sc


def gemm_fp8(aq, a_scale, wq, w_scale, out_dtype, bias=None, *, residual=None, alpha=1.0, lead_cols=0, lead_alpha=1.0, out=None):
    """out[M, N] = alpha * lead * (a_scale[m] w_scale[n] (aq . wq^T) + bias) + residual on the fp8 MFMA (hallo_gemm_fp8)."""
    _chk_dev(aq, wq)
    M, K = aq.shape
    N = wq.shape[0]
    assert aq.dtype == torch.uint8 and wq.dtype == torch.uint8 and wq.shape[1] == K and aq.stride(1) == 1 and wq.stride(1) == 1
    if out is None:
        out = torch.empty((M, N), device=aq.device, dtype=out_dtype)
    d = _l.GemmFp8Desc()
    d.A, d.B, d.C = aq.data_ptr(), wq.data_ptr(), out.data_ptr()
    d.M, d.N, d.K = M, N, K
    d.lda, d.ldb, d.ldc = aq.stride(0), wq.stride(0), out.stride(0)
    d.a_scale, d.w_scale = a_scale.data_ptr(), w_scale.data_ptr()
    d.bias = bias.data_ptr() if bias is not None else None
    d.residual, d.ldr = (residual.data_ptr(), residual.stride(0)) if residual is not None else (None, 0)
    d.alpha, d.lead_cols, d.lead_alpha, d.dtype = float(alpha), int(lead_cols), float(lead_alpha), dtype_code(out.dtype)
    _l.check(_l.load().hallo_gemm_fp8(C.byref(d), _stream()), "hallo_gemm_fp8")
    return out


def ln_stats(x2d, n_out, eps=1e-5, *, geglu=False, bias2_rows_per_group=0, lead_cols=0, given=None):
    """`ln_stats` argument for a LayerNorm-fused gemm(x2d, w[n_out(, x2), K], ...): None when the library's row-stationary
    kernel will take the problem and derive mean / rstd from the A rows it keeps in registers (hallo_gemm_fuses_row_stats),
    else `given` -- what the producer of x2d delivered (a RowParts from gemm(row_parts=True), or [M, 2] from face_xattn) --
    else the statistics from hallo_row_stats (one pass over x2d)."""
    M, K = x2d.shape
    if x2d.is_contiguous() and _l.load().hallo_gemm_fuses_row_stats(M, n_out, K, 1 if geglu else 0, bias2_rows_per_group, lead_cols):
        return None
    if given is not None:
        return given
    return row_stats(x2d, eps)


def producer_stats():
    """hallo_set_option("producer_stats", 0) (A/B) turns the producer-side LayerNorm statistics off altogether."""
    return get_option("producer_stats") > 0


def wants_stats(M, n_out, K, *, geglu=False, bias2_rows_per_group=0, lead_cols=0):
    """Should the producer of an [M, K] tensor emit LayerNorm statistics for the LayerNorm-fused gemm(x, w[n_out(, x2), K]) that
    consumes it?  No when the mechanism is off, or when that consumer runs on the row-stationary kernel (it takes the
    statistics from the A rows it keeps in registers: hallo_gemm_fuses_row_stats)."""
    return producer_stats() and not _l.load().hallo_gemm_fuses_row_stats(M, n_out, K, 1 if geglu else 0, bias2_rows_per_group, lead_cols)


_w2v_ws = {}


def w2v_conv0_gn_gelu(wave, w, gamma, beta, k, stride, eps, dtype):
    """First wav2vec2 feature-encoder layer: fp32 waveform [S] -> [L0, C] = GELU(GroupNorm_C(Conv1d(1 -> C, k, stride)))
    in `dtype` (transformers Wav2Vec2GroupNormConvLayer; see include/hallo_amd.h: hallo_w2v_conv0_gn_gelu)."""
    _chk_dev(wave, w)
    assert wave.dtype == torch.float32 and wave.dim() == 1 and wave.is_contiguous()
    assert w.dtype == torch.float32 and w.is_contiguous() and w.shape[1] == k
    assert gamma.dtype == torch.float32 and beta.dtype == torch.float32
    Cd, S = w.shape[0], wave.numel()
    lib = _l.load()
    need = lib.hallo_w2v_conv0_workspace(S, Cd, k, stride)
    if need < 0:
        raise _l.HalloLibraryError(f"hallo_w2v_conv0_workspace({S}, {Cd}, {k}, {stride}) failed with status {need}")
    key = (wave.device, torch.cuda.current_stream().cuda_stream)
    ws = _w2v_ws.get(key)
    if ws is None or ws.numel() * 4 < need:
        ws = torch.empty(max(need // 4, 1 << 16), device=wave.device, dtype=torch.float32)
        _w2v_ws[key] = ws
    L0 = (S - k) // stride + 1
    out = torch.empty((L0, Cd), device=wave.device, dtype=dtype)
    _l.check(lib.hallo_w2v_conv0_gn_gelu(_p(wave), S, _p(w), _p(gamma), _p(beta), _p(out), _p(ws), Cd, k, stride, float(eps),
                                         dtype_code(dtype), _stream()), "hallo_w2v_conv0_gn_gelu")
    return out


def lerp_rows(x, out_rows):
    """x [L, C] -> [out_rows, C]: F.interpolate(mode="linear", align_corners=True) along the row (time) axis."""
    _chk_dev(x)
    assert x.dim() == 2 and x.is_contiguous()
    out = torch.empty((out_rows, x.shape[1]), device=x.device, dtype=x.dtype)
    _l.check(_l.load().hallo_lerp_rows(_p(x), _p(out), x.shape[0], out_rows, x.shape[1], dtype_code(x.dtype), _stream()),
             "hallo_lerp_rows")
    return out


# ---- transformer-block operators with gradients: LayerNorm, rotary positions, window attention -------------------------------------
# Their workspaces are allocated per call: a captured graph gets them from its own pool, so two graphs never share one, and the
# allocator orders the reuse of a freed one on its stream.  They are not torch functions with a gradient: forward and backward are calls
# of their own, and a forward call refuses tensors that wait for a gradient (where torch records).  Single tokens and short rows are
# host-bound, so messages are only put together where a call is refused.

def _bad(what):
    raise _l.HalloLibraryError(what)


def _call(name, device, *args):
    """One library call on `device`'s current stream, with the device made current for the launch when another one is (a stream only
    takes launches from its own device)."""
    fn = getattr(_l.load(), name)
    i = device.index
    if i == torch.cuda.current_device():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(i):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if status:
        _l.check(status, name)


def _no_graph(*tensors):
    """The forward calls record nothing for torch's differentiation: refused where torch records and one of `tensors` takes part in it."""
    if torch.is_grad_enabled():
        _bad(f"a tensor of shape {next(tuple(t.shape) for t in tensors if t is not None and t.requires_grad)} needs a gradient, which this "
             "call does not record: call it under torch.no_grad() or in an autograd.Function, and its backward operator for the gradients")


def _written(*tensors):
    """Outputs that the caller gave: torch counts the call as a change of them (what it keeps for a gradient is then known to be stale)."""
    for t in tensors:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _like(name, t, like, dtype=None, shape=True):
    """`t` is on `like`'s device, of its type (or `dtype`) and, with `shape`, of its shape."""
    if t.device != like.device:
        _bad(f"{name} is on {t.device}, expected {like.device}")
    if t.dtype != (dtype or like.dtype):
        _bad(f"{name} is {t.dtype}, expected {dtype or like.dtype}")
    if shape and t.shape != like.shape:
        _bad(f"{name}: expected {tuple(like.shape)}, got {tuple(t.shape)}")


class _Places:
    """The memory of a strided tensor, for numpy's overlap test (nothing is read)."""

    def __init__(self, t):
        n = t.element_size()
        self.__array_interface__ = {"data": (t.data_ptr(), False), "shape": tuple(t.shape), "strides": tuple(s * n for s in t.stride()),
                                    "typestr": f"|V{n}", "version": 3}


def _apart(name, out, others, same=()):
    """`out` (given by the caller) shares no memory with `others`, nor with `same` unless it is the same view: rows are written while
    other workgroups still read.  Column slices of one buffer are apart."""
    if not out.numel():
        return
    dims = [(n, s) for n, s in zip(out.shape, out.stride()) if n > 1]
    lo, hi = out.data_ptr(), out.data_ptr() + (1 + sum((n - 1) * s for n, s in dims)) * out.element_size()
    for i, (other, t) in enumerate((*same, *others)):
        if t is None or not t.numel():
            continue
        at = t.data_ptr()
        if at >= hi or at + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size() <= lo:
            continue
        if i < len(same) and at == lo and t.shape == out.shape and [(n, s) for n, s in zip(t.shape, t.stride()) if n > 1] == dims:
            continue
        try:
            met = np.shares_memory(np.asarray(_Places(out)), np.asarray(_Places(t)), max_work=1 << 20)
        except RuntimeError:                     # strides too odd to tell within that work
            met = True
        if met:
            _bad(f"{name}: overlaps {other}")


def _rows2d(name, x):
    """x [..., C] as (rows, C, row pitch): contiguous, or a 2-D view with contiguous rows."""
    sh = x.shape
    if not sh or sh[-1] < 1:
        _bad(f"{name}: expected [..., C] with C >= 1, got {tuple(sh)}")
    Cd, n = sh[-1], x.numel()
    if n == 0 or x.is_contiguous():
        return n // Cd, Cd, Cd
    st = x.stride()
    if len(sh) != 2 or (st[1] != 1 and Cd > 1) or (st[0] < Cd and sh[0] > 1):
        _bad(f"{name}: expected a contiguous tensor or a 2-D view with contiguous rows, got shape {tuple(sh)} strides {st}")
    return sh[0], Cd, max(st[0], Cd)


def _affine(x, gamma, beta):
    """Checks gamma / beta [C] (x's type or fp32, the same for both); returns the library's affine_f32 flag."""
    for name, w in (("gamma", gamma), ("beta", beta)):
        if w is not None and (w.device != x.device or w.dtype not in (x.dtype, torch.float32) or w.shape != x.shape[-1:] or not w.is_contiguous()):
            _bad(f"{name}: expected contiguous [{x.shape[-1]}] of {x.dtype} or float32 on {x.device}, got {tuple(w.shape)} {w.dtype} on {w.device}")
    if gamma is not None and beta is not None and gamma.dtype != beta.dtype:
        _bad("gamma and beta have different types")
    w = beta if gamma is None else gamma
    return 1 if w is not None and w.dtype == torch.float32 else 0


def layernorm_train(x, gamma=None, beta=None, eps=1e-5, *, out=None):
    """(y, stats): y = LayerNorm(x [..., C]) * gamma + beta and the row statistics fp32 [rows, 2] = (mean, rstd) that
    layernorm_backward() takes.  Any C up to 16384.  gamma / beta: [C] of x's type or fp32 (master weights), or None.  out may be x, but not lie
    on part of it."""
    _chk_dev(x, gamma, beta, out)
    if x.requires_grad or gamma is not None and gamma.requires_grad or beta is not None and beta.requires_grad or out is not None and out.requires_grad:
        _no_graph(x, gamma, beta, out)
    code = dtype_code(x.dtype)
    rows, Cd, ldx = _rows2d("x", x)
    f32 = _affine(x, gamma, beta)
    given = out is not None
    if not given:
        out = torch.empty_like(x)
    else:
        _like("out", out, x)
        _apart("out", out, (("gamma", gamma), ("beta", beta)), (("x", x),))
    ldy = _rows2d("out", out)[2]
    stats = torch.empty((rows, 2), device=x.device, dtype=torch.float32)
    _call("hallo_layernorm_train", x.device, x.data_ptr(), ldx, out.data_ptr(), ldy, gamma.data_ptr() if gamma is not None else None,
          beta.data_ptr() if beta is not None else None, f32, stats.data_ptr(), rows, Cd, float(eps), code)
    if given:
        _written(out)
    return out, stats


def layernorm_backward(dy, x, stats, gamma=None, *, weight_grads=True, out=None):
    """(dx, dgamma, dbeta) of layernorm_train(x, gamma, ...) for dy; stats as it returned them.  dgamma / dbeta are fp32 [C] (None with
    weight_grads=False: frozen weights).  out (for dx) may be dy.  Results repeat bit for bit."""
    _chk_dev(dy, x, stats, gamma, out)
    code = dtype_code(x.dtype)
    rows, Cd, ldx = _rows2d("x", x)
    _like("dy", dy, x)
    ldd = _rows2d("dy", dy)[2]
    _like("stats", stats, x, torch.float32, False)
    if stats.shape != (rows, 2) or not stats.is_contiguous():
        _bad(f"stats: expected contiguous ({rows}, 2), got {tuple(stats.shape)}")
    f32 = _affine(x, gamma, None)
    given = out is not None
    if not given:
        out = torch.empty_like(x)
    else:
        _like("out", out, x)
        _apart("out", out, (("stats", stats), ("gamma", gamma)), (("dy", dy), ("x", x)))
    ldo = _rows2d("out", out)[2]
    dg = db = pg = pb = pw = None
    need = 0
    if weight_grads:
        need = _l.load().hallo_layernorm_backward_workspace(rows, Cd)
        if need < 0:
            _l.check(need, "hallo_layernorm_backward_workspace")
        wg = torch.empty((2, Cd), device=x.device, dtype=torch.float32)
        ws = torch.empty(need // 4, device=x.device, dtype=torch.float32)
        dg, db = wg.unbind(0)
        pg = wg.data_ptr()
        pb, pw = pg + 4 * Cd, ws.data_ptr()
    _call("hallo_layernorm_backward", x.device, dy.data_ptr(), ldd, x.data_ptr(), ldx, stats.data_ptr(),
          gamma.data_ptr() if gamma is not None else None, f32, out.data_ptr(), ldo, pg, pb, pw, need, rows, Cd, code)
    if given:
        _written(out)
    return out, dg, db


class RopeAxes:
    """Rotary frequencies of up to four position axes: dims[a] (even) columns of every head for axis a, pair i of them turning by
    position * theta^(-2i / dims[a]).  Built once, on the host, and usable from any stream (not inside a graph capture)."""
    __slots__ = ("dims", "head_dim", "theta", "interleaved", "freq")

    def __init__(self, dims, head_dim, theta=10000.0, interleaved=False, device="cuda"):
        dims = tuple(int(d) for d in dims)
        if not 1 <= len(dims) <= 4 or any(d < 2 or d % 2 for d in dims):
            _bad(f"dims: expected 1 to 4 even widths, got {dims}")
        if head_dim % 2 or not 2 <= head_dim <= 256 or sum(dims) > head_dim:
            _bad(f"dims {dims} do not fit head_dim {head_dim} (even, at most 256)")
        if not theta > 0 or not math.isfinite(theta):
            _bad(f"theta: expected a positive number, got {theta}")
        self.dims, self.head_dim, self.theta, self.interleaved = dims, int(head_dim), float(theta), bool(interleaved)
        try:
            turns = [int(round(self.theta ** (-2.0 * i / d) / (2.0 * math.pi) * 2.0 ** 64)) % (1 << 64) for d in dims for i in range(d // 2)]
        except OverflowError:
            _bad(f"theta {theta}: its frequencies pass the range of a float")
        self.freq = torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in turns], dtype=torch.int64).to(device)


def _entries_meet(B, L, bs, rs, W):
    """Whether rows of different batch entries share elements: rows of W at b * bs + l * rs, rs >= W."""
    if bs >= (L - 1) * rs + W if L > 1 else bs >= W:
        return False
    if L == 1 or bs < W:
        return True
    if rs >= (B - 1) * bs + W:                   # the batch inside of the rows
        return False
    for b in range(1, B):                        # entry b against entry 0, row 0 of either
        l, rest = divmod(b * bs, rs)
        if l >= L:
            break
        if rest < W or (l + 1 < L and rs - rest < W):
            return True
    return False


def rope(x, axes, *, grid=None, origin=None, pos=None, inverse=False, out=None):
    """Rotary positions on x [B, L, heads * head_dim] (any batch / row stride: column slices of a fused q|k|v buffer, q|k together).

    Positions: pos int32 [L, axes] or [B, L, axes]; or grid = the axes' lengths with L cells, the last axis fastest, counted from
    `origin` (default 0).  inverse=True turns back: the gradient with respect to x of rope(x) is rope(dy, inverse=True).  out may be x, but
    not lie on part of it."""
    _chk_dev(x, pos, out, axes.freq)
    if x.requires_grad or out is not None and out.requires_grad:
        _no_graph(x, out)
    code = dtype_code(x.dtype)
    n, hd, sh, st = len(axes.dims), axes.head_dim, x.shape, x.stride()
    if len(sh) != 3 or sh[2] % hd or not sh[2] or st[2] != 1:
        _bad(f"x: expected [B, L, heads * {hd}] with contiguous columns, got {tuple(sh)} strides {st}")
    if axes.freq.device != x.device:
        _bad(f"axes were built on {axes.freq.device}, x is on {x.device}")
    B, L, W = sh
    given = out is not None
    if not given:
        out = torch.empty_like(x)
    else:
        _like("out", out, x)
    if L >= 2 ** 31 - 64 or W // hd > 1 << 16:
        _bad(f"x: at most 2^31 - 65 tokens of 2^16 heads, got {tuple(sh)}")
    so = out.stride()
    if so[2] != 1 or (L > 1 and so[1] < W) or (B > 1 and L and _entries_meet(B, L, so[0], so[1], W)):
        _bad(f"out: expected {tuple(sh)} with rows that do not overlap, got {tuple(out.shape)} strides {so}")
    if given:
        _apart("out", out, (("pos", pos), ("the frequencies", axes.freq)), (("x", x),))
    if (pos is None) == (grid is None):
        _bad("give either pos or grid")
    pp, pbs = None, 0
    if pos is not None:
        if origin is not None:
            _bad("origin goes with grid")
        _like("pos", pos, x, torch.int32, False)
        if pos.shape == (B, L, n):
            pbs = L * n
        elif pos.shape != (L, n):
            _bad(f"pos: expected contiguous ({L}, {n}) or ({B}, {L}, {n}), got {tuple(pos.shape)}")
        if not pos.is_contiguous():
            _bad(f"pos: expected contiguous memory, got strides {pos.stride()}")
        pp = pos.data_ptr()
        grid = origin = ()
    else:
        grid, origin = tuple(grid), tuple(origin) if origin is not None else (0,) * n
        if len(grid) != n or len(origin) != n or min(grid) < 1 or math.prod(grid) != L:
            _bad(f"grid {grid} (origin {origin}): expected {n} lengths with {L} cells")
        if any(o < -2 ** 31 or o + g > 2 ** 31 for o, g in zip(origin, grid)):
            _bad(f"positions from {origin} on pass 32 bits")
    d = _l.RopeDesc(x.data_ptr(), out.data_ptr(), st[0] if B > 1 else 0, st[1] if L > 1 else W, so[0] if B > 1 else 0, so[1] if L > 1 else W,
                    axes.freq.data_ptr(), pp, pbs, B, L, W // hd, hd, n, axes.dims, grid, origin, axes.interleaved, bool(inverse), code)
    _call("hallo_rope", x.device, C.byref(d))
    if given:
        _written(out)
    return out


def _heads4(name, t, heads, hd, writable=False):
    """[B, L, heads * hd] or [B, L, heads, hd] view -> its (batch, row, head) strides."""
    sh, st = t.shape, t.stride()
    if len(sh) == 3:
        ok = sh[2] == heads * hd and st[2] == 1
        bs, rs, hs = st[0], st[1], hd
    else:
        ok = len(sh) == 4 and sh[2] == heads and sh[3] == hd and st[3] == 1
        bs, rs, hs = st[:3] if ok else (0, 0, 0)
    if not ok:
        _bad(f"{name}: expected [B, L, {heads} * {hd}] or [B, L, {heads}, {hd}] with contiguous heads, got {tuple(sh)} strides {st}")
    if writable:
        extent = hd
        for s, n in sorted(((bs, sh[0]), (rs, sh[1]), (hs, heads))):
            if n > 1:
                if s < extent:
                    _bad(f"{name}: overlapping rows, strides {st}")
                extent += (n - 1) * s
    # strides of single or absent rows, entries and heads never count
    if sh[0] <= 1:
        bs = 0
    if sh[1] <= 1:
        rs = 0
    if heads == 1:
        hs = hd
    if (bs | rs | hs) & 7 or rs > 1 << 24 or t.data_ptr() & 15:
        _bad(f"{name}: expected strides that are multiples of 8 (rows at most 2^24 apart) and a 16-byte aligned start, got strides {st}")
    return bs, rs, hs


def _edge(n):
    return -1 if n < 0 else min(int(n), 1 << 29)


def _window_desc(q, k, v, o, lse, heads, kv_heads, left, right, sinks, q_len, kv_len, scale, o_given):
    """(descriptor without workspace, kv_heads, head_dim) of checked arguments."""
    code = dtype_code(q.dtype)
    if kv_heads is None:
        kv_heads = heads
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        _bad(f"{heads} query heads do not share {kv_heads} key heads")
    sq, sk = q.shape, k.shape
    if len(sq) not in (3, 4) or (len(sq) == 3 and sq[2] % heads):
        _bad(f"q: expected [B, L, {heads} * head_dim] or [B, L, {heads}, head_dim], got {tuple(sq)}")
    hd = sq[3] if len(sq) == 4 else sq[2] // heads
    if hd % 8 or not 8 <= hd <= 160:
        _bad(f"head_dim {hd}: expected a multiple of 8 up to 160")
    B, Lq = sq[0], sq[1]
    _like("k", k, q, None, False)
    _like("v", v, q, None, False)
    if len(sk) not in (3, 4) or sk[0] != B:
        _bad(f"k: expected [{B}, L, {kv_heads} * {hd}], got {tuple(sk)}")
    Lk = sk[1]
    if v.shape[:2] != sk[:2]:
        _bad(f"v: expected [{B}, {Lk}, {kv_heads} * {hd}], got {tuple(v.shape)}")
    if Lq > 1 << 29 or Lk > 1 << 29:
        _bad(f"lengths {Lq}, {Lk}: at most 2^29")
    for name, t in (("q_len", q_len), ("kv_len", kv_len)):
        if t is not None:
            _like(name, t, q, torch.int32, False)
            if t.shape != (B,) or not t.is_contiguous():
                _bad(f"{name}: expected contiguous ({B},), got {tuple(t.shape)}")
    if sinks < 0:
        _bad(f"sinks: {sinks}")
    scale = hd ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale < 1e30:
        _bad(f"scale: expected a positive number (1e-30 to 1e30), got {scale}")
    d = _l.WindowAttnDesc(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr() if lse is not None else None,
                          *_heads4("q", q, heads, hd), *_heads4("k", k, kv_heads, hd), *_heads4("v", v, kv_heads, hd),
                          *_heads4("out" if o_given else "o", o, heads, hd, o_given),
                          q_len.data_ptr() if q_len is not None else None, kv_len.data_ptr() if kv_len is not None else None,
                          Lq, Lk, B, heads, kv_heads, hd, _edge(left), _edge(right), _edge(sinks), scale, code)
    return d, kv_heads, hd


def window_attention(q, k, v, heads, *, kv_heads=None, left=-1, right=0, sinks=0, q_len=None, kv_len=None, scale=None, out=None,
                     return_lse=False):
    """softmax(scale q k^T) v over a sliding window and `sinks` always-visible first keys.

    q [B, Lq, heads * head_dim], k / v [B, Lk, kv_heads * head_dim] (or 4-D [B, L, heads, head_dim] views in any order of memory); query
    head h reads key head h // (heads // kv_heads).  Query i stands at p = kv_len - q_len + i and sees key j iff j < kv_len,
    j <= p + right, and j >= p - left or j < sinks; a negative left / right means no limit, so the default is causal attention with the
    queries at the end of the keys -- a prompt, a chunk of new tokens, or one new token against a cache of capacity Lk.  q_len / kv_len:
    int32 [B] on the device (default Lq / Lk), clamped to the tensors' lengths.  Queries that see nothing or are padding get zeros.
    Keys behind kv_len, or outside of every window, may hold anything; a key that some query sees must be finite (others multiply it by 0).
    head_dim: a multiple of 8 up to 160.  out must not overlap q, k or v.

    return_lse: (out, lse), lse fp32 [B, heads, Lq] (-inf where nothing is visible), as window_attention_backward() takes it."""
    _chk_dev(q, k, v, q_len, kv_len, out)
    if q.requires_grad or k.requires_grad or v.requires_grad or out is not None and out.requires_grad:
        _no_graph(q, k, v, out)
    given = out is not None
    if not given:
        out = torch.empty_like(q)
    else:
        _like("out", out, q)
    lse = None
    if return_lse and heads >= 1 and q.dim() > 2:
        lse = torch.empty((q.shape[0], heads, q.shape[1]), device=q.device, dtype=torch.float32)
    d, _, _ = _window_desc(q, k, v, out, lse, heads, kv_heads, left, right, sinks, q_len, kv_len, scale, given)
    if given:
        _apart("out", out, (("q", q), ("k", k), ("v", v), ("q_len", q_len), ("kv_len", kv_len)))
    need = _l.load().hallo_window_attention_workspace(C.byref(d))
    if need:
        if need < 0:
            _l.check(need, "hallo_window_attention_workspace")
        ws = torch.empty(need // 4, device=q.device, dtype=torch.float32)
        d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _call("hallo_window_attention", q.device, C.byref(d))
    if given:
        _written(out)
    return (out, lse) if return_lse else out


def window_attention_backward(do, q, k, v, o, lse, heads, *, kv_heads=None, left=-1, right=0, sinks=0, q_len=None, kv_len=None, scale=None,
                              dq=None, dk=None, dv=None):
    """(dq, dk, dv) of o, lse = window_attention(q, k, v, ..., return_lse=True) for do, with the same arguments.  dk / dv are summed over
    the query heads that share a key head; padded rows get zeros.  dq / dk / dv must overlap neither the inputs nor one another.  Results repeat bit for bit."""
    _chk_dev(do, q, k, v, o, lse, q_len, kv_len, dq, dk, dv)
    _like("o", o, q)
    _like("do", do, q)
    _like("lse", lse, q, torch.float32, False)
    if q.dim() < 3:
        _bad(f"q: expected [B, L, {heads} * head_dim] or [B, L, {heads}, head_dim], got {tuple(q.shape)}")
    if lse.shape != (q.shape[0], heads, q.shape[1]) or not lse.is_contiguous():
        _bad(f"lse: expected contiguous ({q.shape[0]}, {heads}, {q.shape[1]}), got {tuple(lse.shape)}")
    w, kv_heads, hd = _window_desc(q, k, v, o, lse, heads, kv_heads, left, right, sinks, q_len, kv_len, scale, False)
    outs, strides = [], []
    for name, t, like, n in (("dq", dq, q, heads), ("dk", dk, k, kv_heads), ("dv", dv, v, kv_heads)):
        given = t is not None
        if given:
            _like(name, t, like)
        else:
            t = torch.empty(like.shape, device=q.device, dtype=q.dtype)
        outs.append(t)
        strides += _heads4(name, t, n, hd, given)
    inputs = ("do", do), ("q", q), ("k", k), ("v", v), ("o", o), ("lse", lse), ("q_len", q_len), ("kv_len", kv_len)
    if dq is not None:
        _apart("dq", dq, (*inputs, ("dk", dk), ("dv", dv)))
    if dk is not None:
        _apart("dk", dk, (*inputs, ("dv", dv)))
    if dv is not None:
        _apart("dv", dv, inputs)
    given, (dq, dk, dv) = (dq, dk, dv), outs
    d = _l.WindowAttnBwdDesc(w, do.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *_heads4("do", do, heads, hd), *strides)
    need = _l.load().hallo_window_attention_backward_workspace(C.byref(d))
    if need < 0:
        _l.check(need, "hallo_window_attention_backward_workspace")
    ws = torch.empty(max(need // 4, 4), device=q.device, dtype=torch.float32)
    d.fwd.workspace, d.fwd.workspace_bytes = ws.data_ptr(), need
    _call("hallo_window_attention_backward", q.device, C.byref(d))
    _written(*given)
    return dq, dk, dv
