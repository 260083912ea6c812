"""Cases of the transformer-block operators for video and audio token sequences: LayerNorm with its backward pass, rotary
positions over several axes, and attention with a sliding window and always-visible first tokens (forward, backward, and single
tokens against a cache).  `run` computes a case either in its plain form (elementary torch operations) or, with `own` set, through
hallo_amd.ops."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the norm in front of the 64 x 64 level's attentions when four clips of 16 frames train together: 4 * 16 * 4096 tokens of 320
        {"name": "ln_fwd_video", "op": "ln_fwd", "rows": 262144, "C": 320, "dtype": "bf16"},
        # an audio encoder layer on ten seconds of speech (499 feature frames of 768): few rows, launch latency counts
        {"name": "ln_bwd_audio", "op": "ln_bwd", "rows": 499, "C": 768, "dtype": "f16"},
        # the backward pass of the first case, with both weight gradients
        {"name": "ln_bwd_video", "op": "ln_bwd", "rows": 262144, "C": 320, "dtype": "bf16"},
        # one new token for each of eight streams, explicit positions (time, height, width) far into a stream
        {"name": "rope_step", "op": "rope", "B": 8, "L": 1, "heads": 40, "hd": 128, "dims": "32,48,48", "interleaved": True, "grid": "",
         "extra": 0, "inverse": False, "dtype": "bf16"},
        # q | k columns (8 + 8 heads of 40) of the fused q|k|v rows of four 16-frame clips on the 64 x 64 latent grid
        {"name": "rope_video", "op": "rope", "B": 4, "L": 65536, "heads": 16, "hd": 40, "dims": "8,16,16", "interleaved": False,
         "grid": "16,64,64", "extra": 320, "inverse": False, "dtype": "f16"},
        # the gradient of rotated q | k on an odd grid, head dim 80 with columns that no axis turns
        {"name": "rope_odd_grad", "op": "rope", "B": 2, "L": 4255, "heads": 16, "hd": 80, "dims": "12,26,26", "interleaved": False,
         "grid": "5,23,37", "extra": 0, "inverse": True, "dtype": "bf16"},
        # one new token of one stream against 1500 cached ones
        {"name": "attn_step_one", "op": "attn", "B": 1, "Lq": 1, "Lk": 1500, "H": 12, "Hkv": 12, "hd": 64, "left": 1023, "right": 0, "sinks": 4,
         "ragged": False, "dtype": "f16"},
        # 32 streams in one batch, caches of up to 32768 tokens with a window of half of that, four query heads to a key head
        {"name": "attn_step_batch", "op": "attn", "B": 32, "Lq": 1, "Lk": 32768, "H": 32, "Hkv": 8, "hd": 128, "left": 16383, "right": 0,
         "sinks": 16, "ragged": True, "dtype": "bf16"},
        # 16 frames of 32 x 32 tokens, each seeing about four frames around it and the whole first frame
        {"name": "attn_fwd_video", "op": "attn", "B": 2, "Lq": 16384, "Lk": 16384, "H": 8, "Hkv": 8, "hd": 80, "left": 2048, "right": 2048,
         "sinks": 1024, "ragged": False, "dtype": "f16"},
        # a long causal sequence, as a sequence model trains on it or takes it in before it generates
        {"name": "attn_fwd_long", "op": "attn", "B": 2, "Lq": 8192, "Lk": 8192, "H": 32, "Hkv": 8, "hd": 128, "left": 4095, "right": 0,
         "sinks": 4, "ragged": False, "dtype": "bf16"},
        # a padded batch of speech of different lengths, symmetric window, training
        {"name": "attn_bwd_audio", "op": "attn_bwd", "B": 5, "Lq": 1499, "Lk": 1499, "H": 12, "Hkv": 12, "hd": 64, "left": 200, "right": 200,
         "sinks": 1, "ragged": True, "dtype": "f16"},
        # the backward pass of the long causal sequence, key and value gradients shared by four query heads
        {"name": "attn_bwd_long", "op": "attn_bwd", "B": 2, "Lq": 8192, "Lk": 8192, "H": 32, "Hkv": 8, "hd": 128, "left": 4095, "right": 0,
         "sinks": 4, "ragged": False, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "rope", "rope", "step", "step", "attn", "attn_bwd", "attn_bwd"])
    dtype = rng.choice(["f16", "bf16"])
    if op in ("ln_fwd", "ln_bwd"):
        C = rng.choice([rng.choice([320, 640, 768, 1280, 4096]), _log_int(rng, 24, 8192), 8 * _log_int(rng, 8, 1024)])
        rows = min(_log_int(rng, 1, 262144), 80_000_000 // C)
        return {"op": op, "rows": rows, "C": C, "dtype": dtype}
    if op == "rope":
        hd = rng.choice([40, 64, 80, 128, 160, 2 * rng.randint(8, 96)])
        axes = rng.randint(1, 4)
        dims, left = [], hd
        for a in range(axes):
            d = 2 * rng.randint(1, max(1, left // (2 * (axes - a))))
            dims.append(d)
            left -= d
        heads, B = rng.randint(1, 40), rng.randint(1, 4)
        most = max(1, min(65536, 80_000_000 // (hd * heads * B)))
        if axes == 3 and rng.random() < 0.6:
            T, Hh = _log_int(rng, 1, 24), _log_int(rng, 1, 64)
            W = max(1, min(64, most // (T * Hh)))
            L, grid = T * Hh * W, f"{T},{Hh},{W}"
            B = max(1, min(B, 80_000_000 // (hd * heads * L)))
        else:
            L, grid = _log_int(rng, 1, most), ""
        return {"op": "rope", "B": B, "L": L, "heads": heads, "hd": hd, "dims": ",".join(map(str, dims)), "interleaved": rng.random() < 0.5,
                "grid": grid, "extra": 8 * rng.choice([0, rng.randint(1, 40)]), "inverse": rng.random() < 0.5, "dtype": dtype}
    hd = rng.choice([40, 64, 80, 128, 128, 160, 8 * rng.randint(2, 20)])
    Hkv = rng.choice([1, 2, 4, 8, 12])
    G = rng.choice([1, 1, 2, 4, 7, 8])
    if Hkv == 12:
        G = 1
    sinks = rng.choice([0, 1, 4, 16, 100, 1024])
    ragged = rng.random() < 0.6
    if op == "step":
        Lk = _log_int(rng, 1, 32768)
        B = max(1, min(_log_int(rng, 1, 64), 1_000_000_000 // (Lk * Hkv * hd)))
        return {"op": "attn", "B": B, "Lq": rng.choice([1, 1, 1, 2, 5, 16]), "Lk": Lk, "H": Hkv * G, "Hkv": Hkv, "hd": hd,
                "left": rng.choice([-1, _log_int(rng, 1, 32768)]), "right": 0, "sinks": sinks, "ragged": ragged, "dtype": dtype}
    Lk = _log_int(rng, 17, 8192)
    Lq = Lk if rng.random() < 0.7 else _log_int(rng, 17, 8192)
    B = max(1, min(rng.randint(1, 8), int(2 ** 32 / (Lq * Lk * Hkv * G))))
    Hkv = max(1, min(Hkv, int(2 ** 32 / (Lq * Lk * G))))
    left = rng.choice([-1, _log_int(rng, 1, 8192), _log_int(rng, 16, 2048)])
    right = rng.choice([0, 0, -1, left if left >= 0 else 64])
    return {"op": op, "B": B, "Lq": Lq, "Lk": Lk, "H": Hkv * G, "Hkv": Hkv, "hd": hd, "left": left, "right": right, "sinks": sinks,
            "ragged": ragged, "dtype": dtype}


def _lengths(case):
    """Valid queries and keys of each batch entry (part of the case, not of the seed): a ragged batch goes down to about a third."""
    B, Lq, Lk = case["B"], case["Lq"], case["Lk"]
    if not case["ragged"]:
        return [Lq] * B, [Lk] * B
    kl = [max(1, Lk - (Lk * 2 * ((5 * b) % (B + 1))) // (3 * (B + 1))) for b in range(B)]
    ql = [k if Lq == Lk else (Lq if Lq <= 16 else max(1, Lq - (Lq * ((3 * b) % (B + 1))) // (2 * (B + 1)))) for b, k in enumerate(kl)]
    return ql, kl


def _visible(case):
    """(visible query-key pairs, keys that some query sees) of each batch entry."""
    pairs, keys = [], []
    for ql, kl in zip(*_lengths(case)):
        p = np.arange(ql, dtype=np.int64) + (kl - ql)
        hi = np.full_like(p, kl) if case["right"] < 0 else np.clip(p + case["right"] + 1, 0, kl)
        lo = np.zeros_like(p) if case["left"] < 0 else np.clip(p - case["left"], 0, None)
        s = np.minimum(case["sinks"], hi)
        pairs.append(int(np.sum(np.where(lo <= s, hi, hi - lo + s))))
        keys.append(int(hi[-1] - max(lo[0], 0) + min(case["sinks"], max(lo[0], 0))) if ql else 0)
    return pairs, keys


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _visible_mask(s, device):
    """[B, Lq, Lk] truth values: which key each query sees."""
    Lq, Lk = s["Lq"], s["Lk"]
    ql = s["q_len"].view(-1, 1, 1).long()
    kl = s["kv_len"].view(-1, 1, 1).long()
    i = torch.arange(Lq, device=device).view(1, -1, 1)
    j = torch.arange(Lk, device=device).view(1, 1, -1)
    p = kl - ql + i
    ok = (j < kl) & (i < ql)
    if s["right"] >= 0:
        ok = ok & (j <= p + s["right"])
    if s["left"] >= 0:
        ok = ok & ((j >= p - s["left"]) | (j < s["sinks"]))
    return ok


def _grouped(x, Hkv, hd):
    """[B, L, heads * hd] -> fp32 [B, Hkv, G * L, hd] (query rows of the heads that share a key head, head by head)."""
    B, L = x.shape[:2]
    G = x.shape[2] // (Hkv * hd)
    return x.float().view(B, L, Hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * L, hd)


def _ungrouped(x, L):
    B, Hkv, GL, hd = x.shape
    return x.view(B, Hkv, GL // L, L, hd).permute(0, 3, 1, 2, 4).reshape(B, L, -1)


def _plain_scores(s):
    B, Lq, Lk, H, Hkv, hd = (s[k] for k in ("B", "Lq", "Lk", "H", "Hkv", "hd"))
    G = H // Hkv
    q, k = _grouped(s["q"], Hkv, hd), _grouped(s["k"], Hkv, hd)
    sc = torch.matmul(q, k.transpose(2, 3)).mul_(hd ** -0.5)
    ok = _visible_mask(s, q.device)
    sc.view(B, Hkv, G, Lq, Lk).masked_fill_(~ok.view(B, 1, 1, Lq, Lk), float("-inf"))
    return q, k, sc


def _plain_attention(s):
    B, Lq, H, Hkv, hd = (s[k] for k in ("B", "Lq", "H", "Hkv", "hd"))
    _, _, sc = _plain_scores(s)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = torch.exp(sc.sub_(m))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, _grouped(s["v"], Hkv, hd)) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (m + torch.log(total)).view(B, H, Lq)
    return _ungrouped(o, Lq).to(s["q"].dtype), lse


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] in ("ln_fwd", "ln_bwd"):
        rows, C = case["rows"], case["C"]
        s["x"] = (_randn(g, rows, C) * (0.5 + torch.rand(rows, 1, generator=g, device="cuda")) + 0.3 * _randn(g, rows, 1)).to(dt)
        s["gamma"] = (1.0 + 0.1 * _randn(g, C)).to(dt)
        s["beta"] = (0.1 * _randn(g, C)).to(dt)
        if case["op"] == "ln_bwd":
            s["dy"] = (0.02 * _randn(g, rows, C)).to(dt)
            s["stats"] = _plain_stats(s["x"])
        return s
    if case["op"] == "rope":
        B, L, width = case["B"], case["L"], case["heads"] * case["hd"]
        buf = _randn(g, B, L, width + case["extra"]).to(dt)
        s["x"] = buf[..., :width]
        dims = [int(d) for d in case["dims"].split(",")]
        s["dims"] = dims
        if case["grid"]:
            s["grid"] = tuple(int(d) for d in case["grid"].split(","))
            s["origin"] = (1000 * (int(seed) % 50), 0, 0)
        else:
            s["grid"] = None
            s["pos"] = torch.randint(0, 100000, (B, L, len(dims)), generator=g, device="cuda", dtype=torch.int32)
        if own:
            from hallo_amd import ops
            s["axes"] = ops.RopeAxes(dims, case["hd"], theta=10000.0, interleaved=case["interleaved"], device="cuda")
        return s
    B, Lq, Lk, H, Hkv, hd = (case[k] for k in ("B", "Lq", "Lk", "H", "Hkv", "hd"))
    s["q"] = _randn(g, B, Lq, H * hd).to(dt)
    s["k"] = _randn(g, B, Lk, Hkv * hd).to(dt)
    s["v"] = _randn(g, B, Lk, Hkv * hd).to(dt)
    ql, kl = _lengths(case)
    s["q_len"] = torch.tensor(ql, device="cuda", dtype=torch.int32)
    s["kv_len"] = torch.tensor(kl, device="cuda", dtype=torch.int32)
    if case["op"] == "attn_bwd":
        s["o"], s["lse"] = _plain_attention(s)
        s["do"] = (0.05 * _randn(g, B, Lq, H * hd)).to(dt)
    return s


def _plain_stats(x, eps=1e-5):
    xf = x.float()
    mean = xf.mean(-1, keepdim=True)
    var = (xf - mean).square().mean(-1, keepdim=True)
    return torch.cat([mean, torch.rsqrt(var + eps)], -1)


def _plain_ln_fwd(s):
    st = _plain_stats(s["x"])
    y = (s["x"].float() - st[:, :1]) * st[:, 1:] * s["gamma"].float() + s["beta"].float()
    return {"y": y.to(s["x"].dtype), "stats": st}


def _plain_ln_bwd(s):
    dy, mean, rstd = s["dy"].float(), s["stats"][:, :1], s["stats"][:, 1:]
    xh = (s["x"].float() - mean) * rstd
    gy = dy * s["gamma"].float()
    dx = rstd * (gy - gy.mean(-1, keepdim=True) - xh * (gy * xh).mean(-1, keepdim=True))
    return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * xh).sum(0, dtype=torch.float64).float(), "dbeta": dy.sum(0, dtype=torch.float64).float()}


def _rope_positions(s):
    """[B or 1, L, axes] positions."""
    if s["grid"] is None:
        return s["pos"].long()
    ax = [torch.arange(n, device=s["x"].device) + o for n, o in zip(s["grid"], s["origin"])]
    return torch.stack(torch.meshgrid(*ax, indexing="ij"), -1).view(1, -1, len(ax))


def _plain_rope(s):
    x, hd = s["x"], s["hd"]
    B, L = x.shape[:2]
    xf = x.float().view(B, L, -1, hd)
    out = xf.clone()
    pos = _rope_positions(s)
    at = 0
    for a, d in enumerate(s["dims"]):
        freq = 10000.0 ** (-torch.arange(0, d, 2, device=x.device, dtype=torch.float64) / d)
        ang = pos[..., a:a + 1].double() * freq
        cos, sin = ang.cos().float().unsqueeze(2), ang.sin().float().unsqueeze(2)
        if s["inverse"]:
            sin = -sin
        first, second = (slice(at, at + d, 2), slice(at + 1, at + d, 2)) if s["interleaved"] else (slice(at, at + d // 2), slice(at + d // 2, at + d))
        u, v = xf[..., first], xf[..., second]
        out[..., first] = u * cos - v * sin
        out[..., second] = u * sin + v * cos
        at += d
    return out.view(B, L, -1).to(x.dtype)


def _plain_attention_backward(s):
    B, Lq, Lk, Hkv, hd = (s[k] for k in ("B", "Lq", "Lk", "Hkv", "hd"))
    q, k, sc = _plain_scores(s)
    lse = s["lse"].reshape(B, Hkv, -1, 1)
    p = torch.exp(sc.sub_(torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)))
    do, o, v = _grouped(s["do"], Hkv, hd), _grouped(s["o"], Hkv, hd), _grouped(s["v"], Hkv, hd)
    delta = (do * o).sum(-1, keepdim=True)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = p.mul_(torch.matmul(do, v.transpose(2, 3)).sub_(delta))
    dq = torch.matmul(ds, k) * hd ** -0.5
    dk = torch.matmul(ds.transpose(2, 3), q) * hd ** -0.5
    dt = s["q"].dtype
    return {"dq": _ungrouped(dq, Lq).to(dt), "dk": _ungrouped(dk, Lk).to(dt), "dv": _ungrouped(dv, Lk).to(dt)}


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "ln_fwd":
        return _plain_ln_fwd(s)
    if s["op"] == "ln_bwd":
        return _plain_ln_bwd(s)
    if s["op"] == "rope":
        return _plain_rope(s)
    if s["op"] == "attn":
        o, lse = _plain_attention(s)
        return {"o": o, "lse": lse}
    return _plain_attention_backward(s)


def _run_own(s):
    from hallo_amd import ops
    if s["op"] == "ln_fwd":
        y, stats = ops.layernorm_train(s["x"], s["gamma"], s["beta"], 1e-5)
        return {"y": y, "stats": stats}
    if s["op"] == "ln_bwd":
        dx, dgamma, dbeta = ops.layernorm_backward(s["dy"], s["x"], s["stats"], s["gamma"])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if s["op"] == "rope":
        at = {"grid": s["grid"], "origin": s["origin"]} if s["grid"] is not None else {"pos": s["pos"]}
        return ops.rope(s["x"], s["axes"], inverse=s["inverse"], **at)
    kw = dict(kv_heads=s["Hkv"], left=s["left"], right=s["right"], sinks=s["sinks"], q_len=s["q_len"], kv_len=s["kv_len"])
    if s["op"] == "attn":
        o, lse = ops.window_attention(s["q"], s["k"], s["v"], s["H"], return_lse=True, **kw)
        return {"o": o, "lse": lse}
    dq, dk, dv = ops.window_attention_backward(s["do"], s["q"], s["k"], s["v"], s["o"], s["lse"], s["H"], **kw)
    return {"dq": dq, "dk": dk, "dv": dv}


def work(case):
    if case["op"] in ("ln_fwd", "ln_bwd"):
        rows, C = case["rows"], case["C"]
        fwd = case["op"] == "ln_fwd"
        return {"bytes": rows * C * 2 * (2 if fwd else 3) + rows * 8 + C * (4 if fwd else 10), "flops": rows * C * (8 if fwd else 15)}
    if case["op"] == "rope":
        n = case["B"] * case["L"] * case["heads"] * case["hd"]
        pos = 0 if case["grid"] else case["B"] * case["L"] * 4 * len(case["dims"].split(","))
        return {"bytes": 4 * n + pos, "flops": 3 * n}
    pairs, keys = _visible(case)
    ql, _ = _lengths(case)
    q_bytes = case["B"] * case["Lq"] * case["H"] * (case["hd"] * 2)
    kv_bytes = sum(keys) * case["Hkv"] * case["hd"] * 2
    lse = case["B"] * case["Lq"] * case["H"] * 4
    n = sum(pairs) * case["H"] * case["hd"]
    if case["op"] == "attn":
        return {"bytes": 2 * q_bytes + 2 * kv_bytes + lse, "flops": 4 * n}
    return {"bytes": 4 * q_bytes + 2 * kv_bytes + 2 * case["B"] * case["Lk"] * case["Hkv"] * case["hd"] * 2 + lse, "flops": 10 * n}


def _exact_rows(case, s, backward):
    """Attention from its definition in 64 bits, one (batch entry, head) at a time."""
    B, Lq, Lk, H, Hkv, hd = (case[k] for k in ("B", "Lq", "Lk", "H", "Hkv", "hd"))
    f = lambda t, n: t.double().view(B, -1, n, hd)
    q, k, v = f(s["q"], H), f(s["k"], Hkv), f(s["v"], Hkv)
    scale = 1.0 / math.sqrt(hd)
    ql, kl = _lengths(case)
    if backward:
        do, o = f(s["do"], H), f(s["o"], H)
        out = {n: torch.zeros_like(t) for n, t in (("dq", q), ("dk", k), ("dv", v))}
    else:
        out = {"o": torch.zeros_like(q), "lse": torch.full((B, H, Lq), -math.inf, device=q.device, dtype=torch.float64)}
    for b in range(B):
        nq, nk = ql[b], kl[b]
        where = torch.arange(nq, device=q.device)[:, None] + (nk - nq)
        key = torch.arange(nk, device=q.device)[None, :]
        hidden = torch.zeros((nq, nk), device=q.device, dtype=torch.bool)
        if case["right"] >= 0:
            hidden |= key - where > case["right"]
        if case["left"] >= 0:
            hidden |= (where - key > case["left"]) & (key >= case["sinks"])
        for h in range(H):
            c = h // (H // Hkv)
            z = (q[b, :nq, h] @ k[b, :nk, c].t()) * scale
            z[hidden] = -math.inf
            if not backward:
                norm = torch.logsumexp(z, 1)
                out["lse"][b, h, :nq] = norm
                w = torch.exp(z - norm.clamp(min=-1e300)[:, None])
                out["o"][b, :nq, h] = w @ v[b, :nk, c]
                continue
            w = torch.exp(z - s["lse"][b, h, :nq].double().clamp(min=-1e300)[:, None])
            g = do[b, :nq, h]
            out["dv"][b, :nk, c] += w.t() @ g
            w *= g @ v[b, :nk, c].t() - (g * o[b, :nq, h]).sum(1)[:, None]
            out["dq"][b, :nq, h] = (w @ k[b, :nk, c]) * scale
            out["dk"][b, :nk, c] += (w.t() @ q[b, :nq, h]) * scale
    return {n: (t if n == "lse" else t.reshape(B, t.shape[1], -1)) for n, t in out.items()}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ln_fwd":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        rstd = 1.0 / torch.sqrt(var + 1e-5)
        return {"y": torch.addcmul(s["beta"].double(), (x - mean) * rstd, s["gamma"].double()), "stats": torch.cat([mean, rstd], 1)}
    if case["op"] == "ln_bwd":
        x, dy, st = s["x"].double(), s["dy"].double(), s["stats"].double()
        xh = (x - st[:, 0:1]) * st[:, 1:2]
        t = dy * s["gamma"].double()
        C = case["C"]
        dx = (t - t.sum(1, keepdim=True) / C - xh * ((t * xh).sum(1, keepdim=True) / C)) * st[:, 1:2]
        return {"dx": dx, "dgamma": torch.einsum("rc,rc->c", dy, xh), "dbeta": dy.sum(0)}
    if case["op"] == "rope":
        B, L, heads, hd = case["B"], case["L"], case["heads"], case["hd"]
        x = s["x"].double().reshape(B, L, heads, hd)
        if s["grid"] is None:
            pos = s["pos"].double()
        else:
            T, Hh, W = s["grid"]
            n = torch.arange(L, device=x.device)
            pos = torch.stack([n // (Hh * W), n // W % Hh, n % W], 1).double() + torch.tensor(s["origin"], device=x.device).double()
            pos = pos.expand(B, L, 3)
        y, at = x.clone(), 0
        for a, d in enumerate(s["dims"]):
            for i in range(d // 2):
                turn = pos[:, :, a] * math.exp(-math.log(10000.0) * 2 * i / d) * (-1.0 if case["inverse"] else 1.0)
                c, sn = torch.cos(turn)[..., None], torch.sin(turn)[..., None]
                m, n = (at + 2 * i, at + 2 * i + 1) if case["interleaved"] else (at + i, at + i + d // 2)
                y[..., m], y[..., n] = c * x[..., m] - sn * x[..., n], c * x[..., n] + sn * x[..., m]
            at += d
        return y.reshape(B, L, heads * hd)
    if sum(_visible(case)[0]) * case["H"] > 4e9:
        return None
    return _exact_rows(case, s, case["op"] == "attn_bwd")
