// Attention with a sliding window and always-visible first keys: backward pass.
//
//   P = exp(scale q k^T - lse) over the visible pairs,   delta = sum_d(do * o)
//   dV = P^T dO,   dS = P * (dO V^T - delta),   dQ = scale dS K,   dK = scale dS^T Q
// summed over the query heads that share a key head.  Three launches, and one for each kind of parts:
//   prep   delta and lse * log2(e) of every query (fp32; +inf where a query has no visible key, so its P is 0)
//   dkv    a workgroup owns 128 keys: K and V stay in registers as MFMA operands, dK and dV as accumulators, and the query rows that see
//          the keys stream through LDS, for all heads of the group -- shared heads need no atomics
//   dq     a workgroup owns 128 queries of a head (a wave 32), the visible keys stream through LDS
//   join   the sinks are seen by every query: their key tiles' query rows are split over workgroups, fp32 parts are added here in order
//          (also used for all keys when there are too few key tiles to fill the chip, and for dq's keys when there are few queries)
// P (for dV) and dS (for dQ and dK) are rounded to the storage type because the matrix cores take 16-bit operands; P, dP and dS themselves,
// delta and all sums are fp32 (what dkv hands from role to role: see there).  On random inputs the gradients' error against 64 bits is
// 1.4 times that of rounding the exact ones once.
// S and dO V^T are computed in both dkv and dq (7 products where 5 would do with atomics on dQ): results do not depend on timing.
// Bound by the SIMDs' issue as the forward pass (MFMA 40 %, vector 30 - 34 % of all cycles, LDS port 27 - 37 % busy).  2 x 8192 tokens, 32 / 8
// heads of 128, window 4096, bf16: 3.2 ms (dkv 1.79, dq 1.38, prep 0.06), 640 TFLOP/s of the five products that count, 900 of the seven done.
//
// fp16: P is 1/N over long rows and dS smaller still, below fp16's normal numbers.  Both are carried scaled by powers of two that cannot
// overflow and are taken out of the fp32 accumulators at the end: P by 2^14 (P <= 1), dS by 2^e with |dS| = P |do_i . (v_j - o_i)| <=
// 2 |do_i|_2 max_j |v_j|_2 < 2^(15 - e) -- in dkv with the largest |do_i| of the group's queries that see the tile, in dq with the lane's
// own do row, and j over the keys that these queries see.  (A key's own |v_j| bounds nothing: o_i is as long as the longest v that i sees.
// The largest over the whole sequence would do, and lose what is small behind a window in fp16's subnormal numbers.)  bf16 has fp32's range
// and needs neither.
#include <type_traits>
#include "window_args.h"
#include "../../include/hallo_amd.h"

namespace hallo {

bool win_args(const hallo_window_attn_desc* d, WinArgs& a);      // window_attention.hip

namespace {

struct WinBwdArgs {
  WinArgs w;
  const void* dout; void *dq, *dk, *dv;
  long do_bs, do_rs, do_hs, dq_bs, dq_rs, dq_hs, dk_bs, dk_rs, dk_hs, dv_bs, dv_rs, dv_hs;
  float *delta, *lse2;                           // [batch, heads, Lq]
  float *domax, *vmax;                           // fp16: largest row norms of 64 rows, [batch, heads, nq64], [batch, kv_heads, nk64]
  int nq64, nk64;
  int nst, nrt, sps, spr;                        // key tiles of the sinks / of the rest, query splits of each
  float* part;                                   // [batch, kv_heads][nst * sps (if sps > 1) + nrt * spr (if spr > 1)][128][2 hd]
  int nparts;                                    // part tiles of one (batch entry, key head)
  int spq; float* qpart;                         // key splits of dq, [batch, heads, Lq][spq][hd]
};

constexpr int BW_KEYS = 128;                     // keys of a dkv workgroup
constexpr float P_EXP = 14.0f;                   // fp16: P is carried times 2^14

// whether some query of the entry sees key j < kn (the queries stand at shift .. kn - 1); what lies elsewhere may hold anything
__device__ __forceinline__ bool key_seen(const WinArgs& p, int j, int shift, int qn) {
  return qn > 0 && (p.left < 0 || j < p.sinks || shift - p.left <= j);
}

// 2^e with 2 a b 2^e < 2^15
__device__ __forceinline__ float ds_scale(float a, float b) {
  const float bound = 2.0f * a * b;
  if (!(bound > 0.0f) || !(bound < 1e30f)) return 1.0f;
  const int e = 15 - __builtin_amdgcn_frexp_expf(bound);
  return __builtin_amdgcn_ldexpf(1.0f, min(e, 110));
}

template <typename T, int NC>
__global__ __launch_bounds__(256) void win_bwd_prep_kernel(const WinBwdArgs a, int qblocks) {
  using V8 = typename Vec<T>::v8;
  constexpr bool F16 = std::is_same<T, _Float16>::value;
  const WinArgs& p = a.w;
  __shared__ float red[16];
  const int sub = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const bool isq = (int)blockIdx.x < qblocks;
  int bid = isq ? blockIdx.x : blockIdx.x - qblocks;
  const int nb = isq ? a.nq64 : a.nk64, heads = isq ? p.heads : p.kv_heads;
  const int blk = bid % nb; bid /= nb;
  const int h = bid % heads, b = bid / heads;
  const int qn = win_len(p.q_len, b, p.Lq), kn = win_len(p.kv_len, b, p.Lk), n = isq ? qn : kn;
  float big = 0.0f;
  V8 xv[4][NC], ov[4][NC];                       // 16 lanes share a row, a lane's columns start at 8 sub (and 128 + 8 sub); four rows in flight
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = blk * 64 + k * 16 + grp;
    const T* x = isq ? reinterpret_cast<const T*>(a.dout) + (long)b * a.do_bs + (long)h * a.do_hs + (long)i * a.do_rs
                     : reinterpret_cast<const T*>(p.v) + (long)b * p.v_bs + (long)h * p.v_hs + (long)i * p.v_rs;
    const T* o = reinterpret_cast<const T*>(p.o) + (long)b * p.o_bs + (long)h * p.o_hs + (long)i * p.o_rs;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = sub * 8 + 128 * c;
      const bool ok = i < n && d < p.hd && (isq || key_seen(p, i, kn - qn, qn));
      xv[k][c] = ok ? ld8<T>(x + d) : zero8<T>();
      ov[k][c] = ok && isq ? ld8<T>(o + d) : zero8<T>();
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = blk * 64 + k * 16 + grp;
    float dl = 0.0f, sq = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = to_f32(xv[k][c][e]);
        dl += f * to_f32(ov[k][c][e]);
        sq += f * f;
      }
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) {
      dl += __shfl_xor(dl, s, 64);
      if (F16) sq += __shfl_xor(sq, s, 64);
    }
    if (isq && sub == 0 && i < p.Lq) {
      const long at = ((long)b * p.heads + h) * p.Lq + i;
      const float ls = i < n ? p.lse[at] : -__builtin_inff();
      a.delta[at] = dl;
      a.lse2[at] = ls == -__builtin_inff() ? __builtin_inff() : ls * 1.44269504088896340736f;
    }
    if (F16) big = fmaxf(big, sqrtf(sq));
  }
  if (!F16) return;
  if (sub == 0) red[grp] = big;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 1; k < 16; ++k) big = fmaxf(big, red[k]);
    (isq ? a.domax : a.vmax)[((long)b * heads + h) * nb + blk] = big;
  }
}

// Eight waves: four groups of 32 keys times two roles, so that a wave keeps ONE operand and ONE accumulator (HK = 128: 32 + 64
// registers; both in one wave are 400 registers, and hipcc then moves 128 accumulators between its two register files in every tile) and a
// SIMD has a wave of each role, whose matrix and vector work overlap.
//   role 0, tile t:      S = Q K^T, P = exp2(S c - lse2), dV += P^T dO; leaves P for its partner in LDS
//   role 1, tile t - 1:  dP = dO V^T, dS = P * (dP - delta), dK += dS^T Q
// Q and dO tiles are kept for two iterations (three LDS stages), P in two, so one barrier per tile is enough.  P goes over finer than
// dV's product takes it: dS from the rounded P made dK's error 1.7 times that of one rounding.  It is fp32, except for bf16 rows of 112
// and 128 columns: there 64 query rows per tile leave room for 16 bits only, and fp16 of P times 2^14 is 8 times as fine as bf16
// (2 x 8192 tokens, 32 / 8 heads of 128: 3.36 ms; fp32 and 32 query rows per tile: 3.77 ms; P as dV takes it: 3.28 ms).
template <typename T, int HK>
__global__ __launch_bounds__(512, HK <= 64 ? 4 : 2) void win_bwd_dkv_kernel(const WinBwdArgs a) {
  using V8 = typename Vec<T>::v8;
  constexpr bool F16 = std::is_same<T, _Float16>::value;
  constexpr bool HALF_P = !F16 && HK > 96 && HK <= 128, SCALED = F16 || HALF_P;      // SCALED: P is carried times 2^14
  using PT = typename std::conditional<HALF_P, f16x4, f32x4>::type;
  constexpr int QB = HK == 80 || HK == 96 || HALF_P ? 64 : 32;     // query rows of a tile: what three stages and P leave room for
  constexpr int NQ = QB / 32, NKS = HK / 16, NDB = (HK + 31) / 32, CH = HK / 8;
  using Tile = WinTile<HK>;
  constexpr int TB = QB * Tile::PITCH, STAGE = 2 * TB + 2 * QB * 4;        // Q | dO | lse2 | delta
  constexpr int PG = 64 * sizeof(PT), PX = NQ * 4 * PG;  // P of one key group: NQ x [4][64 lanes]
  constexpr int U = (QB * CH + 511) / 512;
  const WinArgs& p = a.w;
  __shared__ __attribute__((aligned(16))) unsigned char smem[3 * STAGE + 2 * 4 * PX];
  win_lds* const lds = (win_lds*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, l31 = lane & 31, kg = wave & 3;
  const bool role = wave >> 2;

  // block -> (key head, batch entry, key tile, query split); the longest tiles come first: the sinks, then the first keys, or the last
  // ones where the queries see everything ahead of them but not everything behind
  int bid = blockIdx.x;
  const int hk = bid % p.kv_heads; bid /= p.kv_heads;
  const int b = bid % p.batch; bid /= p.batch;
  const bool sink = bid < a.nst * a.sps;
  const int loc = sink ? bid : bid - a.nst * a.sps, sp = sink ? a.sps : a.spr;
  const int order = loc / sp, split = loc - order * sp;
  const int tile = !sink && p.right < 0 && p.left >= 0 ? a.nrt - 1 - order : order;
  const int qn = win_len(p.q_len, b, p.Lq), kn = win_len(p.kv_len, b, p.Lk), shift = kn - qn;
  const int s_end = min(p.sinks, p.Lk);
  const int ka = (sink ? 0 : s_end) + tile * BW_KEYS, kz = min(ka + BW_KEYS, sink ? s_end : p.Lk), kb = min(kz, kn);

  // queries that see some key of [ka, kb)
  int ia = 0, ib = 0;
  if (ka < kb) {
    ia = p.right < 0 ? 0 : win_clamp(ka - p.right - shift, 0, qn);
    ib = p.left < 0 || sink ? qn : win_clamp(kb - 1 + p.left - shift + 1, 0, qn);
  }
  const int ntq = ib > ia ? (ib - ia + QB - 1) / QB : 0, its = ntq * p.group;
  const int itb = (int)((long)its * split / sp), ite = (int)((long)its * (split + 1) / sp);

  const T* W = role ? reinterpret_cast<const T*>(p.v) + (long)b * p.v_bs + (long)hk * p.v_hs
                    : reinterpret_cast<const T*>(p.k) + (long)b * p.k_bs + (long)hk * p.k_hs;
  const long w_rs = role ? p.v_rs : p.k_rs;
  const int kw = ka + kg * 32, key = kw + l31;
  const bool seen = key < kb && key_seen(p, key, shift, qn);
  V8 wf[NKS];                                    // this lane's key row of K (role 0) or V (role 1)
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    const int d = ks * 16 + hi * 8;
    wf[ks] = seen && d < p.hd ? ld8<T>(W + (long)key * w_rs + d) : zero8<T>();
  }
  float g = 1.0f;                                // fp16: scale of dS
  if (F16 && role) {
    float dm = 0.0f, vm = 0.0f;
    if (ib > ia) {
      const WinRange r = win_range(p, shift + ia, shift + ib - 1, kn);
      const float* n = a.vmax + ((long)b * p.kv_heads + hk) * a.nk64;
      vm = win_norm(n, r.s1, r.e1, lane, win_norm(n, 0, r.e0, lane, 0.0f));
      for (int h = hk * p.group; h < (hk + 1) * p.group; ++h) dm = win_norm(a.domax + ((long)b * p.heads + h) * a.nq64, ia, ib, lane, dm);
    }
    g = ds_scale(wave_max(dm), wave_max(vm));
  }
  const float gs = g * 0x1p-14f;                 // relative to P's

  // positions that see this lane's key / that all of the group's keys are seen from / that see any of them
  constexpr int FAR = WIN_MAX_LEN * 2 - 1;
  const bool back = p.left < 0 || sink;
  const int plo = p.right < 0 ? -FAR : key - p.right, phi = back ? FAR : key + p.left;
  const int alo = p.right < 0 ? -FAR : kw + 31 - p.right, ahi = back ? FAR : kw + p.left;
  const int nlo = p.right < 0 ? -FAR : kw - p.right, nhi = back ? FAR : kw + 31 + p.left;

  V8 qr[U], gr[U];
  float lr = 0.0f, dr = 0.0f;
  unsigned qo[U], go[U];                         // byte offsets inside a tile, and this thread's places in its LDS image
  int so[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int u = tid + 512 * i, rr = u / CH, ch = u - rr * CH;
    qo[i] = ((unsigned)rr * (unsigned)p.q_rs + ch * 8) * 2;
    go[i] = ((unsigned)rr * (unsigned)a.do_rs + ch * 8) * 2;
    so[i] = Tile::at(rr, ch);
  }
  const bool whole = p.hd == HK;
  int lg = ntq ? itb / ntq : 0, li = itb - lg * ntq;     // head of the group and query tile that load() takes next
  auto load = [&]() {
    const int i0 = ia + li * QB, h = hk * p.group + lg, rem = ib - i0;
    const char* qt = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.q) + (long)b * p.q_bs + (long)h * p.q_hs + (long)i0 * p.q_rs);
    const char* gt = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.dout) + (long)b * a.do_bs + (long)h * a.do_hs + (long)i0 * a.do_rs);
    if (rem >= QB && whole) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (QB * CH % 512 == 0 || i + 1 < U || tid + 512 * i < QB * CH) {
          qr[i] = ld8<T>(reinterpret_cast<const T*>(qt + qo[i]));
          gr[i] = ld8<T>(reinterpret_cast<const T*>(gt + go[i]));
        }
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int u = tid + 512 * i, rr = u / CH, ch = u - rr * CH;
        const bool ok = rr < rem && rr < QB && ch * 8 < p.hd;
        qr[i] = ok ? ld8<T>(reinterpret_cast<const T*>(qt + qo[i])) : zero8<T>();
        gr[i] = ok ? ld8<T>(reinterpret_cast<const T*>(gt + go[i])) : zero8<T>();
      }
    }
    if (tid < QB) {
      const long at = ((long)b * p.heads + h) * p.Lq + i0 + tid;
      lr = tid < rem ? a.lse2[at] : __builtin_inff();
      dr = tid < rem ? a.delta[at] : 0.0f;
    }
    if (++li == ntq) { li = 0; ++lg; }
  };
  auto store = [&](int stage) {
    win_lds* const qt = lds + stage * STAGE;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (QB * CH % 512 == 0 || i + 1 < U || tid + 512 * i < QB * CH) {
        *(__attribute__((address_space(3))) V8*)(qt + so[i]) = qr[i];
        *(__attribute__((address_space(3))) V8*)(qt + TB + so[i]) = gr[i];
      }
    if (tid < QB) {
      *(__attribute__((address_space(3))) float*)(qt + 2 * TB + tid * 4) = lr;
      *(__attribute__((address_space(3))) float*)(qt + 2 * TB + QB * 4 + tid * 4) = dr;
    }
  };

  f32x16 acc[NDB];                               // dV (role 0) or dK (role 1): registers hold keys, lanes columns
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[db][e] = 0.0f;
  const f32x16 zero16 = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  // role 0 takes rows of Q and columns of dO, role 1 rows of dO and columns of Q
  const int rfo = role ? TB : 0, tfo = role ? 0 : TB;
  const Tile tl(lane);
  win_lds* const px = lds + 3 * STAGE + kg * PX + lane * (int)sizeof(PT);
  typedef __attribute__((address_space(3))) PT ldsp;
  const float c = p.c;

  if (itb < ite) { load(); store(0); }
  win_loads_done();
  if (itb + 1 < ite) load();
  __syncthreads();
  int st = 0, ci = ntq ? itb % ntq : 0;          // stage and query tile of role 0; role 1 is one behind
  int prev_p0 = 0;
  for (int it = itb; it <= ite; ++it) {
    const int nst = st == 2 ? 0 : st + 1, pst = st == 0 ? 2 : st - 1;
    if (it + 1 < ite) store(nst);                // last read, by role 1, in the iteration before this one
    if (it + 2 < ite) load();
    const int p0 = role ? prev_p0 : shift + ia + ci * QB;
    prev_p0 = shift + ia + ci * QB;
    const bool mine = role ? it > itb : it < ite;
    if (mine && kw < kb && p0 + QB - 1 >= nlo && p0 <= nhi) {
      const win_lds* const tb = lds + (role ? pst : st) * STAGE;
      const win_lds* const stat = tb + 2 * TB + (role ? QB * 4 : 0) + 16 * hi;
      win_lds* const pt = px + (((it - itb) ^ (role ? 1 : 0)) & 1) * 4 * PX;
      f32x16 s[NQ];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        s[n] = zero16;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
          s[n] = Vec<T>::mfma32(tl.template row<V8>(tb + rfo, n * 32, ks), wf[ks], s[n]);
      }
      win_order<NQ * NKS, 1, NKS < 4 ? NKS : 4>();
      V8 f[NQ][2];
      if (!role) {
        const bool all = p0 >= alo && p0 + QB - 1 <= ahi;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 ls = *(const __attribute__((address_space(3))) f32x4*)(stat + (n * 32 + 8 * g) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][4 * g + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][4 * g + e], c, (SCALED ? P_EXP : 0.0f) - ls[e]));
          }
          if (!all)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const int pe = p0 + n * 32 + 8 * (x >> 2) + 4 * hi + (x & 3);
              s[n][x] = pe >= plo && pe <= phi ? s[n][x] : 0.0f;
            }
#pragma unroll
          for (int x = 0; x < 16; ++x) f[n][x >> 3][x & 7] = from_f32<T>(s[n][x]);
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *(ldsp*)(pt + (n * 4 + g) * PG) = __builtin_convertvector((f32x4{s[n][4 * g], s[n][4 * g + 1], s[n][4 * g + 2], s[n][4 * g + 3]}), PT);
        }
      } else {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 pv = __builtin_convertvector(*(const ldsp*)(pt + (n * 4 + g) * PG), f32x4);
            const f32x4 dl = *(const __attribute__((address_space(3))) f32x4*)(stat + (n * 32 + 8 * g) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float dp = s[n][4 * g + e] - dl[e];
              f[n][g >> 1][4 * (g & 1) + e] = from_f32<T>(pv[e] * (F16 ? dp * gs : dp));
            }
          }
      }
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2) acc[db] = Vec<T>::mfma32(f[n][h2], tl.template col<V8>(tb + tfo, n * 32 + h2 * 16, db), acc[db]);
      win_order<NDB * NQ * 2, 2, NDB * NQ * 2 < 4 ? 2 : 4>();
    }
    __syncthreads();
    st = nst;
    if (++ci == ntq) ci = 0;
  }
  float* part = nullptr;
  if (sp > 1) {
    const int tp = (sink || a.sps == 1 ? 0 : a.nst * a.sps) + tile * sp + split;
    part = a.part + (((long)b * p.kv_heads + hk) * a.nparts + tp) * BW_KEYS * 2 * p.hd + (role ? 0 : p.hd);
  }
  T* D = role ? reinterpret_cast<T*>(a.dk) + (long)b * a.dk_bs + (long)hk * a.dk_hs
              : reinterpret_cast<T*>(a.dv) + (long)b * a.dv_bs + (long)hk * a.dv_hs;
  const long d_rs = role ? a.dk_rs : a.dv_rs;
#pragma unroll
  for (int db = 0; db < NDB; ++db) {
    const int d = db * 32 + l31;
    if (d >= p.hd) continue;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int kl = kg * 32 + (e & 3) + 8 * (e >> 2) + 4 * hi, j = ka + kl;
      const float f = role ? (F16 ? p.scale / g : HALF_P ? p.scale * 0x1p-14f : p.scale) : (SCALED ? 0x1p-14f : 1.0f);
      const float v = j < kb ? acc[db][e] * f : 0.0f;
      if (part) part[(long)kl * 2 * p.hd + d] = v;
      else if (j < kz) D[(long)j * d_rs + d] = from_f32<T>(v);
    }
  }
}

// dK / dV of the tiles whose query rows were split: one workgroup per tile, the parts are added in order
template <typename T>
__global__ __launch_bounds__(256) void win_bwd_join_kernel(const WinBwdArgs a) {
  const WinArgs& p = a.w;
  const int nts = a.sps > 1 ? a.nst : 0, ntr = a.spr > 1 ? a.nrt : 0;
  int bid = blockIdx.x;
  const int rows8 = bid % 16; bid /= 16;         // 8 keys of the tile
  const int tt = bid % (nts + ntr); bid /= (nts + ntr);
  const int hk = bid % p.kv_heads, b = bid / p.kv_heads;
  const bool sink = tt < nts;
  const int tile = sink ? tt : tt - nts, sp = sink ? a.sps : a.spr;
  const int s_end = min(p.sinks, p.Lk);
  const int ka = (sink ? 0 : s_end) + tile * BW_KEYS, kz = min(ka + BW_KEYS, sink ? s_end : p.Lk);
  const int tp = sink ? tile * sp : nts * a.sps + tile * sp;
  const float* part = a.part + (((long)b * p.kv_heads + hk) * a.nparts + tp) * BW_KEYS * 2 * p.hd;
  T* dK = reinterpret_cast<T*>(a.dk) + (long)b * a.dk_bs + (long)hk * a.dk_hs;
  T* dV = reinterpret_cast<T*>(a.dv) + (long)b * a.dv_bs + (long)hk * a.dv_hs;
  using V4 = typename Vec<T>::v4;
  const int w = 2 * p.hd, w4 = w / 4;            // four columns per thread
  for (int k = threadIdx.x; k < 8 * w4; k += 256) {
    const int r = k / w4, d = (k - r * w4) * 4, kl = rows8 * 8 + r, j = ka + kl;
    if (j >= kz) continue;
    const float* q = part + (long)kl * w + d;
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int i = 0; i < sp; ++i) s += *reinterpret_cast<const f32x4*>(q + (long)i * BW_KEYS * w);
    V4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = from_f32<T>(s[e]);
    *reinterpret_cast<V4*>(d < p.hd ? dK + (long)j * a.dk_rs + d : dV + (long)j * a.dv_rs + d - p.hd) = x;
  }
}

template <typename T, int HK>
__global__ __launch_bounds__(256, 2) void win_bwd_dq_kernel(const WinBwdArgs a) {
  using V8 = typename Vec<T>::v8;
  using V4 = typename Vec<T>::v4;
  constexpr bool F16 = std::is_same<T, _Float16>::value;
  constexpr int KB = 32, NKS = HK / 16, NDB = (HK + 31) / 32, CH = HK / 8;
  using Tile = WinTile<HK>;
  constexpr int TB = KB * Tile::PITCH, STAGE = 2 * TB;   // K | V
  constexpr int U = (KB * CH + 255) / 256;
  constexpr int AHEAD = HK > 128 || HK < 32 ? 2 : 4;     // LDS reads ahead of their MFMAs; 160 columns are at the register limit
  const WinArgs& p = a.w;
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * STAGE];
  win_lds* const lds = (win_lds*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, l31 = lane & 31;
  int bid = xcd_remap(blockIdx.x, p.batch * p.heads * p.nqb * a.spq);
  const int split = bid % a.spq;
  bid /= a.spq;
  const int qb = p.nqb - 1 - bid % p.nqb;
  bid /= p.nqb;
  const int h = bid % p.heads, b = bid / p.heads, hk = h / p.group;
  const int qn = win_len(p.q_len, b, p.Lq), kn = win_len(p.kv_len, b, p.Lk), shift = kn - qn;
  const T* K = reinterpret_cast<const T*>(p.k) + (long)b * p.k_bs + (long)hk * p.k_hs;
  const T* V = reinterpret_cast<const T*>(p.v) + (long)b * p.v_bs + (long)hk * p.v_hs;
  const int i0 = qb * 128, iw = i0 + wave * 32, row = iw + l31;
  const T* Q = reinterpret_cast<const T*>(p.q) + (long)b * p.q_bs + (long)h * p.q_hs + (long)row * p.q_rs;
  const T* G = reinterpret_cast<const T*>(a.dout) + (long)b * a.do_bs + (long)h * a.do_hs + (long)row * a.do_rs;

  V8 qf[NKS], gf[NKS];
  float gsq = 0.0f;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    const int d = ks * 16 + hi * 8;
    const bool ok = row < qn && d < p.hd;
    qf[ks] = ok ? ld8<T>(Q + d) : zero8<T>();
    gf[ks] = ok ? ld8<T>(G + d) : zero8<T>();
    if (F16)
#pragma unroll
      for (int e = 0; e < 8; ++e) { const float f = to_f32(gf[ks][e]); gsq += f * f; }
  }
  const long at = ((long)b * p.heads + h) * p.Lq + row;
  float lse = row < qn ? a.lse2[at] : __builtin_inff();
  const float delta = row < qn ? a.delta[at] : 0.0f;
  WinRange r = {0, 0, 0};
  if (i0 < qn) r = win_range(p, shift + i0, shift + min(i0 + 127, qn - 1), kn);
  float undo = p.scale;
  if (F16) {                                     // the scale of dS rides in the exponent of P
    const float* n = a.vmax + ((long)b * p.kv_heads + hk) * a.nk64;
    const float vm = wave_max(win_norm(n, r.s1, r.e1, lane, win_norm(n, 0, r.e0, lane, 0.0f)));
    const float g = ds_scale(sqrtf(win_half_sum(gsq)), vm);
    lse -= __builtin_amdgcn_logf(g);
    undo = p.scale / g;
  }
  const int n0 = (r.e0 + KB - 1) / KB, all_t = n0 + (r.e1 - r.s1 + KB - 1) / KB;
  const int tb = (int)((long)all_t * split / a.spq), nt = (int)((long)all_t * (split + 1) / a.spq);      // tiles tb .. nt - 1
  const int pw0 = shift + iw, pw1 = shift + min(iw + 31, qn - 1), pos = shift + row;
  const int vhi = p.right < 0 ? kn : min(kn, pos + p.right + 1), vlo = p.left < 0 ? 0 : pos - p.left;

  V8 kr[U], vr[U];
  unsigned ko[U], vo[U];                         // byte offsets inside a tile, and this thread's places in its LDS image
  int so[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int u = tid + 256 * i, rr = u / CH, ch = u - rr * CH;
    ko[i] = ((unsigned)rr * (unsigned)p.k_rs + ch * 8) * 2;
    vo[i] = ((unsigned)rr * (unsigned)p.v_rs + ch * 8) * 2;
    so[i] = Tile::at(rr, ch);
  }
  const bool whole = p.hd == HK;
  auto load = [&](int t) {
    const int j0 = t < n0 ? t * KB : r.s1 + (t - n0) * KB, rem = (t < n0 ? r.e0 : r.e1) - j0;
    const char* kt = reinterpret_cast<const char*>(K + (long)j0 * p.k_rs);
    const char* vt = reinterpret_cast<const char*>(V + (long)j0 * p.v_rs);
    if (rem >= KB && whole) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (KB * CH % 256 == 0 || i + 1 < U || tid + 256 * i < KB * CH) {
          kr[i] = ld8<T>(reinterpret_cast<const T*>(kt + ko[i]));
          vr[i] = ld8<T>(reinterpret_cast<const T*>(vt + vo[i]));
        }
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int u = tid + 256 * i, rr = u / CH, ch = u - rr * CH;
        const bool ok = rr < rem && rr < KB && ch * 8 < p.hd;
        kr[i] = ok ? ld8<T>(reinterpret_cast<const T*>(kt + ko[i])) : zero8<T>();
        vr[i] = ok ? ld8<T>(reinterpret_cast<const T*>(vt + vo[i])) : zero8<T>();
      }
    }
  };
  auto store = [&](int stage) {
    win_lds* const kt = lds + stage * STAGE;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (KB * CH % 256 == 0 || i + 1 < U || tid + 256 * i < KB * CH) {
        *(__attribute__((address_space(3))) V8*)(kt + so[i]) = kr[i];
        *(__attribute__((address_space(3))) V8*)(kt + TB + so[i]) = vr[i];
      }
  };
  f32x16 dq[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) dq[db][e] = 0.0f;
  const f32x16 zero16 = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  const Tile tl(lane);
  const float c = p.c;

  if (nt > tb) { load(tb); store(tb & 1); }
  win_loads_done();
  if (nt > tb + 1) load(tb + 1);
  __syncthreads();
  for (int t = tb; t < nt; ++t) {
    const int j0 = t < n0 ? t * KB : r.s1 + (t - n0) * KB, end = t < n0 ? r.e0 : r.e1;
    if (t + 1 < nt) store((t + 1) & 1);
    if (t + 2 < nt) load(t + 2);
    const win_lds* const kt = lds + (t & 1) * STAGE;
    const win_lds* const vt = kt + TB;
    const bool none = iw >= qn || (p.right >= 0 && j0 > pw1 + p.right) || (p.left >= 0 && j0 + KB <= pw0 - p.left && j0 >= p.sinks);
    if (!none) {
      f32x16 s = zero16, dp = zero16;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        s = Vec<T>::mfma32(tl.template row<V8>(kt, 0, ks), qf[ks], s);
        dp = Vec<T>::mfma32(tl.template row<V8>(vt, 0, ks), gf[ks], dp);
      }
      win_order<2 * NKS, 1, AHEAD>();
      const bool all = end - j0 >= KB && (p.right < 0 || j0 + KB - 1 <= pw0 + p.right) &&
                       (p.left < 0 || j0 >= pw1 - p.left || j0 + KB <= p.sinks);
      const int lhi = min(vhi, end);
      V8 df[2];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float pv = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -lse));
        if (!all) {
          const int j = j0 + (e & 3) + 8 * (e >> 2) + 4 * hi;
          pv = j < lhi && (j >= vlo || j < p.sinks) ? pv : 0.0f;
        }
        df[e >> 3][e & 7] = from_f32<T>(pv * (dp[e] - delta));
      }
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) dq[db] = Vec<T>::mfma32(tl.template col<V8>(kt, h2 * 16, db), df[h2], dq[db]);
      win_order<NDB * 2, 2, (AHEAD < NDB * 2 ? AHEAD : NDB * 2)>();
    }
    __syncthreads();
  }
  if (row >= p.Lq) return;
  if (a.spq > 1) {
    float* part = a.qpart + (at * a.spq + split) * p.hd;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = db * 32 + 8 * g + 4 * hi;
        if (d < p.hd)
          *reinterpret_cast<f32x4*>(part + d) = row < qn ? f32x4{dq[db][4 * g] * undo, dq[db][4 * g + 1] * undo, dq[db][4 * g + 2] * undo, dq[db][4 * g + 3] * undo}
                                                        : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    return;
  }
  T* O = reinterpret_cast<T*>(a.dq) + (long)b * a.dq_bs + (long)h * a.dq_hs + (long)row * a.dq_rs;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + 8 * g + 4 * hi;
      if (d < p.hd) {
        V4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = from_f32<T>(row < qn ? dq[db][4 * g + e] * undo : 0.0f);
        *reinterpret_cast<V4*>(O + d) = w;
      }
    }
}

// dq of the query rows whose keys were split: 4 columns per thread, the parts are added in order
template <typename T>
__global__ __launch_bounds__(256) void win_bwd_join_q_kernel(const WinBwdArgs a) {
  using V4 = typename Vec<T>::v4;
  const WinArgs& p = a.w;
  const int per = p.hd / 4;
  const long k = (long)blockIdx.x * 256 + threadIdx.x, at = k / per;
  const int d = (int)(k - at * per) * 4;
  if (at >= (long)p.batch * p.heads * p.Lq) return;
  const float* part = a.qpart + at * a.spq * p.hd + d;
  f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int i = 0; i < a.spq; ++i) s += *reinterpret_cast<const f32x4*>(part + (long)i * p.hd);
  const long bh = at / p.Lq;
  const int i = (int)(at - bh * p.Lq), h = (int)(bh % p.heads), b = (int)(bh / p.heads);
  V4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = from_f32<T>(s[e]);
  *reinterpret_cast<V4*>(reinterpret_cast<T*>(a.dq) + (long)b * a.dq_bs + (long)h * a.dq_hs + (long)i * a.dq_rs + d) = w;
}

// Key tiles and query splits.  A sink tile meets every query, a tile of the rest at most left + right + 128 of them, one of a triangle half
// as many on average, and there may be fewer tiles than the chip takes at once (two workgroups per CU up to 64 columns, else one): queries
// are split so that a workgroup has at most `target` steps of 32 query rows (about 1 us each), with the least of
//   one round: the longest workgroup;   more: all steps / slots + a quarter of the longest (the longest go first),
// a workgroup counting 8 steps more than it has and, with parts to write and to join, 20 (13 where all write at once).  Measured, dkv and
// join: 2 x 2048 causal, 32 / 8 heads of 128, whole / two parts 262 / 177 us; 5 x 7047 without a left edge, 8 heads on one of 128, whole /
// five parts 1765 / 740 us; 5 x 972, 8 / 4 heads of 80, whole / two / three parts 65 / 47 / 53 us; 4 x 1024, 12 heads of
// 64, whole / two parts 44 / 48 us.
int64_t plan_bwd(WinBwdArgs& a) {
  WinArgs& p = a.w;
  p.nqb = (p.Lq + 127) / 128;
  if (p.left < 0) p.sinks = 0;                   // everything up to the right edge is visible anyway
  const int s_end = p.sinks < p.Lk ? p.sinks : p.Lk;
  a.nst = (s_end + BW_KEYS - 1) / BW_KEYS;
  a.nrt = (p.Lk - s_end + BW_KEYS - 1) / BW_KEYS;
  a.nq64 = (p.Lq + 63) / 64;
  a.nk64 = (p.Lk + 63) / 64;
  const long bh = (long)p.batch * p.kv_heads, slots = p.hd <= 64 ? 512 : 256;
  long span = p.Lq;
  if (p.left >= 0 && p.right >= 0 && (long)p.left + p.right + BW_KEYS < span) span = (long)p.left + p.right + BW_KEYS;
  const long it_s = (long)p.group * ((p.Lq + 31) / 32), it_r = (long)p.group * ((span + 31) / 32);
  const auto parts = [](long its, long target) { const long n = (its + target - 1) / target; return n < 1 ? 1L : n; };
  long sum = 0, seen = 0;                        // mean span over up to 64 tiles
  const long shift = (long)p.Lk - p.Lq;
  for (long t = 0, dt = a.nrt / 64 + 1; t < a.nrt; t += dt, ++seen) {
    const long ka = s_end + t * BW_KEYS, kb = ka + BW_KEYS < p.Lk ? ka + BW_KEYS : p.Lk;
    const long ia = p.right < 0 ? 0 : ka - p.right - shift, ib = p.left < 0 ? p.Lq : kb + p.left - shift;
    const long n = (ib < p.Lq ? ib : p.Lq) - (ia > 0 ? ia : 0);
    sum += n > 0 ? n : 0;
  }
  const double all = bh * ((double)a.nst * it_s + (seen ? (double)a.nrt * p.group * sum / (32.0 * seen) : 0.0));
  const long most = a.nst && it_s > it_r ? it_s : it_r;
  long target = most;
  double best = 1e300;
  for (long t = 8;; t += (t + 7) / 8) {
    const long ns = parts(it_s, t), nr = parts(it_r, t), wgs = bh * (a.nst * ns + a.nrt * nr), longest = t < most ? t : most;
    const bool joined = (a.nst && ns > 1) || nr > 1;
    const double extra = joined ? 20.0 : 8.0;
    const double cost = wgs <= slots ? longest + (joined ? 13.0 : 8.0) : (all + wgs * extra) / slots + (longest + extra) / 4;
    if (cost < best) { best = cost; target = t; }
    if (t >= most) break;
  }
  a.sps = a.nst ? (int)parts(it_s, target) : 1;
  a.spr = a.nrt ? (int)parts(it_r, target) : 1;
  // dq: few queries leave CUs idle, then the keys are split (up to 64 columns four workgroups per CU, else two, at least 8 tiles of 32 keys
  // each; 6 x 190 x 3062, 28 heads of 40: 112 -> 61 us and 5 for the join)
  long keys = p.Lk;
  if (p.left >= 0 && p.right >= 0 && (long)p.left + p.right + p.Lq + p.sinks < keys) keys = (long)p.left + p.right + p.Lq + p.sinks;
  const long blocks = (long)p.batch * p.heads * p.nqb, tiles = (keys + 31) / 32;
  const long want = p.hd <= 64 ? 1024 : 512;
  long sq = blocks > 0 && blocks < want / 2 ? want / blocks : 1;
  if (sq > tiles / 8) sq = tiles / 8;
  a.spq = sq < 1 ? 1 : (int)sq;
  a.nparts = (a.sps > 1 ? a.nst * a.sps : 0) + (a.spr > 1 ? a.nrt * a.spr : 0);
  const int64_t rows = (int64_t)p.batch * p.heads * p.Lq;
  int64_t at = 0;
  const auto take = [&](int64_t floats) { const int64_t o = at; at += (floats + 3) / 4 * 4; return o; };
  float* base = a.part;
  a.delta = base + take(rows);
  a.lse2 = base + take(rows);
  a.domax = base + take((int64_t)p.batch * p.heads * a.nq64);
  a.vmax = base + take(bh * a.nk64);
  a.part = base + take(bh * a.nparts * BW_KEYS * 2 * p.hd);
  a.qpart = base + take(a.spq > 1 ? rows * a.spq * p.hd : 0);
  return at * 4;
}

template <typename T, int HK>
int launch_hk(const WinBwdArgs& a, hipStream_t st) {
  const WinArgs& p = a.w;
  const long tiles = (long)p.batch * p.kv_heads * (a.nst * a.sps + a.nrt * a.spr);
  if (tiles > 0) {
    hipLaunchKernelGGL((win_bwd_dkv_kernel<T, HK>), dim3((unsigned)tiles), dim3(512), 0, st, a);
    HALLO_CHECK_LAUNCH();
  }
  if (p.Lq > 0) {
    hipLaunchKernelGGL((win_bwd_dq_kernel<T, HK>), dim3((unsigned)(p.batch * p.heads * p.nqb * a.spq)), dim3(256), 0, st, a);
    HALLO_CHECK_LAUNCH();
  }
  return 0;
}

template <typename T>
int launch(const WinBwdArgs& a, hipStream_t st) {
  const WinArgs& p = a.w;
  const bool f16 = std::is_same<T, _Float16>::value;
  const long qblocks = (long)p.batch * p.heads * a.nq64, kblocks = f16 ? (long)p.batch * p.kv_heads * a.nk64 : 0;
  if (qblocks + kblocks > 0) {
    if (p.hd <= 128) hipLaunchKernelGGL((win_bwd_prep_kernel<T, 1>), dim3((unsigned)(qblocks + kblocks)), dim3(256), 0, st, a, (int)qblocks);
    else hipLaunchKernelGGL((win_bwd_prep_kernel<T, 2>), dim3((unsigned)(qblocks + kblocks)), dim3(256), 0, st, a, (int)qblocks);
    HALLO_CHECK_LAUNCH();
  }
  int rc;
  switch ((p.hd + 15) / 16) {
    case 1: rc = launch_hk<T, 16>(a, st); break;
    case 2: rc = launch_hk<T, 32>(a, st); break;
    case 3: rc = launch_hk<T, 48>(a, st); break;
    case 4: rc = launch_hk<T, 64>(a, st); break;
    case 5: rc = launch_hk<T, 80>(a, st); break;
    case 6: rc = launch_hk<T, 96>(a, st); break;
    case 7: rc = launch_hk<T, 112>(a, st); break;
    case 8: rc = launch_hk<T, 128>(a, st); break;
    case 9: rc = launch_hk<T, 144>(a, st); break;
    default: rc = launch_hk<T, 160>(a, st);
  }
  if (rc) return rc;
  const long nj = (long)p.batch * p.kv_heads * ((a.sps > 1 ? a.nst : 0) + (a.spr > 1 ? a.nrt : 0)) * 16;
  if (nj > 0) {
    hipLaunchKernelGGL((win_bwd_join_kernel<T>), dim3((unsigned)nj), dim3(256), 0, st, a);
    HALLO_CHECK_LAUNCH();
  }
  if (a.spq > 1) {
    const long n = (long)p.batch * p.heads * p.Lq * (p.hd / 4);
    hipLaunchKernelGGL((win_bwd_join_q_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
    HALLO_CHECK_LAUNCH();
  }
  return 0;
}

bool bwd_args(const hallo_window_attn_bwd_desc* d, WinBwdArgs& a) {
  a = WinBwdArgs{};
  if (!d || !win_args(&d->fwd, a.w)) return false;
  const int64_t strides[] = {d->do_bs, d->do_rs, d->do_hs, d->dq_bs, d->dq_rs, d->dq_hs, d->dk_bs, d->dk_rs, d->dk_hs, d->dv_bs, d->dv_rs, d->dv_hs};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return false;
  const int64_t row_strides[] = {d->do_rs, d->dq_rs, d->dk_rs, d->dv_rs};
  for (int64_t s : row_strides)
    if (s > WIN_MAX_STRIDE) return false;
  const void* ptrs[] = {d->dout, d->dq, d->dk, d->dv};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) & 15) return false;
  a.dout = d->dout; a.dq = d->dq; a.dk = d->dk; a.dv = d->dv;
  a.do_bs = d->do_bs; a.do_rs = d->do_rs; a.do_hs = d->do_hs; a.dq_bs = d->dq_bs; a.dq_rs = d->dq_rs; a.dq_hs = d->dq_hs;
  a.dk_bs = d->dk_bs; a.dk_rs = d->dk_rs; a.dk_hs = d->dk_hs; a.dv_bs = d->dv_bs; a.dv_rs = d->dv_rs; a.dv_hs = d->dv_hs;
  return true;
}

}  // namespace
}  // namespace hallo

extern "C" int64_t hallo_window_attention_backward_workspace(const hallo_window_attn_bwd_desc* d) {
  using namespace hallo;
  WinBwdArgs a;
  if (!bwd_args(d, a)) return -22;
  if (a.w.batch == 0) return 0;
  return plan_bwd(a);
}

extern "C" int hallo_window_attention_backward(const hallo_window_attn_bwd_desc* d, void* stream) {
  using namespace hallo;
  WinBwdArgs a;
  if (!bwd_args(d, a)) return -22;
  const WinArgs& p = a.w;
  if (p.batch == 0 || (p.Lq == 0 && p.Lk == 0)) return 0;
  if (p.Lq > 0 && (!p.q || !p.o || !p.lse || !a.dout || !a.dq)) return -22;
  if (p.Lk > 0 && (!p.k || !p.v || !a.dk || !a.dv)) return -22;
  const int64_t need = hallo_window_attention_backward_workspace(d);
  if (need > 0 && (!d->fwd.workspace || d->fwd.workspace_bytes < need || (reinterpret_cast<uintptr_t>(d->fwd.workspace) & 15))) return -22;
  a.part = (float*)d->fwd.workspace;
  plan_bwd(a);
  if ((int64_t)p.batch * p.kv_heads * ((int64_t)a.nst * a.sps + (int64_t)a.nrt * a.spr) * 16 > 0x7fffffff) return -22;
  return d->fwd.dtype == DT_F16 ? launch<_Float16>(a, (hipStream_t)stream) : launch<__bf16>(a, (hipStream_t)stream);
}
