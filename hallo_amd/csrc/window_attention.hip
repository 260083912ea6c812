// Attention with a sliding window and always-visible first keys, shared key heads and per-entry lengths: forward pass.
//
// Two forms.  `win_fwd_kernel` takes 128 queries of one head per workgroup (a wave owns 32) and walks the keys those queries see; K and
// V tiles go global -> registers -> LDS one tile ahead of the MFMAs.  `win_split_kernel` is for few queries (single tokens against a
// cache, prompts of few heads): the query rows of the heads that share a key head are packed into 32-row blocks, the keys are split over
// workgroups and over the waves of each, and `win_join_kernel` joins the parts.
//
// Both contractions run in swapped form, so a lane owns a query and the softmax statistics are lane-local:
//   S^T[key, q] = K[key, :] . Q[q, :]      A = K rows from LDS, B = Q fragments in registers
//   O^T[d, q]   = V^T[d, :] . P^T[:, q]    A = V read transposed from LDS, B = P as the first product left it
// The running maximum moves only when a score exceeds it by more than 6 (log2 units, so P <= 64 and the row sum stays far inside
// fp32).  P is rounded to the storage type for the second product only, because the matrix cores take 16-bit operands at the rate that
// this kernel lives on; the row sum adds the unrounded values, so a rounding is a relative error of half a step in one weight (on random
// inputs the output's error against 64 bits is 1.3 to 1.4 times that of rounding the exact output once).  fp16's
// smallest number would make it more than that: thousands of weights below 2^-25 of the largest one would be in the sum and not in the
// product.  P therefore carries a power of two that rides in the exponent and leaves with the division by the sum (fp16, win_fwd_kernel:
// 2^9, 64 * 2^9 is half of fp16's range; win_split_kernel, whose P is at most 1: 2^14; bf16 has fp32's range: none).
//
// What bounds them: win_fwd_kernel the SIMDs' issue -- MFMA and vector time (exponentials, maxima, sums, conversions) add up rather than
// overlap, 39 + 39 % of all cycles at 128 columns, 41 + 50 % at 80, the LDS port 30 - 35 % busy.  2 x 8192 tokens, 32 / 8 heads of 128,
// window 4096, bf16: 0.96 ms, 860 TFLOP/s; 2 x 16384 tokens, 8 heads of 80, 4097 + 1024 keys a token, fp16: 0.55 - 0.57 ms, 710 - 690 TFLOP/s
// (the second product multiplies 96 columns for 80, 64 for 40, and 16 % of the LDS cycles are conflicts there; 128 columns: none).
// win_split_kernel the bytes of K and V: 32 streams, 16 k window, 8 key heads of 128: 0.36 ms, 5.7 TB/s; 8 key heads of 160, 16 k keys,
// one workgroup per CU: 0.475 ms, 5.65 TB/s.
#include <type_traits>
#include "window_args.h"
#include "../../include/hallo_amd.h"

namespace hallo {

namespace {

constexpr float FWD_P_EXP = 9.0f, SPLIT_P_EXP = 14.0f;       // fp16: exponent of the power of two that P carries

// What the exponents of a row count from: its running maximum in log2 units, less X.  fp16: one step above, so that a rounding of a score
// near 10^8, where a step is 8, cannot take 2^X over the type's range (1.125 * 2^-24 of a number is 0.56 to 1.13 of its step).
template <typename T> __device__ __forceinline__ float win_base(float m, float c, float X) {
  const float b = (m == -__builtin_inff() ? 0.0f : m * c) - X;
  return std::is_same<T, _Float16>::value ? __builtin_fmaf(fabsf(b), 0x1.2p-24f, b) : b;
}

template <typename T, int HK>
__global__ __launch_bounds__(256, 2) void win_fwd_kernel(const WinArgs p) {
  using V8 = typename Vec<T>::v8;
  using V4 = typename Vec<T>::v4;
  constexpr int KB = HK > 128 ? 32 : 64;         // keys per tile
  constexpr int NT = KB / 32, NKS = HK / 16, NDB = (HK + 31) / 32, CH = HK / 8;
  using Tile = WinTile<HK>;
  constexpr int TB = KB * Tile::PITCH, STAGE = 2 * TB;   // K | V
  constexpr int U = (KB * CH + 255) / 256;       // 16-byte pieces per thread and tensor
  constexpr bool F16 = std::is_same<T, _Float16>::value;
  constexpr float NEG_INF = -__builtin_inff(), X = F16 ? FWD_P_EXP : 0.0f;
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * STAGE];
  win_lds* const lds = (win_lds*)smem;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, l31 = lane & 31;
  // the blocks of a key head stay in one XCD's L2, the heads that share it side by side
  int bid = xcd_remap(blockIdx.x, p.batch * p.heads * p.nqb);
  const int gh = bid % p.group;
  bid /= p.group;
  const int qb = p.nqb - 1 - bid % p.nqb;        // causal masks: the blocks with the most keys first
  bid /= p.nqb;
  const int hk = bid % p.kv_heads, b = bid / p.kv_heads, h = hk * p.group + gh;
  const int qn = win_len(p.q_len, b, p.Lq), kn = win_len(p.kv_len, b, p.Lk);
  const T* Q = reinterpret_cast<const T*>(p.q) + (long)b * p.q_bs + (long)h * p.q_hs;
  const T* K = reinterpret_cast<const T*>(p.k) + (long)b * p.k_bs + (long)hk * p.k_hs;
  const T* V = reinterpret_cast<const T*>(p.v) + (long)b * p.v_bs + (long)hk * p.v_hs;
  const int i0 = qb * 128, iw = i0 + wave * 32, row = iw + l31;
  const int shift = kn - qn;                     // position of query 0

  V8 qf[NKS];
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    const int d = ks * 16 + hi * 8;
    qf[ks] = row < qn && d < p.hd ? ld8<T>(Q + (long)row * p.q_rs + d) : zero8<T>();
  }

  WinRange r = {0, 0, 0};
  if (i0 < qn) r = win_range(p, shift + i0, shift + min(i0 + 127, qn - 1), kn);
  const int n0 = (r.e0 + KB - 1) / KB, nt = n0 + (r.e1 - r.s1 + KB - 1) / KB;
  // this wave's positions and this lane's visible keys
  const int pw0 = shift + iw, pw1 = shift + min(iw + 31, qn - 1), pos = shift + row;
  const int vhi = p.right < 0 ? kn : min(kn, pos + p.right + 1), vlo = p.left < 0 ? 0 : pos - p.left;

  V8 kr[U], vr[U];
  unsigned ko[U], vo[U];                         // byte offsets inside a tile (row strides are at most WIN_MAX_STRIDE)
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int u = tid + 256 * i, rr = u / CH, ch = u - rr * CH;
    ko[i] = ((unsigned)rr * (unsigned)p.k_rs + ch * 8) * 2;
    vo[i] = ((unsigned)rr * (unsigned)p.v_rs + ch * 8) * 2;
  }
  const bool whole = p.hd == HK;
  auto load = [&](int t) {
    const int j0 = t < n0 ? t * KB : r.s1 + (t - n0) * KB, rem = (t < n0 ? r.e0 : r.e1) - j0;
    const char* kt = reinterpret_cast<const char*>(K + (long)j0 * p.k_rs);
    const char* vt = reinterpret_cast<const char*>(V + (long)j0 * p.v_rs);
    if (rem >= KB && whole) {                    // vector instructions do not overlap with the MFMAs here: no masks where none are needed
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
        const bool ok = rr < rem && rr < KB && ch * 8 < p.hd;        // rows past the range hold anything: they enter the products as zeros
        kr[i] = ok ? ld8<T>(reinterpret_cast<const T*>(kt + ko[i])) : zero8<T>();
        vr[i] = ok ? ld8<T>(reinterpret_cast<const T*>(vt + vo[i])) : zero8<T>();
      }
    }
  };
  int so[U];                                     // this thread's places in a tile
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int u = tid + 256 * i, rr = u / CH;
    so[i] = Tile::at(rr, u - rr * CH);
  }
  auto store = [&](int stage) {
    win_lds* const kt = lds + stage * STAGE;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (KB * CH % 256 == 0 || i + 1 < U || tid + 256 * i < KB * CH) {
        *(__attribute__((address_space(3))) V8*)(kt + so[i]) = kr[i];
        *(__attribute__((address_space(3))) V8*)(kt + TB + so[i]) = vr[i];
      }
  };

  f32x16 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.0f;
  float m = NEG_INF, l = 0.0f;
  const float c = p.c, slack = 6.0f / p.c;
  const f32x16 zero16 = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  const Tile tl(lane);

  if (nt > 0) { load(0); store(0); }
  win_loads_done();
  if (nt > 1) load(1);
  __syncthreads();
  auto step = [&](auto odd, int t) {             // odd = t & 1
    const int P = odd;
    const int j0 = t < n0 ? t * KB : r.s1 + (t - n0) * KB, end = t < n0 ? r.e0 : r.e1;
    if (t + 1 < nt) store(1 - P);                // read last in iteration t - 1, which the barrier below closed
    if (t + 2 < nt) load(t + 2);
    const win_lds* const kt = lds + P * STAGE;
    const win_lds* const vt = kt + TB;
    const bool none = iw >= qn || (p.right >= 0 && j0 > pw1 + p.right) || (p.left >= 0 && j0 + KB <= pw0 - p.left && j0 >= p.sinks);
    if (!none) {
      f32x16 s[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[n] = zero16;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
          s[n] = Vec<T>::mfma32(tl.template row<V8>(kt, n * 32, ks), qf[ks], s[n]);
      }
      win_order<NT * NKS, 1, NKS < 4 ? NKS : 4>();
      const bool all = end - j0 >= KB && (p.right < 0 || j0 + KB - 1 <= pw0 + p.right) &&
                       (p.left < 0 || j0 >= pw1 - p.left || j0 + KB <= p.sinks);
      if (!all) {
        const int lhi = min(vhi, end);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int j = j0 + n * 32 + (e & 3) + 8 * (e >> 2) + 4 * hi;
            s[n][e] = j < lhi && (j >= vlo || j < p.sinks) ? s[n][e] : NEG_INF;
          }
      }
      float mx[4] = {NEG_INF, NEG_INF, NEG_INF, NEG_INF};    // four chains: a dependent chain of 32 would be latency
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 16; e += 2) mx[e / 2 & 3] = fmaxf(fmaxf(s[n][e], s[n][e + 1]), mx[e / 2 & 3]);
      const float mt = win_half_max(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
      if (__any(mt > m + slack)) {
        const float mn = fmaxf(m, mt);
        const float a = m == mn ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);     // m = -inf: 0
        m = mn;
        l *= a;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[db][e] *= a;
      }
      const float mc = win_base<T>(m, c, X);
      V8 pf[NT][2];
      float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float pv = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][e], c, -mc));
          ls[e & 3] += pv;
          pf[n][e >> 3][e & 7] = from_f32<T>(pv);
        }
      l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2)
            o[db] = Vec<T>::mfma32(tl.template col<V8>(vt, n * 32 + h2 * 16, db), pf[n][h2], o[db]);
      win_order<NDB * NT * 2, 2, NDB * NT * 2 < 4 ? 2 : 4>();
    }
    __syncthreads();
  };
  if constexpr (HK > 96 && HK <= 128) {          // at the register limit, where two copies of the step cost hipcc its order of the LDS reads
    for (int t = 0; t < nt; ++t) step(t & 1, t);
  } else {                                       // the stage as part of the instructions: 2 - 4 % at 64, 80 and 160 columns
    int t = 0;
    for (; t + 1 < nt; t += 2) {
      step(std::integral_constant<int, 0>{}, t);
      step(std::integral_constant<int, 1>{}, t + 1);
    }
    if (t < nt) step(std::integral_constant<int, 0>{}, t);
  }

  l = win_half_sum(l);
  if (row >= p.Lq) return;
  const bool some = row < qn && l > 0.0f;
  // a NaN sum stays NaN
  const float inv = some ? 1.0f / l : (l != l && row < qn ? l : 0.0f);
  if (p.lse && hi == 0)
    p.lse[((long)b * p.heads + h) * p.Lq + row] = some ? ((F16 ? win_base<T>(m, c, X) : m * c) + __builtin_amdgcn_logf(l)) * 0.69314718055994530942f : (inv != 0.0f ? inv : NEG_INF);
  T* O = reinterpret_cast<T*>(p.o) + (long)b * p.o_bs + (long)h * p.o_hs + (long)row * p.o_rs;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + 8 * g + 4 * hi;
      if (d < p.hd) {
        V4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = from_f32<T>(inv == 0.0f ? 0.0f : o[db][4 * g + e] * inv);
        *reinterpret_cast<V4*>(O + d) = w;
      }
    }
}

// ------------------------------------------------------------------------------------------------------------------------------
// Few queries.  Packed row r is query r % Lp of head hk * group + r / Lp: Lp = Lq up to 32 queries (a block of 32 rows holds several heads),
// else the next multiple of 32 (a block over a head's end would walk the keys of all queries).  Bound by the bytes of K and V: a wave reads 32 keys
// at a time, whole rows by neighbouring lanes, into LDS tiles of its own (no barrier), the next 32 keys in flight under the products; the
// four waves take every fourth tile of the split and join through LDS.
// ------------------------------------------------------------------------------------------------------------------------------
template <typename T, int HK>
__global__ __launch_bounds__(256, 2) void win_split_kernel(const WinArgs p) {
  using V8 = typename Vec<T>::v8;
  constexpr int NKS = HK / 16, NDB = (HK + 31) / 32, OP = HK + 4;      // OP: pitch of the joined rows, floats
  constexpr bool F16 = std::is_same<T, _Float16>::value;
  constexpr float NEG_INF = -__builtin_inff(), X = F16 ? SPLIT_P_EXP : 0.0f;
  using Tile = WinTile<HK, HK == 112 || HK == 128 ? 16 : win_chunks(HK)>;      // eight tiles of a workgroup: two workgroups per CU at 128 columns
  constexpr int TB = 32 * Tile::PITCH, WT = 4 * 2 * TB, JT = 32 * OP * 4;      // LDS: K | V of every wave, then the joined rows
  __shared__ __attribute__((aligned(16))) unsigned char smem[WT > JT ? WT : JT];
  __shared__ float sm_m[4][32], sm_l[4][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, l31 = lane & 31;
  int bid = blockIdx.x;
  const int split = bid % p.nsplit; bid /= p.nsplit;
  const int hk = bid % p.kv_heads; bid /= p.kv_heads;
  const int b = bid % p.batch, rb = p.nrb - 1 - bid / p.batch;         // causal masks: the row blocks with the most keys first
  const int qn = win_len(p.q_len, b, p.Lq), kn = win_len(p.kv_len, b, p.Lk), shift = kn - qn;
  const int rows = p.group * p.Lp, r = rb * 32 + l31, gh = r / p.Lp, i = r - gh * p.Lp;
  const bool live = r < rows && i < qn;
  const T* K = reinterpret_cast<const T*>(p.k) + (long)b * p.k_bs + (long)hk * p.k_hs;
  const T* V = reinterpret_cast<const T*>(p.v) + (long)b * p.v_bs + (long)hk * p.v_hs;
  const T* Qr = reinterpret_cast<const T*>(p.q) + (long)b * p.q_bs + (long)(hk * p.group + gh) * p.q_hs + (long)i * p.q_rs;
  V8 qf[NKS];
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    const int d = ks * 16 + hi * 8;
    qf[ks] = live && d < p.hd ? ld8<T>(Qr + d) : zero8<T>();
  }
  // the queries of this block: all of them once it reaches over a head's end
  const int last = min(rb * 32 + 31, rows - 1);
  const bool one = rb * 32 / p.Lp == last / p.Lp;
  const int ilo = one ? rb * 32 % p.Lp : 0, ihi = min(one ? last % p.Lp : p.Lp - 1, qn - 1);
  WinRange w = {0, 0, 0};
  if (ihi >= ilo) w = win_range(p, shift + ilo, shift + ihi, kn);
  const int n0 = (w.e0 + 31) / 32, nt = n0 + (w.e1 - w.s1 + 31) / 32;
  const int tb = (int)((long)nt * split / p.nsplit), te = (int)((long)nt * (split + 1) / p.nsplit);
  const int pos = shift + i;
  const int vhi = !live ? 0 : (p.right < 0 ? kn : min(kn, pos + p.right + 1)), vlo = p.left < 0 ? 0 : pos - p.left;
  const int plo = shift + ilo, phi = shift + ihi;

  // lanes along the rows: a load instruction takes whole rows (HK = 128: four rows of 256 bytes)
  constexpr int CH = HK / 8, U = CH / 2;
  V8 kr[U], vr[U];
  auto load = [&](int t) {
    const int j0 = t < n0 ? t * 32 : w.s1 + (t - n0) * 32, rem = (t < n0 ? w.e0 : w.e1) - j0;
    const T* kt = K + (long)j0 * p.k_rs;
    const T* vt = V + (long)j0 * p.v_rs;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      // 64 % CH == 0: the same lane offset for every i, the rest is uniform
      const int u = 64 % CH ? lane + 64 * i : lane, r0 = 64 % CH ? 0 : 64 / CH * i, rr = u / CH, ch = u - rr * CH;
      const bool ok = rr + r0 < rem && ch * 8 < p.hd;
      kr[i] = ok ? ld8<T>(kt + (long)r0 * p.k_rs + ((unsigned)rr * (unsigned)p.k_rs + ch * 8)) : zero8<T>();
      vr[i] = ok ? ld8<T>(vt + (long)r0 * p.v_rs + ((unsigned)rr * (unsigned)p.v_rs + ch * 8)) : zero8<T>();
    }
  };
  f32x16 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.0f;
  const float c = p.c;
  float m = NEG_INF, mc = win_base<T>(m, c, X), l = 0.0f;
  win_lds* const kt = (win_lds*)smem + wave * 2 * TB;
  win_lds* const vt = kt + TB;
  const Tile tl(lane);

  int t = tb + wave;
  win_loads_done();
  if (t < te) load(t);
  for (; t < te; t += 4) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = lane + 64 * i, rr = u / CH, ch = u - rr * CH;
      *(__attribute__((address_space(3))) V8*)(kt + Tile::at(rr, ch)) = kr[i];
      *(__attribute__((address_space(3))) V8*)(vt + Tile::at(rr, ch)) = vr[i];
    }
    wave_lds_order();
    if (t + 4 < te) load(t + 4);
    f32x16 s = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) s = Vec<T>::mfma32(tl.template row<V8>(kt, 0, ks), qf[ks], s);
    const int j0 = t < n0 ? t * 32 : w.s1 + (t - n0) * 32, end = t < n0 ? w.e0 : w.e1;
    const bool all = end - j0 >= 32 && (p.right < 0 || j0 + 31 <= plo + p.right) && (p.left < 0 || j0 >= phi - p.left || j0 + 32 <= p.sinks);
    if (!all) {
      const int lhi = min(vhi, end);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int j = j0 + (e & 3) + 8 * (e >> 2) + 4 * hi;
        s[e] = j < lhi && (j >= vlo || j < p.sinks) ? s[e] : NEG_INF;
      }
    }
    float mt = NEG_INF;
#pragma unroll
    for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[e]);
    mt = win_half_max(mt);
    if (__any(mt > m)) {
      const float mn = fmaxf(m, mt);
      const float a = m == mn ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      mc = win_base<T>(m, c, X);
      l *= a;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[db][e] *= a;
    }
    V8 pf[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float pv = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -mc));
      l += pv;
      pf[e >> 3][e & 7] = from_f32<T>(pv);
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) o[db] = Vec<T>::mfma32(tl.template col<V8>(vt, h2 * 16, db), pf[h2], o[db]);
    wave_lds_order();
  }
  // what P carried (fp16), to the bit: from here on sums and rows count from m itself
  const float undo = F16 && m != NEG_INF ? __builtin_amdgcn_exp2f(-__builtin_fmaf(m, c, -mc)) : 1.0f;
  l = win_half_sum(l) * undo;
  if (!live) { m = NEG_INF; l = 0.0f; }          // rows without a query went along in the tiles that need no mask
  if (hi == 0) { sm_m[wave][l31] = m; sm_l[wave][l31] = l; }
  __syncthreads();                               // also: every wave is done with its V tile, the joined rows take its place
  const float M = fmaxf(fmaxf(sm_m[0][l31], sm_m[1][l31]), fmaxf(sm_m[2][l31], sm_m[3][l31]));
  const float f = undo * (m == M ? 1.0f : __builtin_amdgcn_exp2f((m - M) * c));       // this wave's share (a wave without a visible key: o = 0)
  float* const jt = reinterpret_cast<float*>(smem);
  for (int w4 = 0; w4 < 4; ++w4) {
    if (wave == w4) {
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = db * 32 + 8 * g + 4 * hi;
          if (d < HK) {
            f32x4* a = reinterpret_cast<f32x4*>(jt + l31 * OP + d);
            f32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = live ? o[db][4 * g + e] * f : 0.0f;
            if (w4) x += *a;
            *a = x;
          }
        }
    }
    __syncthreads();
  }
  // thread -> (row, 32 threads' stride over the columns)
  const int rr = tid >> 3, cc = tid & 7, R = rb * 32 + rr;
  float Mr = NEG_INF, Lr = 0.0f;
#pragma unroll
  for (int w4 = 0; w4 < 4; ++w4) Mr = fmaxf(Mr, sm_m[w4][rr]);
#pragma unroll
  for (int w4 = 0; w4 < 4; ++w4) Lr += sm_l[w4][rr] * (sm_m[w4][rr] == Mr ? 1.0f : __builtin_amdgcn_exp2f((sm_m[w4][rr] - Mr) * c));
  const int gr = R / p.Lp, ir = R - gr * p.Lp, h = hk * p.group + gr;
  if (R >= rows || ir >= p.Lq) return;
  if (p.nsplit > 1) {
    float* part = p.part + (((long)(b * p.kv_heads + hk) * p.nrb + rb) * p.nsplit + split) * 32 * (p.hd + 2) + rr * (p.hd + 2);
    for (int d = cc; d < p.hd; d += 8) part[2 + d] = jt[rr * OP + d];
    if (cc == 0) { part[0] = Mr; part[1] = Lr; }
    return;
  }
  const float inv = Lr > 0.0f ? 1.0f / Lr : (Lr != Lr ? Lr : 0.0f);
  T* O = reinterpret_cast<T*>(p.o) + (long)b * p.o_bs + (long)h * p.o_hs + (long)ir * p.o_rs;
  for (int d = cc * 8; d < p.hd; d += 64) {
    V8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = from_f32<T>(inv == 0.0f ? 0.0f : jt[rr * OP + d + e] * inv);
    st8<T>(O + d, x);
  }
  if (p.lse && cc == 0)
    p.lse[((long)b * p.heads + h) * p.Lq + ir] = Lr > 0.0f ? (Mr * c + __builtin_amdgcn_logf(Lr)) * 0.69314718055994530942f : (inv != 0.0f ? inv : NEG_INF);
}

// one wave per query row: joins the parts of its key splits.  The splits' shares are computed side by side by the lanes, so that the loop
// over the parts is loads that do not wait for one another.
constexpr int WIN_MAX_SPLIT = 512;
template <typename T>
__global__ __launch_bounds__(256) void win_join_kernel(const WinArgs p) {
  __shared__ float share[4][WIN_MAX_SPLIT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rows = p.group * p.Lq;
  const long id = (long)blockIdx.x * 4 + wave;
  if (id >= (long)p.batch * p.kv_heads * rows) return;
  const int row = (int)(id % rows), gr = row / p.Lq, i = row - gr * p.Lq, R = gr * p.Lp + i;
  const long bh = id / rows;
  const int hk = (int)(bh % p.kv_heads), b = (int)(bh / p.kv_heads);
  const int step = 32 * (p.hd + 2);
  const float* part = p.part + (bh * p.nrb + R / 32) * p.nsplit * step + (R % 32) * (p.hd + 2);
  float M = -__builtin_inff();
  for (int s = lane; s < p.nsplit; s += 64) M = fmaxf(M, part[(long)s * step]);
  M = wave_max(M);
  float L = 0.0f;
  for (int s = lane; s < p.nsplit; s += 64) {
    const float m = part[(long)s * step], f = m == M ? 1.0f : __builtin_amdgcn_exp2f((m - M) * p.c);
    share[wave][s] = f;
    L += part[(long)s * step + 1] * f;
  }
  L = wave_sum(L);
  wave_lds_order();                              // share: written and read by this wave alone
  float acc[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int s = 0; s < p.nsplit; ++s) {
    const float f = share[wave][s];
    const float* q = part + (long)s * step + 2;
#pragma unroll
    for (int k = 0; k < 3; ++k) acc[k] += (lane + 64 * k < p.hd ? q[lane + 64 * k] : 0.0f) * f;
  }
  const int h = hk * p.group + gr;
  const float inv = L > 0.0f ? 1.0f / L : (L != L ? L : 0.0f);
  T* O = reinterpret_cast<T*>(p.o) + (long)b * p.o_bs + (long)h * p.o_hs + (long)i * p.o_rs;
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (lane + 64 * k < p.hd) O[lane + 64 * k] = from_f32<T>(inv == 0.0f ? 0.0f : acc[k] * inv);
  if (p.lse && lane == 0)
    p.lse[((long)b * p.heads + h) * p.Lq + i] = L > 0.0f ? (M * p.c + __builtin_amdgcn_logf(L)) * 0.69314718055994530942f : (inv != 0.0f ? inv : -__builtin_inff());
}

// Which form, and how many key splits.
// The row blocks of the split form have four waves on 32 queries, so a long range takes half as long as in blocks of 128 -- as long as all
// of them run at once (three per CU up to 64 columns, else two -- past 128 columns only one has room, which is not counted here; under a causal mask half of the keys on average and the longest first, so
// half as many again, twice as many where a workgroup is long).  Causal, bf16, split form / 128-query blocks: 8192 queries of one head of 64
// (256 row blocks) 40 / 151 us, 2 x 2048 of 8 heads of 64 (1024) 30 / 43 us; of 128 columns: 1024 of 12 heads (384) 21 / 33, 2 x 1024 of
// them (768) 31 / 36, 8192 of four heads (1024) 154 / 247, 1024 of 32 heads (1024) 38 / 34 us.  +- 100 keys, 4 x 500 of 12 heads (768):
// 64 columns 11 / 13, 128 columns 21 / 18 us.
void plan(WinArgs& a) {
  a.nqb = (a.Lq + 127) / 128;
  a.nsplit = 0;                                  // 0: 128-query blocks
  a.Lp = a.Lq > 32 ? (a.Lq + 31) / 32 * 32 : a.Lq;
  const bool causal = a.left < 0 && a.right >= 0 && a.right < a.Lk / 2 && a.Lk < 2L * a.Lq;
  const long nrb = ((long)a.group * a.Lp + 31) / 32, wgs = (long)a.batch * a.kv_heads * nrb;
  const long slots = causal && a.Lk >= 2048 ? 1024 : a.hd <= 64 || causal ? 768 : 512;
  if (a.Lq > 32 && wgs > slots) return;
  a.nrb = (int)nrb;
  long keys = a.Lk;                              // of one row block
  if (a.left >= 0 && a.right >= 0) keys = (long)a.left + a.right + (a.Lq < 32 ? a.Lq : 32) + a.sinks;
  if (keys > a.Lk) keys = a.Lk;
  const long tiles = (keys + 31) / 32;
  // no second round of workgroups for a rest, but where the keys are many: 48 streams of 8 key heads of 128, 16384 keys, one / two
  // pieces 580 / 535 us; 1024 queries of 12 heads 25 / 37 us; five streams, 12 / 13 pieces of 5000 keys, 29 / 35 us
  long ns = 512 / wgs;
  if (ns == 1 && wgs < 512 && tiles >= 128) ns = 2;
  if (ns > tiles / 4) ns = tiles / 4;            // every wave of a split has a tile
  // the second launch and the parts cost what the split saves: one stream of 12 heads of 64 takes 11.4 us against 1024 keys in one piece
  // and in eight, 8.3 and 10.1 us against 512
  if (tiles * a.hd <= 2560) ns = 1;
  if (ns > WIN_MAX_SPLIT) ns = WIN_MAX_SPLIT;
  a.nsplit = ns < 1 ? 1 : (int)ns;
}

template <typename T, int HK>
int launch_hk(const WinArgs& a, hipStream_t st) {
  if (a.nsplit == 0) {
    hipLaunchKernelGGL((win_fwd_kernel<T, HK>), dim3((unsigned)(a.batch * a.heads * a.nqb)), dim3(256), 0, st, a);
    HALLO_CHECK_LAUNCH();
    return 0;
  }
  hipLaunchKernelGGL((win_split_kernel<T, HK>), dim3((unsigned)(a.batch * a.kv_heads * a.nrb * a.nsplit)), dim3(256), 0, st, a);
  HALLO_CHECK_LAUNCH();
  if (a.nsplit > 1) {
    const long rows = (long)a.batch * a.heads * a.Lq;
    hipLaunchKernelGGL((win_join_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
    HALLO_CHECK_LAUNCH();
  }
  return 0;
}

template <typename T>
int launch(const WinArgs& a, hipStream_t st) {
  switch ((a.hd + 15) / 16) {
    case 1: return launch_hk<T, 16>(a, st);
    case 2: return launch_hk<T, 32>(a, st);
    case 3: return launch_hk<T, 48>(a, st);
    case 4: return launch_hk<T, 64>(a, st);
    case 5: return launch_hk<T, 80>(a, st);
    case 6: return launch_hk<T, 96>(a, st);
    case 7: return launch_hk<T, 112>(a, st);
    case 8: return launch_hk<T, 128>(a, st);
    case 9: return launch_hk<T, 144>(a, st);
    default: return launch_hk<T, 160>(a, st);
  }
}

}  // namespace

// shared with the backward pass: checks the sizes, strides and alignment of a descriptor and fills the arguments; false = refused
bool win_args(const hallo_window_attn_desc* d, WinArgs& a) {
  if (!d || (d->dtype != DT_F16 && d->dtype != DT_BF16) || d->batch < 0 || d->heads < 1 || d->kv_heads < 1 || d->heads % d->kv_heads ||
      d->head_dim < 8 || d->head_dim > WIN_MAX_HD || d->head_dim % 8 || d->Lq < 0 || d->Lk < 0 || d->Lq > WIN_MAX_LEN || d->Lk > WIN_MAX_LEN ||
      d->sinks < 0 || !(d->scale >= 1e-30f) || !(d->scale < 1e30f))
    return false;
  const int64_t strides[] = {d->q_bs, d->q_rs, d->q_hs, d->k_bs, d->k_rs, d->k_hs, d->v_bs, d->v_rs, d->v_hs, d->o_bs, d->o_rs, d->o_hs};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return false;
  const int64_t row_strides[] = {d->q_rs, d->k_rs, d->v_rs, d->o_rs};
  for (int64_t s : row_strides)
    if (s > WIN_MAX_STRIDE) return false;
  const void* ptrs[] = {d->q, d->k, d->v, d->o};
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  if ((int64_t)d->batch * d->heads * ((d->Lq + 31) / 32) > 0x7fffffff || (int64_t)d->heads * d->Lq > 0x7fffff00 ||
      (int64_t)d->batch * d->heads * ((d->Lk + 31) / 32) > 0x7fffffff)
    return false;
  const auto cut = [](int x) { return x > WIN_MAX_LEN ? WIN_MAX_LEN : x; };
  a = WinArgs{};
  a.q = d->q; a.k = d->k; a.v = d->v; a.o = d->o; a.lse = d->lse;
  a.q_bs = d->q_bs; a.q_rs = d->q_rs; a.q_hs = d->q_hs; a.k_bs = d->k_bs; a.k_rs = d->k_rs; a.k_hs = d->k_hs;
  a.v_bs = d->v_bs; a.v_rs = d->v_rs; a.v_hs = d->v_hs; a.o_bs = d->o_bs; a.o_rs = d->o_rs; a.o_hs = d->o_hs;
  a.q_len = d->q_len; a.kv_len = d->kv_len;
  a.batch = d->batch; a.heads = d->heads; a.kv_heads = d->kv_heads; a.group = d->heads / d->kv_heads; a.hd = d->head_dim;
  a.Lq = (int)d->Lq; a.Lk = (int)d->Lk;
  a.left = d->left < 0 ? -1 : cut(d->left); a.right = d->right < 0 ? -1 : cut(d->right); a.sinks = cut(d->sinks);
  a.scale = d->scale; a.c = d->scale * 1.44269504088896340736f;
  return true;
}

}  // namespace hallo

extern "C" int64_t hallo_window_attention_workspace(const hallo_window_attn_desc* d) {
  using namespace hallo;
  WinArgs a;
  if (!win_args(d, a)) return -22;
  if (a.batch == 0 || a.Lq == 0) return 0;
  plan(a);
  return a.nsplit > 1 ? (int64_t)a.batch * a.kv_heads * a.nrb * a.nsplit * 32 * (a.hd + 2) * 4 : 0;
}

extern "C" int hallo_window_attention_splits(const hallo_window_attn_desc* d) {
  using namespace hallo;
  WinArgs a;
  if (!win_args(d, a)) return -22;
  if (a.batch == 0 || a.Lq == 0) return 0;
  plan(a);
  return a.nsplit;
}

extern "C" int hallo_window_attention(const hallo_window_attn_desc* d, void* stream) {
  using namespace hallo;
  WinArgs a;
  if (!win_args(d, a)) return -22;
  if (a.batch == 0 || a.Lq == 0) return 0;
  if (!a.q || !a.o || (a.Lk > 0 && (!a.k || !a.v))) return -22;
  const int64_t need = hallo_window_attention_workspace(d);
  if (need > 0 && (!d->workspace || d->workspace_bytes < need)) return -22;
  plan(a);
  a.part = (float*)d->workspace;
  if ((int64_t)a.batch * a.kv_heads * a.nrb * (a.nsplit > 0 ? a.nsplit : 1) > 0x7fffffff) return -22;
  return d->dtype == DT_F16 ? launch<_Float16>(a, (hipStream_t)stream) : launch<__bf16>(a, (hipStream_t)stream);
}
