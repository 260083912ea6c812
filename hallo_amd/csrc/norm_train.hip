// LayerNorm for training: the forward pass that keeps its row statistics, and the backward pass with both weight gradients.
//
//   forward    y = (x - mean) * rstd * gamma + beta,   stats = (mean, rstd) in fp32
//   backward   xh = (x - mean) * rstd,  g = dy * gamma
//              dx = rstd * (g - sum_C(g) / C - xh * sum_C(g xh) / C),   dgamma = sum_rows(dy xh),   dbeta = sum_rows(dy)
//
// Both directions are bound by HBM: x (and dy) is read once, the result written once, everything between lives in registers.  A
// row of nvec = ceil(C / 8) 16-byte vectors is shared by LPR lanes with VPL vectors each, so that a narrow row does not idle lanes
// (C = 320: 16 lanes x 3 vectors, 4 rows per wave) and a wide one stays in registers (LPR = 256: the whole workgroup on a row).
// The row sums go through a fixed tree of lane exchanges, the weight gradients through a fixed sequence -- lane, lanes of a wave,
// waves of a workgroup, workgroups in the second launch -- so a result does not depend on timing (no atomics).
// 262144 rows of 320, bf16: forward 66 us (5.15 TB/s, as fast as a copy of the same bytes), backward with weight gradients 107 us (4.7 TB/s);
// 499 rows of 768, fp16: backward 8 + 2 us, two launches.
#include "common.h"
#include "../../include/hallo_amd.h"

namespace hallo {

namespace {

// 8 elements at their own alignment (rows of odd length or odd pitch): gfx950 global loads and stores take any
template <typename V, int A> struct __attribute__((packed, aligned(A))) Loose { V v; };

// columns col .. col + 7 of a row of C as they are stored, zeros past its end
template <typename T, bool AL>
__device__ __forceinline__ typename Vec<T>::v8 ld_raw8(const T* p, int col, int C) {
  if (AL) return ld8<T>(p + col);
  if (col + 8 <= C) return reinterpret_cast<const Loose<typename Vec<T>::v8, 2>*>(p + col)->v;
  typename Vec<T>::v8 t = zero8<T>();
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (col + e < C) t[e] = p[col + e];
  return t;
}
template <typename T, bool AL>
__device__ __forceinline__ void st_row8(T* p, int col, int C, const float (&f)[8]) {
  typename Vec<T>::v8 t;
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = from_f32<T>(f[e]);
  if (AL) st8<T>(p + col, t);
  else if (col + 8 <= C) reinterpret_cast<Loose<typename Vec<T>::v8, 2>*>(p + col)->v = t;
  else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + e < C) p[col + e] = t[e];
  }
}
// weights: the activations' type or fp32 (master weights), absent = `dflt`
template <typename T>
__device__ __forceinline__ void ld_weight8(const void* w, int f32, int col, int C, float dflt, float (&f)[8]) {
  if (!w) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = dflt;
  } else if (col + 8 > C) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = min(col + e, C - 1);
      f[e] = f32 ? reinterpret_cast<const float*>(w)[c] : to_f32(reinterpret_cast<const T*>(w)[c]);
    }
  } else if (f32) {
    typedef __attribute__((ext_vector_type(8))) float f32x8;
    const f32x8 t = reinterpret_cast<const Loose<f32x8, 4>*>(reinterpret_cast<const float*>(w) + col)->v;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = t[e];
  } else {
    const typename Vec<T>::v8 t = reinterpret_cast<const Loose<typename Vec<T>::v8, 2>*>(reinterpret_cast<const T*>(w) + col)->v;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = to_f32(t[e]);
  }
}

// sum over the LPR lanes that share a row (LPR = 256: over the workgroup; `slot` alternates so that one barrier per sum suffices)
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red, int slot) {
#pragma unroll
  for (int o = (LPR > 64 ? 64 : LPR) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if (LPR > 64) {
    float* r = red + slot * 4;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (r[0] + r[1]) + (r[2] + r[3]);
  }
  return v;
}

template <typename T, int LPR, int VPL, bool AL>
__global__ __launch_bounds__(256) void ln_train_kernel(const T* x, long ldx, T* y, long ldy, const void* gamma, const void* beta,
                                                       int wf32, float2* stats, long rows, int C, float eps) {
  constexpr int RPB = 256 / LPR;                 // rows per workgroup
  __shared__ float red[8];
  const int sub = threadIdx.x % LPR;
  const long row = (long)blockIdx.x * RPB + threadIdx.x / LPR;
  const bool live = row < rows;                  // LPR = 256: one row per workgroup, always live
  const T* xr = x + (live ? row : 0) * ldx;
  const int nvec = (C + 7) / 8;
  typename Vec<T>::v8 raw[VPL];
  float v[VPL][8];
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int vi = sub + LPR * i;
    raw[i] = vi < nvec ? ld_raw8<T, AL>(xr, vi * 8, C) : zero8<T>();
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) { v[i][e] = to_f32(raw[i][e]); sum += v[i][e]; }
  const float mean = row_sum<LPR>(sum, red, 0) / (float)C;
  float sq = 0.0f;
#pragma unroll
  for (int i = 0; i < VPL; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = (sub + LPR * i) * 8 + e < C ? v[i][e] - mean : 0.0f;
      sq += d * d;
    }
  const float rstd = 1.0f / sqrtf(row_sum<LPR>(sq, red, 1) / (float)C + eps);
  if (!live) return;
  if (sub == 0) stats[row] = make_float2(mean, rstd);
  T* yr = y + row * ldy;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int vi = sub + LPR * i;
    if (vi < nvec) {
      float g[8], b[8];
      ld_weight8<T>(gamma, wf32, vi * 8, C, 1.0f, g);
      ld_weight8<T>(beta, wf32, vi * 8, C, 0.0f, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = (v[i][e] - mean) * rstd * g[e] + b[e];
      st_row8<T, AL>(yr, vi * 8, C, v[i]);
    }
  }
}

// Workgroup b takes the row groups b, b + grid, ...; WG: also sums dy xh and dy of its rows and writes them to parts[b] = [dgamma |
// dbeta] (2C floats).  The weight gradients stay in registers over the whole loop: 16 floats per vector and lane.
template <typename T, int LPR, int VPL, bool AL, bool WG>
__global__ __launch_bounds__(256) void ln_bwd_kernel(const T* dy, long ldd, const T* x, long ldx, const float2* __restrict__ stats,
                                                     const void* gamma, int wf32, T* dx, long lddx, float* __restrict__ parts,
                                                     long rows, int C) {
  constexpr int RPB = 256 / LPR;
  extern __shared__ float sm[];                  // WG, LPR <= 64: 4 waves x LPR x VPL x 8 floats (at most 24 KB)
  __shared__ float red[16];
  const int sub = threadIdx.x % LPR;
  const int nvec = (C + 7) / 8;
  const float rC = 1.0f / (float)C;
  float g[VPL][8], ag[VPL][8], ab[VPL][8];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    ld_weight8<T>(gamma, wf32, min(sub + LPR * i, nvec - 1) * 8, C, 1.0f, g[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) ag[i][e] = ab[i][e] = 0.0f;
  }
  // The row group after next is requested before a group is worked on: raw 16-byte vectors wait in registers, and are converted once
  // for the sums and once more for dx (fp32 copies of both inputs would cost the second wave of a SIMD).
  using V8 = typename Vec<T>::v8;
  V8 xr[VPL], dr[VPL];
  float2 st;
  const long step = (long)gridDim.x * RPB;
  auto load = [&](long row) {
    const bool live = row < rows;                // dead lanes (last group) carry zeros through the sums
    st = stats[live ? row : 0];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int vi = sub + LPR * i;
      xr[i] = live && vi < nvec ? ld_raw8<T, AL>(x + row * ldx, vi * 8, C) : zero8<T>();
      dr[i] = live && vi < nvec ? ld_raw8<T, AL>(dy + row * ldd, vi * 8, C) : zero8<T>();
    }
  };
  int slot = 0;
  long row = (long)blockIdx.x * RPB + threadIdx.x / LPR;
  load(row);
  for (long r0 = (long)blockIdx.x * RPB; r0 < rows; r0 += step, row += step) {
    V8 xc[VPL], dc[VPL];
    const float mean = st.x, rstd = st.y;
#pragma unroll
    for (int i = 0; i < VPL; ++i) { xc[i] = xr[i]; dc[i] = dr[i]; }
    if (r0 + step < rows) load(row + step);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xh = (to_f32(xc[i][e]) - mean) * rstd, d = to_f32(dc[i][e]);       // columns past C and dead rows: d = 0
        if (WG) { ag[i][e] += d * xh; ab[i][e] += d; }
        const float gd = d * g[i][e];
        s1 += gd;
        s2 += gd * xh;
      }
    s1 = row_sum<LPR>(s1, red, slot) * rC;
    s2 = row_sum<LPR>(s2, red, slot + 1) * rC;
    slot ^= 2;
#pragma unroll
    for (int i = 0; i < VPL; ++i) asm("" : "+v"(xc[i]), "+v"(dc[i]));      // convert again: keeping the fp32 values costs 16 registers per vector
    if (row < rows) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int vi = sub + LPR * i;
        if (vi < nvec) {
          float o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float xh = (to_f32(xc[i][e]) - mean) * rstd;
            o[e] = rstd * (to_f32(dc[i][e]) * g[i][e] - s1 - xh * s2);
          }
          st_row8<T, AL>(dx + row * lddx, vi * 8, C, o);
        }
      }
    }
  }
  if (!WG) return;
  float* out = parts + (long)blockIdx.x * 2 * C;
  constexpr int W = LPR * VPL * 8;               // columns of a wave's image
#pragma unroll
  for (int half = 0; half < 2; ++half) {         // dgamma, then dbeta, through the same LDS
    auto& acc = half ? ab : ag;
    if (LPR == 256) {                            // every thread holds columns of its own
#pragma unroll
      for (int i = 0; i < VPL; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = (sub + LPR * i) * 8 + e;
          if (c < C) out[half * C + c] = acc[i][e];
        }
      continue;
    }
    float* m = sm + (threadIdx.x >> 6) * W;
    if (half) __syncthreads();
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float a = acc[i][e];
#pragma unroll
        for (int o = 32; o >= LPR; o >>= 1) a += __shfl_xor(a, o, 64);      // the wave's 64 / LPR rows
        if ((threadIdx.x & 63) < LPR) m[(sub + LPR * i) * 8 + e] = a;
      }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += 256) out[half * C + c] = (sm[c] + sm[W + c]) + (sm[2 * W + c] + sm[3 * W + c]);
  }
}

// sums[c] = sum over the workgroups' parts, in order: 16 columns x 64 part groups per workgroup
__global__ __launch_bounds__(1024) void ln_bwd_join_kernel(const float* __restrict__ parts, int nparts, int C, float* dgamma, float* dbeta) {
  __shared__ float sm[64][17];
  const int cl = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + cl;
  float s = 0.0f;
  if (c < 2 * C)
#pragma unroll 4
    for (int p = grp; p < nparts; p += 64) s += parts[(long)p * 2 * C + c];
  sm[grp][cl] = s;
  __syncthreads();
  if (grp >= 4) return;
  float t = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; ++k) t += sm[grp * 16 + k][cl];
  sm[grp * 16][cl] = t;                          // row grp * 16 is read by this thread alone
  wave_lds_order();                              // the four groups are one wave
  if (grp == 0 && c < 2 * C) {
    t = (sm[0][cl] + sm[16][cl]) + (sm[32][cl] + sm[48][cl]);
    if (c < C) dgamma[c] = t; else dbeta[c - C] = t;
  }
}

// Lanes per row and vectors per lane for a row of nvec vectors: the fewest lanes that hold it with at most 3 vectors each, past 192
// vectors the whole workgroup.  3 is for the backward pass -- x and dy twice (now and next), gamma and both gradients in registers --
// on 262144 rows of 320 (bf16): 16 lanes x 3 (a sixth of them idle) 107 us, 8 lanes x 5 (none idle, one wave per SIMD) 147 us.
// Rows that 16 lanes or more hold with 2 take 3 all the same: 262144 rows of 256, fp16, backward 89 us against 93 (forward 42.5 both).  Past 8
// lanes only: 197031 rows of 50, 8 lanes x 1 / x 3, 25 / 50 us.
void pick(int nvec, int& lpr, int& vpl) {
  if (nvec > 192) { lpr = 256; vpl = nvec <= 512 ? 2 : (nvec <= 1024 ? 4 : 8); return; }
  lpr = 8;
  while (lpr * 3 < nvec) lpr *= 2;
  vpl = lpr > 8 ? 3 : (nvec + lpr - 1) / lpr;
}

constexpr int LN_MAX_C = 16384;
constexpr int LN_BWD_WGS = 1024;                 // workgroups of the backward pass: four per CU

template <typename F> int with_shape(int lpr, int vpl, F&& f) {
#define CASE(L, V) if (lpr == L && vpl == V) return f(std::integral_constant<int, L>{}, std::integral_constant<int, V>{});
  CASE(8, 1) CASE(8, 2) CASE(8, 3) CASE(16, 3) CASE(32, 3) CASE(64, 3) CASE(256, 2) CASE(256, 4) CASE(256, 8)
#undef CASE
  return -22;
}

bool aligned16(const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }

template <typename T>
int launch_fwd(const void* x, int64_t ldx, void* y, int64_t ldy, const void* g, const void* b, int wf32, float* stats, int64_t rows, int C,
               float eps, hipStream_t st) {
  const bool al = C % 8 == 0 && aligned16(x, ldx) && aligned16(y, ldy);
  int lpr, vpl;
  pick((C + 7) / 8, lpr, vpl);
  const int64_t grid = (rows * lpr + 255) / 256;
  if (grid > 0x7fffffff) return -22;
  auto go = [&](auto L, auto V, auto A) {
    hipLaunchKernelGGL((ln_train_kernel<T, decltype(L)::value, decltype(V)::value, decltype(A)::value>), dim3((unsigned)grid), dim3(256), 0, st,
                       (const T*)x, (long)ldx, (T*)y, (long)ldy, g, b, wf32, (float2*)stats, (long)rows, C, eps);
    HALLO_CHECK_LAUNCH();
    return 0;
  };
  return al ? with_shape(lpr, vpl, [&](auto L, auto V) { return go(L, V, std::true_type{}); })
            : with_shape(lpr, vpl, [&](auto L, auto V) { return go(L, V, std::false_type{}); });
}

int bwd_wgs(int64_t rows, int lpr) {
  const int64_t need = (rows * lpr + 255) / 256;
  return (int)(need < LN_BWD_WGS ? need : LN_BWD_WGS);
}

template <typename T>
int launch_bwd(const void* dy, int64_t ldd, const void* x, int64_t ldx, const float* stats, const void* g, int wf32, void* dx, int64_t lddx,
               float* dgamma, float* dbeta, float* parts, int64_t rows, int C, hipStream_t st) {
  const bool al = C % 8 == 0 && aligned16(x, ldx) && aligned16(dy, ldd) && aligned16(dx, lddx);
  int lpr, vpl;
  pick((C + 7) / 8, lpr, vpl);
  const int wgs = bwd_wgs(rows, lpr);
  const bool direct = wgs == 1 && dgamma && dbeta == dgamma + C;     // one workgroup: its sums are the result
  float* to = direct ? dgamma : parts;
  auto go = [&](auto L, auto V, auto A, auto W) {
    constexpr int l = decltype(L)::value, v = decltype(V)::value;
    const int lds = decltype(W)::value && l <= 64 ? 4 * l * v * 8 * 4 : 0;
    hipLaunchKernelGGL((ln_bwd_kernel<T, l, v, decltype(A)::value, decltype(W)::value>), dim3(wgs), dim3(256), lds, st, (const T*)dy, (long)ldd,
                       (const T*)x, (long)ldx, (const float2*)stats, g, wf32, (T*)dx, (long)lddx, to, (long)rows, C);
    HALLO_CHECK_LAUNCH();
    return 0;
  };
  if (wgs > 0) {
    auto al_go = [&](auto W) {
      return al ? with_shape(lpr, vpl, [&](auto L, auto V) { return go(L, V, std::true_type{}, W); })
                : with_shape(lpr, vpl, [&](auto L, auto V) { return go(L, V, std::false_type{}, W); });
    };
    const int rc = dgamma ? al_go(std::true_type{}) : al_go(std::false_type{});
    if (rc) return rc;
  }
  if (dgamma && !direct) {
    hipLaunchKernelGGL(ln_bwd_join_kernel, dim3((2 * C + 15) / 16), dim3(1024), 0, st, parts, wgs, C, dgamma, dbeta);
    HALLO_CHECK_LAUNCH();
  }
  return 0;
}

}  // namespace
}  // namespace hallo

extern "C" int hallo_layernorm_train(const void* x, int64_t ldx, void* y, int64_t ldy, const void* gamma, const void* beta, int affine_f32,
                                     float* stats, int64_t rows, int C, float eps, int dtype, void* stream) {
  using namespace hallo;
  if (rows < 0 || C < 1 || C > LN_MAX_C || ldx < C || ldy < C || !(eps >= 0.0f) || (affine_f32 & ~1) || (dtype != DT_F16 && dtype != DT_BF16))
    return -22;
  if (rows == 0) return 0;
  if (!x || !y || !stats || (x == y && ldx != ldy && rows > 1)) return -22;
  hipStream_t st = (hipStream_t)stream;
  return dtype == DT_F16 ? launch_fwd<_Float16>(x, ldx, y, ldy, gamma, beta, affine_f32, stats, rows, C, eps, st)
                         : launch_fwd<__bf16>(x, ldx, y, ldy, gamma, beta, affine_f32, stats, rows, C, eps, st);
}

extern "C" int64_t hallo_layernorm_backward_workspace(int64_t rows, int C) {
  using namespace hallo;
  if (rows < 0 || C < 1 || C > LN_MAX_C) return -22;
  int lpr, vpl;
  pick((C + 7) / 8, lpr, vpl);
  return (int64_t)bwd_wgs(rows, lpr) * 2 * C * 4;
}

extern "C" int hallo_layernorm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* stats, const void* gamma,
                                        int affine_f32, void* dx, int64_t lddx, float* dgamma, float* dbeta, void* workspace,
                                        int64_t workspace_bytes, int64_t rows, int C, int dtype, void* stream) {
  using namespace hallo;
  if (rows < 0 || C < 1 || C > LN_MAX_C || lddy < C || ldx < C || lddx < C || (affine_f32 & ~1) || (dtype != DT_F16 && dtype != DT_BF16))
    return -22;
  if ((dgamma == nullptr) != (dbeta == nullptr)) return -22;
  if (rows > 0 && (!dy || !x || !stats || !dx)) return -22;
  if (rows > 1 && ((dx == dy && lddx != lddy) || (dx == x && lddx != ldx))) return -22;
  if (dgamma && rows > 0 && (!workspace || workspace_bytes < hallo_layernorm_backward_workspace(rows, C))) return -22;
  hipStream_t st = (hipStream_t)stream;
  return dtype == DT_F16
             ? launch_bwd<_Float16>(dy, lddy, x, ldx, stats, gamma, affine_f32, dx, lddx, dgamma, dbeta, (float*)workspace, rows, C, st)
             : launch_bwd<__bf16>(dy, lddy, x, ldx, stats, gamma, affine_f32, dx, lddx, dgamma, dbeta, (float*)workspace, rows, C, st);
}
