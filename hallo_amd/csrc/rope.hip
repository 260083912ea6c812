// Rotary positions over up to four axes (time, height, width, ...).
//
// Axis a owns d_a columns of every head, its pair i turns by pos_a * theta^(-2i / d_a):
//   y_m = x_m cos - x_n sin,   y_n = x_n cos + x_m sin      (m, n) = (2i, 2i + 1) or (i, i + d_a / 2) within the axis' columns
// Columns behind the last axis pass through.  The gradient of a rotation is the rotation by the negative angle (`inverse`).
//
// Angles: a frequency is a 64-bit fixed-point fraction of a turn, so pos * freq modulo 2^64 IS the stored frequency's angle modulo one
// turn, without a rounding at any 32-bit position, where a 32-bit float product is off by whole radians near 10^7.  The stored frequency
// is theta^(..) in a double (53 bits): about 2^-24 of a turn at position 2^31.  The top 32 bits of the angle go to sincospi.
//
// The kernel is bound by HBM (x read once, y written once; 4.5 TB/s on 262144 tokens of 16 heads of 40 in rows of 960, fp16: 149 us).  A workgroup takes `tt` tokens: it computes their cos / sin once into LDS,
// shared by all heads, then walks (token, head, unit); a unit is V columns and, in the half-split form, their V partners, so every
// element is read and written by one thread (y may be x).  V = 8 or 4, whichever divides the axes' (half) widths; other widths go
// through rope_staged_kernel.
#include "common.h"
#include "../../include/hallo_amd.h"

namespace hallo {

namespace {

constexpr int ROPE_MAX_HD = 256;
constexpr int ROPE_PAIRS = 1024;                 // cos / sin pairs a workgroup holds (8 KB)
constexpr int ROPE_TT = 64;                      // most tokens of a workgroup

struct RopeArgs {
  const void* x; void* y;
  long x_bs, x_rs, y_bs, y_rs;
  const unsigned long long* freq;                // [pairs] turns * 2^64
  const int* pos; long pos_bs;                   // [B or 1, L, n_axes]; null: grid
  int n_axes, dims[4], grid[4], origin[4];
  int inverse, heads, hd, pairs, tt, hb;         // hb: heads of a staged tile
  long L, tokens;                                // tokens = B * L
};

// token t0 + i of the workgroup as (batch entry, place): one long division for t0, 32-bit ones for the rest (L < 2^31)
struct RopeWhere {
  long b0; unsigned l0, L;
  __device__ __forceinline__ RopeWhere(const RopeArgs& p, long t0) : b0(t0 / p.L), l0((unsigned)(t0 - b0 * p.L)), L((unsigned)p.L) {}
  __device__ __forceinline__ void at(int i, long& b, unsigned& l) const {
    const unsigned t = l0 + (unsigned)i, q = t / L;
    b = b0 + q;
    l = t - q * L;
  }
};

// cos / sin of every pair of the workgroup's nt tokens
__device__ __forceinline__ void rope_angles(const RopeArgs& p, const RopeWhere& where, int nt, float2* cs) {
  for (int k = threadIdx.x; k < nt * p.pairs; k += 256) {
    const int tt = k / p.pairs, j = k - tt * p.pairs;
    const unsigned long long freq = p.freq[j];
    long b;
    unsigned l;
    where.at(tt, b, l);
    int a = 0, first = 0;
    while (j >= first + p.dims[a] / 2) { first += p.dims[a] / 2; ++a; }
    int pos;
    if (p.pos) pos = p.pos[b * p.pos_bs + (long)l * p.n_axes + a];
    else {
      unsigned r = l;
      for (int c = p.n_axes - 1; c > a; --c) r /= (unsigned)p.grid[c];
      pos = p.origin[a] + (int)(r % (unsigned)p.grid[a]);
    }
    const unsigned long long turn = (unsigned long long)(long long)pos * freq;
    const float half_turns = (float)(int)(unsigned)(turn >> 32) * 0x1p-31f;
    float s, c;
    sincospif(half_turns, &s, &c);
    cs[k] = make_float2(c, p.inverse ? -s : s);
  }
}

template <typename T, int V> struct __attribute__((aligned(2 * V))) PieceA { T v[V]; };
template <typename T, int V> struct __attribute__((packed, aligned(2))) PieceU { T v[V]; };

// IL: interleaved pairs.  AL: every piece of V columns is aligned to its size.
template <typename T, int V, bool IL, bool AL>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs p) {
  using P = typename std::conditional<AL, PieceA<T, V>, PieceU<T, V>>::type;
  __shared__ float2 cs[ROPE_PAIRS];
  __shared__ int ucol[ROPE_MAX_HD / 4], upart[ROPE_MAX_HD / 4], upair[ROPE_MAX_HD / 4];    // unit: first column, partner column (-1: passes through), first pair
  __shared__ long xoff[ROPE_TT], yoff[ROPE_TT];
  const int tid = threadIdx.x;
  const long t0 = (long)blockIdx.x * p.tt;
  const int nt = (int)(p.tokens - t0 < p.tt ? p.tokens - t0 : p.tt);

  // unit table (the axes' sections, then the columns that pass through)
  int units = 0;
  {
    int col = 0, pair = 0;
    for (int a = 0; a < p.n_axes; ++a) {
      const int d = p.dims[a], n = (IL ? d : d / 2) / V;
      for (int u = tid; u < n; u += 256) {
        ucol[units + u] = col + u * V;
        upart[units + u] = IL ? 0 : col + d / 2 + u * V;
        upair[units + u] = pair + (IL ? u * V / 2 : u * V);
      }
      units += n; col += d; pair += d / 2;
    }
    const int n = (p.hd - col) / V;
    for (int u = tid; u < n; u += 256) { ucol[units + u] = col + u * V; upart[units + u] = -1; upair[units + u] = 0; }
    if (p.x != p.y) units += n;                  // in place they stay where they are
  }
  const RopeWhere where(p, t0);
  if (tid < nt) {
    long b;
    unsigned l;
    where.at(tid, b, l);
    xoff[tid] = b * p.x_bs + (long)l * p.x_rs;
    yoff[tid] = b * p.y_bs + (long)l * p.y_rs;
  }
  rope_angles(p, where, nt, cs);
  __syncthreads();

  const T* X = reinterpret_cast<const T*>(p.x);
  T* Y = reinterpret_cast<T*>(p.y);
  const unsigned per = (unsigned)(p.heads * units), items = per * (unsigned)nt;
  constexpr int N = 4;                           // items a thread loads before it stores the first (x and y may be the same memory)
  for (unsigned k0 = tid; k0 < items; k0 += 256 * N) {
    P a[N], b[N];
    unsigned tt[N], hh[N], un[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned k = k0 + 256 * i;
      if (k >= items) break;
      tt[i] = k / per;
      const unsigned r = k - tt[i] * per;
      hh[i] = r / (unsigned)units;
      un[i] = r - hh[i] * (unsigned)units;
      const T* xr = X + xoff[tt[i]] + (long)hh[i] * p.hd;
      a[i] = *reinterpret_cast<const P*>(xr + ucol[un[i]]);
      if (!IL && upart[un[i]] >= 0) b[i] = *reinterpret_cast<const P*>(xr + upart[un[i]]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (k0 + 256 * i >= items) break;
      const int u = un[i], c0 = ucol[u], c1 = upart[u];
      const float2* w = cs + tt[i] * p.pairs + upair[u];
      T* yr = Y + yoff[tt[i]] + (long)hh[i] * p.hd;
      if (c1 < 0) { *reinterpret_cast<P*>(yr + c0) = a[i]; continue; }
      P o;
      if constexpr (IL) {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          const float2 t = w[e];
          const float m = to_f32(a[i].v[2 * e]), n = to_f32(a[i].v[2 * e + 1]);
          o.v[2 * e] = from_f32<T>(m * t.x - n * t.y);
          o.v[2 * e + 1] = from_f32<T>(n * t.x + m * t.y);
        }
        *reinterpret_cast<P*>(yr + c0) = o;
      } else {
        P q;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 t = w[e];
          const float m = to_f32(a[i].v[e]), n = to_f32(b[i].v[e]);
          o.v[e] = from_f32<T>(m * t.x - n * t.y);
          q.v[e] = from_f32<T>(n * t.x + m * t.y);
        }
        *reinterpret_cast<P*>(yr + c0) = o;
        *reinterpret_cast<P*>(yr + c1) = q;
      }
    }
  }
}

// Axes whose (half) widths are odd or twice odd: pieces of 1 or 2 columns would be all address arithmetic.  Here whole rows go through
// LDS in 16-byte chunks (the last one of a row of odd width element by element), and a thread turns the 8 columns of its chunk with the
// partner columns read from LDS, one at a time (interleaved pairs too, although the two lie in one chunk).  Bound by
// vector work: 71 % of the SIMDs' cycles on 8510 tokens of 16 heads of 80 (17.1 us, 2.6 TB/s); the LDS port is busy for 16 %.
constexpr int ROPE_STAGE = 8192;                 // elements of the staged tile (16 KB)

template <typename T, bool AL>
__global__ __launch_bounds__(256) void rope_staged_kernel(const RopeArgs p, int il) {
  using V8 = typename Vec<T>::v8;
  struct __attribute__((packed, aligned(2))) Loose { V8 v; };
  __shared__ float2 cs[ROPE_PAIRS];
  __shared__ __attribute__((aligned(16))) T tile[ROPE_STAGE + 8 * ROPE_TT];
  __shared__ int map[ROPE_MAX_HD];               // column -> partner - column, pair, sign of sin (0: passes through)
  __shared__ long xoff[ROPE_TT], yoff[ROPE_TT];
  const int tid = threadIdx.x;
  const long t0 = (long)blockIdx.x * p.tt;
  const int nt = (int)(p.tokens - t0 < p.tt ? p.tokens - t0 : p.tt);
  for (int c = tid; c < p.hd; c += 256) {
    int at = 0, pair = 0, a = 0, v = 0;
    while (a < p.n_axes && c >= at + p.dims[a]) { at += p.dims[a]; pair += p.dims[a] / 2; ++a; }
    if (a < p.n_axes) {
      const int i = c - at, half = p.dims[a] / 2, up = il ? i & 1 : i >= half, step = il ? 1 : half;
      v = (up ? -step : step) * 65536 + (pair + (il ? i >> 1 : i - up * half)) * 4 + (up ? 1 : 2);
    }
    map[c] = v;
  }
  const RopeWhere where(p, t0);
  if (tid < nt) {
    long b;
    unsigned l;
    where.at(tid, b, l);
    xoff[tid] = b * p.x_bs + (long)l * p.x_rs;
    yoff[tid] = b * p.y_bs + (long)l * p.y_rs;
  }
  __syncthreads();
  const T* X = reinterpret_cast<const T*>(p.x);
  T* Y = reinterpret_cast<T*>(p.y);
  constexpr int N = (ROPE_STAGE / 8 + ROPE_TT + 255) / 256;      // chunks of a thread
  for (int h0 = 0; h0 < p.heads; h0 += p.hb) {
    const int width = min(p.hb, p.heads - h0) * p.hd, nch = (width + 7) / 8;
    const long base = (long)h0 * p.hd;
    V8 in[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = tid + 256 * i, t = k / nch, c = (k - t * nch) * 8;
      if (k < nt * nch) {
        const T* xr = X + xoff[t] + base + c;
        if (c + 8 <= width) in[i] = AL ? ld8<T>(xr) : reinterpret_cast<const Loose*>(xr)->v;
        else {
          in[i] = zero8<T>();
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < width) in[i][e] = xr[e];
        }
      }
    }
    if (h0 == 0) rope_angles(p, where, nt, cs);  // under the first loads
    else __syncthreads();                        // the tile before this one has been read
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = tid + 256 * i;
      if (k < nt * nch) st8<T>(tile + k * 8, in[i]);
    }
    __syncthreads();
    if (p.hd % 8 == 0) {
      // the chunks of a head: a thread keeps the 8 cos, sin and partner distances of its columns over the heads hg, hg + groups, ...
      const int ncc = p.hd / 8, heads = width / p.hd, groups = max(1, min(heads, 256 / (nt * ncc)));
      for (int k = tid; k < nt * groups * ncc; k += 256) {
        const int r = k / ncc, cc = k - r * ncc, t = r / groups, hg = r - t * groups;
        const float2* w = cs + t * p.pairs;
        float co[8], si[8];
        int to[8];
        unsigned turned = 0;                     // columns of an axis (the others pass through)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int m = map[cc * 8 + e];
          const float2 f = w[(m & 0xffff) >> 2];
          co[e] = f.x;
          si[e] = m & 1 ? f.y : -f.y;
          to[e] = e + (m >> 16);
          turned |= (m != 0) << e;
        }
        for (int h = hg; h < heads; h += groups) {
          const T* x = tile + t * nch * 8 + h * p.hd + cc * 8;
          const V8 v = ld8<T>(x);
          V8 o = v;
          if (turned)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (turned >> e & 1) o[e] = from_f32<T>(to_f32(v[e]) * co[e] + to_f32(x[to[e]]) * si[e]);
          T* yr = Y + yoff[t] + base + h * p.hd + cc * 8;
          if (AL) st8<T>(yr, o);
          else reinterpret_cast<Loose*>(yr)->v = o;
        }
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = tid + 256 * i, t = k / nch, c = (k - t * nch) * 8;
      if (k >= nt * nch) break;
      const T* row = tile + t * nch * 8;
      const float2* w = cs + t * p.pairs;
      V8 o;
      int col = c % p.hd;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int m = c + e < width ? map[col] : 0;
        const float2 f = w[(m & 0xffff) >> 2];
        const float s = m & 1 ? f.y : -f.y;
        o[e] = m ? from_f32<T>(to_f32(in[i][e]) * f.x + to_f32(row[c + e + (m >> 16)]) * s) : in[i][e];
        if (++col == p.hd) col = 0;
      }
      T* yr = Y + yoff[t] + base + c;
      if (c + 8 <= width) {
        if (AL) st8<T>(yr, o);
        else reinterpret_cast<Loose*>(yr)->v = o;
      } else
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < width) yr[e] = o[e];
    }
  }
}

template <typename T, int V, bool IL>
int launch_rope(const RopeArgs& a, bool al, hipStream_t st) {
  const long grid = (a.tokens + a.tt - 1) / a.tt;
  if (grid > 0x7fffffff) return -22;
  if (al) hipLaunchKernelGGL((rope_kernel<T, V, IL, true>), dim3((unsigned)grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((rope_kernel<T, V, IL, false>), dim3((unsigned)grid), dim3(256), 0, st, a);
  HALLO_CHECK_LAUNCH();
  return 0;
}

template <typename T>
int launch_staged(const RopeArgs& a, bool il, bool al, hipStream_t st) {
  const long grid = (a.tokens + a.tt - 1) / a.tt;
  if (grid > 0x7fffffff) return -22;
  if (al) hipLaunchKernelGGL((rope_staged_kernel<T, true>), dim3((unsigned)grid), dim3(256), 0, st, a, (int)il);
  else hipLaunchKernelGGL((rope_staged_kernel<T, false>), dim3((unsigned)grid), dim3(256), 0, st, a, (int)il);
  HALLO_CHECK_LAUNCH();
  return 0;
}

template <typename T>
int pick_rope(const RopeArgs& a, int V, bool il, bool al, hipStream_t st) {
  if (il) return V == 8 ? launch_rope<T, 8, true>(a, al, st) : launch_rope<T, 4, true>(a, al, st);
  return V == 8 ? launch_rope<T, 8, false>(a, al, st) : launch_rope<T, 4, false>(a, al, st);
}

}  // namespace
}  // namespace hallo

extern "C" int hallo_rope(const hallo_rope_desc* d, void* stream) {
  using namespace hallo;
  if (!d || (d->dtype != DT_F16 && d->dtype != DT_BF16) || d->batch < 0 || d->L < 0 || d->heads < 1 || d->heads > (1 << 16) || d->head_dim < 2 || d->head_dim % 2 ||
      d->head_dim > ROPE_MAX_HD || d->n_axes < 1 || d->n_axes > 4 || d->batch > 0x7fffffff)
    return -22;
  RopeArgs a = {};
  int sum = 0, g = d->head_dim;                  // g: greatest common divisor that V has to divide
  auto gcd = [](int x, int y) { while (y) { const int t = x % y; x = y; y = t; } return x; };
  const bool il = d->interleaved != 0;
  const bool none = d->batch == 0 || d->L == 0;
  long cells = 1;
  for (int i = 0; i < d->n_axes; ++i) {
    if (d->dims[i] < 2 || d->dims[i] % 2 || d->dims[i] > ROPE_MAX_HD) return -22;
    sum += d->dims[i];
    g = gcd(g, il ? d->dims[i] : d->dims[i] / 2);
    a.dims[i] = d->dims[i];
    if (!d->pos && !none) {
      if (d->grid[i] < 1 || cells > d->L / d->grid[i] + 1 || (int64_t)d->origin[i] + d->grid[i] > 1LL << 31) return -22;
      cells *= d->grid[i];
      a.grid[i] = d->grid[i];
      a.origin[i] = d->origin[i];
    }
  }
  if (sum > d->head_dim || (!d->pos && !none && cells != d->L)) return -22;
  const long width = (long)d->heads * d->head_dim;
  if (d->x_rs < 0 || d->y_rs < width || d->L > 0x7fffffff - ROPE_TT || (d->batch > 0 && d->L > (1L << 46) / d->batch)) return -22;
  if (none) return 0;
  if (d->batch > 1) {                            // rows of different entries must not share elements: two workgroups would write them
    const int64_t ext = d->L > 1 ? (d->L - 1) * d->y_rs + width : width;
    if (d->y_bs < ext) {
      if (d->L == 1 || d->y_bs < width) return -22;
      const bool inside = d->y_rs >= (d->batch - 1) * d->y_bs + width;          // the batch inside of the rows
      for (int64_t b = 1; !inside && b < d->batch && b * d->y_bs / d->y_rs < d->L; ++b) {
        const int64_t l = b * d->y_bs / d->y_rs, rest = b * d->y_bs % d->y_rs;
        if (rest < width || (l + 1 < d->L && d->y_rs - rest < width)) return -22;
      }
    }
  }
  if (!d->x || !d->y || !d->freq) return -22;
  if (d->x == d->y && (d->x_bs != d->y_bs || d->x_rs != d->y_rs)) return -22;
  a.x = d->x; a.y = d->y;
  a.x_bs = d->x_bs; a.x_rs = d->x_rs; a.y_bs = d->y_bs; a.y_rs = d->y_rs;
  a.freq = reinterpret_cast<const unsigned long long*>(d->freq);
  a.pos = d->pos; a.pos_bs = d->pos_bs;
  a.n_axes = d->n_axes; a.inverse = d->inverse != 0; a.heads = d->heads; a.hd = d->head_dim; a.pairs = sum / 2;
  a.L = d->L; a.tokens = d->batch * d->L;
  const int V = g % 8 == 0 ? 8 : g % 4 == 0 ? 4 : g % 2 == 0 ? 2 : 1;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) |
                         (uintptr_t)(2 * (a.x_rs | a.y_rs | a.hd | (d->batch > 1 ? a.x_bs | a.y_bs : 0)));
  // tokens of a workgroup: enough to fill its lanes and the cos / sin table, few enough to spread over the 256 CUs
  // pieces of 4 columns: 150 us direct, 214 us staged (262144 tokens, 16 heads of 40); pieces of 1: 26 us direct, 18 us staged (8510
  // tokens, 16 heads of 80)
  const bool staged = V <= 2;
  int tt = ROPE_PAIRS / a.pairs;
  if (tt > ROPE_TT) tt = ROPE_TT;
  if (staged && tt * width > ROPE_STAGE) tt = width <= ROPE_STAGE ? (int)(ROPE_STAGE / width) : 1;      // all heads of a token in one tile
  while (tt > 1 && (a.tokens + tt - 1) / tt < 1024) tt = (tt + 1) / 2;
  a.tt = tt;
  hipStream_t st = (hipStream_t)stream;
  if (staged) {
    a.hb = ROPE_STAGE / (tt * a.hd);
    if (a.hb >= a.heads) a.hb = a.heads;
    else if (a.hb >= 8) a.hb = a.hb / 8 * 8;     // later tiles start at multiples of 8 columns
    const uintptr_t rows = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) |
                           (uintptr_t)(2 * (a.x_rs | a.y_rs | (d->batch > 1 ? a.x_bs | a.y_bs : 0) | (a.hb < a.heads ? a.hb * a.hd : 0)));
    return d->dtype == DT_F16 ? launch_staged<_Float16>(a, il, rows % 16 == 0, st) : launch_staged<__bf16>(a, il, rows % 16 == 0, st);
  }
  const bool al = bits % (2 * V) == 0;
  return d->dtype == DT_F16 ? pick_rope<_Float16>(a, V, il, al, st) : pick_rope<__bf16>(a, V, il, al, st);
}
