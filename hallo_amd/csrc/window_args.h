// What the window attention kernels share: arguments, visible ranges, LDS pitches, MFMA operand reads.
//
// A query i of batch entry b stands at position p = kv_len - q_len + i and sees key j iff
//   j < kv_len,  j <= p + right (right >= 0),  and  j >= p - left (left >= 0) or j < sinks.
#pragma once
#include "common.h"

namespace hallo {

struct WinArgs {
  const void *q, *k, *v; void* o; float* lse;
  long q_bs, q_rs, q_hs, k_bs, k_rs, k_hs, v_bs, v_rs, v_hs, o_bs, o_rs, o_hs;
  const int *q_len, *kv_len;                     // [batch] or null (= Lq, Lk)
  int batch, heads, kv_heads, group, hd, Lq, Lk, left, right, sinks;
  float scale, c;                                // c = scale * log2(e)
  int nqb;                                       // query blocks of one (batch entry, head)
  // split form (few queries): row blocks of 32 packed rows, key splits, partial results [row block][split][32][hd + 2]
  int nrb, nsplit, Lp; float* part;              // Lp: packed rows of a head
};

constexpr int WIN_MAX_LEN = 1 << 29;             // sums of two positions / window edges stay inside int
constexpr int WIN_MAX_HD = 160;
constexpr int WIN_MAX_STRIDE = 1 << 24;          // elements between rows: 32-bit offsets inside a tile of 128 rows

typedef __attribute__((ext_vector_type(4))) short win_s16x4;
typedef __attribute__((ext_vector_type(8))) short win_s16x8;
typedef __attribute__((address_space(3))) unsigned char win_lds;

__device__ __forceinline__ int win_clamp(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }
__device__ __forceinline__ int win_len(const int* len, int b, int most) { return len ? win_clamp(len[b], 0, most) : most; }

// keys that some query at positions plo .. phi sees: [0, e0) and [s1, e1), the second empty when the first reaches to the end
struct WinRange { int e0, s1, e1; };
__device__ __forceinline__ WinRange win_range(const WinArgs& p, int plo, int phi, int kn) {
  const int hi = p.right < 0 ? kn : win_clamp(phi + p.right + 1, 0, kn);
  const int lo = p.left < 0 ? 0 : win_clamp(plo - p.left, 0, hi);
  const int se = min(p.sinks, hi);
  return lo <= se ? WinRange{hi, hi, hi} : WinRange{se, lo, hi};
}

// largest of the row norms n[i], one for every 64 rows, over the rows lo .. hi - 1 and those beside them in their blocks
__device__ __forceinline__ float win_norm(const float* n, int lo, int hi, int lane, float big) {
  for (int i = lo / 64 + lane; i * 64 < hi; i += 64) big = fmaxf(big, n[i]);
  return big;
}

// LDS tiles of rows of HK elements (a multiple of 16): rows of C 16-byte chunks, chunk c of row r stored at c ^ swz(r).  A tile is read
// along its rows (MFMA operand, 16 bytes per lane, lane = row: 16 consecutive rows at one chunk) and transposed (32 lanes: 4 consecutive
// rows x 64 aligned bytes); the swizzle puts both kinds of 256 bytes on all 64 banks once.  It repeats every 16 rows, so a fragment
// further down the tile is an immediate offset away.  (Padded pitches without a swizzle serve one kind only: a quarter of the forward
// kernel's LDS cycles were conflicts.)
// C = 4, 12 or 20: consecutive rows start four chunks apart (mod 16) and the swizzle stays within four chunks, so two lane offsets of
// each kind serve all columns and the rest is part of the instruction.  C = 16 is denser, for the kernel that is short of LDS.
constexpr int win_chunks(int HK) { return HK <= 32 ? 4 : HK <= 96 ? 12 : 20; }
template <int HK, int C = win_chunks(HK)> struct WinTile {
  static_assert(C * 8 >= HK && (C % 8 == 4 || C == 16), "");
  static constexpr bool NEAR = C % 8 == 4;
  static constexpr int PITCH = C * 16, NKS = HK / 16, NDB = (HK + 31) / 32;
  static constexpr int NA = NEAR ? 2 : NKS, NB = NEAR ? 1 : NDB;
  static __device__ __forceinline__ int swz(int r) { return NEAR ? r >> 2 & 3 : (r & 3) << 2 | (r >> 2 & 3); }
  static __device__ __forceinline__ int at(int r, int c) { return r * PITCH + ((c ^ swz(r)) << 4); }
  // this lane's byte offsets: of row (lane & 31), columns 16 ks + 8 hi, and of rows 8 k + .. read transposed
  int along[NA], trans[NB][2];
  __device__ __forceinline__ WinTile(int lane) {
    const int hi = lane >> 5, l31 = lane & 31, gi = lane & 15, gdh = lane >> 4 & 1;
#pragma unroll
    for (int ks = 0; ks < NA; ++ks) along[ks] = at(l31, ks * 2 + hi);
#pragma unroll
    for (int db = 0; db < NB; ++db)
#pragma unroll
      for (int k = 0; k < 2; ++k)                // columns past HK lie in the padding: operand rows whose products are not stored
        trans[db][k] = at(8 * k + 4 * hi + (gi >> 2), db * 4 + gdh * 2 + (gi >> 1 & 1)) + (gi & 1) * 8;
  }
  template <typename V8> __device__ __forceinline__ V8 row(const win_lds* tile, int row0, int ks) const {
    return *(const __attribute__((address_space(3))) V8*)(tile + along[ks % NA] + row0 * PITCH + (NEAR ? (ks >> 1) * 64 : 0));
  }
  // Operand of a 32x32x16 MFMA whose 16-deep contraction runs over 16 LDS rows, read transposed: lane l holds column db * 32 + (l & 31)
  // of rows row0 + 4 hi + (e & 3) + 8 (e >> 2) (e = 0..7) -- the rows in which a 32x32 accumulator of the same wave holds its
  // registers, so a converted accumulator is the other operand as it stands.  row0: a multiple of 16
  template <typename V8> __device__ __forceinline__ V8 col(const win_lds* tile, int row0, int db) const {
    typedef __attribute__((address_space(3))) win_s16x4 lds4;
    const win_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + trans[NEAR ? 0 : db][0] + row0 * PITCH + (NEAR ? db * 64 : 0)));
    const win_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + trans[NEAR ? 0 : db][1] + row0 * PITCH + (NEAR ? db * 64 : 0)));
    return __builtin_bit_cast(V8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// Order of a stretch of code that holds `mfmas` MFMAs with `per` LDS reads each and nothing else of either kind: `ahead` MFMAs' reads
// first, then an MFMA and the reads of the one `ahead` places later, in turn.  (hipcc's own order puts each read right in front of its
// MFMA, so that every MFMA waits for a read's whole latency.)
template <int mfmas, int per, int ahead> __device__ __forceinline__ void win_order() {
  __builtin_amdgcn_sched_group_barrier(0x100, per * ahead, 0);
#pragma unroll
  for (int i = 0; i < mfmas - ahead; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, per, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, ahead, 0);
}

// Wait for all loads issued so far (vmcnt 0).  Put behind the loads that stay in registers for a whole loop: hipcc cannot see that they
// have arrived once loads of the loop's own are in flight on the way round, and would wait for those in every iteration.
__device__ __forceinline__ void win_loads_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// maximum / sum with the partner lane (l ^ 32).  The swap is written out: s_nop 1 covers the VALU write -> permlane read hazard, and
// through the builtin hipcc folds max(a, b) of the swapped pair to a.
__device__ __forceinline__ float win_half_max(float v) {
  float w = v;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\tv_max_f32 %0, %0, %1" : "+v"(v), "+v"(w));
  return v;
}
__device__ __forceinline__ float win_half_sum(float v) { return v + __shfl_xor(v, 32, 64); }

}  // namespace hallo
