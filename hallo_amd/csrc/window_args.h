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
  int nrb, nsplit; float* part;
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

// LDS row pitches in bytes for rows of HK elements (a multiple of 16).  Rows that are only read as MFMA fragments along the row (16
// bytes per lane, lane = row): an odd number of 16-byte slots, so consecutive rows start on different banks.  Rows that are read
// transposed (4 rows x 32 bytes per 16 lanes): twice an odd number, so that those four pieces are on different banks.
constexpr int win_pitch_row(int HK) { return HK * 2 + 16; }
constexpr int win_pitch_tr(int HK) { return HK * 2 + ((HK / 16) % 2 ? 0 : 32); }

// Operand of a 32x32x16 MFMA whose 16-deep contraction runs over 16 LDS rows, read transposed: lane l holds column
// col0 + (l & 31) of rows row0 + 4 hi + (e & 3) + 8 (e >> 2) (hi = l >> 5, e = 0..7) -- the rows in which a 32x32 accumulator of the
// same wave holds its registers, so a converted accumulator is the other operand as it stands.
// `base`: tile + ((l >> 5) * 4 + ((l & 15) >> 2)) * pitch + (l & 3) * 8 ; colb: byte offset of this lane's 16-column group
template <typename V8, int PITCH>
__device__ __forceinline__ V8 win_tr8(const win_lds* base, int row0, int colb) {
  const win_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) win_s16x4*)(base + row0 * PITCH + colb));
  const win_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) win_s16x4*)(base + (row0 + 8) * PITCH + colb));
  return __builtin_bit_cast(V8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// maximum / sum with the partner lane (l ^ 32).  The swap is written out: s_nop 1 covers the VALU write -> permlane read hazard, and
// through the builtin hipcc folds max(a, b) of the swapped pair to a.
__device__ __forceinline__ float win_half_max(float v) {
  float w = v;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\tv_max_f32 %0, %0, %1" : "+v"(v), "+v"(w));
  return v;
}
__device__ __forceinline__ float win_half_sum(float v) { return v + __shfl_xor(v, 32, 64); }

}  // namespace hallo
