// What the prefill kernels (varlen_prefill.hip, paged_chunk.hip) share of their
// 64-key tile: K and V staged in LDS, read as operands of mfma_f32_32x32x16_bf16.
//
//  * LDS tile layout: 64 key rows of 256 B, the 16-byte chunk c of row r at
//    slot c ^ swz(r).  K uses swz = r % 16 (the QK operand reads one chunk
//    of 16 consecutive rows per LDS cycle); V uses swz = 4 (r % 4) (the PV
//    operand reads 64 B of 4 consecutive rows).  Both are conflict-free.
//  * Off: a lane's LDS offsets kread and vread (read_offsets).
#pragma once

#include "common.hpp"

namespace {

constexpr int kD = 128;
constexpr int kBN = 64;                   // keys per staged K/V tile
constexpr int kRowBytes = kD * 2;         // one staged key row (256 B)
constexpr int kTileElems = kBN * kD;      // one staged K or V tile (16 KiB)

typedef __attribute__((address_space(3))) void lds_void_t;
typedef short i16x4 __attribute__((__vector_size__(4 * sizeof(short))));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4_t;

// This lane's LDS offsets of the two MFMA operands.
template <typename Off>
__device__ __forceinline__ void read_offsets(Off& o, int lane) {
  // QK A operand (mfma 32x32x16): lane reads key row lane % 32, chunk 2t + lane / 32
  // at chunk (2t + h) ^ (r % 16) = (h ^ (r % 16)) ^ 2t: d step t is kread ^ (t << 5)
  // (the XOR stays inside the row's 256 bytes).
  const int r = lane & 31, h = lane >> 5;
  o.kread = r * kRowBytes + ((h ^ (r & 15)) << 4);
  // PV A operand (V^T) through ds_read_b64_tr_b16: in 16-lane group g, lane
  // m supplies row 4 (g / 2) + m / 4 (+ 8 for the second read, + 16 per key
  // chunk) and dims 32 db + 16 (g % 2) + 4 (m % 4) .. +3.
  // Slot 4 (db ^ (m / 4)) + ..: d block db is vread ^ (db << 6).
  const int g = lane >> 4, m = lane & 15;
  const int vrow = 4 * (g >> 1) + (m >> 2);
  const int slot = 4 * (m >> 2) + 2 * (g & 1) + ((m & 3) >> 1);
  o.vread = vrow * kRowBytes + slot * 16 + 8 * (m & 1);
}

__device__ __forceinline__ q3::bf16x8 lds_ld16(const uint16_t* base, uint32_t byte_off) {
  return q3::as_bf16x8(
      *reinterpret_cast<const q3::u32x4*>(reinterpret_cast<const char*>(base) + byte_off));
}

// V^T operand: two transposing 8-byte reads (keys +0..3 and +8..11 of the
// lane half's key set).
__device__ __forceinline__ q3::bf16x8 lds_vt(const uint16_t* base, uint32_t byte_off) {
  const char* p = reinterpret_cast<const char*>(base) + byte_off;
  const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(p));
  const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(p + 8 * kRowBytes));
  typedef short i16x8 __attribute__((__vector_size__(8 * sizeof(short))));
  const i16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(q3::bf16x8, both);
}

// LDS operand distance of the MFMA loops (steps read ahead).
constexpr int kAhead = 2;

// Byte offset of the K operand of QK step u (key block u % 2, d step u / 2).
template <typename Off>
__device__ __forceinline__ uint32_t qk_operand(const Off& off, int u) {
  return (off.kread ^ static_cast<uint32_t>((u >> 1) << 5)) + (u & 1) * 32 * kRowBytes;
}

// Byte offset of the V^T operand of PV step u (key chunk u / 4, d block u % 4).
template <typename Off>
__device__ __forceinline__ uint32_t pv_operand(const Off& off, int u) {
  return (off.vread ^ static_cast<uint32_t>((u & 3) << 6)) + (u >> 2) * 16 * kRowBytes;
}

// Maximum of the 32 scores s[0..1][0..15] of one lane: four interleaved
// v_max3 chains of eight scores and a final combine (depth 6).  Written as
// one asm block because fmaxf would first canonicalize every MFMA result;
// a NaN score makes P, and so the output, NaN either way.
__device__ __forceinline__ float max3_scores(const q3::f32x16 (&s)[2]) {
  const q3::f32x16& a = s[0];
  const q3::f32x16& b = s[1];
  float m, t1, t2, t3;
  asm volatile(
      "v_max3_f32 %0, %4, %5, %6\n\t"
      "v_max3_f32 %1, %12, %13, %14\n\t"
      "v_max3_f32 %2, %20, %21, %22\n\t"
      "v_max3_f32 %3, %28, %29, %30\n\t"
      "v_max3_f32 %0, %0, %7, %8\n\t"
      "v_max3_f32 %1, %1, %15, %16\n\t"
      "v_max3_f32 %2, %2, %23, %24\n\t"
      "v_max3_f32 %3, %3, %31, %32\n\t"
      "v_max3_f32 %0, %0, %9, %10\n\t"
      "v_max3_f32 %1, %1, %17, %18\n\t"
      "v_max3_f32 %2, %2, %25, %26\n\t"
      "v_max3_f32 %3, %3, %33, %34\n\t"
      "v_max3_f32 %0, %0, %11, %19\n\t"
      "v_max3_f32 %2, %2, %27, %35\n\t"
      "v_max3_f32 %0, %0, %1, %2\n\t"
      "v_max_f32 %0, %0, %3"
      : "=&v"(m), "=&v"(t1), "=&v"(t2), "=&v"(t3)
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]),
        "v"(a[8]), "v"(a[9]), "v"(a[10]), "v"(a[11]), "v"(a[12]), "v"(a[13]), "v"(a[14]),
        "v"(a[15]), "v"(b[0]), "v"(b[1]), "v"(b[2]), "v"(b[3]), "v"(b[4]), "v"(b[5]), "v"(b[6]),
        "v"(b[7]), "v"(b[8]), "v"(b[9]), "v"(b[10]), "v"(b[11]), "v"(b[12]), "v"(b[13]),
        "v"(b[14]), "v"(b[15]));
  return m;
}

// x combined with the value lane l ^ 32 holds: v_permlane32_swap of x with
// itself leaves the lower-half value in r[0] and the upper-half value in
// r[1] on every lane.
__device__ __forceinline__ float cross_half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float cross_half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ void wait_loads() {
  // vmcnt(0) with expcnt / lgkmcnt left at their maxima.
  __builtin_amdgcn_s_waitcnt(0x0f70);
}

}  // namespace
