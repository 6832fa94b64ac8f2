// K/V tiles of a paged cache in LDS (paged_chunk.hip; paged_shared.hip takes the groups, the
// read offsets and the slack): pages to 64-key tiles by buffer loads that write LDS, and a
// tile's fold into 32 query rows of a wave.  Args: a kernel's arguments, with k, k_blk, k_sh,
// k_slot (elements), the same for v, num_blocks, bt, bt_stride, max_pages, and gpb and
// per_group (groups of kGroup keys of a block, and its reciprocal).
#pragma once

#include "prefill_tile.hpp"

namespace {

constexpr float kRescaleSlack = 8.f;  // log2 headroom before the running maximum is raised
constexpr int kGroup = 16;           // keys a wave loads of a tile: inside one page

// x / d by its reciprocal: x + 1/2 over d lies 1 / (2 d) or more from every integer, far
// more than the product's rounding (3 instructions where a division takes 20, and every
// instruction before the first tile is fetched for the first time).
__device__ __forceinline__ int divide(uint32_t x, double per) {
  return static_cast<int>(__builtin_fma(static_cast<double>(x), per, 0.5 * per));
}

// 16-byte loads a lane issues of a K or V tile.
template <int W>
constexpr int dma_per_wave() { return kBN * kRowBytes / (W * 64 * 16); }
constexpr int kMaxDma = dma_per_wave<4>();

struct LaneOffsets {
  uint32_t kdma[kMaxDma], vdma[kMaxDma];  // source offsets within a group of 16 keys
  uint32_t kread, vread;
};

template <int W, typename Args>
__device__ __forceinline__ LaneOffsets lane_offsets(const Args& a, int lane, int wave) {
  LaneOffsets o;
  // Load j of wave w fills LDS rows 4 n .. 4 n + 3, n = D w + j (D loads a wave);
  // lane i writes slot i % 16 of row 4 n + i / 16, i.e. source chunk slot ^ swz(row).
  constexpr int D = dma_per_wave<W>();
#pragma unroll
  for (int j = 0; j < D; ++j) {
    const int row = (4 * (D * wave + j) + (lane >> 4)) % kGroup;
    const int slot = lane & 15;
    o.kdma[j] = static_cast<uint32_t>(row * a.k_slot * 2) + ((slot ^ (row & 15)) << 4);
    o.vdma[j] = static_cast<uint32_t>(row * a.v_slot * 2) + ((slot ^ (4 * (row & 3))) << 4);
  }
  read_offsets(o, lane);
  return o;
}

// Where the item's next 64 groups of 16 keys (16 tiles) lie, a lane each, and the 64
// after them: the page, and the group's place inside it.
struct PageWindow {
  int base;                // group of lane 0
  int32_t page, next_page;
  uint32_t sub, next_sub;
  uint64_t ok;             // groups of the window whose page is a block of the pool
};

template <typename Args>
__device__ __forceinline__ void group_at(const Args& a, int64_t row, int group, int32_t& page,
                                         uint32_t& sub) {
  const uint32_t p = divide(group, a.per_group);
  sub = static_cast<uint32_t>(group) - p * a.gpb;
  page = row >= 0 && p < a.max_pages ? a.bt[row * a.bt_stride + p] : -1;
}
template <typename Args>
__device__ __forceinline__ void window_check(PageWindow& w, const Args& a) {
  w.ok = __ballot(w.page >= 0 && w.page < a.num_blocks);
}
// (window_check before its first use: the loads may be on their way until then.)
template <typename Args>
__device__ __forceinline__ void window_start(PageWindow& w, const Args& a, int64_t row,
                                             int tile, int lane) {
  w.base = tile * (kBN / kGroup);
  group_at(a, row, w.base + lane, w.page, w.sub);
  group_at(a, row, w.base + 64 + lane, w.next_page, w.next_sub);
}
// Moves on once `tile` lies behind the window (tiles come in order).
template <typename Args>
__device__ __forceinline__ void window_to(PageWindow& w, const Args& a, int64_t row, int tile,
                                          int lane) {
  if (tile * (kBN / kGroup) < w.base + 64) return;
  w.base += 64;
  w.page = w.next_page;
  w.sub = w.next_sub;
  group_at(a, row, w.base + 64 + lane, w.next_page, w.next_sub);
  window_check(w, a);
}

// An item's keys.
struct ItemKeys {
  const uint16_t* k;  // the KV head of block 0
  const uint16_t* v;
  int64_t row;        // of the block table
  int cap;            // keys of the sequence
};

// Issues this wave's share of the loads of key tile `tile` into (sk, sv).  Returns
// which of the tile's four groups lie in the pool's blocks.
template <int W, typename Args>
__device__ __forceinline__ uint32_t tile_dma(const Args& a, const LaneOffsets& off,
                                             PageWindow& w, const ItemKeys& ks, int tile,
                                             uint16_t* sk, uint16_t* sv, int wave, int lane) {
  window_to(w, a, ks.row, tile, lane);
  const int g0 = tile * (kBN / kGroup) - w.base;
  const int g = wave * (kBN / kGroup) / W;  // this wave's group
  const int64_t page = __builtin_amdgcn_readlane(w.page, g0 + g);
  const int sub = __builtin_amdgcn_readlane(w.sub, g0 + g) * kGroup;
  const uint32_t ok = static_cast<uint32_t>(w.ok >> g0) & 15u;
  const int rows = (ok >> g) & 1u ? min(kGroup, ks.cap - tile * kBN - g * kGroup) : 0;
  const uint16_t* kb = ks.k;
  const uint16_t* vb = ks.v;
  if (rows > 0) {
    kb += page * a.k_blk + static_cast<int64_t>(sub) * a.k_slot;
    vb += page * a.v_blk + static_cast<int64_t>(sub) * a.v_slot;
  }
  // rows behind the last key lie outside the descriptor and read as zero
  const int k_bytes = rows > 0 ? (rows - 1) * a.k_slot * 2 + kRowBytes : 0;
  const int v_bytes = rows > 0 ? (rows - 1) * a.v_slot * 2 + kRowBytes : 0;
  const __amdgpu_buffer_rsrc_t kr =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(kb), 0, k_bytes, 0x00020000);
  const __amdgpu_buffer_rsrc_t vr =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(vb), 0, v_bytes, 0x00020000);
  constexpr int D = dma_per_wave<W>();
#pragma unroll
  for (int j = 0; j < D; ++j) {
    const int blk = (D * wave + j) * 512;  // elements: 1 KiB per load
    __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void_t*)(sk + blk), 16, off.kdma[j], 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void_t*)(sv + blk), 16, off.vdma[j], 0, 0, 0);
  }
  return ok;
}

// One 64-key tile (staged in kt / vt) folded into this wave's online softmax
// state; c: the softmax scale times log2(e).  mask(s) sets the scores of masked
// keys to -inf: s[kb][r] of a lane is key 32 kb + 8 (r / 4) + r % 4 + 4 (lane / 32)
// of the tile.
template <typename Off, typename Mask>
__device__ __forceinline__ void tile_fold(const Off& off, float c, const Mask& mask,
                                          const uint16_t* kt, const uint16_t* vt, const q3::bf16x8 (&qv)[8],
                                          float& m_run, float& l_run, q3::f32x16 (&acc)[4]) {
  // ---- S^T = K Q^T for two 32-key blocks ----
  // Step u covers key block u % 2, dims 16 (u / 2) .. +15; the two blocks'
  // chains alternate and K operands are read kAhead steps ahead (the scheduling
  // fences keep that distance).
  q3::f32x16 s[2];
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
  {
    q3::bf16x8 kf[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) kf[u] = lds_ld16(kt, qk_operand(off, u));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      s[u & 1] = q3::mfma32x32x16(kf[u % kAhead], qv[u >> 1], s[u & 1]);
      if (u + kAhead < 16) kf[u % kAhead] = lds_ld16(kt, qk_operand(off, u + kAhead));
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  mask(s);
  // Row max as a v_max3 chain over the lane's 32 scores.  The scores were
  // written by the QK MFMAs just above: 24 wait states cover the
  // MFMA-to-VALU dependency.
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");
  float bm = max3_scores(s);
  bm = cross_half_max(bm);
  const float m_cand = bm * c;
  const bool raise = m_cand > m_run + kRescaleSlack;
  if (__any(raise)) {
    const float m_new = raise ? m_cand : m_run;
    const float alpha = raise ? q3::fast_exp2(m_run - m_new) : 1.f;
    m_run = m_new;
    l_run *= alpha;
#pragma unroll
    for (int db = 0; db < 4; ++db) acc[db] *= alpha;
  }
  // V^T operands of the first PV steps are read before the exponentials,
  // which hide their latency.
  q3::bf16x8 vf[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) vf[u] = lds_vt(vt, pv_operand(off, u));
  __builtin_amdgcn_sched_barrier(0);
  const float m_use = m_run == q3::kNegInf ? 0.f : m_run;
  // ---- P = exp2(s * c - m) as P^T B operands (chunk g = 2 kb + kc:
  // scores s[kb][8 kc .. 8 kc + 7]) and O^T += V^T P^T, step u covering
  // key chunk u / 4, dims 32 (u % 4) .. +31.  Chunk 0 is computed first;
  // the exponentials of chunk g + 1 are issued between the four MFMAs of
  // chunk g, two per step, so the VALU works while the matrix core runs.
  q3::u32x4 pk[4];
  float psum[4];  // four independent sum chains, started by chunk 0
  auto exp_pair = [&](int g, int h) {  // scores 2h, 2h + 1 of chunk g
    const int kb = g >> 1, kc = g & 1;
    const float e0 = q3::fast_exp2(__builtin_fmaf(s[kb][8 * kc + 2 * h], c, -m_use));
    const float e1 = q3::fast_exp2(__builtin_fmaf(s[kb][8 * kc + 2 * h + 1], c, -m_use));
    if (g == 0 && h < 2) {
      psum[2 * h] = e0;
      psum[2 * h + 1] = e1;
    } else {
      psum[(2 * h) & 3] += e0;
      psum[(2 * h + 1) & 3] += e1;
    }
    pk[g][h] = q3::pack_bf16x2(e0, e1);
  };
#pragma unroll
  for (int h = 0; h < 4; ++h) exp_pair(0, h);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    acc[u & 3] = q3::mfma32x32x16(vf[u % kAhead], q3::as_bf16x8(pk[u >> 2]), acc[u & 3]);
    if (u + kAhead < 16) vf[u % kAhead] = lds_vt(vt, pv_operand(off, u + kAhead));
    if (u < 12) exp_pair((u >> 2) + 1, u & 3);
    __builtin_amdgcn_sched_barrier(0);
  }
  l_run += (psum[0] + psum[1]) + (psum[2] + psum[3]);
}

}  // namespace
