// Attention of a chunk of new tokens over the paged cache, for gfx950 (GQA).
//
// Sequence s of the batch has n_s new tokens, packed in q from row cu[s], and
// c_s = seq_lens[row_s] tokens before them; the new tokens' keys and values are
// in its pages already.  Token i attends the keys j <= c_s + i of its row of the
// block table:
//   o_i = sum_j exp(scale q_i k_j) v_j / sum_j exp(scale q_i k_j),
// in one pass with a running maximum and sum in fp32; here P is rounded to bf16 for
// the PV product, as in the prefill (a relative error of at most 2^-8 per term of a
// weighted mean), the output once to bf16.  A row without keys is zero.  P as two bf16
// terms, as paged_chunk_stream.hip carries it where loads are the bound, is a second PV
// product here: 2,048 tokens behind 64,000 2.00 -> 2.69 ms, 509 behind 12,000 115 -> 149 us,
// 40 behind 100,000 113 -> 138, twelve turns 160 -> 197.  One term: outputs 0.0023 off 64 bits
// (root mean square, relative), of which 0.0017 are their own rounding.
//
//  * Query rows of one KV head are packed: row r is token r / G, head r % G of
//    the group, so one staged K/V tile serves every head of the group whatever
//    G is.  A work item is (sequence, KV head, 128 or 256 packed rows); each of the
//    four or eight waves of a workgroup owns 32 of them.
//  * K/V tiles of 64 keys go from HBM into LDS by buffer loads that write LDS,
//    16 or 8 keys a wave, so a wave reads one page per tile: its base is a scalar and
//    the lanes' offsets never change.  The descriptor ends at the sequence's
//    last key (or holds nothing where the table names no page of the pool), so
//    slots behind it are never read.  Page ids come 64 at a time into a
//    register (16 tiles' worth), the next 64 before they are needed.
//
// Long chunks are bound by the matrix cores and the softmax's VALU work, which the two
// waves of a SIMD do largely in turns: 2,048 tokens behind 64,000, 32/8 heads, 1.95-2.05
// ms, 1,063-1,127 TFLOP/s (an 8,192-cubed library product: 1,159), 55% MFMA-busy.  Few
// rows behind much are bound by HBM (40 tokens behind 100,000: 107 us for 410 MB, and 10
// of joins), few rows behind little by the chain of loads before the first tile, about 9
// us, and a second launch.
#include <algorithm>

#include "paged_chunk_stream.hpp"
#include "prefill_tile.hpp"

namespace {

// Workgroups of W = 4 or 8 waves: packed query rows of an item.
template <int W>
constexpr int rows_of() { return 32 * W; }
constexpr int kMaxG = 16;
constexpr float kRescaleSlack = 8.f;  // log2 headroom before the running maximum is raised
constexpr int kGroup = 16;           // keys a wave loads of a tile: inside one page

// A cut item, noted by the range v that holds its first tile: its parts lie in slot
// 2 v + 1 and in slots 2 (v + 1), 2 (v + 2), ... of the next ranges.
struct CutItem {
  int32_t parts;  // 0: this range holds no cut item's first tile
  int32_t rows;   // packed rows of the item
  int32_t r0;     // the first one
  int32_t kvh;
  int64_t q0;     // first row of q of its sequence
};

struct ChunkArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint16_t* k;
  int64_t k_blk, k_sh;
  int k_slot;
  const uint16_t* v;
  int64_t v_blk, v_sh;
  int v_slot;
  int64_t num_blocks;
  const int32_t* bt;
  int64_t bt_stride, max_rows, max_pages;
  const int32_t* seq_lens;
  const int32_t* row_ids;  // nullable: identity
  const int32_t* cu;
  uint16_t* o;
  int64_t o_st, o_sh;
  int64_t total;   // rows of q
  int B, Hkv, G;
  int gpb;         // groups of kGroup keys of a block
  int reach;       // positions that a row of the table addresses
  int n_mtiles;    // items of the longest chunk of one KV head
  double per_head, per_group;  // 1 / G, 1 / gpb
  float scale_log2;
  // range schedule
  double per_range;  // 1 / ranges
  float* po;       // [2 ranges][rows][kD] partial outputs, not normalised, 32 rows mixed
  float2* pml;     // [2 ranges][rows] their running maximum (log2 domain) and sum
  CutItem* cuts;   // [ranges]
};

// x / d by its reciprocal: x + 1/2 over d lies 1 / (2 d) or more from every integer, far
// more than the product's rounding (3 instructions where a division takes 20, and every
// instruction before the first tile is fetched for the first time).
__device__ __forceinline__ int divide(uint32_t x, double per) {
  return static_cast<int>(__builtin_fma(static_cast<double>(x), per, 0.5 * per));
}

// One sequence of the batch.
struct Seq {
  int64_t q0;   // its first row of q
  int n;        // its new tokens (0: nothing is computed)
  int64_t row;  // its row of the block table, -1: none
  int ctx;      // tokens before the new ones
  int cap;      // keys that may be attended: at most what its tokens reach and a row holds
};

// The same, as a table keeps it.
struct SeqEntry {
  int32_t q0, n, row, ctx;
};

__device__ __forceinline__ Seq seq_of(const ChunkArgs& a, const SeqEntry& e) {
  Seq s{e.q0, e.n, e.row, e.ctx, 0};
  const int64_t len = static_cast<int64_t>(e.ctx) + e.n;
  const int cap = static_cast<int>(len < a.reach ? len : a.reach);
  s.cap = e.row >= 0 && cap > 0 ? cap : 0;
  return s;
}

__device__ __forceinline__ Seq seq_at(const ChunkArgs& a, int b) {
  const int64_t s0 = a.cu[b], s1 = a.cu[b + 1];
  const int64_t row = a.row_ids ? a.row_ids[b] : b;
  const bool ok = s0 >= 0 && s1 > s0 && s1 <= a.total;
  const bool listed = row >= 0 && row < a.max_rows;
  SeqEntry e;
  e.q0 = ok ? static_cast<int32_t>(s0) : 0;
  e.n = ok ? static_cast<int32_t>(s1 - s0) : 0;
  e.row = listed ? static_cast<int32_t>(row) : -1;
  e.ctx = listed ? a.seq_lens[row] : 0;
  return seq_of(a, e);
}

// Keys that packed rows r0 .. r1 - 1 of a sequence reach.
__device__ __forceinline__ int keys_of(const ChunkArgs& a, const Seq& s, int r1) {
  const int tokens = min(s.n, divide(r1 + a.G - 1, a.per_head));
  const int64_t reach = static_cast<int64_t>(s.ctx) + tokens;
  return static_cast<int>(reach < 0 ? 0 : reach < s.cap ? reach : s.cap);
}

struct TileBufs {
  uint16_t* k0;
  uint16_t* v0;
  uint16_t* k1;
  uint16_t* v1;
};

// 16-byte loads a lane issues of a K or V tile.
template <int W>
constexpr int dma_per_wave() { return kBN * kRowBytes / (W * 64 * 16); }
constexpr int kMaxDma = dma_per_wave<4>();

struct LaneOffsets {
  uint32_t kdma[kMaxDma], vdma[kMaxDma];  // source offsets within a group of 16 keys
  uint32_t kread, vread;
};

template <int W>
__device__ __forceinline__ LaneOffsets lane_offsets(const ChunkArgs& a, int lane, int wave) {
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

__device__ __forceinline__ void group_at(const ChunkArgs& a, int64_t row, int group, int32_t& page,
                                         uint32_t& sub) {
  const uint32_t p = divide(group, a.per_group);
  sub = static_cast<uint32_t>(group) - p * a.gpb;
  page = row >= 0 && p < a.max_pages ? a.bt[row * a.bt_stride + p] : -1;
}
__device__ __forceinline__ void window_check(PageWindow& w, const ChunkArgs& a) {
  w.ok = __ballot(w.page >= 0 && w.page < a.num_blocks);
}
// (window_check before its first use: the loads may be on their way until then.)
__device__ __forceinline__ void window_start(PageWindow& w, const ChunkArgs& a, int64_t row,
                                             int tile, int lane) {
  w.base = tile * (kBN / kGroup);
  group_at(a, row, w.base + lane, w.page, w.sub);
  group_at(a, row, w.base + 64 + lane, w.next_page, w.next_sub);
}
// Moves on once `tile` lies behind the window (tiles come in order).
__device__ __forceinline__ void window_to(PageWindow& w, const ChunkArgs& a, int64_t row, int tile,
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
template <int W>
__device__ __forceinline__ uint32_t tile_dma(const ChunkArgs& a, const LaneOffsets& off,
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

// A wave's 32 packed rows: lane l holds row r0 + l % 32.
struct WaveRows {
  int r0;         // first packed row
  int tok, head;  // this lane's token and head of the group
  int last;       // last key of this lane's token (-1: none)
  int lo, hi;     // least and greatest such key of the wave's rows (uniform)
  bool active;    // the wave has rows of the sequence
};

template <int W>
__device__ __forceinline__ WaveRows wave_rows(const ChunkArgs& a, const Seq& s, int mt, int wave,
                                              int lane) {
  WaveRows w;
  w.r0 = mt * rows_of<W>() + wave * 32;
  const int r = w.r0 + (lane & 31);
  w.tok = divide(r, a.per_head);
  w.head = r - w.tok * a.G;
  auto last = [&](int tok) {
    const int64_t p = static_cast<int64_t>(s.ctx) + min(tok, s.n - 1);
    return static_cast<int>(p < s.cap - 1 ? (p < -1 ? -1 : p) : s.cap - 1);
  };
  w.last = last(w.tok);
  w.lo = last(divide(w.r0, a.per_head));
  w.hi = last(divide(w.r0 + 31, a.per_head));
  w.active = w.r0 < s.n * a.G;
  return w;
}

__device__ __forceinline__ void load_q(const ChunkArgs& a, const Seq& s, const WaveRows& w,
                                       int kvh, int lane, q3::bf16x8 (&qv)[8]) {
  const bool ok = w.tok < s.n;
  const uint16_t* p = a.q + (s.q0 + (ok ? w.tok : 0)) * a.q_st +
                      (static_cast<int64_t>(kvh) * a.G + (ok ? w.head : 0)) * a.q_sh +
                      8 * (lane >> 5);
#pragma unroll
  for (int c = 0; c < 8; ++c)
    qv[c] = q3::as_bf16x8(ok ? q3::ld16(p + 16 * c) : q3::u32x4{0u, 0u, 0u, 0u});
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

// Key tiles [t0, t1) of an item folded into a fresh state; pw: window_start of t0.  Every
// thread of the workgroup calls it; the tile buffers are free when it returns.
template <int W>
__device__ __forceinline__ void run_tiles(const ChunkArgs& a, const LaneOffsets& off, const Seq& s,
                                          const WaveRows& w, int kvh, int t0, int t1,
                                          PageWindow pw, const TileBufs& tb, int lane, int wave,
                                          float& m_run, float& l_run, q3::f32x16 (&acc)[4]) {
  m_run = q3::kNegInf;
  l_run = 0.f;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;
  if (t0 >= t1) return;
  window_check(pw, a);
  const ItemKeys ks{a.k + kvh * a.k_sh, a.v + kvh * a.v_sh, s.row, s.cap};
  uint32_t ok = tile_dma<W>(a, off, pw, ks, t0, tb.k0, tb.v0, wave, lane);
  q3::bf16x8 qv[8];
  load_q(a, s, w, kvh, lane, qv);
  wait_loads();
  __syncthreads();
  auto tile = [&](int it, const uint16_t* kt, const uint16_t* vt, uint16_t* nk, uint16_t* nv) {
    const uint32_t here = ok;
    if (it + 1 < t1) ok = tile_dma<W>(a, off, pw, ks, it + 1, nk, nv, wave, lane);
    const int n0 = it * kBN;
    if (w.active && n0 <= w.hi) {
      auto mask = [&](q3::f32x16 (&x)[2]) {
        if (n0 + kBN - 1 > w.lo || here != 15u) {
          // score (kb, r): key n0 + 4 (lane / 32) + kr of group 2 kb + r / 8
          const int lim = w.last - n0 - 4 * (lane >> 5);
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int kr = kb * 32 + 8 * (r / 4) + (r % 4);
              const int l = (here >> (2 * kb + r / 8)) & 1u ? lim : -1;
              x[kb][r] = kr <= l ? x[kb][r] : q3::kNegInf;
            }
        }
      };
      tile_fold(off, a.scale_log2, mask, kt, vt, qv, m_run, l_run, acc);
    }
    wait_loads();
    __syncthreads();
  };
  for (int it = t0; it < t1; it += 2) {
    tile(it, tb.k0, tb.v0, tb.k1, tb.v1);
    if (it + 1 < t1) tile(it + 1, tb.k1, tb.v1, tb.k0, tb.v0);
  }
}

// Normalises this wave's rows (l: a row's full sum) and writes those of the
// sequence, through 8 KiB of LDS at `stage` so that 16 lanes write a head row.
__device__ __forceinline__ void store_output(const ChunkArgs& a, const Seq& s, const WaveRows& w,
                                             int kvh, int lane, float l,
                                             const q3::f32x16 (&acc)[4], char* stage) {
  const int l32 = lane & 31, hl = lane >> 5;
  const float inv = l > 0.f ? 1.f / l : 0.f;  // 0: no key
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const int ch = 4 * db + g4;
      q3::u32x2 x = {q3::pack_bf16x2(acc[db][4 * g4] * inv, acc[db][4 * g4 + 1] * inv),
                     q3::pack_bf16x2(acc[db][4 * g4 + 2] * inv, acc[db][4 * g4 + 3] * inv)};
      *reinterpret_cast<q3::u32x2*>(stage + l32 * 256 + ((ch ^ (l32 & 15)) << 4) + hl * 8) = x;
    }
  const int oc = lane & 15;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int rr = 4 * j + (lane >> 4);
    const q3::u32x4 x =
        *reinterpret_cast<const q3::u32x4*>(stage + rr * 256 + ((oc ^ (rr & 15)) << 4));
    const int r = w.r0 + rr;
    const int tok = divide(r, a.per_head);
    if (tok < s.n)
      q3::st16(a.o + (s.q0 + tok) * a.o_st +
                   (static_cast<int64_t>(kvh) * a.G + (r - tok * a.G)) * a.o_sh + 8 * oc,
               x);
  }
}

__device__ __forceinline__ char* stage_of(const TileBufs& tb, int wave) {
  const int sb = wave >> 1;
  return reinterpret_cast<char*>(sb == 0 ? tb.k0 : sb == 1 ? tb.v0 : sb == 2 ? tb.k1 : tb.v1) +
         (wave & 1) * 8192;
}

#define Q3_CHUNK_TILE_BUFFERS                                          \
  __shared__ __attribute__((aligned(1024))) uint16_t s_k0[kTileElems]; \
  __shared__ __attribute__((aligned(1024))) uint16_t s_v0[kTileElems]; \
  __shared__ __attribute__((aligned(1024))) uint16_t s_k1[kTileElems]; \
  __shared__ __attribute__((aligned(1024))) uint16_t s_v1[kTileElems]; \
  const TileBufs tb{s_k0, s_v0, s_k1, s_v1}

// Batches that no workgroup can tabulate: one workgroup per item, KV head fastest
// (neighbouring workgroups go to different XCDs, and an XCD's L2 holds few heads), the
// last row tiles first.
template <int W>
__global__ __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_chunk_flat_kernel(ChunkArgs a) {
  Q3_CHUNK_TILE_BUFFERS;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t id = blockIdx.x, per_tile = static_cast<uint32_t>(a.Hkv) * a.B;
  const int mt = a.n_mtiles - 1 - static_cast<int>(id / per_tile);
  const uint32_t rest = id % per_tile;
  const int b = static_cast<int>(rest / a.Hkv);
  const int kvh = static_cast<int>(rest % a.Hkv);
  const Seq s = seq_at(a, b);
  if (mt * rows_of<W>() >= static_cast<int64_t>(s.n) * a.G) return;
  const LaneOffsets off = lane_offsets<W>(a, lane, wave);
  const WaveRows w = wave_rows<W>(a, s, mt, wave, lane);
  const int tiles = (keys_of(a, s, (mt + 1) * rows_of<W>()) + kBN - 1) / kBN;
  float m_run, l_run;
  q3::f32x16 acc[4];
  PageWindow pw;
  window_start(pw, a, s.row, 0, lane);
  run_tiles<W>(a, off, s, w, kvh, 0, tiles, pw, tb, lane, wave, m_run, l_run, acc);
  l_run = cross_half_sum(l_run);
  if (w.active) store_output(a, s, w, kvh, lane, l_run, acc, stage_of(tb, wave));
}

// ---------------------------------------------------------------------------
// Range schedule: too few items for the device (a few long contexts).  The items'
// key tiles, each of weight kUnits, with kItemUnits for an item's start and end, lie
// end to end, KV head by KV head; they are cut into equal ranges, one per resident
// workgroup.  Neighbouring ranges run on one XCD, so its L2 serves one KV head.  A
// tile belongs to the range that holds its midpoint.  An item cut by a border leaves
// a partial state per part, which a second launch joins: with up to a part for each
// workgroup, joining inside one of them would take as long as the tiles.
// A range is at least kMinRangeTiles long, where few rows meet few keys: 202 tokens
// behind 53 take 21.1 us with four tiles, 17.7 with two, 17.1 with one, seven sequences
// of 6 tokens behind 300 keys 19.7, 18.6 and 23.7.
constexpr int kUnits = 16;          // a tile with more than four waves' rows, or of W = 4
constexpr int kFewUnits = 12;       // a tile of W = 8 that no SIMD computes two waves of
constexpr int kItemUnits = 40;
constexpr int kMinRangeTiles = 2;
constexpr int kWholeSlack = 20;     // an uncut item: one part in 20, and six tiles, above
constexpr int kWholeUnits = 96;     // an equal share
constexpr int kMaxSeqs = 256;       // sequences and (sequence, row tile) pairs
constexpr int kMaxEntries = 1024;   // tabulated in LDS

// A key tile's weight in an item of `rows` packed rows.
template <int W>
__device__ __forceinline__ int tile_units(int rows) {
  return W == 8 && rows <= rows_of<4>() ? kFewUnits : kUnits;
}

// Exclusive prefix sum of v[0 .. n) in LDS, in place, n <= kMaxEntries; returns the
// total.  Every thread of the workgroup calls it.
template <int W, typename T>
__device__ __forceinline__ T block_scan(T* v, int n, T* s_wsum) {
  constexpr int kPer = kMaxEntries / (W * 64);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  T x[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    x[i] = tid * kPer + i < n ? v[tid * kPer + i] : 0;
    sum += x[i];
  }
  T incl;
  if constexpr (sizeof(T) == 8)  // a thread's weights are below 2^31, a wave's in two halves
    incl = (static_cast<int64_t>(q3::wave_prefix_sum(static_cast<int>(sum >> 16))) << 16) +
           q3::wave_prefix_sum(static_cast<int>(sum & 0xffff));
  else
    incl = q3::wave_prefix_sum(sum);
  if (lane == 63) s_wsum[wave] = incl;
  __syncthreads();
  T run = incl - sum, total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    run += w < wave ? s_wsum[w] : 0;
    total += s_wsum[w];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (tid * kPer + i < n) v[tid * kPer + i] = run;
    run += x[i];
  }
  __syncthreads();
  return total;
}

// Largest index i < n with v[i] <= p (v ascending, v[0] <= p).
template <typename T>
__device__ __forceinline__ int last_at_most(const T* v, int n, T p) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (v[mid] <= p) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// floor(x / y) below 2^20, x >= 0: an estimate in 32 bits, less than one off, put right.
__device__ __forceinline__ int quotient(int64_t x, int64_t y) {
  int q = static_cast<int>(static_cast<float>(x) * __builtin_amdgcn_rcpf(static_cast<float>(y)));
  if (q * y > x) --q;
  if ((q + 1) * y <= x) ++q;
  return __builtin_amdgcn_readfirstlane(q);
}

// Tabulates the batch, its sequences and the row tiles before each; returns the row tiles
// of all.  Every workgroup waits for this before its first K/V load: one chain of two
// memory round trips (row_ids, then seq_lens), the rest is in LDS.
template <int W>
__device__ __forceinline__ int tabulate(const ChunkArgs& a, int* s_first, SeqEntry* s_seq,
                                        int* s_wsum) {
  for (int b = threadIdx.x; b < a.B; b += W * 64) {
    const Seq s = seq_at(a, b);
    s_seq[b] = SeqEntry{static_cast<int32_t>(s.q0), s.n, static_cast<int32_t>(s.row), s.ctx};
    s_first[b] = static_cast<int>((static_cast<int64_t>(s.n) * a.G + rows_of<W>() - 1) / rows_of<W>());
  }
  __syncthreads();
  // (the bound matters only where cu_seqlens is not ascending)
  return min(kMaxEntries, block_scan<W, int>(s_first, a.B, s_wsum));
}

// A tabulated sequence, in scalar registers.
__device__ __forceinline__ Seq tabulated(const ChunkArgs& a, SeqEntry se) {
  se.q0 = __builtin_amdgcn_readfirstlane(se.q0);
  se.n = __builtin_amdgcn_readfirstlane(se.n);
  se.row = __builtin_amdgcn_readfirstlane(se.row);
  se.ctx = __builtin_amdgcn_readfirstlane(se.ctx);
  return seq_of(a, se);
}

template <int W>
__global__ __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_chunk_range_kernel(ChunkArgs a) {
  Q3_CHUNK_TILE_BUFFERS;
  __shared__ int64_t s_pos[kMaxEntries];  // weight before each (sequence, row tile)
  __shared__ int s_first[kMaxSeqs];       // row tiles before each sequence
  __shared__ SeqEntry s_seq[kMaxSeqs];
  __shared__ uint8_t s_of[kMaxEntries];   // a pair's sequence
  static_assert(kMaxSeqs <= 256, "s_of holds a sequence");
  __shared__ int64_t s_wsum[W];
  __shared__ int s_most;                  // key tiles of the longest item
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (tid == 0) s_most = 0;
  const int E = tabulate<W>(a, s_first, s_seq, reinterpret_cast<int*>(s_wsum));
  for (int e = tid; e < E; e += W * 64) {
    const int b = last_at_most(s_first, a.B, e);
    const Seq s = seq_of(a, s_seq[b]);
    const int mt = e - s_first[b];
    const int tiles = (keys_of(a, s, (mt + 1) * rows_of<W>()) + kBN - 1) / kBN;
    s_of[e] = static_cast<uint8_t>(b);
    s_pos[e] = static_cast<int64_t>(tile_units<W>(s.n * a.G - mt * rows_of<W>())) * tiles + kItemUnits;
    atomicMax(&s_most, tiles);
  }
  __syncthreads();
  const int64_t H = block_scan<W, int64_t>(s_pos, E, s_wsum);
  const int nwg = gridDim.x;
  const int64_t U = H * a.Hkv;
  // a range's width: every workgroup's share (its product with the workgroups is U or more:
  // the rounding below is far less than the step to the next multiple), at least
  // kMinRangeTiles tiles
  const int64_t share = static_cast<int64_t>(static_cast<double>(U) * a.per_range) + 1;
  const int64_t width = share < kMinRangeTiles * kUnits ? kMinRangeTiles * kUnits : share;
  const int w = blockIdx.x;
  // Items that are no more than the workgroups and nearly as long as each other are not
  // cut: the longest takes little more than an equal share, and a cut costs its saves
  // and the second launch's reads (2,048 tokens behind 64,000: 1.92 ms against 2.04).
  const int64_t longest = static_cast<int64_t>(kUnits) * s_most + kItemUnits;
  const bool whole = static_cast<int64_t>(E) * a.Hkv <= nwg &&
                     longest <= share + share / kWholeSlack + kWholeUnits;
  const int v = (whole || width == share) && nwg % 8 == 0 ? (w % 8) * (nwg / 8) + w / 8 : w;
  int64_t p_lo = v * width < U ? v * width : U;
  int64_t p_hi = p_lo + width < U ? p_lo + width : U;
  if (whole) {
    const int kvh = E > 0 ? v / E : a.Hkv, e = E > 0 ? v - kvh * E : 0;
    p_lo = kvh < a.Hkv ? kvh * H + uniform64(s_pos[e]) : U;
    p_hi = kvh >= a.Hkv ? U : (e + 1 < E ? kvh * H + uniform64(s_pos[e + 1]) : (kvh + 1) * H);
  }
  CutItem cut{};
  if (p_lo < p_hi) {
    const LaneOffsets off = lane_offsets<W>(a, lane, wave);
    int kvh = quotient(p_lo, H);
    int e = __builtin_amdgcn_readfirstlane(last_at_most(s_pos, E, p_lo - kvh * H));
    auto seq_of_pair = [&](int entry, int& tile) {
      const int b = __builtin_amdgcn_readfirstlane(static_cast<int>(s_of[entry]));
      tile = entry - __builtin_amdgcn_readfirstlane(s_first[b]);
      return tabulated(a, s_seq[b]);
    };
    int mt;
    Seq s = seq_of_pair(e, mt);
    PageWindow ahead;
    bool have = false;  // `ahead` is this item's first window
    while (true) {
      const int64_t P = kvh * H + uniform64(s_pos[e]);  // the item's position
      if (P >= p_hi) break;
      const int units = tile_units<W>(s.n * a.G - mt * rows_of<W>());
      const int tiles = (keys_of(a, s, (mt + 1) * rows_of<W>()) + kBN - 1) / kBN;
      // tile j's midpoint: P + kItemUnits + units j + units / 2; an item without tiles
      // belongs to the range that holds its position
      const int64_t base = P + kItemUnits + units / 2;
      auto first_at = [&](int64_t p) {
        const int64_t d = p - base;
        if (d <= 0) return 0;
        if (d > static_cast<int64_t>(units) * (tiles - 1)) return tiles;
        const uint32_t x = static_cast<uint32_t>(d) + units - 1;
        return static_cast<int>(units == kUnits ? x / kUnits : x / kFewUnits);
      };
      const int j0 = first_at(p_lo), j1 = first_at(p_hi);
      if (j0 < j1 || (tiles == 0 && P >= p_lo)) {
        const WaveRows wr = wave_rows<W>(a, s, mt, wave, lane);
        float m_run, l_run;
        q3::f32x16 acc[4];
        PageWindow pw = ahead;
        if (!have) window_start(pw, a, s.row, j0, lane);
        // the next item's first window, on its way while this one's tiles run
        const int next = e + 1 == E ? 0 : e + 1;
        window_start(ahead, a, __builtin_amdgcn_readfirstlane(s_seq[s_of[next]].row), 0, lane);
        have = true;
        run_tiles<W>(a, off, s, wr, kvh, j0, j1, pw, tb, lane, wave, m_run, l_run, acc);
        l_run = cross_half_sum(l_run);
        if (j0 == 0 && j1 == tiles) {
          if (wr.active) store_output(a, s, wr, kvh, lane, l_run, acc, stage_of(tb, wave));
        } else {
          const int slot = j0 == 0 ? 2 * v + 1 : 2 * v;
          if (wr.active) {
            // [wave][16 chunks of 8 elements][2 halves][32 rows][4]: every store whole lines
            const int64_t row = static_cast<int64_t>(slot) * rows_of<W>() + wave * 32;
            q3::f32x4* po = reinterpret_cast<q3::f32x4*>(a.po + row * kD) + lane;
#pragma unroll
            for (int i = 0; i < 16; ++i)
              po[64 * i] = q3::f32x4{acc[i >> 2][4 * (i & 3)], acc[i >> 2][4 * (i & 3) + 1],
                                     acc[i >> 2][4 * (i & 3) + 2], acc[i >> 2][4 * (i & 3) + 3]};
            if (lane < 32) a.pml[row + lane] = float2{m_run, l_run};
          }
          if (j0 == 0) {
            const int64_t last = base + static_cast<int64_t>(units) * (tiles - 1);
            cut.parts = quotient(last, width) - v + 1;
            cut.r0 = mt * rows_of<W>();
            cut.rows = min(rows_of<W>(), s.n * a.G - cut.r0);
            cut.kvh = kvh;
            cut.q0 = s.q0;
          }
        }
        __syncthreads();  // the staging buffers are read before the next loads refill them
      }
      if (++e == E) {
        e = 0;
        if (++kvh == a.Hkv) break;
      }
      s = seq_of_pair(e, mt);
    }
  }
  if (tid == 0) a.cuts[v] = cut;
}

// ---------------------------------------------------------------------------
// Dealt schedule: more items than cutting pays for.  Every workgroup sorts the (sequence,
// row tile) pairs by their weight, the longest first, and takes one item of each round of
// as many items as there are workgroups, in the rounds' order to and fro: who had the
// longest of one round has the shortest of the next.  The sort is by 64 classes of
// weight, by counting and stable, so every workgroup has the same order.
template <int W>
__global__ __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_chunk_deal_kernel(ChunkArgs a) {
  Q3_CHUNK_TILE_BUFFERS;
  __shared__ int s_first[kMaxSeqs];  // row tiles before each sequence
  __shared__ SeqEntry s_seq[kMaxSeqs];
  __shared__ int s_slot[kMaxEntries];  // [class][64 pairs]: those of the class, then the ones before
  __shared__ uint32_t s_order[kMaxEntries];  // the sequence, and 16 bits of its row tile
  __shared__ int s_wsum[W];
  __shared__ int s_most;               // weight of the longest
  constexpr int kGroups = kMaxEntries / 64, kPer = kGroups / W;
  constexpr int kClasses = 64;
  static_assert(kClasses * kGroups == kMaxEntries, "the counts fill s_slot");
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (tid == 0) s_most = 0;
  for (int i = tid; i < kMaxEntries; i += W * 64) s_slot[i] = 0;
  const int E = tabulate<W>(a, s_first, s_seq, s_wsum);
  int weight[kPer], rank[kPer];
  uint32_t pair[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = (wave + W * i) * 64 + lane;
    weight[i] = 0;
    pair[i] = 0;
    if (e < E) {
      const int b = last_at_most(s_first, a.B, e);
      const Seq s = seq_of(a, s_seq[b]);
      const int mt = e - s_first[b];
      pair[i] = static_cast<uint32_t>(b) << 16 | static_cast<uint32_t>(mt);
      const int tiles = (keys_of(a, s, (mt + 1) * rows_of<W>()) + kBN - 1) / kBN;
      weight[i] = tile_units<W>(s.n * a.G - mt * rows_of<W>()) * tiles + kItemUnits;
      atomicMax(&s_most, weight[i]);
    }
  }
  __syncthreads();
  const float per_class = (kClasses - 1) / static_cast<float>(max(s_most, 1));
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = (wave + W * i) * 64 + lane;
    const int c = kClasses - 1 -
                  min(kClasses - 1, static_cast<int>(static_cast<float>(weight[i]) * per_class));
    uint64_t same = __ballot(e < E);
#pragma unroll
    for (int bit = 1; bit < kClasses; bit <<= 1) {
      const uint64_t set = __ballot((c & bit) != 0);
      same &= (c & bit) != 0 ? set : ~set;
    }
    rank[i] = __popcll(same & ((uint64_t{1} << lane) - 1));
    weight[i] = c * kGroups + wave + W * i;
    if (e < E && rank[i] == 0) s_slot[weight[i]] = __popcll(same);
  }
  __syncthreads();
  block_scan<W, int>(s_slot, kMaxEntries, s_wsum);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = (wave + W * i) * 64 + lane;
    if (e < E) s_order[s_slot[weight[i]] + rank[i]] = pair[i];
  }
  __syncthreads();

  const LaneOffsets off = lane_offsets<W>(a, lane, wave);
  const int nwg = gridDim.x, w = blockIdx.x;
  const int items = E * a.Hkv;
  // an XCD's neighbours share KV heads where their number allows it, else sequences
  const int p = a.Hkv % 8 != 0 && nwg % 8 == 0 ? (w % 8) * (nwg / 8) + w / 8 : w;
  auto item_of = [&](int round) { return round * nwg + ((round & 1) ? nwg - 1 - p : p); };
  auto pair_of = [&](int item) {
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(s_order[item / a.Hkv])));
  };
  PageWindow ahead;
  for (int round = 0, item = item_of(0); item < items; ++round) {
    const uint32_t pr = pair_of(item);
    const Seq s = tabulated(a, s_seq[pr >> 16]);
    const int mt = pr & 0xffff;
    const int kvh = item % a.Hkv;
    const WaveRows wr = wave_rows<W>(a, s, mt, wave, lane);
    const int tiles = (keys_of(a, s, (mt + 1) * rows_of<W>()) + kBN - 1) / kBN;
    float m_run, l_run;
    q3::f32x16 acc[4];
    PageWindow pw = ahead;
    if (round == 0) window_start(pw, a, s.row, 0, lane);
    // the next item's first window, on its way while this one's tiles run
    item = item_of(round + 1);
    const int next = item < items ? item : item_of(round);
    window_start(ahead, a, __builtin_amdgcn_readfirstlane(s_seq[pair_of(next) >> 16].row), 0, lane);
    run_tiles<W>(a, off, s, wr, kvh, 0, tiles, pw, tb, lane, wave, m_run, l_run, acc);
    l_run = cross_half_sum(l_run);
    if (wr.active) store_output(a, s, wr, kvh, lane, l_run, acc, stage_of(tb, wave));
    __syncthreads();  // the staging buffers are read before the next loads refill them
  }
}

// Joins the parts of the cut items: a lane takes eight elements of a row.  A task is 32
// rows of an item of up to six parts by half their elements (a wave takes an eighth, all
// parts' loads in flight at once), or 32 rows by a quarter of the elements of an item
// with more parts, which the four waves share.  (Items of four to six parts on the second
// path: 1,001 tokens behind 650 take 45.5 us instead of 38.9, 509 behind 12,000 take 132
// instead of 125.)  The workgroups deal the tasks among themselves from the list of cut
// items: a workgroup for each possible task (ranges x rows) costs more in workgroups that
// find nothing to do than the joins take.
constexpr int kJoinParts = 8;
constexpr int kJoinWaves = 4;
constexpr int kJoinFew = 6;

// A lane's eight elements of a row, joined so far.
struct Joined {
  float m, l, o[8];
};

// Joins the next K of n further parts, from slot `slot` on (slot0 in place of the first,
// and read with weight 0 where there are fewer: other slots may hold anything).
template <int K, int W>
__device__ __forceinline__ void join_parts(const ChunkArgs& a, Joined& j, int slot0, int slot, int n,
                                           int row, int e) {
  float2 ml[K];
  q3::f32x4 x[K][2];
#pragma unroll
  for (int u = 0; u < K; ++u) {
    const int64_t first =
        static_cast<int64_t>(u == 0 || u >= n ? slot0 : slot + 2 * u) * rows_of<W>() + (row & ~31);
    ml[u] = a.pml[first + (row & 31)];
    // elements e .. e + 3 of 32 rows, then e + 4 .. e + 7 of them
    const q3::f32x4* src = reinterpret_cast<const q3::f32x4*>(a.po + first * kD) + 8 * e + (row & 31);
    x[u][0] = src[0];
    x[u][1] = src[32];
  }
  __builtin_amdgcn_sched_barrier(0);  // every load is issued before the first is waited for
  float m = j.m;
#pragma unroll
  for (int u = 0; u < K; ++u) m = fmaxf(m, ml[u].x);
  const float use = m == q3::kNegInf ? 0.f : m;
  const float f = q3::fast_exp2(j.m - use);
  j.m = m;
  j.l *= f;
#pragma unroll
  for (int i = 0; i < 8; ++i) j.o[i] *= f;
#pragma unroll
  for (int u = 0; u < K; ++u) {
    const float g = u < n ? q3::fast_exp2(ml[u].x - use) : 0.f;
    j.l += g * ml[u].y;
#pragma unroll
    for (int i = 0; i < 8; ++i) j.o[i] += g * x[u][i >> 2][i & 3];
  }
}

__device__ __forceinline__ void store_joined(const ChunkArgs& a, const CutItem& c, const Joined& j,
                                             int row, int e) {
  const float inv = j.l > 0.f ? 1.f / j.l : 0.f;
  const int r = c.r0 + row;
  const int tok = divide(r, a.per_head);
  q3::st16(a.o + (c.q0 + tok) * a.o_st +
               (static_cast<int64_t>(c.kvh) * a.G + (r - tok * a.G)) * a.o_sh + e,
           q3::u32x4{q3::pack_bf16x2(j.o[0] * inv, j.o[1] * inv),
                     q3::pack_bf16x2(j.o[2] * inv, j.o[3] * inv),
                     q3::pack_bf16x2(j.o[4] * inv, j.o[5] * inv),
                     q3::pack_bf16x2(j.o[6] * inv, j.o[7] * inv)});
}

template <int W>
__global__ __launch_bounds__(kJoinWaves * 64) void paged_chunk_join_kernel(ChunkArgs a, int ranges) {
  __shared__ int s_task[kMaxEntries];  // tasks before each range's item
  __shared__ int s_wsum[kJoinWaves];
  __shared__ Joined s_j[kJoinWaves - 1][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  for (int v = tid; v < ranges; v += kJoinWaves * 64) {
    const CutItem c = a.cuts[v];
    const int blocks = (c.rows + 31) / 32;
    s_task[v] = c.parts == 0 ? 0 : c.parts <= kJoinFew ? 2 * blocks : 4 * blocks;
  }
  __syncthreads();
  const int tasks = block_scan<kJoinWaves, int>(s_task, ranges, s_wsum);
  for (int task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int v = __builtin_amdgcn_readfirstlane(last_at_most(s_task, ranges, task));
    const CutItem c = a.cuts[v];
    const int k = task - s_task[v];
    if (c.parts <= kJoinFew) {
      const int row = 32 * (k >> 1) + (lane & 31);
      if (row >= c.rows) continue;
      const int e = 64 * (k & 1) + 16 * wave + 8 * (lane >> 5);
      Joined j{q3::kNegInf, 0.f, {}};
      if (c.parts <= 3)
        join_parts<3, W>(a, j, 2 * v + 1, 2 * v, c.parts, row, e);
      else
        join_parts<kJoinFew, W>(a, j, 2 * v + 1, 2 * v, c.parts, row, e);
      store_joined(a, c, j, row, e);
      continue;
    }
    const int row = 32 * (k >> 2) + (lane & 31);
    const int each = (c.parts + kJoinWaves - 1) / kJoinWaves;
    const int p1 = min(c.parts, (wave + 1) * each);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = 32 * (k & 3) + 16 * i + 8 * (lane >> 5);
      Joined j{q3::kNegInf, 0.f, {}};
      if (row < c.rows)
        for (int p = wave * each; p < p1; p += kJoinParts)
          join_parts<kJoinParts, W>(a, j, p == 0 ? 2 * v + 1 : 2 * (v + p), 2 * (v + p), p1 - p, row,
                                    e);
      if (wave > 0) s_j[wave - 1][lane] = j;
      __syncthreads();
      if (wave == 0 && row < c.rows) {
#pragma unroll
        for (int s = 0; s < kJoinWaves - 1; ++s) {
          const Joined& x = s_j[s][lane];
          const float m = fmaxf(j.m, x.m), use = m == q3::kNegInf ? 0.f : m;
          const float f = q3::fast_exp2(j.m - use), g = q3::fast_exp2(x.m - use);
          j.m = m;
          j.l = j.l * f + x.l * g;
#pragma unroll
          for (int o = 0; o < 8; ++o) j.o[o] = j.o[o] * f + x.o[o] * g;
        }
        store_joined(a, c, j, row, e);
      }
      __syncthreads();  // s_j is read before it is written again
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.

int cu_count() {
  static int cached[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 0;
  if (cached[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
      return 0;
    cached[dev] = n;
  }
  return cached[dev];
}

// Resident workgroups of the range schedule (two waves a SIMD); 256 CUs where no device
// can be asked.
int range_workgroups(int W) {
  const int cus = cu_count();
  const int wgs = (cus > 0 ? cus : 256) * 8 / W;
  return wgs < kMaxEntries ? wgs : kMaxEntries;
}

struct ChunkLayout {
  int64_t po, pml, cuts, total;
};
ChunkLayout chunk_layout(int W) {
  const int64_t ranges = range_workgroups(W), rows = 2 * ranges * 32 * W;
  ChunkLayout l;
  l.po = 0;
  l.pml = l.po + rows * kD * sizeof(float);
  l.cuts = l.pml + rows * sizeof(float2);
  l.total = l.cuts + (ranges * sizeof(CutItem) + 255) / 256 * 256;
  return l;
}

// How a call runs; a rule on its launch shape, so that a captured call stays valid.
//  - few packed rows a KV head: the streaming kernel (paged_chunk_stream.hip);
//  - chunks of more than four waves' rows: eight-wave workgroups, which stage each K/V
//    tile once for twice the rows (2,048 tokens behind 64,000, 32/8 heads: 1.92 ms
//    against 2.03; eight chunks of 100-500 behind 100-9,000: 313 us against 318; 16
//    single tokens behind 4,000 in the same kernels: 54 against 51);
//  - ranges for up to 1.75 items a workgroup, dealt items above: one prompt of 4,096 (2.03
//    items) 141 us dealt, 165 in ranges; eight chunks of about 1,000 (2.2) 71 and 77;
//    twelve turns of 20-700 behind 0-6,000 (1.44) 186 and 165.  How unequal the items are
//    decides too, and the lengths lie on the device: by the count alone, eight of 200-800
//    behind 1,000-8,000 (2.2) take 309 where ranges take 300, and six chunks with groups of
//    five heads (1.31) 218 where dealt items take 205;
//  - items in order where the batch is too large to be tabulated in LDS.  (Where it is
//    not, order alone costs: 16 chunks of 200-800 behind 1,000-8,000 825 us, dealt 658;
//    100 of 30-100 behind 200-2,000 213 and 196; one prompt of 4,096 146 and 141.)
struct Variant {
  bool stream;
  int waves;
  bool ranges, dealt;
};
Variant variant_of(int B, int max_chunk, int64_t total, int G, int Hkv) {
  const int64_t rows = std::min<int64_t>(max_chunk, total) * G;
  Variant v{q3::chunk_streams(B, rows), rows > rows_of<4>() ? 8 : 4, false, false};
  const int64_t entries = q3::cdiv(total * G, 32 * v.waves) + B;
  const bool listed = B <= kMaxSeqs && entries <= kMaxEntries && Hkv <= (1 << 20);
  v.ranges = listed && 4 * entries * Hkv <= 7 * static_cast<int64_t>(range_workgroups(v.waves));
  v.dealt = listed && !v.ranges;
  return v;
}

template <int W>
int launch_tiles(ChunkArgs a, const Variant& var, int max_chunk, void* workspace, hipStream_t s,
                 const char* who) {
  q3::clear_error();
  if (var.ranges) {
    const int wgs = range_workgroups(W);
    const ChunkLayout l = chunk_layout(W);
    char* ws = static_cast<char*>(workspace);
    a.po = reinterpret_cast<float*>(ws + l.po);
    a.pml = reinterpret_cast<float2*>(ws + l.pml);
    a.cuts = reinterpret_cast<CutItem*>(ws + l.cuts);
    a.per_range = 1. / wgs;
    hipLaunchKernelGGL(paged_chunk_range_kernel<W>, dim3(wgs), dim3(W * 64), 0, s, a);
    if (const int rc = q3::launch_status(who)) return rc;
    hipLaunchKernelGGL(paged_chunk_join_kernel<W>, dim3(4 * (wgs * W / 8)), dim3(kJoinWaves * 64), 0,
                       s, a, wgs);
    return q3::launch_status(who);
  }
  if (var.dealt) {
    hipLaunchKernelGGL(paged_chunk_deal_kernel<W>, dim3(range_workgroups(W)), dim3(W * 64), 0, s, a);
    return q3::launch_status(who);
  }
  const int64_t longest = max_chunk < a.total ? max_chunk : a.total;
  a.n_mtiles = static_cast<int>(q3::cdiv(longest * a.G, rows_of<W>()));
  const int64_t items = static_cast<int64_t>(a.Hkv) * a.B * a.n_mtiles;
  if (items > q3::kMaxThreads / (W * 64))
    return q3::fail(QWEN3_EINVAL, "%s: grid too large (KV heads %d, batch %d, max_chunk %d)", who,
                    a.Hkv, a.B, max_chunk);
  hipLaunchKernelGGL(paged_chunk_flat_kernel<W>, dim3(static_cast<unsigned>(items)), dim3(W * 64), 0,
                     s, a);
  return q3::launch_status(who);
}

}  // namespace

extern "C" size_t qwen3_paged_chunk_workspace_bytes(int B, int max_chunk, int64_t total_tokens,
                                                    int num_heads, int num_kv_heads,
                                                    int head_dim) {
  if (B <= 0 || total_tokens <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      num_heads / num_kv_heads > kMaxG || head_dim != kD || max_chunk <= 0)
    return 0;
  const Variant v =
      variant_of(B, max_chunk, total_tokens, num_heads / num_kv_heads, num_kv_heads);
  if (v.stream)
    return q3::chunk_stream_workspace(
        B, static_cast<int>(std::min<int64_t>(max_chunk, total_tokens) * (num_heads / num_kv_heads)));
  return v.ranges ? chunk_layout(v.waves).total : 256;
}

extern "C" int qwen3_paged_chunk_bf16(
    const void* q, const int64_t q_strides[2], const void* k_cache, const int64_t k_strides[3],
    const void* v_cache, const int64_t v_strides[3], int64_t num_blocks,
    const int32_t* block_table, int64_t bt_row_stride, int64_t max_rows, int64_t max_pages,
    const int32_t* seq_lens, const int32_t* row_ids, const int32_t* cu_seqlens, void* out,
    const int64_t out_strides[2], int B, int max_chunk, int64_t total_tokens, int num_heads,
    int num_kv_heads, int head_dim, int block_size, float scale, void* workspace,
    size_t workspace_bytes, void* stream) {
  const char* who = "qwen3_paged_chunk_bf16";
  if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !cu_seqlens || !out ||
      !q_strides || !k_strides || !v_strides || !out_strides)
    return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  if (head_dim != kD)
    return q3::fail(QWEN3_EUNSUPPORTED, "%s: head_dim %d not supported (built for %d)", who,
                    head_dim, kD);
  if (block_size <= 0 || block_size % kGroup != 0)
    return q3::fail(QWEN3_EUNSUPPORTED, "%s: block_size %d must be a multiple of %d", who,
                    block_size, kGroup);
  if (num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 ||
      num_heads / num_kv_heads > kMaxG)
    return q3::fail(QWEN3_EUNSUPPORTED, "%s: num_heads %d / num_kv_heads %d unsupported", who,
                    num_heads, num_kv_heads);
  if (B < 0 || max_chunk < 0 || total_tokens < 0 || total_tokens > 0x7fffffff ||
      num_blocks <= 0 || max_rows <= 0 || max_pages <= 0 || bt_row_stride < max_pages)
    return q3::fail(QWEN3_EINVAL, "%s: bad sizes (B=%d max_chunk=%d total_tokens=%lld "
                    "num_blocks=%lld max_rows=%lld max_pages=%lld bt_row_stride=%lld)", who, B,
                    max_chunk, (long long)total_tokens, (long long)num_blocks,
                    (long long)max_rows, (long long)max_pages, (long long)bt_row_stride);
  if (!(scale > 0.f) || !(scale < __builtin_inff()))
    return q3::fail(QWEN3_EINVAL, "%s: scale must be positive and finite", who);
  if (max_pages * block_size > (int64_t(1) << 30))
    return q3::fail(QWEN3_EINVAL, "%s: max_pages * block_size too large", who);
  const int64_t vec_strides[] = {q_strides[0], q_strides[1], k_strides[0], k_strides[1],
                                 k_strides[2], v_strides[0], v_strides[1], v_strides[2],
                                 out_strides[0], out_strides[1]};
  bool ok = q3::aligned16(q) && q3::aligned16(k_cache) && q3::aligned16(v_cache) &&
            q3::aligned16(out);
  for (int64_t st : vec_strides) ok = ok && st % 8 == 0;
  if (!ok)
    return q3::fail(QWEN3_EALIGN, "%s: q/K/V/out need 16-byte aligned rows (strides multiple "
                    "of 8 elements)", who);
  // Rows behind a descriptor's end must lie outside it, and 16 of them inside 32-bit offsets.
  for (int64_t st : {k_strides[2], v_strides[2]})
    if (st < kD || st > (int64_t(1) << 24))
      return q3::fail(QWEN3_EUNSUPPORTED, "%s: slot stride %lld outside %d..2^24", who,
                      (long long)st, kD);
  const int64_t total_rows = total_tokens * (num_heads / num_kv_heads);
  if (total_rows > 0x7fffffff - 256)
    return q3::fail(QWEN3_EINVAL, "%s: too many tokens", who);
  if (B == 0 || max_chunk == 0 || total_tokens == 0) return QWEN3_OK;
  const size_t need = qwen3_paged_chunk_workspace_bytes(B, max_chunk, total_tokens, num_heads,
                                                        num_kv_heads, head_dim);
  if (!workspace || workspace_bytes < need)
    return q3::fail(QWEN3_EWORKSPACE, "%s: workspace of %zu bytes needed, %zu given", who, need,
                    workspace ? workspace_bytes : (size_t)0);
  if (!q3::aligned16(workspace))
    return q3::fail(QWEN3_EALIGN, "%s: workspace must be 16-byte aligned", who);
  ChunkArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_st = q_strides[0];
  a.q_sh = q_strides[1];
  a.k = static_cast<const uint16_t*>(k_cache);
  a.k_blk = k_strides[0];
  a.k_sh = k_strides[1];
  a.k_slot = static_cast<int>(k_strides[2]);
  a.v = static_cast<const uint16_t*>(v_cache);
  a.v_blk = v_strides[0];
  a.v_sh = v_strides[1];
  a.v_slot = static_cast<int>(v_strides[2]);
  a.num_blocks = num_blocks;
  a.bt = block_table;
  a.bt_stride = bt_row_stride;
  a.max_rows = max_rows;
  a.max_pages = max_pages;
  a.seq_lens = seq_lens;
  a.row_ids = row_ids;
  a.cu = cu_seqlens;
  a.o = static_cast<uint16_t*>(out);
  a.o_st = out_strides[0];
  a.o_sh = out_strides[1];
  a.total = total_tokens;
  a.B = B;
  a.Hkv = num_kv_heads;
  a.G = num_heads / num_kv_heads;
  a.gpb = block_size / kGroup;
  a.per_head = 1. / a.G;
  a.per_group = 1. / a.gpb;
  a.reach = static_cast<int>(max_pages * block_size);
  a.scale_log2 = scale * q3::kLog2e;
  const Variant var = variant_of(B, max_chunk, total_tokens, a.G, a.Hkv);
  const auto s = static_cast<hipStream_t>(stream);
  if (var.stream) {
    const q3::ChunkStreamCall call{
        a.q, a.q_st, a.q_sh, a.k, a.k_blk, a.k_sh, a.k_slot, a.v, a.v_blk, a.v_sh, a.v_slot,
        a.num_blocks, a.bt, a.bt_stride, a.max_rows, a.max_pages, a.seq_lens, a.row_ids, a.cu,
        a.o, a.o_st, a.o_sh, a.total, a.B, a.Hkv, a.G, block_size,
        static_cast<int>(std::min<int64_t>(max_chunk, total_tokens) * a.G), a.scale_log2};
    return q3::launch_chunk_stream(call, workspace, s, who);
  }
  return var.waves == 8 ? launch_tiles<8>(a, var, max_chunk, workspace, s, who)
                        : launch_tiles<4>(a, var, max_chunk, workspace, s, who);
}
