// Chunk attention where a sequence's new tokens and their heads are few: at most 16
// packed query rows (token, head of the group) per KV head -- draft tokens being
// verified, or decoding sequences.  The streaming decode's schedule and loads
// (paged_decode.hip): the (sequence, KV head, 16-key tile) triples lie end to end and
// are cut into equal ranges, one per resident wave; K and V go from HBM straight into
// MFMA operands, two batches of tiles in flight per wave; a sequence-head that straddles
// ranges is joined by a second launch.  Here the 16 columns of a product are the packed
// rows of a sequence, each with its own last key.  P meets V as two bf16 terms, as in the
// decode: 16 bits, for a second product that the loads hide (48 sequences of four tokens
// 156 us with one term and with two).
//
// Bound by HBM: K and V are read once for all rows of a sequence (48 sequences of four
// tokens behind 1,024-8,192, 32/8 heads: 862 MB algorithmic, 872 MB fetched, 153 us and 8
// of merge, 5.5 TB/s).  The same batch in the tile kernels, whose loads
// pass through LDS: 193 us.  Two column groups a wave, to 32 rows: 78 us against 55 for 16
// sequences of eight tokens behind 4,000 (registers for one batch of tiles less in
// flight), so 17 rows and more go to the tile kernels.  A few rows behind little are
// latency: a dependent load each for rows, lengths, page ids, keys and the queries, then
// code that no cache holds yet (one sequence of five tokens behind 900: 9.5 us, and 5 of merge).
#include "paged_chunk_stream.hpp"
#include "paged_decode_merge.hpp"
#include "paged_decode_tile.hpp"

namespace {

struct StreamArgs {
  DecodeArgs d;       // q, pool, tables, out, scale, partials (G: rows of a partial)
  const int32_t* cu;
  int64_t total;      // rows of q
  int group;          // query heads per KV head
};

// A sequence of the batch as the table keeps it.
struct StreamSeq {
  int32_t q0, n;      // its rows of q
  int32_t row;        // of the block table
  int32_t ctx;        // tokens before the new ones
};

// Keys that the sequence's last token reaches.
__device__ __forceinline__ int keys_of(const StreamArgs& a, const StreamSeq& s) {
  const int64_t len = static_cast<int64_t>(s.ctx) + s.n, cap = a.d.max_pages * a.d.bs;
  const int64_t L = len < cap ? len : cap;
  return s.row >= 0 && s.n > 0 && L > 0 ? static_cast<int>(L) : 0;
}

__device__ __forceinline__ StreamSeq seq_at(const StreamArgs& a, int b) {
  const int64_t s0 = a.cu[b], s1 = a.cu[b + 1];
  const int64_t row = row_of(a.d, b);
  const bool ok = s0 >= 0 && s1 > s0 && s1 <= a.total;
  StreamSeq s;
  s.q0 = ok ? static_cast<int32_t>(s0) : 0;
  s.n = ok ? static_cast<int32_t>(s1 - s0) : 0;
  s.row = static_cast<int32_t>(row);
  s.ctx = row >= 0 ? a.d.seq_lens[row] : 0;
  return s;
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ StreamSeq uniform_seq(const StreamSeq& s) {
  return {uniform(s.q0), uniform(s.n), uniform(s.row), uniform(s.ctx)};
}

// Tabulates the batch: the sequences, and the exclusive prefix of their tiles.
template <int kRounds>
__device__ __forceinline__ int tabulate_chunks(const StreamArgs& a, int32_t* s_pref,
                                               StreamSeq* s_seq, int32_t (*s_wsum)[kWaves]) {
  constexpr int kThreads = kWaves * 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int B = a.d.B;
  const int rounds = (B + kThreads - 1) / kThreads;
  int n[kRounds], incl[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    if (kRounds > 1 && i >= rounds) break;
    const int b = i * kThreads + tid;
    const StreamSeq s = seq_at(a, min(b, B - 1));
    n[i] = b < B ? (keys_of(a, s) + kTile - 1) / kTile : 0;
    if (b < B) s_seq[b] = s;
    incl[i] = wave_prefix_sum(n[i]);
    if (lane == 63) s_wsum[i][wave] = incl[i];
  }
  __syncthreads();
  int run = 0;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    if (kRounds > 1 && i >= rounds) break;
    int before = run;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int ws = s_wsum[i][w];
      before += w < wave ? ws : 0;
      run += ws;
    }
    const int b = i * kThreads + tid;
    if (b < B) s_pref[b] = before + incl[i] - n[i];
  }
  if (tid == 0) s_pref[B] = run;
  __syncthreads();
  return run;
}

// Load-side cursor of a wave.
struct ChunkCursor {
  int64_t g, g1;
  int b, hkv, t;
  int n, L;
};

__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_chunk_stream_kernel(StreamArgs a) {
  __shared__ int32_t s_pref[kStreamMaxB + 1];
  __shared__ StreamSeq s_seq[kStreamMaxB];
  __shared__ int32_t s_wsum[kStreamMaxB / (kWaves * 64)][kWaves];
  const DecodeArgs& d = a.d;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = uniform(tid >> 6);  // what follows from it stays in scalar registers
  const int lo = lane & 15;
  const int hi = lane >> 4;
  const int B = d.B;
  const int total_v = B <= kWaves * 64
                        ? tabulate_chunks<1>(a, s_pref, s_seq, s_wsum)
                        : tabulate_chunks<kStreamMaxB / (kWaves * 64)>(a, s_pref, s_seq, s_wsum);
  const int64_t T = static_cast<int64_t>(d.Hkv) * uniform(total_v);
  const int64_t W = static_cast<int64_t>(gridDim.x) * kWaves;
  int64_t pw = q3::cdiv(T, W);
  pw = pw < kMinTilesPerWave ? kMinTilesPerWave : pw;
  if (blockIdx.x == 0) {
    for (int b = tid; b <= B; b += kWaves * 64) d.s_pref[b] = s_pref[b];
    if (tid == 0) d.s_meta[0] = static_cast<int32_t>(pw);
  }
  const int64_t w = wave_index(T, W, pw, wave);
  const int64_t g0 = w * pw;
  if (g0 >= T) return;

  ChunkCursor cur;
  {
    int lo_b = 0, hi_b = B - 1;  // largest b with Hkv * pref[b] <= g0
    while (lo_b < hi_b) {
      const int mid = (lo_b + hi_b + 1) >> 1;
      if (static_cast<int64_t>(d.Hkv) * s_pref[mid] <= g0) lo_b = mid; else hi_b = mid - 1;
    }
    lo_b = uniform(lo_b);
    cur.b = lo_b;
    const int before = uniform(s_pref[lo_b]);
    cur.n = uniform(s_pref[lo_b + 1]) - before;
    cur.L = keys_of(a, uniform_seq(s_seq[lo_b]));
    const int64_t off = g0 - static_cast<int64_t>(d.Hkv) * before;
    cur.hkv = static_cast<int>(off / cur.n);
    cur.t = static_cast<int>(off % cur.n);
    cur.g = g0;
    cur.g1 = g0 + pw < T ? g0 + pw : T;
  }
  TableWindow tw;
  window_load(tw, d, uniform(s_seq[cur.b].row), (cur.t * kTile) / d.bs, lane);

  auto issue = [&](Chunk& c) {
    c.n = 0;
    if (cur.g >= cur.g1) return;
    if (cur.t >= cur.n) {  // next sequence-head
      if (++cur.hkv == d.Hkv) {
        cur.hkv = 0;
        do {
          ++cur.b;
          cur.n = uniform(s_pref[cur.b + 1] - s_pref[cur.b]);
        } while (cur.n == 0);
        cur.L = keys_of(a, uniform_seq(s_seq[cur.b]));
      }
      cur.t = 0;
      window_load(tw, d, uniform(s_seq[cur.b].row), 0, lane);
    }
    const int64_t left = cur.g1 - cur.g;
    int n = cur.n - cur.t;
    n = n < kChunk ? n : kChunk;
    n = left < n ? static_cast<int>(left) : n;
    c.n = n;
    c.t0 = cur.t;
    c.seg = cur.b * d.Hkv + cur.hkv;
    c.ntiles = cur.n;
    c.L = cur.L;
    const uint16_t* kbase = d.k + static_cast<int64_t>(cur.hkv) * d.k_sh;
    const uint16_t* vbase = d.v + static_cast<int64_t>(cur.hkv) * d.v_sh;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      int64_t phys = -1;
      int sub = 0;
      if (i < n) {
        const int tok0 = (cur.t + i) * kTile;
        phys = window_phys(tw, d, tok0 / d.bs, lane);
        sub = tok0 % d.bs;
      }
      load_tile(c, i, d, kbase, vbase, phys, sub, lo, hi);
    }
    cur.t += n;
    cur.g += n;
  };

  // Compute-side state: the sequence-head being accumulated.
  int cseg = -1, chkv = 0, ct_lo = 0, ct_hi = 0, cn = 0;
  bool cfirst = true;
  StreamSeq cs{0, 0, -1, 0};
  Columns col;

  auto begin = [&](const Chunk& c) {
    cs = uniform_seq(s_seq[c.seg / d.Hkv]);
    chkv = c.seg % d.Hkv;
    ct_lo = c.t0;
    cn = c.ntiles;
    const int tok = lo / a.group, head = lo - tok * a.group;
    const bool ok = tok < cs.n;
    const int64_t last = static_cast<int64_t>(cs.ctx) + (ok ? tok : 0);
    col.last = static_cast<int>(last < c.L - 1 ? (last < -1 ? -1 : last) : c.L - 1);
    reset(col.st);
    const uint16_t* qp = d.q + (static_cast<int64_t>(cs.q0) + (ok ? tok : 0)) * d.q_sb +
                         (static_cast<int64_t>(chkv) * a.group + (ok ? head : 0)) * d.q_sh + hi * 8;
#pragma unroll
    for (int cc = 0; cc < 4; ++cc)
      col.q[cc] = q3::as_bf16x8(ok ? q3::ld16(qp + cc * 32) : q3::u32x4{0u, 0u, 0u, 0u});
  };

  auto finalize = [&]() {
    const float l = q3::sum_xor32(q3::sum_xor16(col.st.l));
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int tok = lo / a.group;
    if (tok >= cs.n || lo >= d.G) return;
    const q3::f32x4 (&acc)[8] = col.st.acc;
    if (ct_lo == 0 && ct_hi == cn) {
      store_out_bf16(d, cs.q0 + tok, chkv * a.group + (lo - tok * a.group), acc, inv, hi);
      return;
    }
    const int64_t slot = (w * 2 + (cfirst ? 0 : 1)) * d.G + lo;
    float* po = d.s_po + slot * kD + 32 * hi;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      *reinterpret_cast<q3::f32x4*>(po + 8 * r) =
          q3::f32x4{acc[0][r] * inv, acc[1][r] * inv, acc[2][r] * inv, acc[3][r] * inv};
      *reinterpret_cast<q3::f32x4*>(po + 8 * r + 4) =
          q3::f32x4{acc[4][r] * inv, acc[5][r] * inv, acc[6][r] * inv, acc[7][r] * inv};
    }
    if (hi == 0) d.s_plse[slot] = l > 0.f ? col.st.m + __builtin_log2f(l) : q3::kNegInf;
  };

  auto process = [&](Chunk& c) {
    if (c.seg != cseg) {
      if (cseg >= 0) {
        finalize();
        cfirst = false;
      }
      cseg = c.seg;
      begin(c);
    }
    fold_chunk(c, d.scale_log2, hi, col);
    ct_hi = c.t0 + c.n;
  };

  Chunk ca, cbuf;
  issue(ca);
  issue(cbuf);
  while (true) {
    if (ca.n == 0) break;
    process(ca);
    issue(ca);
    if (cbuf.n == 0) break;
    process(cbuf);
    issue(cbuf);
  }
  if (cseg >= 0) finalize();
}

// Joins the partials of every sequence-head split across waves, and writes zeros for
// tokens without keys: one workgroup per (KV head, sequence), a wave per row.
__global__ __launch_bounds__(q3::kChunkStreamRows * 64) void paged_chunk_stream_merge_kernel(StreamArgs a) {
  const DecodeArgs& d = a.d;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hkv = blockIdx.x, b = blockIdx.y;
  const StreamPartials parts{d.s_po, d.s_plse, d.s_pref, d.s_meta, d.Hkv, d.G};
  const int64_t s0 = a.cu[b], s1 = a.cu[b + 1];
  const int n = s0 >= 0 && s1 > s0 && s1 <= a.total ? static_cast<int>(s1 - s0) : 0;
  const int rows = min(n * a.group, d.G);
  if (wave >= rows) return;
  uint32_t y;
  if (!merge_partials(parts, b, static_cast<int64_t>(hkv) * d.G + wave, lane, y)) return;
  const int tok = wave / a.group;
  *reinterpret_cast<uint32_t*>(
      d.out + (s0 + tok) * d.o_sb +
      (static_cast<int64_t>(hkv) * a.group + (wave - tok * a.group)) * d.o_sh + 2 * lane) = y;
}

StreamLayout layout_of(int B, int rows) {
  const int wgs = stream_workgroups();
  return stream_layout(B, int64_t(wgs > 0 ? wgs : kStreamMaxWgs) * kWaves, rows);
}

}  // namespace

namespace q3 {

bool chunk_streams(int B, int64_t rows) {
  return B <= kStreamMaxB && rows <= kChunkStreamRows && stream_workgroups() > 0;
}

size_t chunk_stream_workspace(int B, int rows) {
  return static_cast<size_t>(layout_of(B, rows).total);
}

int launch_chunk_stream(const ChunkStreamCall& c, void* workspace, hipStream_t s, const char* who) {
  StreamArgs a{};
  DecodeArgs& d = a.d;
  d.q = c.q;
  d.q_sb = c.q_st;
  d.q_sh = c.q_sh;
  d.k = c.k;
  d.k_sblk = c.k_blk;
  d.k_sh = c.k_sh;
  d.k_sslot = c.k_slot;
  d.v = c.v;
  d.v_sblk = c.v_blk;
  d.v_sh = c.v_sh;
  d.v_sslot = c.v_slot;
  d.num_blocks = c.num_blocks;
  d.bt = c.bt;
  d.bt_stride = c.bt_stride;
  d.max_rows = c.max_rows;
  d.max_pages = c.max_pages;
  d.seq_lens = c.seq_lens;
  d.row_ids = c.row_ids;
  d.out = c.o;
  d.o_sb = c.o_st;
  d.o_sh = c.o_sh;
  d.B = c.B;
  d.Hkv = c.Hkv;
  d.G = c.rows;
  d.bs = c.block_size;
  d.scale_log2 = c.scale_log2;
  a.cu = c.cu;
  a.total = c.total;
  a.group = c.G;
  char* ws = static_cast<char*>(workspace);
  const StreamLayout l = layout_of(c.B, c.rows);
  d.s_po = reinterpret_cast<float*>(ws + l.po);
  d.s_plse = reinterpret_cast<float*>(ws + l.plse);
  d.s_pref = reinterpret_cast<int32_t*>(ws + l.pref);
  d.s_meta = reinterpret_cast<int32_t*>(ws + l.meta);
  const int wgs = stream_workgroups();
  clear_error();
  hipLaunchKernelGGL(paged_chunk_stream_kernel, dim3(wgs), dim3(kWaves * 64), 0, s, a);
  if (const int rc = launch_status(who)) return rc;
  hipLaunchKernelGGL(paged_chunk_stream_merge_kernel, dim3(c.Hkv, c.B),
                     dim3(64 * c.rows), 0, s, a);
  return launch_status(who);
}

}  // namespace q3
