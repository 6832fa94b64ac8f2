// Paged decode attention of a batch whose groups of sequences share a prefix, for gfx950
// (GQA, one query token a sequence).
//
// Sequence b attends the keys j < L_b of its row of the block table; the first P of them
// lie in the same pages for all sequences of a group.  With m, l, o the running maximum,
// sum and weighted mean of some keys,
//   (m, l, o)[0, L_b) = join((m, l, o)[0, P), (m, l, o)[P, L_b)),
// so the prefix is attended once, by the rows (sequence, head) of all of the group's
// sequences packed together, and its K and V are read once instead of once a sequence.
//
// One launch attends, a second joins.  In the first, a workgroup does one of two things:
//  * prefixes of more than 16 rows: K/V tiles of 64 keys staged in LDS, four stages, so
//    that the loads of three tiles are on their way while one is computed; eight waves, 128
//    rows an item.  The items' tiles lie end to end and are cut into equal ranges, a
//    workgroup each;
//  * what each sequence has of its own, and prefixes of up to 16 rows: the streaming
//    decode's loop (paged_decode.hip), K and V straight into MFMA operands, the 16-key
//    tiles of all items end to end, cut into equal ranges, a wave each.  (Staged instead,
//    prefixes of 4 sequences and 4 query heads a KV head: one group behind 30,000 tokens
//    39.9 us for 41.3, behind 100,000 99 for 85, sixteen behind 2,048 60.0 for 54.4.)
// The workgroups are divided by the tiles' weights.  Parts of cut items, and whole ones
// that have another half, are left in the workspace (normalised, with the log2 of their
// sum), and the second launch joins each row's.  P is floored to whole tiles of 16 keys
// and bounded by what the group's first sequence holds; the rest counts as each
// sequence's own, and so does all of a sequence that ends inside P.  The probabilities meet
// the values as two bf16 terms, as in the decode: what both leave of a probability is below
// 2^-16 of it (each term's half step, 2^-8), against 2^-8 of the output's own rounding; one
// term alone would be as far off as that.  A third would cost the staged tiles 8 more MFMAs
// of 24.
//
// What bounds it: HBM, where sequences have much of their own (256 of 50-2,500 tokens behind
// 2,000, 16/8 heads: 225 us, 5.7 TB/s); behind long prefixes the staged tiles, 1.87 us each
// on each CU, where their loads alone take 1.4 (5.9 TB/s) and their products and softmax
// alone 1.45: a SIMD's two waves issue 48 MFMAs of 32 cycles and 340 other vector
// instructions a tile, near the sum of the two, 3,300 cycles, however they are interleaved.
// The other 0.4 us are loads and products that wait for one another at the barrier of every
// tile (32 sequences behind 100,000, 32/8 heads: 115-120 us, 3.7 TB/s; 64 behind 8,192 and
// 1-1,000 tokens of their own 47-50 us, 3.1 TB/s); in small calls the latency of the
// steps, 2.5 us until the batch is tabulated, 10 of the first tiles, 5 of the join (4 behind
// 896, 16/8 heads: 14 us).
// Attended one by one (paged_decode.hip) the same batches take 489, 1,817, 296 and 15 us.
//
// Measured against it (32 behind 100,000; 64 behind 8,192): the values' products of both
// halves of a tile's keys after the scores 117.7 us for 115.2; scores of one half taken a tile
// ahead in stages of their own 113 for 113, 48 for 48, and all operands read from LDS a step
// before they are used 121 for 119, 48 for 48; items of 256 rows 2.65 us a tile, for 3.74 of two
// of 128 rows (not timed in a whole call of a batch that large); parts
// stored past the caches 54.8 us for 52.6; waves' priorities no difference.
#include <algorithm>

#include "paged_decode_merge.hpp"
#include "paged_decode_tile.hpp"
#include "paged_kv_tile.hpp"

namespace {

constexpr int kThreads = 512;
constexpr int kShWaves = kThreads / 64;
constexpr int kMaxSeqs = 1024;        // sequences, and groups, tabulated in LDS
constexpr int kRounds = kMaxSeqs / kThreads;
constexpr int kRowsT = 128;           // rows of an item whose tiles are staged
constexpr int kRowsS = 16;            // rows of one that is streamed
constexpr int kMaxWgs = 512;
constexpr int kStages = 4;
// Weight, in streamed tiles of 16 keys, of a staged tile of 64 (64 behind 8,192: 47.4 us; of
// 4 51.3, of 6 49.8); what an item's start and end weigh, in tiles of its kind (staged, none
// 51.6, of 8 48.3; streamed, none 52.7, of 3 48.7), all swept on that batch, whose items have
// 128 rows, and taken for smaller ones too; tiles that a range takes at least
// (staged, 1 to 4 the same; streamed, a chunk: 4 behind 4,096 23.8 us for 21.8, 16 behind
// 4,096 23.2 for 23.8; four chunks 23.5 and 26.2).
constexpr int kStagedUnits = 5;
constexpr int kItemTiles = 4;
constexpr int kSegTiles = 1;
constexpr int kMinStaged = 2;
constexpr int kMinStreamed = 2 * kChunk;

// What the second launch needs of a sequence.
struct SeqMeta {
  int32_t own_at, own_n;  // its own tiles of one head: before them in the list, their number
  int32_t pre_at, pre_n;  // its prefix's, in the list that `kind` says
  int32_t pre_row;        // first row of the sequence in its group
  int32_t kind;           // 0: no prefix, 1: streamed, 2: staged
};
struct CallMeta {
  int32_t pw;       // tiles of a wave's range
  int32_t pt;       // tiles of a workgroup's range
  int32_t all_t;    // staged tiles of one KV head
  int32_t pad;
};

struct SharedArgs {
  DecodeArgs d;
  // as the staged tiles' code calls them
  const uint16_t* k;
  int64_t k_blk, k_sh;
  int k_slot;
  const uint16_t* v;
  int64_t v_blk, v_sh;
  int v_slot;
  int64_t num_blocks;
  const int32_t* bt;
  int64_t bt_stride, max_pages;
  int gpb;
  double per_group, per_head;
  // groups
  const int32_t* cu;      // (groups + 1)
  const int32_t* shared;  // (groups)
  int groups;
  // workspace
  float* po_s;      // [waves][2][kRowsS][kD] streamed parts
  float* lse_s;
  float* po_t;      // [workgroups][2][rows_t][kD] staged parts
  float* lse_t;
  float* po_own;    // [B][Hq][kD] whole items that have a prefix
  float* lse_own;
  float* po_pre;    // [B][Hq][kD] whole prefixes
  float* lse_pre;
  SeqMeta* seqs;
  CallMeta* call;
  int rows_t;       // rows of a staged part: kRowsT, or all of a smaller batch
};

constexpr int kNoGroup = 0xffff;
struct Tables {
  // Tiles of one head before each, with kSegTiles (kItemTiles) for each item:
  int32_t own[kMaxSeqs + 1];   // of sequences
  int32_t row[kMaxSeqs];
  int32_t len[kMaxSeqs];
  int32_t gs[kMaxSeqs + 1];    // of groups, streamed
  int32_t gt[kMaxSeqs + 1];    // of groups, staged
  int32_t gp[kMaxSeqs];        // tiles of 16 keys of the prefix
  uint16_t grp[kMaxSeqs];      // the group whose prefix a sequence shares
  int16_t g0[kMaxSeqs + 2];    // first sequence (-1, B + 1: outside the batch)
  int32_t wsum[3][kRounds][kShWaves];
  int32_t falling;             // whether the groups' bounds do not ascend
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Last index i < n with v[i] <= p (v ascending); -1: none.
template <typename T>
__device__ __forceinline__ int last_at_most(const T* v, int n, int p) {
  int lo = -1, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (v[mid] <= p) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Sequences of group g (0: not a range of the batch).
__device__ __forceinline__ int members(const Tables& t, int g, int B) {
  const int s0 = t.g0[g], s1 = t.g0[g + 1];
  return s0 >= 0 && s1 > s0 && s1 <= B ? s1 - s0 : 0;
}
// Tiles of the prefix that sequence b shares.
__device__ __forceinline__ int skipped(const Tables& t, int b) {
  const int g = t.grp[b];
  return g == kNoGroup ? 0 : t.gp[g];
}
__device__ __forceinline__ int staged_tiles(int gp) { return (gp * kTile + kBN - 1) / kBN; }

// Tabulates the batch; returns streamed own tiles, streamed prefix tiles and staged tiles
// of one head.
template <int R>
__device__ __forceinline__ void tabulate_shared(const SharedArgs& a, Tables& t, int& all_own,
                                                int& all_gs, int& all_gt) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int B = a.d.B, NG = a.groups;
  if (tid == 0) t.falling = 0;
  int64_t row[R];
  int32_t cap[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int b = i * kThreads + tid;
    row[i] = row_of(a.d, min(b, B - 1));
    if (b <= NG) t.g0[b] = static_cast<int16_t>(max(-1, min(a.cu[b], B + 1)));
    cap[i] = b < NG ? a.shared[b] : 0;
  }
  if (R * kThreads == NG && tid == 0)
    t.g0[NG] = static_cast<int16_t>(max(-1, min(a.cu[NG], B + 1)));
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int b = i * kThreads + tid;
    const int32_t len = a.d.seq_lens[row[i] >= 0 ? row[i] : 0];
    if (b < B) {
      t.row[b] = static_cast<int32_t>(row[i]);
      t.len[b] = static_cast<int32_t>(row[i] >= 0 ? clamp_len(a.d, len) : 0);
    }
  }
  __syncthreads();
  // a group's prefix: whole tiles of what its first sequence holds
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int g = i * kThreads + tid;
    if (g < NG) {
      if (t.g0[g] > t.g0[g + 1]) t.falling = 1;
      const int n = members(t, g, B);
      const int most = n > 1 ? min(cap[i], t.len[t.g0[g]]) : 0;
      t.gp[g] = most > 0 ? most / kTile : 0;
    }
  }
  __syncthreads();
  // (bounds that fall back make groups overlap: two prefixes of one row, whose parts share
  // their places, and more tiles than the host has counted on.  There are no groups then)
  const bool falling = t.falling != 0;
  int own[R], gs[R], gt[R], own_i[R], gs_i[R], gt_i[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int b = i * kThreads + tid;
    int skip = 0;
    own[i] = gs[i] = gt[i] = 0;
    if (b < B) {
      const int g = falling ? -1 : last_at_most(t.g0, NG, b);
      const bool in = g >= 0 && b < t.g0[g] + members(t, g, B);
      // (one that ends inside the prefix attends alone: masked, infinities and NaN among the
      // values behind its end would reach it by their products with zero)
      const bool shares = in && t.len[b] >= t.gp[g] * kTile;
      if (shares) skip = t.gp[g];
      t.grp[b] = static_cast<uint16_t>(shares ? g : kNoGroup);
      const int tiles = (t.len[b] + kTile - 1) / kTile;
      own[i] = tiles > skip ? tiles - skip + kSegTiles : 0;
    }
    if (b < NG) {
      const int rows = members(t, b, B) * a.d.G, gp = falling ? 0 : t.gp[b];
      const int items = (rows + kRowsT - 1) / kRowsT;
      if (gp > 0 && rows > kRowsS) gt[i] = (staged_tiles(gp) + kItemTiles) * items;
      else if (gp > 0) gs[i] = gp + kSegTiles;
    }
    own_i[i] = wave_prefix_sum(own[i]);
    gs_i[i] = wave_prefix_sum(gs[i]);
    gt_i[i] = wave_prefix_sum(gt[i]);
    if (lane == 63) {
      t.wsum[0][i][wave] = own_i[i];
      t.wsum[1][i][wave] = gs_i[i];
      t.wsum[2][i][wave] = gt_i[i];
    }
  }
  __syncthreads();
  int run[3] = {0, 0, 0};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    int before[3] = {run[0], run[1], run[2]};
#pragma unroll
    for (int x = 0; x < 3; ++x)
#pragma unroll
      for (int w = 0; w < kShWaves; ++w) {
        const int s = t.wsum[x][i][w];
        before[x] += w < wave ? s : 0;
        run[x] += s;
      }
    const int b = i * kThreads + tid;
    if (b < B) t.own[b] = before[0] + own_i[i] - own[i];
    if (b < NG) {
      t.gs[b] = before[1] + gs_i[i] - gs[i];
      t.gt[b] = before[2] + gt_i[i] - gt[i];
    }
  }
  if (tid == 0) {
    t.own[B] = run[0];
    t.gs[NG] = run[1];
    t.gt[NG] = run[2];
  }
  __syncthreads();
  all_own = uniform(run[0]);
  all_gs = uniform(run[1]);
  all_gt = uniform(run[2]);
}

// How the tiles are divided among the workgroups and waves (all of it in scalar registers:
// the compiler takes what LDS and floats give for a lane's own).
struct Plan {
  int streamed, staged;  // tiles of all KV heads
  int wgs_t;             // workgroups of staged tiles, the grid's first ones
  int pw, pt;            // tiles of a wave's, of a workgroup's range
};
__device__ __forceinline__ Plan plan_of(const SharedArgs& a, int all_s, int all_t) {
  Plan p;
  const int N = gridDim.x;
  p.streamed = all_s * a.d.Hkv;
  p.staged = all_t * a.d.Hkv;
  const float wt = static_cast<float>(p.staged) * kStagedUnits, ws = static_cast<float>(p.streamed);
  int n = all_t == 0 ? 0 : static_cast<int>(N * (wt / (wt + ws)) + 0.5f);
  if (all_t > 0) n = n < 1 ? 1 : n;
  if (all_s > 0) n = n > N - 1 ? N - 1 : n;
  n = uniform(n);
  p.wgs_t = n;
  p.pt = n > 0 ? uniform((p.staged + n - 1) / n) : kMinStaged;
  p.pt = p.pt < kMinStaged ? kMinStaged : p.pt;
  const int waves = (N - n) * kShWaves;
  p.pw = waves > 0 ? uniform((p.streamed + waves - 1) / waves) : kMinStreamed;
  p.pw = p.pw < kMinStreamed ? kMinStreamed : p.pw;
  return p;
}

// The normalised state of column lo (dims 32 hi ..) into a part's row.
__device__ __forceinline__ void store_part(float* po, const q3::f32x4 (&acc)[8], float inv, int hi) {
  po += 32 * hi;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    *reinterpret_cast<q3::f32x4*>(po + 8 * r) =
        q3::f32x4{acc[0][r] * inv, acc[1][r] * inv, acc[2][r] * inv, acc[3][r] * inv};
    *reinterpret_cast<q3::f32x4*>(po + 8 * r + 4) =
        q3::f32x4{acc[4][r] * inv, acc[5][r] * inv, acc[6][r] * inv, acc[7][r] * inv};
  }
}

// ---- streamed tiles: one wave --------------------------------------------------------

// An item of the streamed list: a sequence's own keys, or a group's prefix.
struct StreamItem {
  int e;       // sequence, or B + group
  int n;       // tiles (below 1: none)
  int t0;      // first tile of the sequence
  int L;       // end of its keys
  int row;     // of the block table
};

__device__ __forceinline__ StreamItem stream_item(const SharedArgs& a, const Tables& t, int e) {
  const int B = a.d.B;
  StreamItem s;
  s.e = e;
  if (e < B) {
    s.n = uniform(t.own[e + 1] - t.own[e]) - kSegTiles;
    s.t0 = uniform(skipped(t, e));
    s.L = uniform(t.len[e]);
    s.row = uniform(t.row[e]);
  } else {
    const int g = e - B;
    s.n = uniform(t.gs[g + 1] - t.gs[g]) - kSegTiles;
    s.t0 = 0;
    s.L = s.n * kTile;
    s.row = s.n > 0 ? uniform(t.row[t.g0[g]]) : -1;
  }
  return s;
}

__device__ __forceinline__ void stream_range(const SharedArgs& a, const Tables& t, int all_own, int w, int g0,
                             int g1) {
  const DecodeArgs& d = a.d;
  const int lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  const int B = d.B, entries = B + a.groups;
  const int own_end = d.Hkv * all_own;

  StreamItem load;  // the item of the next tile to load: its KV head, the tile's place in it
  int hkv, at;
  int g = g0;       // its place in the list (an item's tiles lie behind its kSegTiles)
  {
    int e, before;
    if (g0 < own_end) {
      e = uniform(last_at_most(t.own, B, g0 / d.Hkv));
      before = uniform(t.own[e]);
    } else {
      const int p = (g0 - own_end) / d.Hkv;
      e = uniform(last_at_most(t.gs, a.groups, p));
      before = all_own + uniform(t.gs[e]);
      e += B;
    }
    load = stream_item(a, t, e);
    const int off = g0 - d.Hkv * before;
    hkv = uniform(off / (load.n + kSegTiles));
    at = off - hkv * (load.n + kSegTiles) - kSegTiles;
    if (at < 0) {
      g -= at;
      at = 0;
    }
  }
  TableWindow tw;
  window_load(tw, d, load.row, ((load.t0 + at) * kTile) / d.bs, lane);

  auto issue = [&](Chunk& c) {
    c.n = 0;
    if (g >= g1) return;
    if (at >= load.n) {  // the next item
      if (++hkv == d.Hkv) {
        hkv = 0;
        int e = load.e;
        do {
          ++e;
          load = stream_item(a, t, e);
        } while (load.n <= 0 && e + 1 < entries);
      }
      at = 0;
      g += kSegTiles;
      if (g >= g1) return;
      window_load(tw, d, load.row, (load.t0 * kTile) / d.bs, lane);
    }
    int n = load.n - at;
    n = n < kChunk ? n : kChunk;
    n = g1 - g < n ? g1 - g : n;
    c.n = n;
    c.t0 = load.t0 + at;
    c.seg = load.e * d.Hkv + hkv;
    c.ntiles = load.n;
    c.L = load.L;
    const uint16_t* kbase = d.k + static_cast<int64_t>(hkv) * d.k_sh;
    const uint16_t* vbase = d.v + static_cast<int64_t>(hkv) * d.v_sh;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      int64_t phys = -1;
      int sub = 0;
      if (i < n) {
        const int tok0 = (c.t0 + i) * kTile;
        phys = window_phys(tw, d, tok0 / d.bs, lane);
        sub = tok0 % d.bs;
      }
      load_tile(c, i, d, kbase, vbase, phys, sub, lo, hi);
    }
    at += n;
    g += n;
  };

  // the item being accumulated
  int cseg = -1, ce = 0, ct_lo = 0, ct_hi = 0, cn = 0, first = 0;
  int cb = 0, chead = 0;     // this lane's sequence and query head
  bool mine = false;         // its column is a row of the item
  Columns col;

  auto begin = [&](const Chunk& c) {
    ce = c.seg / d.Hkv;
    const int kvh = c.seg - ce * d.Hkv;
    ct_lo = c.t0;
    cn = c.ntiles;
    int head = lo;
    if (ce < B) {
      cb = ce;
      mine = lo < d.G;
      first = uniform(skipped(t, ce));
    } else {
      const int grp = ce - B, s = divide(lo, a.per_head);
      head = lo - s * d.G;
      mine = s < uniform(t.g0[grp + 1] - t.g0[grp]);
      cb = uniform(t.g0[grp]) + (mine ? s : 0);
      first = 0;
    }
    chead = kvh * d.G + (mine ? head : 0);
    col.last = c.L - 1;
    reset(col.st);
    const uint16_t* qp = d.q + cb * d.q_sb + static_cast<int64_t>(chead) * d.q_sh + hi * 8;
#pragma unroll
    for (int cc = 0; cc < 4; ++cc)
      col.q[cc] = q3::as_bf16x8(mine ? q3::ld16(qp + cc * 32) : q3::u32x4{0u, 0u, 0u, 0u});
  };

  auto finish = [&]() {
    const float l = q3::sum_xor32(q3::sum_xor16(col.st.l));
    const float inv = l > 0.f ? 1.f / l : 0.f;
    if (!mine) return;
    const bool whole = ct_hi - ct_lo == cn;
    if (whole && ce < B && first == 0) {
      store_out_bf16(d, cb, chead, col.st.acc, inv, hi);
      return;
    }
    const float lse = l > 0.f ? col.st.m + __builtin_log2f(l) : q3::kNegInf;
    float* po;
    float* pl;
    if (whole) {
      const int64_t row = static_cast<int64_t>(cb) * d.Hq + chead;
      po = (ce < B ? a.po_own : a.po_pre) + row * kD;
      pl = (ce < B ? a.lse_own : a.lse_pre) + row;
    } else {
      // a range's first item may go on from the one before, its last one into the next
      const int64_t slot = (static_cast<int64_t>(w) * 2 + (ct_lo == first ? 1 : 0)) * kRowsS + lo;
      po = a.po_s + slot * kD;
      pl = a.lse_s + slot;
    }
    store_part(po, col.st.acc, inv, hi);
    if (hi == 0) *pl = lse;
  };

  auto process = [&](Chunk& c) {
    if (c.seg != cseg) {
      if (cseg >= 0) finish();
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
  if (cseg >= 0) finish();
}

// ---- staged tiles: one workgroup ------------------------------------------------------

constexpr int kStageElems = 2 * kTileElems;  // a tile's keys, then its values

// A buffer load that writes LDS, 16 bytes a lane from LDS byte `to` on.  In assembly: with
// the builtin the compiler waits, before it reads one stage, for the loads into all of
// them.  Whoever reads the stage waits for it by count (staged_range), and nothing else
// here uses M0.
__device__ __forceinline__ void load_lds16(q3::u32x4 rsrc, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(to), "v"(offset), "s"(rsrc)
               : "memory");
}
__device__ __forceinline__ q3::u32x4 descriptor(const uint16_t* p, int bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  return q3::u32x4{static_cast<uint32_t>(at), static_cast<uint32_t>(at >> 32) & 0xffffu,
                   static_cast<uint32_t>(bytes), 0x00020000u};
}
// LDS byte of a shared array's element.
__device__ __forceinline__ uint32_t lds_byte(const uint16_t* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_t*)const_cast<uint16_t*>(p)));
}

// Where a range's next tiles lie, in LDS: for each group of 16 keys the page (-1: the table
// names no block of the pool) and the place in it, for each tile which of its groups have
// one.  (Held in registers, as the chunk kernels have them, the wait for the next pages'
// load would be a wait for the tiles ahead.)
constexpr int kPageTiles = 64;
constexpr int kTileGroups = kBN / kGroup;
struct Pages {
  int2 at[kPageTiles * kTileGroups];
  uint32_t ok[kPageTiles];
};

__device__ __forceinline__ void fill_pages(const SharedArgs& a, Pages& pages, int64_t row, int tile,
                                           int n) {
  const int tid = threadIdx.x;
  const int group = tile * kTileGroups + tid;
  if (tid >= kPageTiles * kTileGroups) return;
  const uint32_t p = divide(group, a.per_group);
  int32_t id = tid < n * kTileGroups && p < a.max_pages ? a.bt[row * a.bt_stride + p] : -1;
  id = id >= 0 && id < a.num_blocks ? id : -1;
  pages.at[tid] = int2{id, (group - static_cast<int>(p) * a.gpb) * kGroup};
  const uint64_t ok = __ballot(id >= 0);
  if (tid % kTileGroups == 0) pages.ok[tid / kTileGroups] = static_cast<uint32_t>(ok >> (tid & 63)) & 15u;
}

// A wave's part of a tile's loads, as read from Pages before they are issued.
struct Next {
  int page, sub;
  uint32_t ok;
};
// What a wave loads: waves 0 .. 3 a group of keys each, waves 4 .. 7 of values.
struct Loader {
  const uint16_t* base;  // the KV head of block 0
  int64_t blk;
  int slot;
  int group;             // of a tile
  uint32_t from[4];      // a lane's source offsets within a group
};
constexpr int kShare = 4;  // a wave's loads of a tile

__device__ __forceinline__ Loader loader_of(const SharedArgs& a, int lane, int wave) {
  Loader l;
  const bool keys = wave < 4;
  l.base = keys ? a.k : a.v;
  l.blk = keys ? a.k_blk : a.v_blk;
  l.slot = keys ? a.k_slot : a.v_slot;
  l.group = wave & 3;
#pragma unroll
  for (int j = 0; j < kShare; ++j) {
    // load j fills LDS rows 4 j .. 4 j + 3 of the group, lane i slot i % 16 of row 4 j + i / 16
    // (prefill_tile.hpp: the source chunk is slot ^ swz(row))
    const int row = 4 * j + (lane >> 4), slot = lane & 15;
    l.from[j] = static_cast<uint32_t>(row * l.slot * 2) +
                ((slot ^ (keys ? row & 15 : 4 * (row & 3))) << 4);
  }
  return l;
}

__device__ __forceinline__ Next next_tile(const Pages& pages, int i, const Loader& l) {
  const int2 at = pages.at[i * kTileGroups + l.group];
  return Next{at.x, at.y, pages.ok[i]};
}

// Issues this wave's share of a tile's loads: `keys` keys from its first on, head: the KV
// head's place.  Returns which of its groups lie in the pool.
__device__ __forceinline__ uint32_t stage_tile(const Loader& l, const uint16_t* head, int keys,
                                               const Next& n, const uint16_t* to) {
  const int page = uniform(n.page), sub = uniform(n.sub);
  const int rows = page >= 0 ? min(kGroup, keys - l.group * kGroup) : 0;
  const uint16_t* p = head;
  if (rows > 0) p += page * l.blk + static_cast<int64_t>(sub) * l.slot;
  // rows behind the last key lie outside the descriptor and read as zero
  const q3::u32x4 r = descriptor(p, rows > 0 ? (rows - 1) * l.slot * 2 + kRowBytes : 0);
  const uint32_t at = lds_byte(to) + l.group * (kGroup * kRowBytes);
#pragma unroll
  for (int j = 0; j < kShare; ++j) load_lds16(r, l.from[j], at + j * 1024);
  return uniform(n.ok);
}

// Maximum of a lane's 16 scores (as max3_scores, of half a tile).
__device__ __forceinline__ float max3_half(const q3::f32x16& a) {
  float m, t;
  asm volatile(
      "v_max3_f32 %0, %2, %3, %4\n\t"
      "v_max3_f32 %1, %10, %11, %12\n\t"
      "v_max3_f32 %0, %0, %5, %6\n\t"
      "v_max3_f32 %1, %1, %13, %14\n\t"
      "v_max3_f32 %0, %0, %7, %8\n\t"
      "v_max3_f32 %1, %1, %15, %16\n\t"
      "v_max3_f32 %0, %0, %9, %17\n\t"
      "v_max_f32 %0, %0, %1"
      : "=&v"(m), "=&v"(t)
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]),
        "v"(a[8]), "v"(a[9]), "v"(a[10]), "v"(a[11]), "v"(a[12]), "v"(a[13]), "v"(a[14]),
        "v"(a[15]));
  return m;
}

// (The builtin alone is no memory operation to the compiler.)
__device__ __forceinline__ void wait_all_waves() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A wave's probabilities of 32 keys, in two bf16 terms, not yet met with their values.
struct Probs {
  q3::u32x4 hi[2], lo[2];
};
__device__ __forceinline__ void prob_pair(Probs& p, float (&sums)[4], const q3::f32x16& s, int i,
                                          float c, float m) {
  const int g = i >> 2, h = i & 3;  // scores 2 h, 2 h + 1 of the 16 keys g
  const float e0 = q3::fast_exp2(__builtin_fmaf(s[8 * g + 2 * h], c, -m));
  const float e1 = q3::fast_exp2(__builtin_fmaf(s[8 * g + 2 * h + 1], c, -m));
  sums[(2 * h) & 3] += e0;
  sums[(2 * h + 1) & 3] += e1;
  uint32_t hi = q3::pack_bf16x2(e0, e1);
  asm("" : "+v"(hi));  // (or each half is rounded once more instead of taken from the pair)
  uint32_t lo = q3::pack_bf16x2(e0 - q3::bf16_lo(hi), e1 - q3::bf16_hi(hi));
  asm volatile("" : "+v"(lo));  // (or it is put off until the products have ended)
  p.hi[g][h] = hi;
  p.lo[g][h] = lo;
}

// Scores of the 32 keys that kt begins with: s[r] of a lane is key 8 (r / 4) + r % 4 +
// 4 (lane / 32).
__device__ __forceinline__ q3::f32x16 score(const LaneOffsets& off, const uint16_t* kt,
                                            const q3::bf16x8 (&qv)[8]) {
  q3::bf16x8 kf[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) kf[u] = lds_ld16(kt, off.kread ^ static_cast<uint32_t>(u << 5));
  __builtin_amdgcn_sched_barrier(0);  // (all reads on their way, not one by one)
  q3::f32x16 s;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
  for (int u = 0; u < 8; ++u) s = q3::mfma32x32x16(kf[u], qv[u], s);
  return s;
}

// Raises the running maximum to what scores s reach where that is far above it; returns
// the factor of what was summed under the old one.
__device__ __forceinline__ float raise_max(const q3::f32x16& s, float c, float& m_run) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");  // the products before a read in assembly
  const float m_cand = cross_half_max(max3_half(s)) * c;
  const bool raise = m_cand > m_run + kRescaleSlack;
  const float m_new = raise ? m_cand : m_run;
  const float alpha = raise ? q3::fast_exp2(m_run - m_new) : 1.f;
  m_run = m_new;
  return alpha;
}
__device__ __forceinline__ float finite_max(float m) { return m == q3::kNegInf ? 0.f : m; }

// O^T += V^T P^T of the 32 keys whose values vt begins with; between(i) is called after
// every second of the 16 products: work that runs beside them.
template <typename Between>
__device__ __forceinline__ void add_values(const LaneOffsets& off, const uint16_t* vt,
                                           const Probs& p, const Between& between,
                                           q3::f32x16 (&acc)[4]) {
  q3::bf16x8 vf[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) vf[u] = lds_vt(vt, pv_operand(off, u));
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int term = 0; term < 2; ++term)
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        // (the two terms' products of one accumulator lie four apart: the second would
        // wait for the first)
        acc[db] = q3::mfma32x32x16(vf[db], q3::as_bf16x8(term == 0 ? p.hi[g] : p.lo[g]), acc[db]);
        if (g == 0 && term == 1) vf[db] = lds_vt(vt, pv_operand(off, 4 + db));
        if (db & 1) between(4 * g + 2 * term + (db >> 1));
        __builtin_amdgcn_sched_barrier(0);
      }
}

// Staged tiles [p0, p1) of the list, by one workgroup.  A wave takes 32 of an item's rows
// and 32 of a tile's keys, so that each SIMD has work of up to 64 rows on; the two halves of
// the keys are joined when the item ends.
__device__ __forceinline__ void staged_range(const SharedArgs& a, const Tables& t, int all_t, int v,
                                             int p0, int p1, uint16_t* tiles_at, Pages& pages) {
  const DecodeArgs& d = a.d;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform(tid >> 6);
  LaneOffsets off;
  read_offsets(off, lane);
  const Loader loader = loader_of(a, lane, wave);
  int p = p0;
  while (p < p1) {
    const int kvh = uniform(p / all_t);
    const int in = p - kvh * all_t;
    const int grp = uniform(last_at_most(t.gt, a.groups, in));
    const int keys = uniform(t.gp[grp]) * kTile;
    const int tiles = (keys + kBN - 1) / kBN;
    const int s0 = uniform(t.g0[grp]), rows = uniform(t.g0[grp + 1] - t.g0[grp]) * d.G;
    const int before = uniform(t.gt[grp]);
    // (an item's tiles lie behind its kItemTiles)
    const int mt = uniform((in - before) / (tiles + kItemTiles));
    const int at0 = in - before - mt * (tiles + kItemTiles) - kItemTiles;
    const int j0 = at0 > 0 ? at0 : 0, j1 = min(tiles, at0 + p1 - p);
    p += tiles - at0;  // the next item
    if (j0 >= j1) continue;
    // waves 0 .. 3 lie on a SIMD each, 4 .. 7 on the same again
    const bool few = rows - mt * kRowsT <= kRowsT / 2;
    const int part = few ? wave & 1 : wave & 3;    // of the rows
    const int half = few ? wave >> 1 : wave >> 2;  // of the keys

    // this wave's 32 rows: lane l holds row r0 + l % 32
    const int r0 = mt * kRowsT + part * 32, r = r0 + (lane & 31);
    const bool active = r0 < rows && half < 2, mine = r < rows;
    const int s = divide(mine ? r : 0, a.per_head);
    const int b = s0 + s, head = kvh * d.G + ((mine ? r : 0) - s * d.G);
    q3::bf16x8 qv[8];
    {
      const uint16_t* qp = d.q + b * d.q_sb + static_cast<int64_t>(head) * d.q_sh + 8 * (lane >> 5);
#pragma unroll
      for (int c = 0; c < 8; ++c)
        qv[c] = q3::as_bf16x8(mine ? q3::ld16(qp + 16 * c) : q3::u32x4{0u, 0u, 0u, 0u});
    }
    const int64_t row = uniform(t.row[s0]);
    const uint16_t* kv = loader.base + kvh * (wave < 4 ? a.k_sh : a.v_sh);
    float m_run = q3::kNegInf, l_run = 0.f;
    q3::f32x16 acc[4];
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[db][x] = 0.f;

    for (int ja = j0; ja < j1; ja += kPageTiles) {
      const int je = min(ja + kPageTiles, j1);
      fill_pages(a, pages, row, ja, je - ja);
      __syncthreads();
      // (the queries too have arrived: that wait inside the loop would be one for the
      // tiles ahead)
#pragma unroll
      for (int c = 0; c < 8; ++c) asm volatile("" : "+v"(qv[c]));
      // stage i: tile ja + i of this round, then every fourth
      auto stage = [&](int j, const Next& n) {
        const uint16_t* to = tiles_at + ((j - ja) % kStages) * kStageElems;
        return stage_tile(loader, kv, keys - j * kBN, n, wave < 4 ? to : to + kTileElems);
      };
      uint32_t ok[kStages - 1] = {0u, 0u, 0u};  // of the next tiles
#pragma unroll
      for (int u = 0; u < kStages - 1; ++u)
        if (ja + u < je) ok[u] = stage(ja + u, next_tile(pages, u, loader));
      Next ahead = next_tile(pages, min(kStages - 1, je - ja - 1), loader);

      // a tile's scores, masked: x[i] is a key of group 2 half + i / 8, and the prefix ends
      // with a group
      auto mask = [&](q3::f32x16& x, int j, uint32_t okj) {
        const int left = keys - j * kBN;
        if (left < kBN) okj &= (1u << (left / kGroup)) - 1u;
        if (okj != 15u) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            x[i] = (okj >> (2 * half + i / 8)) & 1u ? x[i] : q3::kNegInf;
        }
      };
      const int rest = half < 2 ? half * 32 * kD : 0;  // where a wave's keys begin in a tile
      // the first tile has arrived (its loads are the oldest), at every wave's
      if (ja + 2 < je) __builtin_amdgcn_s_waitcnt(0x0f70 | 2 * kShare);
      else if (ja + 1 < je) __builtin_amdgcn_s_waitcnt(0x0f70 | kShare);
      else wait_loads();
      wait_all_waves();
      Probs probs;
      if (active) {
        q3::f32x16 x = score(off, tiles_at + rest, qv);
        mask(x, ja, ok[0]);
        const float alpha = raise_max(x, d.scale_log2, m_run), use = finite_max(m_run);
        float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 8; ++i) prob_pair(probs, sums, x, i, d.scale_log2, use);
        l_run = l_run * alpha + ((sums[0] + sums[1]) + (sums[2] + sums[3]));
#pragma unroll
        for (int db = 0; db < 4; ++db) acc[db] *= alpha;
      }
      const uint16_t* here = tiles_at;
      // Tile j's values meet their probabilities while the next tile's are computed.
      for (int j = ja; j + 1 < je; ++j) {
        const uint16_t* next = tiles_at + ((j + 1 - ja) % kStages) * kStageElems;
        // this wave's share of tile j + 1 has arrived (its loads of tile j + 2 are newer),
        // then everybody's has, and nobody reads tile j - 1 any more
        if (j + 2 < je) __builtin_amdgcn_s_waitcnt(0x0f70 | kShare);
        else wait_loads();
        wait_all_waves();
        const uint32_t ok1 = ok[1];
        ok[1] = ok[2];
        if (j + kStages - 1 < je) {
          ok[2] = stage(j + kStages - 1, ahead);
          ahead = next_tile(pages, min(j + kStages, je - 1) - ja, loader);
        }
        if (active) {
          const uint16_t* vt = here + kTileElems + rest;
          // (the halves in different order, or a SIMD's two waves are at the same step)
          if (half == 1) add_values(off, vt, probs, [](int) {}, acc);
          q3::f32x16 x = score(off, next + rest, qv);
          mask(x, j + 1, ok1);
          const float alpha = raise_max(x, d.scale_log2, m_run), use = finite_max(m_run);
          Probs p;
          float sums[4] = {0.f, 0.f, 0.f, 0.f};
          auto pair = [&](int i) { prob_pair(p, sums, x, i, d.scale_log2, use); };
          if (half == 0) {
            add_values(off, vt, probs, pair, acc);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) pair(i);
          }
          l_run = l_run * alpha + ((sums[0] + sums[1]) + (sums[2] + sums[3]));
          if (__any(alpha != 1.f)) {
#pragma unroll
            for (int db = 0; db < 4; ++db) acc[db] *= alpha;
          }
          probs = p;
        }
        here = next;
      }
      if (active) {
        add_values(off, here + kTileElems + rest, probs, [](int) {}, acc);
      }
      __syncthreads();  // pages and stages are read before they are filled again
    }
    // the second half's state, through the stages
    q3::f32x4* hold = reinterpret_cast<q3::f32x4*>(tiles_at + part * kTileElems) + lane;
    float2* ml = reinterpret_cast<float2*>(tiles_at + 4 * kTileElems) + part * 64 + lane;
    if (half == 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        hold[64 * i] = q3::f32x4{acc[i >> 2][4 * (i & 3)], acc[i >> 2][4 * (i & 3) + 1],
                               acc[i >> 2][4 * (i & 3) + 2], acc[i >> 2][4 * (i & 3) + 3]};
      *ml = float2{m_run, l_run};
    }
    __syncthreads();
    if (half == 0) {
      const float2 o = *ml;
      const float m = fmaxf(m_run, o.x), use = m == q3::kNegInf ? 0.f : m;
      const float f = q3::fast_exp2(m_run - use), g = q3::fast_exp2(o.x - use);
      const float l = q3::sum_xor32(l_run * f + o.y * g), inv = l > 0.f ? 1.f / l : 0.f;
      const float fi = f * inv, gi = g * inv;
      float* po;
      float* pl;
      if (j1 - j0 == tiles) {
        const int64_t to = static_cast<int64_t>(b) * d.Hq + head;
        po = a.po_pre + to * kD;
        pl = a.lse_pre + to;
      } else {
        const int64_t to = (2 * static_cast<int64_t>(v) + (j0 == 0 ? 1 : 0)) * a.rows_t + (r - mt * kRowsT);
        po = a.po_t + to * kD;
        pl = a.lse_t + to;
      }
      po += 4 * (lane >> 5);
      if (mine) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const q3::f32x4 x = hold[64 * i];
          q3::f32x4 y;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = acc[i >> 2][4 * (i & 3) + e] * fi + x[e] * gi;
          *reinterpret_cast<q3::f32x4*>(po + 8 * i) = y;
        }
        if (lane < 32) *pl = l > 0.f ? m + __builtin_log2f(l) : q3::kNegInf;
      }
    }
    __syncthreads();  // the stages are read before the next item's loads refill them
  }
}

__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_shared_kernel(SharedArgs a) {
  __shared__ __attribute__((aligned(1024))) uint16_t s_tiles[kStages * kStageElems];
  __shared__ Tables t;
  __shared__ Pages s_pages;
  const int tid = threadIdx.x, wave = uniform(tid >> 6);
  int all_own, all_gs, all_t;
  if (a.d.B <= kThreads && a.groups < kThreads)
    tabulate_shared<1>(a, t, all_own, all_gs, all_t);
  else
    tabulate_shared<kRounds>(a, t, all_own, all_gs, all_t);
  const Plan plan = plan_of(a, all_own + all_gs, all_t);
  if (blockIdx.x == gridDim.x - 1) {
    for (int b = tid; b < a.d.B; b += kThreads) {
      SeqMeta m{};
      m.own_at = t.own[b];
      m.own_n = max(0, t.own[b + 1] - t.own[b] - kSegTiles);
      if (skipped(t, b) > 0) {
        const int g = t.grp[b];
        const int rows = members(t, g, a.d.B) * a.d.G;
        m.kind = rows > kRowsS ? 2 : 1;
        m.pre_at = m.kind == 2 ? t.gt[g] : all_own + t.gs[g];
        m.pre_n = m.kind == 2 ? staged_tiles(t.gp[g]) : t.gp[g];
        m.pre_row = (b - t.g0[g]) * a.d.G;
      }
      a.seqs[b] = m;
    }
    if (tid == 0)
      *a.call = CallMeta{plan.pw, plan.pt, all_t, 0};
  }
  const int v = blockIdx.x;
  if (v < plan.wgs_t) {
    const int p0 = v * plan.pt;
    if (p0 < plan.staged)
      staged_range(a, t, all_t, v, p0, min(p0 + plan.pt, plan.staged), s_tiles, s_pages);
    return;
  }
  // a batch too small for every wave is dealt one wave a workgroup first
  const int N = gridDim.x - plan.wgs_t, at = v - plan.wgs_t;
  const bool spread = plan.streamed <= (N * kShWaves - 1) * plan.pw;
  const int w = spread ? wave * N + at : at * kShWaves + wave;
  const int g0 = w * plan.pw;
  if (g0 < plan.streamed)
    stream_range(a, t, all_own, w, g0, min(g0 + plan.pw, plan.streamed));
}

// ---- the join ---------------------------------------------------------------------------

// Rows (query heads of sequences) up to which a row's parts are dealt to eight waves, a CU
// reading what a few do too slowly: 4 sequences behind 30,000 tokens 41.7 us for 62.3, 40
// behind 30,000, 640 rows, 51 for 51; of 2,048 rows 57 for 48.
constexpr int kSplitRows = 512;

// Parts of a row: `n` slots from `first` on, `step` apart; the first one may lie elsewhere.
struct Parts {
  const float* po;
  const float* lse;
  int64_t first, next;  // rows of po: of part 0, of part i > 0: next + i * step
  int step, n;
};

// One workgroup of kSplit waves per (query head, sequence): lane i of a wave fetches the
// sum of the i-th of its parts, of up to 64 at once, then every lane owns two dimensions and
// sums the weighted parts, kBatch loads in flight; the waves are joined in LDS.
template <int kSplit>
__global__ __launch_bounds__(kSplit * 64) void paged_shared_join_kernel(SharedArgs a) {
  constexpr int kBatch = 8;
  const DecodeArgs& d = a.d;
  const int lane = threadIdx.x & 63;
  const int split = uniform(threadIdx.x >> 6);
  const int hq = blockIdx.x, b = blockIdx.y;
  const int hkv = hq / d.G, g = hq - hkv * d.G;
  const SeqMeta m = a.seqs[b];
  const CallMeta call = *a.call;
  const int64_t direct = static_cast<int64_t>(b) * d.Hq + hq;

  Parts part[2];
  part[0].n = part[1].n = 0;
  // a streamed item's parts: `col` its column of this row
  auto streamed = [&](Parts& x, const float* po, const float* lse, int before, int n, int col) {
    if (n == 0) return;
    const int S = d.Hkv * before + hkv * (n + kSegTiles) + kSegTiles;
    const int64_t wf = S / call.pw, wl = (S + n - 1) / call.pw;
    x.n = static_cast<int>(wl - wf + 1);
    if (wf == wl) {
      x.po = po;
      x.lse = lse;
      x.first = x.next = direct;
      x.step = 0;
      return;
    }
    x.po = a.po_s;
    x.lse = a.lse_s;
    x.first = (2 * wf + 1) * kRowsS + col;
    x.step = 2 * kRowsS;
    x.next = 2 * wf * kRowsS + col;
  };
  streamed(part[0], a.po_own, a.lse_own, m.own_at, m.own_n, g);
  if (m.kind == 0 && part[0].n == 1) return;  // written whole
  if (m.kind == 1) {
    streamed(part[1], a.po_pre, a.lse_pre, m.pre_at, m.pre_n, m.pre_row + g);
  } else if (m.kind == 2) {
    const int r = m.pre_row + g, mt = r / kRowsT;
    const int S = hkv * call.all_t + m.pre_at + mt * (m.pre_n + kItemTiles) + kItemTiles;
    const int64_t vf = S / call.pt, vl = (S + m.pre_n - 1) / call.pt;
    Parts& x = part[1];
    x.n = static_cast<int>(vl - vf + 1);
    if (vf == vl) {
      x.po = a.po_pre;
      x.lse = a.lse_pre;
      x.first = x.next = direct;
      x.step = 0;
    } else {
      x.po = a.po_t;
      x.lse = a.lse_t;
      const int row = r - mt * kRowsT;
      x.first = (2 * vf + 1) * a.rows_t + row;
      x.step = 2 * a.rows_t;
      x.next = 2 * vf * a.rows_t + row;
    }
  }
  const int all = part[0].n + part[1].n;
  auto row_at = [&](int i) {  // part i, in its own list
    const Parts& x = part[i < part[0].n ? 0 : 1];
    const int k = i < part[0].n ? i : i - part[0].n;
    return k == 0 ? x.first : x.next + static_cast<int64_t>(k) * x.step;
  };
  float M = q3::kNegInf, sw = 0.f, o0 = 0.f, o1 = 0.f;
  for (int i0 = split; i0 < all; i0 += 64 * kSplit) {
    const int i = i0 + kSplit * lane;
    const float lse = i < all ? (i < part[0].n ? part[0].lse : part[1].lse)[row_at(i)] : q3::kNegInf;
    float top = lse;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, q3::shfl_xor(top, o));
    const float m_new = fmaxf(M, top), use = m_new == q3::kNegInf ? 0.f : m_new;
    const float f = q3::fast_exp2(M - use);
    M = m_new;
    const float wt = q3::fast_exp2(lse - use);
    float wsum = wt;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) wsum += q3::shfl_xor(wsum, o);
    sw = sw * f + wsum;
    o0 *= f;
    o1 *= f;
    const int cnt = min(64, (all - i0 + kSplit - 1) / kSplit);
    for (int j0 = 0; j0 < cnt; j0 += kBatch) {
      float2 ov[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + kSplit * min(j0 + j, cnt - 1);
        const float* po = i < part[0].n ? part[0].po : part[1].po;
        ov[j] = *reinterpret_cast<const float2*>(po + row_at(i) * kD + 2 * lane);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const float u = j0 + j < cnt ? __shfl(wt, j0 + j, 64) : 0.f;
        o0 += u * ov[j].x;
        o1 += u * ov[j].y;
      }
    }
  }
  if constexpr (kSplit > 1) {
    __shared__ float s_m[kSplit], s_w[kSplit];
    __shared__ float2 s_o[kSplit][64];
    s_o[split][lane] = float2{o0, o1};
    if (lane == 0) {
      s_m[split] = M;
      s_w[split] = sw;
    }
    __syncthreads();
    if (split != 0) return;
#pragma unroll
    for (int x = 1; x < kSplit; ++x) M = fmaxf(M, s_m[x]);
    const float use = M == q3::kNegInf ? 0.f : M;
    sw = o0 = o1 = 0.f;
#pragma unroll
    for (int x = 0; x < kSplit; ++x) {
      const float f = q3::fast_exp2(s_m[x] - use);
      const float2 o = s_o[x][lane];
      sw += f * s_w[x];
      o0 += f * o.x;
      o1 += f * o.y;
    }
  }
  const float inv = sw > 0.f ? 1.f / sw : 0.f;
  *reinterpret_cast<uint32_t*>(d.out + b * d.o_sb + hq * d.o_sh + 2 * lane) =
      q3::pack_bf16x2(o0 * inv, o1 * inv);
}

// ---------------------------------------------------------------------------
// Host side.

// One workgroup a CU (its LDS); 256 where no device can be asked.
int shared_workgroups() {
  const int cus = cu_count();
  const int wgs = cus > 0 ? cus : 256;
  return wgs < kMaxWgs ? wgs : kMaxWgs;
}

struct SharedLayout {
  int64_t po_s, lse_s, po_t, lse_t, po_own, lse_own, po_pre, lse_pre, seqs, call, total;
  int rows_t;
};
SharedLayout shared_layout(int B, int num_heads, int G) {
  const int64_t wgs = shared_workgroups();
  const int64_t slots = wgs * kShWaves * 2 * kRowsS, rows = static_cast<int64_t>(B) * num_heads;
  SharedLayout l;
  l.rows_t = static_cast<int>(std::min<int64_t>(kRowsT, static_cast<int64_t>(B) * G));
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  };
  l.po_s = take(slots * kD * 4);
  l.lse_s = take(slots * 4);
  l.po_t = take(wgs * 2 * l.rows_t * kD * 4);
  l.lse_t = take(wgs * 2 * l.rows_t * 4);
  l.po_own = take(rows * kD * 4);
  l.lse_own = take(rows * 4);
  l.po_pre = take(rows * kD * 4);
  l.lse_pre = take(rows * 4);
  l.seqs = take(B * static_cast<int64_t>(sizeof(SeqMeta)));
  l.call = take(sizeof(CallMeta));
  l.total = at;
  return l;
}

}  // namespace

extern "C" size_t qwen3_paged_decode_shared_workspace_bytes(int B, int num_heads,
                                                            int num_kv_heads, int head_dim) {
  if (B <= 0 || B > kMaxSeqs || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads != 0 || num_heads / num_kv_heads > kMaxG || head_dim != kD)
    return 0;
  return static_cast<size_t>(shared_layout(B, num_heads, num_heads / num_kv_heads).total);
}

extern "C" int qwen3_paged_decode_shared_bf16(
    const void* q, const int64_t q_strides[2], const void* k_cache, const int64_t k_strides[3],
    const void* v_cache, const int64_t v_strides[3], int64_t num_blocks,
    const int32_t* block_table, int64_t bt_row_stride, int64_t max_rows, int64_t max_pages,
    const int32_t* seq_lens, int seq_len_bias, const int32_t* row_ids, const int32_t* cu_groups,
    const int32_t* shared_lens, int num_groups, void* out, const int64_t out_strides[2], int B,
    int num_heads, int num_kv_heads, int head_dim, int block_size, float scale, void* workspace,
    size_t workspace_bytes, void* stream) {
  const char* who = "qwen3_paged_decode_shared_bf16";
  SharedArgs a{};
  if (int rc = prepare(a.d, who, q, q_strides, k_cache, k_strides, v_cache, v_strides, num_blocks,
                       block_table, bt_row_stride, max_rows, max_pages, seq_lens,
                       seq_len_bias, row_ids, out, out_strides, B, num_heads, num_kv_heads,
                       head_dim, block_size, scale))
    return rc;
  if (!cu_groups || (num_groups > 0 && !shared_lens))
    return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  if (num_groups < 0 || num_groups > B)
    return q3::fail(QWEN3_EINVAL, "%s: %d groups of %d sequences", who, num_groups, B);
  if (B > kMaxSeqs)
    return q3::fail(QWEN3_EUNSUPPORTED, "%s: %d sequences (at most %d)", who, B, kMaxSeqs);
  if (!(scale > 0.f) || !(scale < __builtin_inff()))
    return q3::fail(QWEN3_EINVAL, "%s: scale must be positive and finite", who);
  // Rows behind a descriptor's end must lie outside it, and 16 of them inside 32-bit offsets.
  for (int64_t st : {k_strides[2], v_strides[2]})
    if (st < kD || st > (int64_t(1) << 24))
      return q3::fail(QWEN3_EUNSUPPORTED, "%s: slot stride %lld outside %d..2^24", who,
                      (long long)st, kD);
  // tiles are counted in 32 bits, and products of them with a range's width
  if (static_cast<int64_t>(B) * 2 * max_pages * (block_size / kTile) * num_kv_heads > (1 << 30))
    return q3::fail(QWEN3_EINVAL, "%s: batch %d times %lld pages, %d KV heads too large", who, B,
                    (long long)max_pages, num_kv_heads);
  if (B == 0) return QWEN3_OK;
  const SharedLayout l = shared_layout(B, num_heads, a.d.G);
  if (!workspace || workspace_bytes < static_cast<size_t>(l.total))
    return q3::fail(QWEN3_EWORKSPACE, "%s: workspace of %lld bytes needed, %zu given", who,
                    (long long)l.total, workspace ? workspace_bytes : (size_t)0);
  if (!q3::aligned16(workspace))
    return q3::fail(QWEN3_EALIGN, "%s: workspace must be 16-byte aligned", who);
  a.k = a.d.k;
  a.k_blk = a.d.k_sblk;
  a.k_sh = a.d.k_sh;
  a.k_slot = static_cast<int>(a.d.k_sslot);
  a.v = a.d.v;
  a.v_blk = a.d.v_sblk;
  a.v_sh = a.d.v_sh;
  a.v_slot = static_cast<int>(a.d.v_sslot);
  a.num_blocks = num_blocks;
  a.bt = block_table;
  a.bt_stride = bt_row_stride;
  a.max_pages = max_pages;
  a.gpb = block_size / kGroup;
  a.per_group = 1. / a.gpb;
  a.per_head = 1. / a.d.G;
  a.cu = cu_groups;
  a.shared = shared_lens;
  a.groups = num_groups;
  char* ws = static_cast<char*>(workspace);
  a.po_s = reinterpret_cast<float*>(ws + l.po_s);
  a.lse_s = reinterpret_cast<float*>(ws + l.lse_s);
  a.po_t = reinterpret_cast<float*>(ws + l.po_t);
  a.lse_t = reinterpret_cast<float*>(ws + l.lse_t);
  a.po_own = reinterpret_cast<float*>(ws + l.po_own);
  a.lse_own = reinterpret_cast<float*>(ws + l.lse_own);
  a.po_pre = reinterpret_cast<float*>(ws + l.po_pre);
  a.lse_pre = reinterpret_cast<float*>(ws + l.lse_pre);
  a.seqs = reinterpret_cast<SeqMeta*>(ws + l.seqs);
  a.call = reinterpret_cast<CallMeta*>(ws + l.call);
  a.rows_t = l.rows_t;
  const auto s = static_cast<hipStream_t>(stream);
  q3::clear_error();
  hipLaunchKernelGGL(paged_shared_kernel, dim3(shared_workgroups()), dim3(kThreads), 0, s, a);
  if (const int rc = q3::launch_status(who)) return rc;
  const dim3 grid(num_heads, B);
  if (B * num_heads <= kSplitRows)
    hipLaunchKernelGGL(paged_shared_join_kernel<8>, grid, dim3(8 * 64), 0, s, a);
  else
    hipLaunchKernelGGL(paged_shared_join_kernel<1>, grid, dim3(64), 0, s, a);
  return q3::launch_status(who);
}
