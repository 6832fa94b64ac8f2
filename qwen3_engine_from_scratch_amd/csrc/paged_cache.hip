// Pages of the cache copied, forked and moved: whole blocks of the pool
// (num_blocks, layers x heads x slots x head_dim contiguous per block), and the
// block-table entries that name them.
//
// Pure copies: bound by HBM (every byte read once and written once) or, for a page
// or two, by the launch.  The plan (which block goes where) is host data and
// travels in the launch's arguments, so a call is its launches and nothing else: no
// staging copy to wait for, and it can be captured.
#include <algorithm>
#include <memory>
#include <new>

#include "common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxJobs = 240;   // copies of one launch: their plan is a launch argument
// 16-byte chunks a thread copies.  200 moves of 1.8 MB: 130 us with one, 135 with two, 140
// with four (a plain copy of as many bytes: 137); with cached loads and stores 139, 141
// and 148: nothing reads a moved page before the caches have turned over.
constexpr int kUnroll = 1;
constexpr int kPiece = kThreads * kUnroll;  // chunks of a block that one workgroup copies

struct CopyJobs {
  int32_t src[kMaxJobs];
  int32_t dst[kMaxJobs];
  int32_t tokens[kMaxJobs];  // slots copied; the others of the block are zeroed
};

struct Pool {
  uint16_t* k;
  uint16_t* v;
  int64_t block_chunks;  // 16-byte chunks of one block
  int slot_chunks;       // of one slot
  int block_size;
};

// One piece of one block of K or of V.  kOnce: no other copy of the call reads the source
// (forks of one request do: 24 forks of eight, 17.7 us with streaming loads, 10.8 without).
template <bool kOnce>
__device__ __forceinline__ void copy_piece(const Pool& p, int64_t piece, int which, int64_t src,
                                           int64_t dst, int tokens) {
  uint16_t* base = which ? p.v : p.k;
  const uint16_t* s = base + src * p.block_chunks * 8;
  uint16_t* d = base + dst * p.block_chunks * 8;
  const int64_t c0 = piece * kPiece + threadIdx.x;
  q3::u32x4 x[kUnroll];
  const bool whole = tokens >= p.block_size;
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int64_t c = c0 + i * kThreads;
    x[i] = q3::u32x4{0u, 0u, 0u, 0u};
    if (c < p.block_chunks &&
        (whole || static_cast<uint32_t>(c) / p.slot_chunks % p.block_size <
                      static_cast<uint32_t>(tokens)))
      x[i] = kOnce ? q3::ld16_nt(s + 8 * c) : q3::ld16(s + 8 * c);
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int64_t c = c0 + i * kThreads;
    if (c < p.block_chunks)
      __builtin_nontemporal_store(x[i], reinterpret_cast<q3::u32x4*>(d + 8 * c));
  }
}

__global__ __launch_bounds__(kThreads) void page_copy_kernel(Pool p, CopyJobs jobs) {
  const int j = blockIdx.y;
  copy_piece<false>(p, blockIdx.x, blockIdx.z, jobs.src[j], jobs.dst[j], jobs.tokens[j]);
}

// Forks: row dst takes over the entries of row src for the first tokens[j] tokens.
struct ForkJobs {
  int32_t src[kMaxJobs];
  int32_t dst[kMaxJobs];
  int32_t tokens[kMaxJobs];
  int32_t block[kMaxJobs];   // the copy of a partly filled last page
};

struct Table {
  int32_t* bt;
  int64_t stride, rows, pages;
  int32_t* seq_lens;
  int64_t num_blocks;
};

__global__ __launch_bounds__(kThreads) void page_fork_kernel(Pool p, Table t, ForkJobs jobs,
                                                             int pieces) {
  const int j = blockIdx.y;
  const int64_t src = jobs.src[j], dst = jobs.dst[j];
  const int tokens = jobs.tokens[j];
  const int full = tokens / p.block_size, rest = tokens - full * p.block_size;
  if (blockIdx.x < 2 * static_cast<unsigned>(pieces)) {
    if (rest == 0) return;
    const int32_t from = t.bt[src * t.stride + full];
    if (from < 0 || from >= t.num_blocks) return;
    copy_piece<false>(p, blockIdx.x >> 1, blockIdx.x & 1, from, jobs.block[j], rest);
    return;
  }
  // the table row, one workgroup
  for (int64_t i = threadIdx.x; i < t.pages; i += kThreads)
    t.bt[dst * t.stride + i] =
        i < full ? t.bt[src * t.stride + i] : (i == full && rest > 0 ? jobs.block[j] : -1);
  if (threadIdx.x == 0) t.seq_lens[dst] = tokens;
}

// Moves: block src[i] goes to dst[i]; src ascending, so an entry finds its move.
struct MoveJobs {
  int32_t src[kMaxJobs];
  int32_t dst[kMaxJobs];
};

// The first `scans` workgroups of a launch relabel the table, the others copy: a
// move is one launch.
__global__ __launch_bounds__(kThreads) void page_move_kernel(Pool p, Table t, MoveJobs jobs, int n,
                                                             int scans, int pieces) {
  if (blockIdx.x >= static_cast<unsigned>(scans)) {
    const int64_t i = blockIdx.x - scans;  // (job, K or V, piece)
    const int piece = static_cast<int>(i % pieces);
    const int j = static_cast<int>(i / pieces);
    copy_piece<true>(p, piece, j & 1, jobs.src[j >> 1], jobs.dst[j >> 1], p.block_size);
    return;
  }
  __shared__ int32_t s_src[kMaxJobs], s_dst[kMaxJobs];
  for (int i = threadIdx.x; i < n; i += kThreads) {
    s_src[i] = jobs.src[i];
    s_dst[i] = jobs.dst[i];
  }
  __syncthreads();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t row = i / t.pages, col = i - row * t.pages;
  if (row >= t.rows) return;
  int32_t* e = t.bt + row * t.stride + col;
  const int32_t b = *e;
  int lo = 0, hi = n - 1;  // least index with src >= b, or the last
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (s_src[mid] < b) lo = mid + 1; else hi = mid;
  }
  if (s_src[lo] == b) *e = s_dst[lo];
}

int check_pool(Pool& p, void* k_cache, void* v_cache, int64_t block_elems, int slot_elems,
               int block_size, int64_t num_blocks, const char* who) {
  if (!k_cache || !v_cache) return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  if (block_elems <= 0 || slot_elems <= 0 || block_size <= 0 || num_blocks <= 0 ||
      num_blocks > 0x7fffffff || block_elems % (static_cast<int64_t>(slot_elems) * block_size) != 0)
    return q3::fail(QWEN3_EINVAL, "%s: bad sizes", who);
  if (slot_elems % 8 != 0 || !q3::aligned16(k_cache) || !q3::aligned16(v_cache))
    return q3::fail(QWEN3_EALIGN, "%s: slots must be whole 16-byte chunks", who);
  if (block_elems > (int64_t(1) << 31))
    return q3::fail(QWEN3_EUNSUPPORTED, "%s: blocks of %lld elements", who, (long long)block_elems);
  p.k = static_cast<uint16_t*>(k_cache);
  p.v = static_cast<uint16_t*>(v_cache);
  p.block_chunks = block_elems / 8;
  p.slot_chunks = slot_elems / 8;
  p.block_size = block_size;
  return QWEN3_OK;
}

// Every id a block of the pool, no destination twice and none that is also a
// source: the copies of a call run at the same time.  plan: the copies, src ascending.
struct Plan {
  std::unique_ptr<int32_t[]> src, dst;
};

int check_plan(Plan& plan, const int32_t* src, const int32_t* dst, int n, int64_t num_blocks,
               bool src_once, const char* who) {
  if (n > num_blocks)
    return q3::fail(QWEN3_EINVAL, "%s: %d destinations among %lld", who, n, (long long)num_blocks);
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= num_blocks || dst[i] < 0 || dst[i] >= num_blocks)
      return q3::fail(QWEN3_EINVAL, "%s: entry %d (%d -> %d) outside 0 .. %lld", who, i,
                      src[i], dst[i], (long long)num_blocks - 1);
  std::unique_ptr<int64_t[]> pairs(new (std::nothrow) int64_t[n]);
  plan.src.reset(new (std::nothrow) int32_t[n]);
  plan.dst.reset(new (std::nothrow) int32_t[n]);
  if (!pairs || !plan.src || !plan.dst) return q3::fail(QWEN3_EINVAL, "%s: out of memory", who);
  for (int i = 0; i < n; ++i) plan.dst[i] = dst[i];
  std::sort(plan.dst.get(), plan.dst.get() + n);
  for (int i = 1; i < n; ++i)
    if (plan.dst[i] == plan.dst[i - 1])
      return q3::fail(QWEN3_EINVAL, "%s: %d is written twice", who, plan.dst[i]);
  for (int i = 0; i < n; ++i)
    if (std::binary_search(plan.dst.get(), plan.dst.get() + n, src[i]))
      return q3::fail(QWEN3_EINVAL, "%s: %d is read and written", who, src[i]);
  for (int i = 0; i < n; ++i) pairs[i] = (static_cast<int64_t>(src[i]) << 32) | dst[i];
  std::sort(pairs.get(), pairs.get() + n);
  for (int i = 0; i < n; ++i) {
    plan.src[i] = static_cast<int32_t>(pairs[i] >> 32);
    plan.dst[i] = static_cast<int32_t>(pairs[i] & 0xffffffff);
    if (src_once && i > 0 && plan.src[i] == plan.src[i - 1])
      return q3::fail(QWEN3_EINVAL, "%s: %d moves twice", who, plan.src[i]);
  }
  return QWEN3_OK;
}

int check_table(Table& t, int32_t* block_table, int64_t bt_row_stride, int64_t max_rows,
                int64_t max_pages, int64_t num_blocks, const char* who) {
  if (!block_table) return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  if (max_rows <= 0 || max_pages <= 0 || bt_row_stride < max_pages || max_rows > 0x7fffffff ||
      max_pages > 0x7fffffff)
    return q3::fail(QWEN3_EINVAL, "%s: bad table sizes", who);
  t.bt = block_table;
  t.stride = bt_row_stride;
  t.rows = max_rows;
  t.pages = max_pages;
  t.num_blocks = num_blocks;
  return QWEN3_OK;
}

}  // namespace

extern "C" int qwen3_page_copy_bf16(void* k_cache, void* v_cache, int64_t block_elems,
                                    int slot_elems, int block_size, int64_t num_blocks,
                                    const int32_t* src, const int32_t* dst, const int32_t* tokens,
                                    int n, void* stream) {
  const char* who = "qwen3_page_copy_bf16";
  Pool p{};
  if (const int rc = check_pool(p, k_cache, v_cache, block_elems, slot_elems, block_size,
                                num_blocks, who))
    return rc;
  if (n < 0 || (n > 0 && (!src || !dst)))
    return q3::fail(QWEN3_EINVAL, "%s: bad list of copies", who);
  if (n == 0) return QWEN3_OK;
  Plan plan;
  if (const int rc = check_plan(plan, src, dst, n, num_blocks, false, who)) return rc;
  if (tokens)
    for (int i = 0; i < n; ++i)
      if (tokens[i] < 0 || tokens[i] > block_size)
        return q3::fail(QWEN3_EINVAL, "%s: %d tokens of a block of %d", who, tokens[i], block_size);
  const int64_t pieces = q3::cdiv(p.block_chunks, kPiece);
  q3::clear_error();
  for (int at = 0; at < n; at += kMaxJobs) {
    const int m = std::min(kMaxJobs, n - at);
    CopyJobs jobs{};
    for (int i = 0; i < m; ++i) {
      jobs.src[i] = src[at + i];
      jobs.dst[i] = dst[at + i];
      jobs.tokens[i] = tokens ? tokens[at + i] : block_size;
    }
    hipLaunchKernelGGL(page_copy_kernel, dim3(static_cast<unsigned>(pieces), m, 2), dim3(kThreads),
                       0, static_cast<hipStream_t>(stream), p, jobs);
    if (const int rc = q3::launch_status(who)) return rc;
  }
  return QWEN3_OK;
}

extern "C" int qwen3_page_fork_bf16(void* k_cache, void* v_cache, int64_t block_elems,
                                    int slot_elems, int block_size, int64_t num_blocks,
                                    int32_t* block_table, int64_t bt_row_stride, int64_t max_rows,
                                    int64_t max_pages, int32_t* seq_lens, const int32_t* src_rows,
                                    const int32_t* dst_rows, const int32_t* tokens,
                                    const int32_t* new_blocks, int n, void* stream) {
  const char* who = "qwen3_page_fork_bf16";
  Pool p{};
  if (const int rc = check_pool(p, k_cache, v_cache, block_elems, slot_elems, block_size,
                                num_blocks, who))
    return rc;
  Table t{};
  if (const int rc = check_table(t, block_table, bt_row_stride, max_rows, max_pages, num_blocks, who))
    return rc;
  if (!seq_lens || n < 0 || (n > 0 && (!src_rows || !dst_rows || !tokens || !new_blocks)))
    return q3::fail(QWEN3_EINVAL, "%s: bad list of forks", who);
  if (n == 0) return QWEN3_OK;
  t.seq_lens = seq_lens;
  Plan plan;  // rows instead of blocks: the same rules
  if (const int rc = check_plan(plan, src_rows, dst_rows, n, max_rows, false, who)) return rc;
  std::unique_ptr<int32_t[]> fresh(new (std::nothrow) int32_t[n]);
  if (!fresh) return q3::fail(QWEN3_EINVAL, "%s: out of memory", who);
  int parts = 0;
  for (int i = 0; i < n; ++i) {
    if (tokens[i] < 0 || tokens[i] > max_pages * block_size)
      return q3::fail(QWEN3_EINVAL, "%s: fork %d of %d tokens: a table row holds %lld", who, i,
                      tokens[i], (long long)(max_pages * block_size));
    if (tokens[i] % block_size == 0) continue;
    if (new_blocks[i] < 0 || new_blocks[i] >= num_blocks)
      return q3::fail(QWEN3_EINVAL, "%s: fork %d needs a block for its last page, got %d", who, i,
                      new_blocks[i]);
    fresh[parts++] = new_blocks[i];
  }
  std::sort(fresh.get(), fresh.get() + parts);
  for (int i = 1; i < parts; ++i)
    if (fresh[i] == fresh[i - 1])
      return q3::fail(QWEN3_EINVAL, "%s: block %d is written twice", who, fresh[i]);
  const int64_t pieces = q3::cdiv(p.block_chunks, kPiece);
  q3::clear_error();
  for (int at = 0; at < n; at += kMaxJobs) {
    const int m = std::min(kMaxJobs, n - at);
    ForkJobs jobs{};
    for (int i = 0; i < m; ++i) {
      jobs.src[i] = src_rows[at + i];
      jobs.dst[i] = dst_rows[at + i];
      jobs.tokens[i] = tokens[at + i];
      jobs.block[i] = new_blocks[at + i];
    }
    hipLaunchKernelGGL(page_fork_kernel, dim3(static_cast<unsigned>(2 * pieces + 1), m),
                       dim3(kThreads), 0, static_cast<hipStream_t>(stream), p, t, jobs,
                       static_cast<int>(pieces));
    if (const int rc = q3::launch_status(who)) return rc;
  }
  return QWEN3_OK;
}

extern "C" int qwen3_page_move_bf16(void* k_cache, void* v_cache, int64_t block_elems,
                                    int slot_elems, int block_size, int64_t num_blocks,
                                    int32_t* block_table, int64_t bt_row_stride, int64_t max_rows,
                                    int64_t max_pages, const int32_t* src, const int32_t* dst,
                                    int n, void* stream) {
  const char* who = "qwen3_page_move_bf16";
  Pool p{};
  if (const int rc = check_pool(p, k_cache, v_cache, block_elems, slot_elems, block_size,
                                num_blocks, who))
    return rc;
  Table t{};
  if (const int rc = check_table(t, block_table, bt_row_stride, max_rows, max_pages, num_blocks, who))
    return rc;
  if (n < 0 || (n > 0 && (!src || !dst)))
    return q3::fail(QWEN3_EINVAL, "%s: bad list of moves", who);
  if (n == 0) return QWEN3_OK;
  Plan plan;
  if (const int rc = check_plan(plan, src, dst, n, num_blocks, true, who)) return rc;
  const int64_t pieces = q3::cdiv(p.block_chunks, kPiece);
  const int64_t scans = q3::cdiv(max_rows * max_pages, kThreads);
  const int64_t most = scans + 2 * pieces * std::min(n, kMaxJobs);
  if (most > q3::kMaxThreads / kThreads) return q3::fail(QWEN3_EINVAL, "%s: table or blocks too large", who);
  q3::clear_error();
  for (int at = 0; at < n; at += kMaxJobs) {
    const int m = std::min(kMaxJobs, n - at);
    MoveJobs jobs{};
    for (int i = 0; i < m; ++i) {
      jobs.src[i] = plan.src[at + i];
      jobs.dst[i] = plan.dst[at + i];
    }
    hipLaunchKernelGGL(page_move_kernel, dim3(static_cast<unsigned>(scans + 2 * pieces * m)),
                       dim3(kThreads), 0, static_cast<hipStream_t>(stream), p, t, jobs, m,
                       static_cast<int>(scans), static_cast<int>(pieces));
    if (const int rc = q3::launch_status(who)) return rc;
  }
  return QWEN3_OK;
}
