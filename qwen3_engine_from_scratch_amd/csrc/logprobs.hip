// Log probabilities of given tokens, the entropy of their distribution and its most
// likely tokens, from rows of logits, and the logits' gradient.
//
// With z = x / T and c = log2(e) / T, in one pass over a row: a thread keeps the largest x
// so far, m, a point P beside m c, s = sum 2^(x c - P) and s1 = sum 2^(x c - P) (x c - P).
// Two such states join with f = 2^(P - P'): s' = f s, s1' = f (s1 + s (P - P')).  Then
//   log p_t = (x_t - m) / T - ln 2 (log2 s - (m c - P)),   H = ln 2 (log2 s - s1 / s).
// P is m c rounded, so that x c - P is one multiply-add; what it is off, m c - P, is a factor
// of the sums, known and taken out again.  P's half step is 1/2 up to 2^24, doubles with
// every power of two behind it and would leave the exponents' range from 2^31 on: where
// |m c| is 2^24 or more (finite masks, small temperatures) P is m c itself and the exponents
// are (x - m) c.  (That form everywhere: 4,096 x 151,936 bf16 206 us for 200; sums of far
// rows in a second pass: 64 rows of a step masked by -1e9 26.4 us for 20.)
//
// The n most likely tokens come out of the same pass: a thread keeps the maximum of its
// own tokens, and the n-th largest of these maxima, T, is a bound that n tokens reach.  Only
// threads whose maximum reaches it hold tokens that do, so their tokens alone are read
// again (a few dozen 16-byte pieces each) and the few that reach T are ranked.  Where many
// threads reach T by equal values (a row masked but for fewer than n tokens), those above
// T are gathered this way and the lowest indices at T by walking the row from its start.
// Rows with NaN (which ranks above every number, as torch sorts) or +inf, and rows whose
// candidates overflow their list, are ranked one token a round.
//
// A row is cut into parts of whole rounds where there are too few rows for the device; a
// second launch joins the parts.
//
// What bounds it: HBM where there are rows enough (4,096 x 151,936 bf16 200 us, 6.2 TB/s, with
// 5 listed 226, with 20 listed 292; 1,003 x 50,021 fp32, 4 given, 8 listed, 41 us, 4.9 TB/s, of
// which the list some 5),
// latency in a decode step (64 rows, 20 listed: 12.7 us, of which the list 4, and 6.2 of the
// join; one row, 5 listed, 7.3 and 4.4) and, with a list, in short rows.  The gradient reads
// and writes 1.25 GB of 2,048 x 151,936 in 222 us, 5.6 TB/s, after 100 of the log
// probabilities.
#include "common.hpp"

namespace {

// Threads of a workgroup (512: 20 listed of 2,000 x 16,000 bf16 40 us for 30, of 1 and of 64
// rows of a step 17.4 and 24.3 for 16.0 and 22.1; 64 listed of 12 x 151,936 37 for 42), and
// where whole rows have up to kShort 16-byte pieces (256 there: 5,571 x 796, 50 listed, 40
// us for 27, 2,000 x 8,000, 20 listed, 26 for 21; 128 for 3,000 x 8,000 fp32, 50 listed, 42
// for 38).
constexpr int kThreads = 256;
constexpr int kShortThreads = 128;
constexpr int kShort = 1024;
constexpr int kMaxTop = 64;      // most likely tokens a row
constexpr int kMaxGiven = 64;    // given tokens a row
constexpr int kMaxParts = 64;
constexpr int kResident = 512;   // parts of all rows: 2 a CU (1,024: 64 rows 24.6 us for 22.1)
constexpr int kCap = 1024;       // candidates of a part
constexpr int kFewThreads = 64;  // threads that reach T and are read again one by one
constexpr int kBatchTokens = 16; // a thread's tokens of a load (64 rows of a step 22.6 us, of 32 24.2)
constexpr int kFewPieces = 256;  // pieces that are read again for a bound looser than n needs
constexpr uint32_t kMinusInf = 0x007fffffu;  // key of -inf
constexpr float kFar = 0x1p24f;  // |m c| from which P is m c itself
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kTiny = -200.f;  // 2^x is zero below it: keeps 0 * -inf out of the sums

typedef uint32_t piece_t __attribute__((__vector_size__(16), __aligned__(2)));
typedef unsigned long long u64;

struct Bf16 {
  static constexpr int kE = 8, kBytes = 2;
  static __device__ __forceinline__ void unpack(q3::u32x4 w, float (&x)[kE]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = q3::bf16_lo(w[i]);
      x[2 * i + 1] = q3::bf16_hi(w[i]);
    }
  }
  static __device__ __forceinline__ float one(const char* p) {
    return q3::bf16_lo(*reinterpret_cast<const uint16_t*>(p));
  }
  static __device__ __forceinline__ q3::u32x4 pack(const float (&x)[kE]) {
    return q3::u32x4{q3::pack_bf16x2(x[0], x[1]), q3::pack_bf16x2(x[2], x[3]),
                     q3::pack_bf16x2(x[4], x[5]), q3::pack_bf16x2(x[6], x[7])};
  }
  static __device__ __forceinline__ void put(char* p, float x) {
    *reinterpret_cast<uint16_t*>(p) = q3::bf16_bits(x);
  }
};
struct Fp16 {
  static constexpr int kE = 8, kBytes = 2;
  typedef _Float16 h8 __attribute__((__vector_size__(16)));
  static __device__ __forceinline__ void unpack(q3::u32x4 w, float (&x)[kE]) {
    const h8 h = __builtin_bit_cast(h8, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(h[i]);
  }
  static __device__ __forceinline__ float one(const char* p) {
    return static_cast<float>(*reinterpret_cast<const _Float16*>(p));
  }
  static __device__ __forceinline__ q3::u32x4 pack(const float (&x)[kE]) {
    h8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = static_cast<_Float16>(x[i]);
    return __builtin_bit_cast(q3::u32x4, h);
  }
  static __device__ __forceinline__ void put(char* p, float x) {
    *reinterpret_cast<_Float16*>(p) = static_cast<_Float16>(x);
  }
};
struct Fp32 {
  static constexpr int kE = 4, kBytes = 4;
  static __device__ __forceinline__ void unpack(q3::u32x4 w, float (&x)[kE]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ float one(const char* p) {
    return *reinterpret_cast<const float*>(p);
  }
  static __device__ __forceinline__ q3::u32x4 pack(const float (&x)[kE]) {
    return q3::u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                     __float_as_uint(x[3])};
  }
  static __device__ __forceinline__ void put(char* p, float x) {
    *reinterpret_cast<float*>(p) = x;
  }
};

// A row's (or part's) sums.
struct alignas(16) Sums {
  float max;  // largest logit (-inf: none above it)
  float s, s1;
};

struct LogprobArgs {
  const char* x;
  int64_t row_bytes;
  int vocab;
  int pieces;            // 16-byte pieces of a row, the last one maybe shorter
  int parts, per_part;   // parts of a row, pieces of a part
  float c, inv_t;        // log2(e) / temperature, 1 / temperature
  const int64_t* tokens; // (rows, given), nullable
  int given;
  float* logprobs;
  float* entropy;        // nullable
  int top;
  int64_t* top_ids;
  float* top_logprobs;
  float2* stats;         // (rows) maximum, log2 s; nullable
  Sums* part_sums;       // (rows, parts)
  u64* part_top;         // (rows, parts, top), descending, 0: none
};

// Order of logits as whole numbers: larger value, larger key; equal zeros, NaN on top (one
// above the key of +inf, so that no token ranks as high as the ~0 that bounds a search).
constexpr uint32_t kNanKey = 0xff800001u;
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return kNanKey;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}
// A token among others: the larger logit first, the lower index among equal ones.
__device__ __forceinline__ u64 ranked(uint32_t key, uint32_t idx) {
  return static_cast<u64>(key) << 32 | static_cast<uint32_t>(~idx);
}
__device__ __forceinline__ uint32_t key_in(u64 r) { return static_cast<uint32_t>(r >> 32); }
__device__ __forceinline__ uint32_t index_in(u64 r) { return ~static_cast<uint32_t>(r); }

// First token that a piece's 16 bytes are loaded from: the row's last piece is loaded
// from the row's last 16 bytes, and its tokens before the piece's own first are skipped.
template <typename Tr>
__device__ __forceinline__ int piece_start(const LogprobArgs& a, int p) {
  return min(p * Tr::kE, a.vocab - Tr::kE);
}
// (Rows shorter than 16 bytes are read one token at a time; the tokens behind the row's
// end count as skipped ones.)
template <typename Tr>
__device__ __forceinline__ q3::u32x4 load_piece(const LogprobArgs& a, const char* xr, int p) {
  if (a.vocab < Tr::kE) {
    float x[Tr::kE];
    for (int e = 0; e < Tr::kE; ++e) x[e] = e < a.vocab ? Tr::one(xr + e * Tr::kBytes) : 0.f;
    return Tr::pack(x);
  }
  const piece_t* src = reinterpret_cast<const piece_t*>(
      xr + static_cast<int64_t>(piece_start<Tr>(a, p)) * Tr::kBytes);
  return __builtin_bit_cast(q3::u32x4, __builtin_nontemporal_load(src));
}
// Whether element e of piece p is a token of its own, and which.
template <typename Tr>
__device__ __forceinline__ bool token_at(const LogprobArgs& a, int p, int e, int& idx) {
  if (a.vocab < Tr::kE) {
    idx = e;
    return e < a.vocab;
  }
  idx = piece_start<Tr>(a, p) + e;
  return idx >= p * Tr::kE;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;  // (fmaxf would first quiet each operand)
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
  return m;
}

// Whether P of the largest logit `max` is max c itself.
__device__ __forceinline__ bool far(float max, float c) {
  return !(__builtin_fabsf(max * c) < kFar) && __builtin_fabsf(max) < __builtin_inff();
}
// P where it is not (of no logit but -inf the least that one can be).
__device__ __forceinline__ float point(float max, float c) { return fmaxf(max * c, -kFar); }

// The states' join: a with a larger maximum, by d = P - P'.
__device__ __forceinline__ void raise_by(Sums& a, float max, float d) {
  d = fmaxf(d, -3e38f);
  const float f = q3::fast_exp2(d);
  a.s1 = f * (a.s1 + a.s * fmaxf(d, 2.f * kTiny));
  a.s *= f;
  a.max = max;
}
// The same where either may be far.
__device__ __forceinline__ void raise(Sums& a, float max, float c) {
  float d = point(a.max, c) - point(max, c);
  if (far(max, c))
    d = far(a.max, c) ? (a.max - max) * c : -__builtin_fmaf(max, c, -point(a.max, c));
  else if (far(a.max, c))
    d = __builtin_fmaf(a.max, c, -point(max, c));
  // (a state of -inf alone: s is 0, whatever its point)
  raise_by(a, max, a.max == q3::kNegInf ? -3e38f : d);
}

// Adds N tokens (-inf: none) at y(x) = x c - P.
template <int N, bool kEnt, typename Y>
__device__ __forceinline__ void add(Sums& st, const float (&x)[N], const Y& exponent) {
  float s[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = exponent(x[i]);
    const float e = q3::fast_exp2(y);
    s[i & 3] += e;
    if constexpr (kEnt) s1[i & 3] = __builtin_fmaf(e, fmaxf(y, kTiny), s1[i & 3]);
  }
  st.s += (s[0] + s[1]) + (s[2] + s[3]);
  if constexpr (kEnt) st.s1 += (s1[0] + s1[1]) + (s1[2] + s1[3]);
}

// Folds N tokens into a state.
template <int N, bool kEnt>
__device__ __forceinline__ void fold(Sums& st, const float (&x)[N], float c) {
  float m = st.max;
#pragma unroll
  for (int i = 0; i < N; i += 2) m = max3(m, x[i], x[i + 1]);
  const float p = point(m, c);
  if (!__any(far(st.max, c) || far(m, c))) {
    raise_by(st, m, point(st.max, c) - p);
    add<N, kEnt>(st, x, [&](float v) { return __builtin_fmaf(v, c, -p); });
  } else {
    const bool off = far(m, c);
    raise(st, m, c);
    add<N, kEnt>(st, x, [&](float v) { return off ? (v - m) * c : __builtin_fmaf(v, c, -p); });
  }
}

template <int kT>
struct Shared {
  static constexpr int kWaves = kT / 64;
  static_assert(kMaxTop <= kFewThreads && kT / 4 <= kFewThreads);
  Sums sums[kWaves];
  u64 best[kWaves];
  uint32_t key[kT];
  int count[kWaves];
  u64 cand[kCap];
  u64 top[kMaxTop];
  int few[kFewThreads];  // threads that are read again
  int n_few, n_cand;
  uint32_t bound;
};

__device__ __forceinline__ void join_wave(Sums& st, float c) {
  float max = st.max;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) max = fmaxf(max, q3::shfl_xor(max, o));
  raise(st, max, c);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    st.s += q3::shfl_xor(st.s, o);
    st.s1 += q3::shfl_xor(st.s1, o);
  }
}

// The block's threads' states in one, on every thread.
template <int kT>
__device__ __forceinline__ void join_block(Sums& st, float c, Shared<kT>& sh) {
  constexpr int kWaves = kT / 64;
  join_wave(st, c);
  if ((threadIdx.x & 63) == 0) sh.sums[threadIdx.x >> 6] = st;
  __syncthreads();
  Sums r = sh.sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) r.max = fmaxf(r.max, sh.sums[w].max);
  r.s = r.s1 = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    Sums o = sh.sums[w];
    raise(o, r.max, c);
    r.s += o.s;
    r.s1 += o.s1;
  }
  st = r;
  __syncthreads();
}

template <int kT>
__device__ __forceinline__ u64 block_max(u64 v, Shared<kT>& sh) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 y = __shfl_xor(v, o, 64);
    v = y > v ? y : v;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.best[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kT / 64; ++w) v = sh.best[w] > v ? sh.best[w] : v;
  return v;
}

// How many of a wave's keys are at least t.
template <int kPer>
__device__ __forceinline__ int reaching(const uint32_t (&k)[kPer], uint32_t t) {
  int cnt = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) cnt += __popcll(__ballot(k[i] >= t));
  return cnt;
}

// A bound that n to `most` of the keys reach, or the n-th largest key itself where equal
// ones leave no such bound (0: fewer than n keys).  Bit by bit, by one wave, kPer keys a
// lane.
template <int kPer>
__device__ __forceinline__ uint32_t nth_bound(const uint32_t (&k)[kPer], int n, int most) {
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cand = t | 1u << bit;
    const int cnt = reaching(k, cand);
    if (cnt >= n) t = cand;
    if (cnt >= n && cnt <= most) break;
  }
  return t;
}

// The same of the block's threads' keys.  Fewer finite ones than n are told beforehand: the
// search for -inf or 0 would pass all 32 bits (rows masked but for 12 tokens: 4 us of 24).
template <int kPer>
__device__ __forceinline__ uint32_t bound_of(const uint32_t (&k)[kPer], int n, int most) {
  if (reaching(k, kMinusInf + 1u) < n) return reaching(k, kMinusInf) < n ? 0u : kMinusInf;
  return nth_bound(k, n, most);
}

// Largest x of a wave's lanes, on every lane: four steps inside each row of 16 lanes, then
// the rows' own into the rows above.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  auto take = [&](uint32_t y) { x = y > x ? y : x; };
  take(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x111, 0xF, 0xF, true));   // row_shr:1
  take(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x112, 0xF, 0xF, true));   // row_shr:2
  take(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x114, 0xF, 0xF, true));   // row_shr:4
  take(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x118, 0xF, 0xF, true));   // row_shr:8
  take(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x142, 0xA, 0xF, false));  // row_bcast:15
  take(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x143, 0xC, 0xF, false));  // row_bcast:31
  return __builtin_amdgcn_readlane(x, 63);
}

// Appends a part's token to the candidates (counted, not kept, behind the list's end).
template <int kT>
__device__ __forceinline__ void append(Shared<kT>& sh, uint32_t key, int idx) {
  const int at = atomicAdd(&sh.n_cand, 1);
  if (at < kCap) sh.cand[at] = ranked(key, static_cast<uint32_t>(idx));
}

// The tokens of the threads in sh.few whose key is at least `least`: their pieces dealt to
// all threads, so that the loads are one round trip (or few).
template <typename Tr, int kT>
__device__ __forceinline__ void gather_few(const LogprobArgs& a, const char* xr, int p0, int p1,
                                           uint32_t least, Shared<kT>& sh) {
  const int each = (p1 - p0 + kT - 1) / kT;  // a thread's pieces
  const int all = min(sh.n_few, kFewThreads) * each;
  for (int i = threadIdx.x; i < all; i += kT) {
    const int of = i / each;
    const int p = p0 + sh.few[of] + (i - of * each) * kT;
    if (p >= p1) continue;
    float x[Tr::kE];
    Tr::unpack(load_piece<Tr>(a, xr, p), x);
#pragma unroll
    for (int e = 0; e < Tr::kE; ++e) {
      int idx;
      const bool ok = token_at<Tr>(a, p, e, idx);
      const uint32_t k = key_of(x[e]);
      if (ok && k >= least) append(sh, k, idx);
    }
  }
}

// Lists the threads where q holds.
template <int kT>
__device__ __forceinline__ void list_few(bool q, Shared<kT>& sh) {
  if (q) {
    const int at = atomicAdd(&sh.n_few, 1);
    if (at < kFewThreads) sh.few[at] = threadIdx.x;
  }
}

// Largest token of piece p that ranks below `below`; 0: none.
template <typename Tr>
__device__ __forceinline__ u64 best_in_piece(const LogprobArgs& a, const char* xr, int p,
                                             u64 below) {
  float x[Tr::kE];
  Tr::unpack(load_piece<Tr>(a, xr, p), x);
  u64 best = 0;
#pragma unroll
  for (int e = 0; e < Tr::kE; ++e) {
    int idx;
    const bool ok = token_at<Tr>(a, p, e, idx);
    const u64 r = ranked(key_of(x[e]), static_cast<uint32_t>(idx));
    if (ok && r < below && r > best) best = r;
  }
  return best;
}

// sh.top: the part's most likely tokens.  max: this thread's; nan: the part holds NaN or
// +inf.  Every thread of the block calls it.
template <typename Tr, int kT>
__device__ __forceinline__ void top_tokens(const LogprobArgs& a, const char* xr, int p0, int p1,
                                           float max, bool nan, Shared<kT>& sh) {
  constexpr int kWaves = kT / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = a.top;
  const bool some = p0 + tid < p1;
  const uint32_t mine = some ? key_of(max) : 0u;
  sh.key[tid] = mine;
  if (tid < kMaxTop) sh.top[tid] = 0;
  if (tid == 0) sh.n_few = sh.n_cand = 0;
  __syncthreads();
  bool done = false;
  if (!nan) {
    if (wave == 0) {
      uint32_t k[kWaves];
#pragma unroll
      for (int i = 0; i < kWaves; ++i) k[i] = sh.key[64 * i + lane];
      const int each = (p1 - p0 + kT - 1) / kT;
      // (looser than a quarter of the threads, each that reaches it holds several tokens)
      const int most = each > 0 ? min(min(p1 - p0, kT) / 4, kFewPieces / each) : n;
      const uint32_t t = bound_of(k, n, most > n ? most : n);
      if (lane == 0) sh.bound = t;
    }
    __syncthreads();
    const uint32_t t = sh.bound;
    const bool reaches = mine >= (t > 1u ? t : 1u);
    int cnt = __popcll(__ballot(reaches));
    if (lane == 0) sh.count[wave] = cnt;
    __syncthreads();
    cnt = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) cnt += sh.count[w];
    const bool few = cnt <= (n > kT / 4 ? n : kT / 4);
    list_few(few ? reaches : mine > t, sh);
    __syncthreads();
    gather_few<Tr, kT>(a, xr, p0, p1, few ? t : t + 1u, sh);
    __syncthreads();
    // (many reach t by equal values: t is the n-th largest itself, not below it)
    if (!few && sh.n_cand < n) {  // the lowest indices at t itself
      int left = n - sh.n_cand;
      for (int p = p0 + tid; left > 0 && p - tid < p1; p += kT) {
        uint32_t hit = 0;
        if (p < p1) {
          float x[Tr::kE];
          Tr::unpack(load_piece<Tr>(a, xr, p), x);
#pragma unroll
          for (int e = 0; e < Tr::kE; ++e) {
            int idx;
            if (token_at<Tr>(a, p, e, idx) && key_of(x[e]) == t) hit |= 1u << e;
          }
        }
        const int h = __popc(hit), incl = q3::wave_prefix_sum(h);
        __syncthreads();
        if (lane == 63) sh.count[wave] = incl;
        __syncthreads();
        int before = incl - h, all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          before += w < wave ? sh.count[w] : 0;
          all += sh.count[w];
        }
#pragma unroll
        for (int e = 0; e < Tr::kE; ++e)
          if (hit >> e & 1u) {
            int idx;
            token_at<Tr>(a, p, e, idx);
            if (before < left) append(sh, t, idx);
            ++before;
          }
        left -= all;
      }
      __syncthreads();
    }
    const int nc = sh.n_cand;
    done = nc <= kCap;
    if (done) {
      for (int i = tid; i < nc; i += kT) {
        const u64 r = sh.cand[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < nc; ++j) rank += sh.cand[j] > r ? 1 : 0;
        if (rank < n) sh.top[rank] = r;
      }
    }
  }
  if (!done) {  // one token a round
    u64 best = 0;
    for (int p = p0 + tid; p < p1; p += kT) {
      const u64 b = best_in_piece<Tr>(a, xr, p, ~0ull);
      best = b > best ? b : best;
    }
    for (int r = 0; r < n; ++r) {
      const u64 w = block_max(best, sh);
      if (w == 0) break;  // (the same for every thread)
      if (tid == 0) sh.top[r] = w;
      const int owner = (static_cast<int>(index_in(w)) / Tr::kE - p0) % kT;
      u64 next = 0;
      for (int64_t p = static_cast<int64_t>(p0) + owner + static_cast<int64_t>(tid) * kT;
           p < p1; p += static_cast<int64_t>(kT) * kT) {
        const u64 b = best_in_piece<Tr>(a, xr, static_cast<int>(p), w);
        next = b > next ? b : next;
      }
      next = block_max(next, sh);
      if (tid == owner) best = next;
    }
  }
  __syncthreads();
}

// log p of a logit: (x - max) / T - log(sum exp((x' - max) / T)), the sum from s.
__device__ __forceinline__ float logprob_of(const LogprobArgs& a, float x, float max,
                                            float log2s) {
  const float shift = far(max, a.c) ? 0.f : __builtin_fmaf(max, a.c, -point(max, a.c));
  const float r = __builtin_fmaf(x - max, a.inv_t, -kLn2 * (log2s - shift));
  return r > 0.f ? 0.f : r;  // by a rounding of the sum
}

// What a row's sums give, by the threads of a block; top: its most likely tokens in LDS.
template <typename Tr>
__device__ __forceinline__ void write_row(const LogprobArgs& a, const char* xr, int64_t row,
                                          const Sums& st, const u64* top) {
  const int tid = threadIdx.x, step = blockDim.x;
  const float log2s = __builtin_log2f(st.s);
  if (tid == 0) {
    if (a.entropy) {
      const float h = kLn2 * (log2s - st.s1 / st.s);
      a.entropy[row] = h < 0.f ? 0.f : h;  // (one token left: the difference's rounding)
    }
    if (a.stats) a.stats[row] = float2{st.max, log2s};
  }
  for (int k = tid; k < a.given; k += step) {
    const int64_t t = a.tokens[row * a.given + k];
    float r = 0.f;  // below zero: no token
    if (t >= a.vocab) r = __builtin_nanf("");
    else if (t >= 0) r = logprob_of(a, Tr::one(xr + t * Tr::kBytes), st.max, log2s);
    a.logprobs[row * a.given + k] = r;
  }
  for (int k = tid; k < a.top; k += step) {
    const u64 r = top[k];
    a.top_ids[row * a.top + k] = index_in(r);
    a.top_logprobs[row * a.top + k] = logprob_of(a, value_of(key_in(r)), st.max, log2s);
  }
}

template <typename Tr, int kT, bool kEnt, bool kTop>
__global__ __launch_bounds__(kT) void logprobs_kernel(LogprobArgs a) {
  __shared__ Shared<kT> sh;
  constexpr int E = Tr::kE, kBatch = kBatchTokens / E;
  const int tid = threadIdx.x;
  const uint32_t row = blockIdx.x / static_cast<uint32_t>(a.parts);
  const int part = static_cast<int>(blockIdx.x - row * static_cast<uint32_t>(a.parts));
  const char* xr = a.x + static_cast<int64_t>(row) * a.row_bytes;
  const int p0 = min(part * a.per_part, a.pieces), p1 = min(p0 + a.per_part, a.pieces);
  const int whole = min(p1, a.vocab / E);  // pieces before it are whole ones

  Sums st{q3::kNegInf, 0.f, 0.f};
  auto load = [&](int p, q3::u32x4 (&w)[kBatch]) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      // (a piece that this thread does not have: another one of the part, not used)
      const int q = p + u * kT;
      w[u] = load_piece<Tr>(a, xr, q < p1 ? q : p0);
    }
  };
  if (p0 < p1) {
    q3::u32x4 next[kBatch];
    load(p0 + tid, next);
    for (int base = p0; base < p1; base += kBatch * kT) {
      q3::u32x4 w[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) w[u] = next[u];
      if (base + kBatch * kT < p1) load(base + kBatch * kT + tid, next);
      float x[kBatch * E];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        float y[E];
        Tr::unpack(w[u], y);
#pragma unroll
        for (int e = 0; e < E; ++e) x[u * E + e] = y[e];
      }
      if (base + kBatch * kT > whole) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int p = base + tid + u * kT;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            int idx;
            if (p >= p1 || !token_at<Tr>(a, p, e, idx)) x[u * E + e] = q3::kNegInf;
          }
        }
      }
      fold<kBatch * E, kEnt>(st, x, a.c);
    }
  }
  const float mine = st.max;
  join_block(st, a.c, sh);
  if constexpr (kTop) top_tokens<Tr, kT>(a, xr, p0, p1, mine, st.s != st.s, sh);
  if (a.parts == 1) {
    write_row<Tr>(a, xr, row, st, sh.top);
    return;
  }
  const int64_t at = static_cast<int64_t>(row) * a.parts + part;
  if (tid == 0) a.part_sums[at] = st;
  if constexpr (kTop)
    for (int k = tid; k < a.top; k += kT) a.part_top[at * a.top + k] = sh.top[k];
}

// Joins a row's parts.
constexpr int kJoinThreads = 256;

// Whether the parts' most likely tokens are joined by rank, some 0.9 us for eight lists and
// a token a thread, or head by head, some 0.1 us each: 64 rows of 8 parts, 64 tokens 34.8 us
// by rank and 40.4 by heads, 20 tokens 22.0 and 22.6, 5 tokens 20.2 and 19.4; 16 rows of 32
// parts, 20 tokens 37.6 and 21.6.
__device__ __forceinline__ bool ranked_join(int parts, int top) {
  return 9 * ((parts + 7) / 8) * ((parts * top + kJoinThreads - 1) / kJoinThreads) <= top;
}

template <typename Tr>
__global__ __launch_bounds__(kJoinThreads) void logprobs_join_kernel(LogprobArgs a) {
  __shared__ u64 s_top[kMaxTop];
  __shared__ u64 s_all[kMaxParts * kMaxTop];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const char* xr = a.x + row * a.row_bytes;
  Sums st{q3::kNegInf, 0.f, 0.f};
  if (lane < a.parts) st = a.part_sums[row * a.parts + lane];  // (every wave)
  join_wave(st, a.c);
  const int all = a.parts * a.top;
  if (a.top) {
    for (int i = tid; i < all; i += kJoinThreads) s_all[i] = a.part_top[row * all + i];
    if (tid < kMaxTop) s_top[tid] = 0;
    __syncthreads();
    if (ranked_join(a.parts, a.top)) {
      // a token's rank is how many rank above it in each list, by halving, eight lists at
      // once
      const int first = 1 << (31 - __clz(a.top));
      for (int i = tid; i < all; i += kJoinThreads) {
        const u64 r = s_all[i];
        int rank = 0;
        for (int q = 0; q < a.parts; q += 8) {
          int above[8] = {0, 0, 0, 0, 0, 0, 0, 0};
          for (int step = first; step > 0; step >>= 1) {
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const int at = above[u] + step - 1;
              const bool in = q + u < a.parts && at < a.top;
              const u64 x = s_all[in ? (q + u) * a.top + at : 0];
              above[u] += in && x > r ? step : 0;
            }
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) rank += above[u];
        }
        if (r != 0 && rank < a.top) s_top[rank] = r;
      }
    } else if (tid < 64) {
      // the largest of the lists' heads, n times, a list a lane
      int at = lane * a.top;
      const int end = lane < a.parts ? at + a.top : at;
      u64 head = at < end ? s_all[at] : 0;
      for (int r = 0; r < a.top; ++r) {
        const uint32_t key = key_in(head), low = static_cast<uint32_t>(head);
        const uint32_t best = wave_max(key);
        const uint32_t first = wave_max(key == best ? low : 0u);
        if (key == best && low == first && head != 0) {
          s_top[r] = head;
          ++at;
          head = at < end ? s_all[at] : 0;
        }
      }
    }
    __syncthreads();
  }
  write_row<Tr>(a, xr, row, st, s_top);
}

// ---------------------------------------------------------------------------
// Gradient.  With p_i = softmax(z)_i, the row's H, g_k of its given tokens, h_j of its most
// likely ones and g_H of its entropy:
//   dx_i = (sum g_k 1[i = t_k] + sum h_j 1[i = id_j] - p_i (sum g + sum h + g_H (log p_i + H))) / T
// One pass, 16 bytes in and out a piece; pieces that hold a given or listed token are
// marked in a bitmap and add their terms before the one rounding.
constexpr int kGradThreads = 256;
constexpr int kGradPieces = 8;  // a thread's
constexpr int kGradSpan = kGradThreads * kGradPieces;

struct GradArgs {
  LogprobArgs r;              // logits, tokens, top_ids
  const float* entropy;       // the row's H (nullable with g_entropy)
  const float2* stats;
  const float* g_logprobs;    // nullable
  const float* g_entropy;     // nullable
  const float* g_top;         // nullable
  char* dx;
  int64_t dx_row_bytes;
  int segments;
};

template <typename Tr>
__global__ __launch_bounds__(kGradThreads) void logprobs_grad_kernel(GradArgs g) {
  const LogprobArgs& a = g.r;
  constexpr int E = Tr::kE;
  __shared__ uint32_t s_mark[kGradSpan / 32];
  __shared__ int s_idx[kMaxGiven + kMaxTop];
  __shared__ float s_g[kMaxGiven + kMaxTop];
  const int tid = threadIdx.x;
  const uint32_t row = blockIdx.x / static_cast<uint32_t>(g.segments);
  const int seg = static_cast<int>(blockIdx.x - row * static_cast<uint32_t>(g.segments));
  const int p0 = seg * kGradSpan, p1 = min(p0 + kGradSpan, a.pieces);
  const char* xr = a.x + static_cast<int64_t>(row) * a.row_bytes;
  char* dr = g.dx + static_cast<int64_t>(row) * g.dx_row_bytes;
  q3::u32x4 w[kGradPieces];
#pragma unroll
  for (int u = 0; u < kGradPieces; ++u) {
    const int p = p0 + tid + u * kGradThreads;
    w[u] = load_piece<Tr>(a, xr, p < p1 ? p : p0);
  }
  for (int i = tid; i < kGradSpan / 32; i += kGradThreads) s_mark[i] = 0;
  const int n_given = g.g_logprobs ? a.given : 0, n_top = g.g_top ? a.top : 0;
  const int special = n_given + n_top;
  __syncthreads();
  for (int k = tid; k < special; k += kGradThreads) {
    const int64_t t = k < n_given ? a.tokens[static_cast<int64_t>(row) * a.given + k]
                                  : a.top_ids[static_cast<int64_t>(row) * a.top + k - n_given];
    const bool ok = t >= 0 && t < a.vocab;
    s_idx[k] = ok ? static_cast<int>(t) : -1;
    s_g[k] = !ok ? 0.f
                 : k < n_given ? g.g_logprobs[static_cast<int64_t>(row) * a.given + k]
                               : g.g_top[static_cast<int64_t>(row) * a.top + k - n_given];
    const int p = ok ? static_cast<int>(t) / E - p0 : -1;
    if (p >= 0 && p < kGradSpan) atomicOr(&s_mark[p >> 5], 1u << (p & 31));
  }
  __syncthreads();
  float sum = 0.f;
  for (int k = 0; k < special; ++k) sum += s_g[k];
  const float gh = g.g_entropy ? g.g_entropy[row] : 0.f;
  const float2 stats = g.stats[row];
  const bool off = far(stats.x, a.c);
  const float p_max = point(stats.x, a.c), log2s = stats.y;
  // p_i (b + gh ln 2 log2 p_i)
  const float b = sum + (g.g_entropy ? gh * g.entropy[row] : 0.f), gl = gh * kLn2;
#pragma unroll
  for (int u = 0; u < kGradPieces; ++u) {
    const int p = p0 + tid + u * kGradThreads;
    if (p >= p1) break;
    float x[E];
    Tr::unpack(w[u], x);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float y = (off ? (x[e] - stats.x) * a.c : __builtin_fmaf(x[e], a.c, -p_max)) - log2s;
      const float pr = q3::fast_exp2(y);
      x[e] = -pr * __builtin_fmaf(gl, fmaxf(y, kTiny), b);
    }
    const int at = p - p0;
    if (s_mark[at >> 5] >> (at & 31) & 1u) {
      for (int k = 0; k < special; ++k) {
        const int i = s_idx[k];
        if (i < 0 || i / E != p) continue;
        const int el = a.vocab < E ? i : i - piece_start<Tr>(a, p);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] += e == el ? s_g[k] : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] *= a.inv_t;
    if (p < a.vocab / E) {
      piece_t* dst = reinterpret_cast<piece_t*>(dr + static_cast<int64_t>(p) * 16);
      __builtin_nontemporal_store(__builtin_bit_cast(piece_t, Tr::pack(x)), dst);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        int idx;
        if (token_at<Tr>(a, p, e, idx)) Tr::put(dr + static_cast<int64_t>(idx) * Tr::kBytes, x[e]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.

int elements_of(int dtype) { return dtype == 2 ? 4 : 8; }
int bytes_of(int dtype) { return dtype == 2 ? 4 : 2; }

// Parts of a row: as many workgroups as the device holds at once where the rows are fewer,
// of a round each (kThreads pieces) at least.
int parts_for(int64_t rows, int64_t pieces) {
  const int64_t most = q3::cdiv(pieces, kThreads);
  int64_t p = kResident / rows;
  p = p < most ? p : most;
  p = p < kMaxParts ? p : kMaxParts;
  return static_cast<int>(p < 1 ? 1 : p);
}

struct LogprobLayout {
  int64_t sums, top, total;
};
LogprobLayout layout_of(int64_t rows, int parts, int top) {
  LogprobLayout l;
  l.sums = 0;
  l.top = parts > 1 ? rows * parts * static_cast<int64_t>(sizeof(Sums)) : 0;
  l.total = l.top + (parts > 1 ? rows * parts * top * 8 : 0);
  return l;
}

int check_shape(const char* who, const void* logits, int64_t row_stride, int dtype, int64_t rows,
                int64_t vocab, int given, int top, float temperature) {
  if (!logits) return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  if (dtype < 0 || dtype > 2)
    return q3::fail(QWEN3_EUNSUPPORTED, "%s: dtype %d not supported", who, dtype);
  if (rows < 0 || vocab <= 0 || vocab > (int64_t(1) << 30) || (rows > 1 && row_stride < vocab))
    return q3::fail(QWEN3_EINVAL, "%s: bad sizes (rows=%lld vocab=%lld row_stride=%lld)", who,
                    (long long)rows, (long long)vocab, (long long)row_stride);
  if (given < 0 || given > kMaxGiven || top < 0 || top > kMaxTop || top > vocab)
    return q3::fail(QWEN3_EUNSUPPORTED, "%s: %d given tokens, %d most likely ones (at most %d, "
                    "%d and the vocabulary's)", who, given, top, kMaxGiven, kMaxTop);
  if (!(temperature > 0.f) || !(temperature < __builtin_inff()) ||
      !(q3::kLog2e / temperature < __builtin_inff()))
    return q3::fail(QWEN3_EINVAL, "%s: temperature must be positive and finite", who);
  if (reinterpret_cast<uintptr_t>(logits) % bytes_of(dtype) != 0)
    return q3::fail(QWEN3_EALIGN, "%s: logits must be aligned to their type", who);
  return QWEN3_OK;
}

LogprobArgs args_of(const void* logits, int64_t row_stride, int dtype, int64_t vocab,
                    const int64_t* tokens, int given, float temperature, int top) {
  LogprobArgs a{};
  a.x = static_cast<const char*>(logits);
  a.row_bytes = row_stride * bytes_of(dtype);
  a.vocab = static_cast<int>(vocab);
  a.pieces = static_cast<int>(q3::cdiv(vocab, elements_of(dtype)));
  a.c = static_cast<float>(1.4426950408889634 / static_cast<double>(temperature));
  a.inv_t = 1.f / temperature;
  a.tokens = tokens;
  a.given = tokens ? given : 0;
  a.top = top;
  return a;
}

template <typename Tr, int kT>
void launch_rows(const LogprobArgs& a, int64_t rows, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(rows * a.parts)), block(kT);
  if (a.entropy) {
    if (a.top) hipLaunchKernelGGL((logprobs_kernel<Tr, kT, true, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((logprobs_kernel<Tr, kT, true, false>), grid, block, 0, s, a);
  } else {
    if (a.top) hipLaunchKernelGGL((logprobs_kernel<Tr, kT, false, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((logprobs_kernel<Tr, kT, false, false>), grid, block, 0, s, a);
  }
}

template <typename Tr>
int launch(const LogprobArgs& a, int64_t rows, hipStream_t s, const char* who) {
  q3::clear_error();
  if (a.parts > 1 || a.pieces > kShort) launch_rows<Tr, kThreads>(a, rows, s);
  else launch_rows<Tr, kShortThreads>(a, rows, s);
  if (const int rc = q3::launch_status(who)) return rc;
  if (a.parts == 1) return QWEN3_OK;
  hipLaunchKernelGGL(logprobs_join_kernel<Tr>, dim3(static_cast<unsigned>(rows)),
                     dim3(kJoinThreads), 0, s, a);
  return q3::launch_status(who);
}

}  // namespace

extern "C" size_t qwen3_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int dtype,
                                                       int top_n) {
  if (rows <= 0 || vocab <= 0 || vocab > (int64_t(1) << 30) || dtype < 0 || dtype > 2 ||
      top_n < 0 || top_n > kMaxTop)
    return 0;
  const int parts = parts_for(rows, q3::cdiv(vocab, elements_of(dtype)));
  return static_cast<size_t>(layout_of(rows, parts, top_n).total);
}

extern "C" int qwen3_token_logprobs(const void* logits, int64_t row_stride, int dtype,
                                    int64_t rows, int64_t vocab, const int64_t* tokens, int given,
                                    float temperature, float* logprobs, float* entropy, int top_n,
                                    int64_t* top_ids, float* top_logprobs, float* stats,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "qwen3_token_logprobs";
  if (const int rc = check_shape(who, logits, row_stride, dtype, rows, vocab, given, top_n,
                                 temperature))
    return rc;
  if ((given > 0 && (!tokens || !logprobs)) || (top_n > 0 && (!top_ids || !top_logprobs)))
    return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  LogprobArgs a = args_of(logits, row_stride, dtype, vocab, tokens, given, temperature, top_n);
  a.given = given;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  a.stats = reinterpret_cast<float2*>(stats);
  if (rows == 0) return QWEN3_OK;
  a.parts = parts_for(rows, a.pieces);
  a.per_part = static_cast<int>(q3::cdiv(q3::cdiv(a.pieces, a.parts), kThreads) * kThreads);
  a.parts = static_cast<int>(q3::cdiv(a.pieces, a.per_part));
  if (rows * a.parts > q3::kMaxThreads / kThreads)
    return q3::fail(QWEN3_EINVAL, "%s: %lld rows are too many for one launch", who,
                    (long long)rows);
  const size_t need = qwen3_token_logprobs_workspace_bytes(rows, vocab, dtype, top_n);
  if (need && (!workspace || workspace_bytes < need))
    return q3::fail(QWEN3_EWORKSPACE, "%s: workspace of %zu bytes needed, %zu given", who, need,
                    workspace ? workspace_bytes : (size_t)0);
  if (need && !q3::aligned16(workspace))
    return q3::fail(QWEN3_EALIGN, "%s: workspace must be 16-byte aligned", who);
  const LogprobLayout l = layout_of(rows, a.parts, top_n);
  char* ws = static_cast<char*>(workspace);
  a.part_sums = reinterpret_cast<Sums*>(ws + l.sums);
  a.part_top = reinterpret_cast<u64*>(ws + l.top);
  const auto s = static_cast<hipStream_t>(stream);
  return dtype == 0 ? launch<Bf16>(a, rows, s, who)
                    : dtype == 1 ? launch<Fp16>(a, rows, s, who) : launch<Fp32>(a, rows, s, who);
}

extern "C" int qwen3_token_logprobs_grad(
    const void* logits, int64_t row_stride, int dtype, int64_t rows, int64_t vocab,
    const int64_t* tokens, int given, float temperature, const float* entropy, int top_n,
    const int64_t* top_ids, const float* stats, const float* g_logprobs, const float* g_entropy,
    const float* g_top, void* grad, int64_t grad_row_stride, void* stream) {
  const char* who = "qwen3_token_logprobs_grad";
  if (const int rc = check_shape(who, logits, row_stride, dtype, rows, vocab, given, top_n,
                                 temperature))
    return rc;
  if (!stats || !grad || (g_logprobs && !tokens) || (g_entropy && !entropy) || (g_top && !top_ids))
    return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  if (rows > 1 && grad_row_stride < vocab)
    return q3::fail(QWEN3_EINVAL, "%s: gradient rows overlap", who);
  if (reinterpret_cast<uintptr_t>(grad) % bytes_of(dtype) != 0)
    return q3::fail(QWEN3_EALIGN, "%s: the gradient must be aligned to its type", who);
  if (rows == 0) return QWEN3_OK;
  GradArgs g{};
  g.r = args_of(logits, row_stride, dtype, vocab, tokens, given, temperature, top_n);
  g.r.top_ids = const_cast<int64_t*>(top_ids);
  g.entropy = entropy;
  g.stats = reinterpret_cast<const float2*>(stats);
  g.g_logprobs = g_logprobs;
  g.g_entropy = g_entropy;
  g.g_top = g_top;
  g.dx = static_cast<char*>(grad);
  g.dx_row_bytes = grad_row_stride * bytes_of(dtype);
  g.segments = static_cast<int>(q3::cdiv(g.r.pieces, kGradSpan));
  if (rows * g.segments > q3::kMaxThreads / kGradThreads)
    return q3::fail(QWEN3_EINVAL, "%s: %lld rows are too many for one launch", who,
                    (long long)rows);
  const dim3 grid(static_cast<unsigned>(rows * g.segments)), block(kGradThreads);
  const auto s = static_cast<hipStream_t>(stream);
  q3::clear_error();
  if (dtype == 0) hipLaunchKernelGGL(logprobs_grad_kernel<Bf16>, grid, block, 0, s, g);
  else if (dtype == 1) hipLaunchKernelGGL(logprobs_grad_kernel<Fp16>, grid, block, 0, s, g);
  else hipLaunchKernelGGL(logprobs_grad_kernel<Fp32>, grid, block, 0, s, g);
  return q3::launch_status(who);
}
