// Rotary positions of q and k, with or without the write of k and v into the
// paged pool, for models without QK-norm (pre_attention.hip has the fused form with
// it) and for positions that no table holds.
//
//   y_a = m (x_a cos t - x_b sin t),  y_b = m (x_b cos t + x_a sin t),  t = pos f_i
// for the pairs i < r / 2 of the first r = rotary_dim elements of a head: (a, b) =
// (i, i + r / 2) in the half layout, (2 i, 2 i + 1) in the interleaved one.  The other
// elements pass through unchanged.  inverse: -t, the transpose of the same map (the
// gradient, and the rotation back but for m^2).
//
// Angles come from the position itself: f_i in 64 bits, pos f_i / (2 pi) reduced to
// one turn in 64 bits (at position 2^31 still exact to 2^-22 of a turn and better
// below), then cos and sin in 32.  Everything else is fp32, rounded once at the end.
//
// Bound by HBM: each q, k (and v) element is read once and written once.  The rows of
// all tokens are one list of work units, 16-byte chunks or (half layout) the two chunks
// of eight pairs, so that nothing crosses lanes; a workgroup takes kThreads x
// units_of units of it, all loaded before the angles of the tokens they belong to are
// formed, once each, in LDS.  8,115 tokens of 32 + 8 heads of 128 with the pool write,
// cold: 41.5 us, 5.2 TB/s, the rate of a plain copy of as many bytes.
#include "common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;      // rotary_dim up to 512
// Units a thread has in flight: 64 bytes.
template <bool kHalf>
constexpr int units_of() { return kHalf ? 2 : 4; }

enum class Addr { None, Slots, Decode };

struct RotaryArgs {
  const char* q;
  int64_t q_s0, q_s1;
  const char* k;  // nullable
  int64_t k_s0, k_s1;
  const uint16_t* v;
  int64_t v_s0, v_s1;
  char* q_out;
  int64_t qo_s0, qo_s1;
  char* k_out;  // nullable with a pool
  int64_t ko_s0, ko_s1;
  const double* inv_freq;
  float factor;
  float sign;   // of sin: -1 for the inverse
  const int64_t* positions;  // Decode: nullable
  uint16_t* k_cache;
  uint16_t* v_cache;
  int64_t kc[4], vc[4];
  int64_t num_blocks;
  int layer;
  const int64_t* slots;
  const int32_t* seq_lens;
  const int32_t* block_table;
  int64_t bt_stride, max_rows, max_pages;
  const int32_t* row_ids;
  int64_t n_tokens;
  int Hq, Hkv, D, r, bs;
  // Work units of a head row: a pair of chunks (half layout) or one chunk of the
  // rotated part, then one chunk each of what passes through.
  int rot_units, row_units;
  int units;           // of a token
  uint32_t row_magic, unit_magic;  // ceil(2^32 / row_units), ceil(2^32 / units)
  int span;            // tokens that a workgroup's units belong to, at most
};

// x / d for the magic ceil(2^32 / d), where x d < 2^32 (d = 1: the magic is 0).
__device__ __forceinline__ int divide(int x, uint32_t magic) {
  return magic == 0 ? x : static_cast<int>(__umulhi(static_cast<uint32_t>(x), magic));
}

// More than the L2 of all XCDs holds: outputs that the next kernel would not find there,
// written past it (8,115 tokens with the pool write, cold: 45.9 -> 41.5 us, the time of a
// plain copy; loads without reuse are marked so always).
constexpr int64_t kStreamBytes = int64_t(32) << 20;

template <bool kStreams>
__device__ __forceinline__ void put16(void* p, q3::u32x4 x) {
  if constexpr (kStreams)  // (at run time the compiler joins both into a plain store)
    __builtin_nontemporal_store(x, reinterpret_cast<q3::u32x4*>(p));
  else
    q3::st16(p, x);
}

// 16 bytes of T as floats and back.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void get(q3::u32x4 w, float* x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(w[e]);
  }
  static __device__ __forceinline__ q3::u32x4 put(const float* x) {
    return q3::u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                     __float_as_uint(x[3])};
  }
};
template <>
struct Vec<__bf16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void get(q3::u32x4 w, float* x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = q3::bf16_lo(w[e]);
      x[2 * e + 1] = q3::bf16_hi(w[e]);
    }
  }
  static __device__ __forceinline__ q3::u32x4 put(const float* x) {
    return q3::u32x4{q3::pack_bf16x2(x[0], x[1]), q3::pack_bf16x2(x[2], x[3]),
                     q3::pack_bf16x2(x[4], x[5]), q3::pack_bf16x2(x[6], x[7])};
  }
};
template <>
struct Vec<_Float16> {
  static constexpr int n = 8;
  typedef _Float16 f16x2 __attribute__((__vector_size__(2 * sizeof(_Float16))));
  static __device__ __forceinline__ void get(q3::u32x4 w, float* x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f16x2 h = __builtin_bit_cast(f16x2, static_cast<uint32_t>(w[e]));
      x[2 * e] = static_cast<float>(h[0]);
      x[2 * e + 1] = static_cast<float>(h[1]);
    }
  }
  static __device__ __forceinline__ q3::u32x4 put(const float* x) {
    q3::u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f16x2 h = {static_cast<_Float16>(x[2 * e]), static_cast<_Float16>(x[2 * e + 1])};
      w[e] = __builtin_bit_cast(uint32_t, h);
    }
    return w;
  }
};

// A token's position, and where its k and v go in the pool (off < 0: nowhere).
struct Where {
  int64_t pos;
  int64_t kc, vc;  // element offsets of (head 0, element 0); -1: not written
};

template <Addr A>
__device__ __forceinline__ Where where(const RotaryArgs& a, int64_t t) {
  Where w{0, -1, -1};
  int64_t phys = -1, off = 0;
  if constexpr (A == Addr::Decode) {
    const int64_t row = a.row_ids ? a.row_ids[t] : t;
    if (row >= 0 && row < a.max_rows) {
      const int64_t at = a.seq_lens[row];
      if (at >= 0 && at / a.bs < a.max_pages) {
        phys = a.block_table[row * a.bt_stride + at / a.bs];
        off = at % a.bs;
      }
      w.pos = at;
    }
    if (a.positions) w.pos = a.positions[t];
  } else {
    w.pos = a.positions[t];
    if constexpr (A == Addr::Slots) {
      const int64_t slot = a.slots[t];
      if (slot >= 0) {
        phys = slot / a.bs;
        off = slot % a.bs;
      }
    }
  }
  if (A != Addr::None && phys >= 0 && phys < a.num_blocks) {
    w.kc = phys * a.kc[0] + a.layer * a.kc[1] + off * a.kc[3];
    w.vc = phys * a.vc[0] + a.layer * a.vc[1] + off * a.vc[3];
  }
  return w;
}

template <typename T, bool kHalf, Addr A, bool kStreams>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float2 s_cs[];  // [span][r / 2], then the tokens' places in the pool
  constexpr int kN = Vec<T>::n;  // elements of a chunk
  constexpr int kU = units_of<kHalf>();
  const int tid = threadIdx.x;
  const int pairs = a.r / 2;
  const int heads = a.Hq + (a.k ? a.Hkv : 0);
  const int64_t g0 = static_cast<int64_t>(blockIdx.x) * (kThreads * kU);
  const int64_t t0 = g0 / a.units;  // the first unit's token
  const int rest = static_cast<int>(g0 - t0 * a.units);
  const int left = static_cast<int>(min(a.n_tokens - t0, static_cast<int64_t>(a.span)));

  struct Unit {
    int tok, row, e;   // token (from t0 on), head row (q, then k, then v), first element
    bool rot;
    q3::u32x4 x1, x2;  // x2: the half layout's other chunk, e + r / 2
  };
  Unit n[kU];
#pragma unroll
  for (int b = 0; b < kU; ++b) {
    const int l = rest + b * kThreads + tid;
    n[b].tok = divide(l, a.unit_magic);
    if (n[b].tok >= left) continue;
    const int i = l - n[b].tok * a.units;
    n[b].row = divide(i, a.row_magic);
    const int u = i - n[b].row * a.row_units;
    n[b].rot = u < a.rot_units;
    n[b].e = n[b].rot ? u * kN : a.r + (u - a.rot_units) * kN;
    const int64_t tok = t0 + n[b].tok;
    const T* src =
        n[b].row < a.Hq
            ? reinterpret_cast<const T*>(a.q) + tok * a.q_s0 + n[b].row * a.q_s1
        : n[b].row < heads
            ? reinterpret_cast<const T*>(a.k) + tok * a.k_s0 + (n[b].row - a.Hq) * a.k_s1
            : reinterpret_cast<const T*>(a.v) + tok * a.v_s0 + (n[b].row - heads) * a.v_s1;
    n[b].x1 = q3::ld16_nt(src + n[b].e);  // read once
    if (kHalf && n[b].rot) n[b].x2 = q3::ld16_nt(src + n[b].e + pairs);
  }

  int64_t* s_kc = reinterpret_cast<int64_t*>(s_cs + a.span * pairs);  // pool offsets, -1: none
  int64_t* s_vc = s_kc + a.span;
  double* s_pos = reinterpret_cast<double*>(s_vc + a.span);
  for (int i = tid; i < left; i += kThreads) {
    const Where w = where<A>(a, t0 + i);
    s_kc[i] = w.kc;
    s_vc[i] = w.vc;
    s_pos[i] = static_cast<double>(w.pos);
  }
  __syncthreads();
  for (int i = tid; i < left * pairs; i += kThreads) {
    const int t = i / pairs, p = i - t * pairs;
    constexpr double kInvTwoPi = 0.15915494309189533577;
    double turn = s_pos[t] * (a.inv_freq[p] * kInvTwoPi);
    turn -= __builtin_rint(turn);
    float s, c;
    sincospif(2.f * static_cast<float>(turn), &s, &c);
    s_cs[i] = float2{c * a.factor, s * a.factor * a.sign};
  }
  __syncthreads();

#pragma unroll
  for (int b = 0; b < kU; ++b) {
    const Unit& x = n[b];
    if (x.tok >= left) continue;
    const int64_t tok = t0 + x.tok;
    T* out = nullptr;
    uint16_t* pool = nullptr;
    bool rot = x.rot;
    if (x.row < a.Hq) {
      out = reinterpret_cast<T*>(a.q_out) + tok * a.qo_s0 + x.row * a.qo_s1;
    } else if (x.row < heads) {
      const int h = x.row - a.Hq;
      if (a.k_out) out = reinterpret_cast<T*>(a.k_out) + tok * a.ko_s0 + h * a.ko_s1;
      if (A != Addr::None && s_kc[x.tok] >= 0) pool = a.k_cache + s_kc[x.tok] + h * a.kc[2];
    } else {  // v: bits into the pool
      rot = false;
      if (s_vc[x.tok] >= 0) pool = a.v_cache + s_vc[x.tok] + (x.row - heads) * a.vc[2];
    }
    auto store = [&](int e, q3::u32x4 y) {
      if (out) put16<kStreams>(out + e, y);
      if (A != Addr::None && pool) put16<kStreams>(pool + e, y);
    };
    q3::u32x4 y1 = x.x1, y2 = x.x2;
    if (rot) {
      const float2* cs = s_cs + x.tok * pairs;
      float x1[kN], o1[kN];
      Vec<T>::get(x.x1, x1);
      if constexpr (kHalf) {
        float x2[kN], o2[kN];
        Vec<T>::get(x.x2, x2);
#pragma unroll
        for (int m = 0; m < kN; ++m) {
          const float2 f = cs[x.e + m];
          o1[m] = x1[m] * f.x - x2[m] * f.y;
          o2[m] = x2[m] * f.x + x1[m] * f.y;
        }
        y2 = Vec<T>::put(o2);
      } else {
#pragma unroll
        for (int m = 0; m < kN / 2; ++m) {
          const float2 f = cs[x.e / 2 + m];
          o1[2 * m] = x1[2 * m] * f.x - x1[2 * m + 1] * f.y;
          o1[2 * m + 1] = x1[2 * m + 1] * f.x + x1[2 * m] * f.y;
        }
      }
      y1 = Vec<T>::put(o1);
    }
    store(x.e, y1);
    if (kHalf && x.rot) store(x.e + pairs, y2);
  }
}

template <typename T, Addr A>
void launch(const RotaryArgs& a, bool half, bool streams, unsigned blocks, size_t lds,
            hipStream_t s) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), lds, s, a);
  };
  if (half)
    streams ? go(rotary_kernel<T, true, A, true>) : go(rotary_kernel<T, true, A, false>);
  else
    streams ? go(rotary_kernel<T, false, A, true>) : go(rotary_kernel<T, false, A, false>);
}

// Checks what the three entry points share, and launches.
template <Addr A>
int run(RotaryArgs a, int dtype, int layout, int inverse, int num_layers, void* stream,
        const char* who) {
  if (!a.q || !a.q_out || !a.inv_freq || (A != Addr::Decode && !a.positions) ||
      (A == Addr::None && (a.k != nullptr) != (a.k_out != nullptr)))
    return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  if (A != Addr::None && (!a.k || !a.v || !a.k_cache || !a.v_cache))
    return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  if (dtype < 0 || dtype > 2 || (A != Addr::None && dtype != 0))
    return q3::fail(QWEN3_EUNSUPPORTED, "%s: dtype %d not supported", who, dtype);
  if (layout != 0 && layout != 1)
    return q3::fail(QWEN3_EINVAL, "%s: layout %d (0: half, 1: interleaved)", who, layout);
  const int size = dtype == 2 ? 4 : 2, n = 16 / size;
  if (a.D <= 0 || a.D % 8 != 0 || a.r <= 0 || a.r > a.D || a.r > 2 * kMaxPairs || a.r % 16 != 0)
    return q3::fail(QWEN3_EUNSUPPORTED, "%s: head_dim %d must be a multiple of 8, rotary_dim %d of "
                    "16 and at most head_dim and %d", who, a.D, a.r, 2 * kMaxPairs);
  if (a.Hq <= 0 || a.Hkv < 0 || (a.k && a.Hkv == 0) || a.n_tokens < 0 ||
      static_cast<int64_t>(a.Hq + 2 * static_cast<int64_t>(a.Hkv)) * a.D > (1 << 24))
    return q3::fail(QWEN3_EINVAL, "%s: bad sizes", who);
  if (A != Addr::None && (a.bs <= 0 || a.num_blocks <= 0 || a.layer < 0 || a.layer >= num_layers))
    return q3::fail(QWEN3_EINVAL, "%s: bad pool sizes", who);
  if (!(a.factor > 0.f) || !(a.factor < __builtin_inff()))
    return q3::fail(QWEN3_EINVAL, "%s: the factor must be positive and finite", who);
  bool ok = true;
  for (const void* p : {static_cast<const void*>(a.q), static_cast<const void*>(a.k),
                        static_cast<const void*>(a.q_out), static_cast<const void*>(a.k_out),
                        static_cast<const void*>(a.v), static_cast<const void*>(a.k_cache),
                        static_cast<const void*>(a.v_cache)})
    ok = ok && q3::aligned16(p);
  for (int64_t st : {a.q_s0, a.q_s1, a.k_s0, a.k_s1, a.qo_s0, a.qo_s1, a.ko_s0, a.ko_s1, a.v_s0,
                     a.v_s1, a.kc[0], a.kc[1], a.kc[2], a.kc[3], a.vc[0], a.vc[1], a.vc[2],
                     a.vc[3]})
    ok = ok && st % n == 0;
  if (!ok)
    return q3::fail(QWEN3_EALIGN, "%s: rows must be 16-byte aligned (strides multiple of %d)", who,
                    n);
  if (a.n_tokens == 0) return QWEN3_OK;
  a.sign = inverse ? -1.f : 1.f;
  a.rot_units = layout == 0 ? a.r / 2 / n : a.r / n;
  a.row_units = a.rot_units + (a.D - a.r) / n;
  a.units = (a.Hq + (a.k ? a.Hkv : 0) + (A != Addr::None ? a.Hkv : 0)) * a.row_units;
  const int group = kThreads * (layout == 0 ? units_of<true>() : units_of<false>());
  // the kernel's divisions: of at most units + group by units, of units by row_units
  if (static_cast<int64_t>(a.units + group) * a.units >= (int64_t(1) << 32))
    return q3::fail(QWEN3_EINVAL, "%s: bad sizes", who);
  auto magic = [](int d) {
    return d == 1 ? 0u : static_cast<uint32_t>(((uint64_t(1) << 32) + d - 1) / d);
  };
  a.row_magic = magic(a.row_units);
  a.unit_magic = magic(a.units);
  a.span = (group - 1) / a.units + 2;
  const bool streams = a.n_tokens * (a.Hq + static_cast<int64_t>(a.Hkv)) * a.D * size > kStreamBytes;
  const int64_t blocks = q3::cdiv(a.n_tokens * a.units, group);
  if (a.n_tokens > (int64_t(1) << 40) / a.units || blocks > q3::kMaxThreads / kThreads)
    return q3::fail(QWEN3_EINVAL, "%s: too many tokens", who);
  const size_t lds =
      static_cast<size_t>(a.span) * (static_cast<size_t>(a.r / 2) * sizeof(float2) + 24);
  q3::clear_error();
  const auto s = static_cast<hipStream_t>(stream);
  const auto g = static_cast<unsigned>(blocks);
  if constexpr (A == Addr::None) {
    if (dtype == 1) launch<_Float16, A>(a, layout == 0, streams, g, lds, s);
    if (dtype == 2) launch<float, A>(a, layout == 0, streams, g, lds, s);
  }
  if (dtype == 0) launch<__bf16, A>(a, layout == 0, streams, g, lds, s);
  return q3::launch_status(who);
}

void fill(RotaryArgs& a, const void* q, const int64_t* q_strides, const void* k,
          const int64_t* k_strides, void* q_out, const int64_t* q_out_strides, void* k_out,
          const int64_t* k_out_strides, const double* inv_freq, float factor, int64_t tokens,
          int num_heads, int num_kv_heads, int head_dim, int rotary_dim) {
  a.q = static_cast<const char*>(q);
  a.q_s0 = q_strides[0];
  a.q_s1 = q_strides[1];
  a.k = static_cast<const char*>(k);
  if (k) {
    a.k_s0 = k_strides[0];
    a.k_s1 = k_strides[1];
  }
  a.q_out = static_cast<char*>(q_out);
  a.qo_s0 = q_out_strides[0];
  a.qo_s1 = q_out_strides[1];
  a.k_out = static_cast<char*>(k_out);
  if (k_out) {
    a.ko_s0 = k_out_strides[0];
    a.ko_s1 = k_out_strides[1];
  }
  a.inv_freq = inv_freq;
  a.factor = factor;
  a.n_tokens = tokens;
  a.Hq = num_heads;
  a.Hkv = num_kv_heads;
  a.D = head_dim;
  a.r = rotary_dim;
}

void fill_pool(RotaryArgs& a, const void* v, const int64_t* v_strides, void* k_cache,
               const int64_t* kc, void* v_cache, const int64_t* vc, int64_t num_blocks, int layer,
               int block_size) {
  a.v = static_cast<const uint16_t*>(v);
  a.v_s0 = v_strides[0];
  a.v_s1 = v_strides[1];
  a.k_cache = static_cast<uint16_t*>(k_cache);
  a.v_cache = static_cast<uint16_t*>(v_cache);
  for (int i = 0; i < 4; ++i) {
    a.kc[i] = kc[i];
    a.vc[i] = vc[i];
  }
  a.num_blocks = num_blocks;
  a.layer = layer;
  a.bs = block_size;
}

}  // namespace

extern "C" int qwen3_rotary(const void* q, const int64_t q_strides[2], const void* k,
                            const int64_t k_strides[2], void* q_out,
                            const int64_t q_out_strides[2], void* k_out,
                            const int64_t k_out_strides[2], int dtype, const double* inv_freq,
                            float factor, int layout, int inverse, const int64_t* positions,
                            int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim,
                            int rotary_dim, void* stream) {
  const char* who = "qwen3_rotary";
  if (!q_strides || !q_out_strides || (k && !k_strides) || (k_out && !k_out_strides))
    return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  RotaryArgs a{};
  fill(a, q, q_strides, k, k_strides, q_out, q_out_strides, k_out, k_out_strides, inv_freq, factor,
       num_tokens, num_heads, num_kv_heads, head_dim, rotary_dim);
  a.positions = positions;
  return run<Addr::None>(a, dtype, layout, inverse, 0, stream, who);
}

extern "C" int qwen3_rotary_slots_bf16(
    const void* q, const int64_t q_strides[2], const void* k, const int64_t k_strides[2],
    const void* v, const int64_t v_strides[2], void* q_out, const int64_t q_out_strides[2],
    void* k_out, const int64_t k_out_strides[2], const double* inv_freq, float factor, int layout,
    const int64_t* positions, const int64_t* slot_mapping, void* k_cache,
    const int64_t k_cache_strides[4], void* v_cache, const int64_t v_cache_strides[4],
    int64_t num_blocks, int layer_idx, int num_layers, int64_t num_tokens, int num_heads,
    int num_kv_heads, int head_dim, int rotary_dim, int block_size, void* stream) {
  const char* who = "qwen3_rotary_slots_bf16";
  if (!q_strides || !k_strides || !v_strides || !q_out_strides || (k_out && !k_out_strides) ||
      !k_cache_strides || !v_cache_strides || !slot_mapping)
    return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  RotaryArgs a{};
  fill(a, q, q_strides, k, k_strides, q_out, q_out_strides, k_out, k_out_strides, inv_freq, factor,
       num_tokens, num_heads, num_kv_heads, head_dim, rotary_dim);
  fill_pool(a, v, v_strides, k_cache, k_cache_strides, v_cache, v_cache_strides, num_blocks,
            layer_idx, block_size);
  a.positions = positions;
  a.slots = slot_mapping;
  return run<Addr::Slots>(a, 0, layout, 0, num_layers, stream, who);
}

extern "C" int qwen3_rotary_decode_bf16(
    const void* q, const int64_t q_strides[2], const void* k, const int64_t k_strides[2],
    const void* v, const int64_t v_strides[2], void* q_out, const int64_t q_out_strides[2],
    const double* inv_freq, float factor, int layout, void* k_cache,
    const int64_t k_cache_strides[4], void* v_cache, const int64_t v_cache_strides[4],
    int64_t num_blocks, int layer_idx, int num_layers, const int32_t* seq_lens,
    const int32_t* block_table, int64_t bt_row_stride, int64_t max_rows, int64_t max_pages,
    const int32_t* row_ids, const int64_t* positions, int B, int num_heads, int num_kv_heads,
    int head_dim, int rotary_dim, int block_size, void* stream) {
  const char* who = "qwen3_rotary_decode_bf16";
  if (!q_strides || !k_strides || !v_strides || !q_out_strides || !k_cache_strides ||
      !v_cache_strides || !seq_lens || !block_table)
    return q3::fail(QWEN3_EINVAL, "%s: null pointer argument", who);
  if (B < 0 || max_rows <= 0 || max_pages <= 0 || bt_row_stride < max_pages)
    return q3::fail(QWEN3_EINVAL, "%s: bad table sizes", who);
  RotaryArgs a{};
  fill(a, q, q_strides, k, k_strides, q_out, q_out_strides, nullptr, nullptr, inv_freq, factor, B,
       num_heads, num_kv_heads, head_dim, rotary_dim);
  fill_pool(a, v, v_strides, k_cache, k_cache_strides, v_cache, v_cache_strides, num_blocks,
            layer_idx, block_size);
  a.seq_lens = seq_lens;
  a.block_table = block_table;
  a.bt_stride = bt_row_stride;
  a.max_rows = max_rows;
  a.max_pages = max_pages;
  a.row_ids = row_ids;
  a.positions = positions;
  return run<Addr::Decode>(a, 0, layout, 0, num_layers, stream, who);
}
