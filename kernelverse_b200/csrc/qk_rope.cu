// Per-head RMSNorm and rotary position embedding of queries and keys, and their append to a paged
// KV cache on the way.
//
// Mathematics, in float32 with one rounding at the end.  For each head x of D elements:
//   y = x * rsqrt(mean(x^2) + eps) * w                     (only where a weight is given)
//   the pair (i, j) of angle n < R / 2 becomes (y_i c_n - y_j s_n, y_j c_n + y_i s_n), where
//   (c, s) is row positions[token] of the cos/sin table and (i, j) = (n, n + R / 2), or
//   (2 n, 2 n + 1) when interleaved; elements R..D pass unrotated.
// The append stores keys and values at slot slot_mapping[token] as they are or as
// e4m3(clamp(y / scale[h], +-448)), quantised from the float32 value with the correctly rounded
// quotient.
//
// What bounds it: HBM for prompts (each element is read once and written once), the launch for
// decode steps.  A head is held by a team of a few lanes, each with the two V-element vectors
// whose elements pair up, so the rotation needs no exchange and the norm one shuffle tree; a lane
// keeps the same element range for every head it serves, so cos, sin and the weights are loaded
// once per token and lane.
#include "kvb_common.cuh"
#include "kvb_async.cuh"

namespace kvb {
namespace {

constexpr unsigned int kStatusBadRopeIndex = 2u;   // a position or slot out of range
constexpr int kRopeThreads = 256;

struct RopeArgs {
  const void* q;
  const void* k;
  const void* v;              // null: norm and rotation only
  const void* positions;      // [tokens]
  const void* slots;          // [tokens] (append)
  const float* cos_sin;       // [max_pos, R]: R/2 cosines, R/2 sines
  const void* q_weight;       // [D] or null
  const void* k_weight;
  const float* k_scale;       // [hkv] (e4m3 caches)
  const float* v_scale;
  void* q_out;                // [tokens, hq, D]
  void* k_out;                // [tokens, hkv, D], or the K cache
  void* v_out;                // the V cache
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;   // input strides (elements) of a token and of a head
  int64_t max_pos, tokens, num_slots, k_bs, v_bs;  // k_bs / v_bs: cache elements of one block
  int hq, hkv, D, R, bs;
  int pos64, slot64, interleaved, e4m3;
  float eps;
};

__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t)reinterpret_cast<const int32_t*>(p)[i];
}

// V elements of T moved with the widest accesses their size allows (16 bytes each at most).
template <typename T, int V> struct VecN {
  static constexpr int kBytes = V * (int)sizeof(T);
  static constexpr int kWords = kBytes / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWords % 4 == 0) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
      }
    } else {
      static_assert(kWords == 2, "8- or 16-byte vectors");
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = x.x; w[1] = x.y;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kWords % 4 == 0) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    }
  }
  __device__ __forceinline__ void unpack(float (&f)[V]) const {
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = Elem<T>::to_f(e[i]);
  }
  __device__ __forceinline__ void pack(const float (&f)[V]) {
    T* e = reinterpret_cast<T*>(w);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = Elem<T>::from_f(f[i]);
  }
};

template <int V>
__device__ __forceinline__ void load_floats(const float* p, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 2) {   // 8-byte aligned: the table's rows have an even number of floats
    const float2 x = __ldg(reinterpret_cast<const float2*>(p + i));
    f[i] = x.x; f[i + 1] = x.y;
  }
}

template <int V>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&f)[V], const Divisor& d) {
  uint32_t c[V / 4];
#pragma unroll
  for (int i = 0; i < V / 4; ++i)
    c[i] = quant_e4m3x2(f[4 * i], f[4 * i + 1], d) | ((uint32_t)quant_e4m3x2(f[4 * i + 2], f[4 * i + 3], d) << 16);
  if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(c[0], c[1]);
  else *reinterpret_cast<uint32_t*>(p) = c[0];
}

// A team of `lanes` lanes (a power of two) serves HPT consecutive heads of one token, queries
// first, then keys, then values.
template <typename T, int V, int HPT>
__global__ void __launch_bounds__(kRopeThreads) qk_rope_kernel(const __grid_constant__ RopeArgs a, int lanes, int pairs,
                                                               int groups) {
  pdl_trigger();
  pdl_wait();            // launched as a programmatic dependent: global data from here on
  const int64_t team = ((int64_t)blockIdx.x * kRopeThreads + threadIdx.x) / lanes;
  const int li = threadIdx.x & (lanes - 1);
  const int64_t tok = team / groups;
  if (tok >= a.tokens) return;   // whole teams leave; the shuffles below name the team's own lanes
  const int h0 = (int)(team - tok * groups) * HPT;
  const uint32_t mask = (lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u)) << ((threadIdx.x & 31) & ~(lanes - 1));
  const int heads = a.hq + a.hkv + (a.v ? a.hkv : 0);
  const int half = a.R >> 1;

  // This lane's two vectors: elements [ea, ea + V) and [eb, eb + V).
  const bool active = li < pairs;
  int ea, eb;
  bool rot_a, rot_b;
  if (a.interleaved) {
    ea = 2 * V * li;
    eb = ea + V;
    rot_a = ea < a.R;
    rot_b = eb < a.R;
  } else {
    const int rp = half / V;               // lanes that hold rotated pairs
    rot_a = rot_b = li < rp;
    ea = rot_a ? V * li : a.R + 2 * V * (li - rp);
    eb = rot_a ? half + V * li : ea + V;
  }
  const bool has_a = active && ea < a.D, has_b = active && eb < a.D;

  // Every load of the team's heads is issued before the first is used.
  VecN<T, V> xa[HPT], xb[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = h0 + i;
    if (h >= heads) break;
    const T* src;
    if (h < a.hq) src = reinterpret_cast<const T*>(a.q) + tok * a.q_ts + h * a.q_hs;
    else if (h < a.hq + a.hkv) src = reinterpret_cast<const T*>(a.k) + tok * a.k_ts + (h - a.hq) * a.k_hs;
    else src = reinterpret_cast<const T*>(a.v) + tok * a.v_ts + (h - a.hq - a.hkv) * a.v_hs;
    if (has_a) xa[i].load(src + ea);
    if (has_b) xb[i].load(src + eb);
  }
  const int64_t pos = load_index(a.positions, a.pos64, tok);
  const bool pos_ok = pos >= 0 && pos < a.max_pos;
  int64_t slot = -1;
  if (a.v) {
    slot = load_index(a.slots, a.slot64, tok);
    if (slot >= a.num_slots || !pos_ok) {
      if (slot >= a.num_slots && li == 0) atomicOr(&g_tu_status, kStatusBadRopeIndex);
      slot = -1;
    }
  }
  if (!pos_ok && li == 0) atomicOr(&g_tu_status, kStatusBadRopeIndex);

  // cos / sin: V values each; interleaved, the first half belongs to xa and the second to xb
  float c[V], s[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    c[i] = 1.0f;
    s[i] = 0.0f;
  }
  if (pos_ok && active && h0 < a.hq + a.hkv) {
    const float* row = a.cos_sin + pos * a.R;
    if (!a.interleaved) {
      if (rot_a) {
        load_floats<V>(row + ea, c);
        load_floats<V>(row + half + ea, s);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = i < V / 2 ? ea + 2 * i : eb + 2 * (i - V / 2);   // first element of the pair
        if (e < a.R) {
          c[i] = __ldg(row + (e >> 1));
          s[i] = __ldg(row + half + (e >> 1));
        }
      }
    }
  }
  int64_t koff = 0, voff = 0;
  if (slot >= 0) {
    const int64_t blk = slot / a.bs, in = slot - blk * a.bs;
    koff = blk * a.k_bs + in * a.hkv * (int64_t)a.D;
    voff = blk * a.v_bs + in * a.hkv * (int64_t)a.D;
  }

#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = h0 + i;
    if (h >= heads) break;
    float fa[V], fb[V];
#pragma unroll
    for (int e = 0; e < V; ++e) fa[e] = fb[e] = 0.0f;
    if (has_a) xa[i].unpack(fa);
    if (has_b) xb[i].unpack(fb);
    const bool is_v = h >= a.hq + a.hkv;
    const bool is_k = !is_v && h >= a.hq;
    if (!is_v) {
      const T* w = reinterpret_cast<const T*>(is_k ? a.k_weight : a.q_weight);
      if (w) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) ss += fa[e] * fa[e] + fb[e] * fb[e];
        for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float r = rsqrtf(ss / (float)a.D + a.eps);
        VecN<T, V> wv;
        float wf[V];
        if (has_a) {
          wv.load(w + ea);
          wv.unpack(wf);
#pragma unroll
          for (int e = 0; e < V; ++e) fa[e] = fa[e] * r * wf[e];
        }
        if (has_b) {
          wv.load(w + eb);
          wv.unpack(wf);
#pragma unroll
          for (int e = 0; e < V; ++e) fb[e] = fb[e] * r * wf[e];
        }
      }
      if (!a.interleaved) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float y = fa[e], z = fb[e];
          fa[e] = y * c[e] - z * s[e];
          fb[e] = z * c[e] + y * s[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          const float y = fa[2 * e], z = fa[2 * e + 1];
          fa[2 * e] = y * c[e] - z * s[e];
          fa[2 * e + 1] = z * c[e] + y * s[e];
          const float u = fb[2 * e], t = fb[2 * e + 1];
          fb[2 * e] = u * c[V / 2 + e] - t * s[V / 2 + e];
          fb[2 * e + 1] = t * c[V / 2 + e] + u * s[V / 2 + e];
        }
      }
      if (!pos_ok) {
#pragma unroll
        for (int e = 0; e < V; ++e) fa[e] = fb[e] = __int_as_float(0x7fc00000);
      }
    }
    VecN<T, V> o;
    if (h < a.hq) {
      T* dst = reinterpret_cast<T*>(a.q_out) + (tok * a.hq + h) * a.D;
      if (has_a) { o.pack(fa); o.store(dst + ea); }
      if (has_b) { o.pack(fb); o.store(dst + eb); }
    } else if (!a.v) {
      T* dst = reinterpret_cast<T*>(a.k_out) + (tok * a.hkv + (h - a.hq)) * a.D;
      if (has_a) { o.pack(fa); o.store(dst + ea); }
      if (has_b) { o.pack(fb); o.store(dst + eb); }
    } else if (slot >= 0) {
      const int kh = is_v ? h - a.hq - a.hkv : h - a.hq;
      const int64_t off = (is_v ? voff : koff) + (int64_t)kh * a.D;
      if (a.e4m3) {
        uint8_t* dst = reinterpret_cast<uint8_t*>(is_v ? a.v_out : a.k_out) + off;
        const Divisor d = make_divisor(__ldg((is_v ? a.v_scale : a.k_scale) + kh));
        if (has_a) store_codes<V>(dst + ea, fa, d);
        if (has_b) store_codes<V>(dst + eb, fb, d);
      } else {
        T* dst = reinterpret_cast<T*>(is_v ? a.v_out : a.k_out) + off;
        if (has_a) { o.pack(fa); o.store(dst + ea); }
        if (has_b) { o.pack(fb); o.store(dst + eb); }
      }
    }
  }
}

// Any even head and rotary dim, any alignment: one warp per (token, head), element by element; the
// head is read once for the norm and once more (from L1) for the rotation.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) qk_rope_any_kernel(const __grid_constant__ RopeArgs a) {
  pdl_trigger();
  pdl_wait();
  const int heads = a.hq + a.hkv + (a.v ? a.hkv : 0);
  const int64_t unit = ((int64_t)blockIdx.x * kRopeThreads + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int64_t tok = unit / heads;
  if (tok >= a.tokens) return;
  const int h = (int)(unit - tok * heads);
  const bool is_v = h >= a.hq + a.hkv, is_k = !is_v && h >= a.hq;
  const int64_t pos = load_index(a.positions, a.pos64, tok);
  const bool pos_ok = pos >= 0 && pos < a.max_pos;
  int64_t slot = -1;
  if (a.v) {
    slot = load_index(a.slots, a.slot64, tok);
    if (slot >= a.num_slots || !pos_ok) {
      if (slot >= a.num_slots && lane == 0) atomicOr(&g_tu_status, kStatusBadRopeIndex);
      slot = -1;
    }
  }
  if (!pos_ok && lane == 0) atomicOr(&g_tu_status, kStatusBadRopeIndex);
  const int kh = is_v ? h - a.hq - a.hkv : h - a.hq;
  const T* src = is_v ? reinterpret_cast<const T*>(a.v) + tok * a.v_ts + kh * a.v_hs
                      : is_k ? reinterpret_cast<const T*>(a.k) + tok * a.k_ts + kh * a.k_hs
                             : reinterpret_cast<const T*>(a.q) + tok * a.q_ts + h * a.q_hs;
  const T* w = is_v ? nullptr : reinterpret_cast<const T*>(is_k ? a.k_weight : a.q_weight);
  float r = 1.0f;
  if (w) {
    float ss = 0.0f;
    for (int e = lane; e < a.D; e += 32) {
      const float x = Elem<T>::to_f(src[e]);
      ss += x * x;
    }
    r = rsqrtf(warp_sum(ss) / (float)a.D + a.eps);
  }
  void* out;
  int64_t off;
  bool codes = false;
  Divisor d = make_divisor(1.0f);
  if (h < a.hq) {
    out = a.q_out;
    off = (tok * a.hq + h) * a.D;
  } else if (!a.v) {
    out = a.k_out;
    off = (tok * a.hkv + kh) * a.D;
  } else {
    if (slot < 0) return;
    const int64_t blk = slot / a.bs;
    out = is_v ? a.v_out : a.k_out;
    off = blk * (is_v ? a.v_bs : a.k_bs) + ((slot - blk * a.bs) * a.hkv + kh) * (int64_t)a.D;
    codes = a.e4m3;
    if (codes) d = make_divisor((is_v ? a.v_scale : a.k_scale)[kh]);
  }
  auto put = [&](int e, float f) {
    if (codes) reinterpret_cast<uint8_t*>(out)[off + e] = (uint8_t)(quant_e4m3x2(f, 0.0f, d) & 0xffu);
    else reinterpret_cast<T*>(out)[off + e] = Elem<T>::from_f(f);
  };
  auto get = [&](int e) -> float {
    const float x = Elem<T>::to_f(src[e]);
    return w ? x * r * Elem<T>::to_f(w[e]) : x;
  };
  const int half = a.R >> 1;
  const float* row = a.cos_sin + (pos_ok ? pos : 0) * a.R;
  if (is_v) {
    for (int e = lane; e < a.D; e += 32) put(e, Elem<T>::to_f(src[e]));
    return;
  }
  const float nan = __int_as_float(0x7fc00000);
  for (int n = lane; n < half; n += 32) {
    const int i = a.interleaved ? 2 * n : n, j = a.interleaved ? 2 * n + 1 : n + half;
    const float y = get(i), z = get(j);
    const float c = pos_ok ? row[n] : nan, s = pos_ok ? row[half + n] : nan;
    put(i, y * c - z * s);
    put(j, z * c + y * s);
  }
  for (int e = a.R + lane; e < a.D; e += 32) put(e, pos_ok ? get(e) : nan);
}

template <typename T, int V>
cudaError_t launch_rope(const RopeArgs& a, cudaStream_t st) {
  const int heads = a.hq + a.hkv + (a.v ? a.hkv : 0);
  const int pairs = a.interleaved ? (a.D + 2 * V - 1) / (2 * V) : a.R / (2 * V) + (a.D - a.R + 2 * V - 1) / (2 * V);
  int lanes = 1;
  while (lanes < pairs) lanes <<= 1;
  // Four heads a team once that still gives every SM several blocks: cos and sin are then loaded
  // once for four heads and eight vector loads are in flight per lane.
  const bool four = a.tokens * ((heads + 3) / 4) * lanes >= 148LL * 4 * kRopeThreads;
  const int groups = four ? (heads + 3) / 4 : heads;
  const int64_t blocks = (a.tokens * groups * lanes + kRopeThreads - 1) / kRopeThreads;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  if (four) return launch_pdl(qk_rope_kernel<T, V, 4>, dim3((unsigned)blocks), dim3(kRopeThreads), 0, st, a, lanes, pairs, groups);
  return launch_pdl(qk_rope_kernel<T, V, 1>, dim3((unsigned)blocks), dim3(kRopeThreads), 0, st, a, lanes, pairs, groups);
}

template <typename T>
cudaError_t dispatch_rope(const RopeArgs& a, int vec, cudaStream_t st) {
  if (vec == 8) return launch_rope<T, 8>(a, st);
  if (vec == 4) return launch_rope<T, 4>(a, st);
  const int64_t units = a.tokens * (a.hq + a.hkv + (a.v ? a.hkv : 0));
  const int64_t blocks = (units * 32 + kRopeThreads - 1) / kRopeThreads;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  return launch_pdl(qk_rope_any_kernel<T>, dim3((unsigned)blocks), dim3(kRopeThreads), 0, st, a);
}

// Checks what the two entry points share, picks the vector width and launches.
int run_rope(const char* what, RopeArgs& a, int dtype, cudaStream_t st) {
  if (!is_float_dtype(dtype)) return set_error(KVB_E_DTYPE, "%s: dtype %d", what, dtype);
  if (a.tokens < 0 || a.hq <= 0 || a.hkv <= 0 || a.D <= 0 || a.R < 0 || a.max_pos < 0)
    return set_error(KVB_E_ARG, "%s: bad sizes", what);
  if (a.D % 2 || a.R % 2 || a.R > a.D || a.D > 1024)
    return set_error(KVB_E_SHAPE, "%s: head_dim (even, <= 1024) and rotary_dim (even, <= head_dim), got %d and %d", what,
                     a.D, a.R);
  if (a.tokens == 0) return KVB_OK;
  const int es = dtype_size(dtype);
  if ((reinterpret_cast<uintptr_t>(a.cos_sin) & 7) != 0) return set_error(KVB_E_ALIGN, "%s: cos_sin needs 8-byte alignment", what);
  // The widest vectors that every row starts on: V elements, 16 bytes at most a load.
  int vec = 0;
  for (int v : {8, 4}) {
    const int unit = a.interleaved ? v : 2 * v;
    const uintptr_t ab = v * es < 16 ? (uintptr_t)(v * es) : 16;
    auto on = [&](const void* p) { return (reinterpret_cast<uintptr_t>(p) & (ab - 1)) == 0; };
    auto even = [&](int64_t s) { return (s * es) % (int64_t)ab == 0; };
    const int64_t cache_al = a.e4m3 ? v : (int64_t)ab / es;      // elements
    const bool ok = a.D % v == 0 && a.R % unit == 0 && a.D <= 64 * v && on(a.q) && on(a.k) && on(a.q_out) &&
                    (!a.q_weight || on(a.q_weight)) && (!a.k_weight || on(a.k_weight)) && even(a.q_ts) && even(a.q_hs) &&
                    even(a.k_ts) && even(a.k_hs) &&
                    (a.v ? on(a.v) && even(a.v_ts) && even(a.v_hs) && a.k_bs % cache_al == 0 && a.v_bs % cache_al == 0 &&
                               (a.e4m3 ? ((reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out)) &
                                          (uintptr_t)(v - 1)) == 0
                                       : on(a.k_out) && on(a.v_out))
                         : on(a.k_out));
    if (ok) {
      vec = v;
      break;
    }
  }
  cudaError_t e;
  switch (dtype) {
    case KVB_BF16: e = dispatch_rope<__nv_bfloat16>(a, vec, st); break;
    case KVB_F16: e = dispatch_rope<__half>(a, vec, st); break;
    default: e = dispatch_rope<float>(a, vec, st); break;
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(KVB_E_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  }
  return check_launch(what);
}

}  // namespace
}  // namespace kvb

using namespace kvb;

extern "C" int kvb_qk_norm_rope(const void* q, const void* k, int dtype, int64_t q_token_stride, int64_t q_head_stride,
                                int64_t k_token_stride, int64_t k_head_stride, const void* positions, int positions_dtype,
                                const float* cos_sin, int64_t max_positions, int rotary_dim, int interleaved,
                                const void* q_weight, const void* k_weight, float eps, int64_t num_tokens, int num_q_heads,
                                int num_kv_heads, int head_dim, void* q_out, void* k_out, void* stream) {
  if (positions_dtype != KVB_I32 && positions_dtype != KVB_I64) return set_error(KVB_E_DTYPE, "qk_norm_rope: positions dtype");
  if (num_tokens > 0 && (!q || !k || !positions || !q_out || !k_out || (!cos_sin && rotary_dim > 0)))
    return set_error(KVB_E_ARG, "qk_norm_rope: null pointer");
  RopeArgs a{};
  a.q = q; a.k = k; a.positions = positions; a.cos_sin = cos_sin; a.q_weight = q_weight; a.k_weight = k_weight;
  a.q_out = q_out; a.k_out = k_out;
  a.q_ts = q_token_stride; a.q_hs = q_head_stride; a.k_ts = k_token_stride; a.k_hs = k_head_stride;
  a.max_pos = max_positions; a.tokens = num_tokens; a.hq = num_q_heads; a.hkv = num_kv_heads; a.D = head_dim;
  a.R = rotary_dim; a.pos64 = positions_dtype == KVB_I64; a.interleaved = interleaved != 0; a.eps = eps; a.bs = 1;
  return run_rope("qk_norm_rope", a, dtype, as_stream(stream));
}

extern "C" int kvb_rope_paged_kv_append(const void* q, const void* k, const void* v, int dtype, int64_t q_token_stride,
                                        int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                                        int64_t v_token_stride, int64_t v_head_stride, const void* positions,
                                        int positions_dtype, const void* slot_mapping, int slot_dtype, const float* cos_sin,
                                        int64_t max_positions, int rotary_dim, int interleaved, const void* q_weight,
                                        const void* k_weight, float eps, int64_t num_tokens, int num_q_heads,
                                        int num_kv_heads, int head_dim, void* k_cache, void* v_cache, int cache_dtype,
                                        int block_size, int64_t num_blocks, int64_t k_block_stride, int64_t v_block_stride,
                                        const float* k_scale, const float* v_scale, void* q_out, void* stream) {
  if ((positions_dtype != KVB_I32 && positions_dtype != KVB_I64) || (slot_dtype != KVB_I32 && slot_dtype != KVB_I64))
    return set_error(KVB_E_DTYPE, "rope_paged_kv_append: positions / slot dtype");
  if (cache_dtype != dtype && cache_dtype != KVB_E4M3)
    return set_error(KVB_E_DTYPE, "rope_paged_kv_append: the cache holds the input type or e4m3 codes, not dtype %d", cache_dtype);
  if (block_size <= 0 || num_blocks < 0) return set_error(KVB_E_ARG, "rope_paged_kv_append: bad cache sizes");
  if (num_tokens > 0 && (!q || !k || !v || !positions || !slot_mapping || !q_out || !k_cache || !v_cache ||
                         (!cos_sin && rotary_dim > 0) || (cache_dtype == KVB_E4M3 && (!k_scale || !v_scale))))
    return set_error(KVB_E_ARG, "rope_paged_kv_append: null pointer");
  const int64_t block = (int64_t)block_size * num_kv_heads * head_dim;
  if (num_blocks > 1 && (k_block_stride < block || v_block_stride < block))
    return set_error(KVB_E_SHAPE, "rope_paged_kv_append: cache blocks overlap");
  RopeArgs a{};
  a.q = q; a.k = k; a.v = v; a.positions = positions; a.slots = slot_mapping; a.cos_sin = cos_sin;
  a.q_weight = q_weight; a.k_weight = k_weight; a.k_scale = k_scale; a.v_scale = v_scale;
  a.q_out = q_out; a.k_out = k_cache; a.v_out = v_cache;
  a.q_ts = q_token_stride; a.q_hs = q_head_stride; a.k_ts = k_token_stride; a.k_hs = k_head_stride;
  a.v_ts = v_token_stride; a.v_hs = v_head_stride;
  a.max_pos = max_positions; a.tokens = num_tokens; a.num_slots = num_blocks * block_size;
  a.k_bs = k_block_stride; a.v_bs = v_block_stride; a.hq = num_q_heads; a.hkv = num_kv_heads; a.D = head_dim;
  a.R = rotary_dim; a.bs = block_size; a.pos64 = positions_dtype == KVB_I64; a.slot64 = slot_dtype == KVB_I64;
  a.interleaved = interleaved != 0; a.e4m3 = cache_dtype == KVB_E4M3; a.eps = eps;
  return run_rope("rope_paged_kv_append", a, dtype, as_stream(stream));
}
