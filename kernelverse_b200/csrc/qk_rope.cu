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
// Each element is read once and written once.  What bounds it: the launch for decode steps; for
// prompts latency (3.7 of 6.55 TB/s; DRAM 31 %, issue slots 60 %: a block lives for one round of
// loads, so none of the next heads' are in flight while it computes).  A head is held by a team of
// a few lanes, each with the two V-element vectors whose elements pair up, so the rotation needs no
// exchange and the norm one shuffle tree; a lane keeps the same element range for every head it
// serves, so cos and sin are loaded once per token and lane; the weights are loaded for each head,
// from L1.
#include <type_traits>

#include "kvb_common.cuh"
#include "kvb_async.cuh"

namespace kvb {
namespace {

constexpr unsigned int kStatusBadRopeIndex = 2u;   // a position or slot out of range
constexpr int kRopeThreads = 256;
constexpr int kRopeHeads = 2, kRopeBlocks = 4;   // heads a team, blocks an SM for long inputs

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
  template <bool kOnce = false>            // kOnce: read-once data, not kept in L1 beside the table's rows
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWords % 4 == 0) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4* q = reinterpret_cast<const uint4*>(p) + i;
        const uint4 x = kOnce ? __ldcs(q) : __ldg(q);
        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
      }
    } else {
      static_assert(kWords == 2, "8- or 16-byte vectors");
      const uint2* q = reinterpret_cast<const uint2*>(p);
      const uint2 x = kOnce ? __ldcs(q) : __ldg(q);
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
  // The elements as packed float32 pairs, and back with one rounding.
  __device__ __forceinline__ void unpack(uint64_t (&f)[V / 2]) const {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = f2_pack(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f[i] = f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      } else {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[i] = f2_pack(x.x, x.y);
      }
    }
  }
  __device__ __forceinline__ void pack(const uint64_t (&f)[V / 2]) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 x = f2_unpack(f[i]);
      if constexpr (sizeof(T) == 4) {
        w[2 * i] = __float_as_uint(x.x);
        w[2 * i + 1] = __float_as_uint(x.y);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x.x, x.y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(x.x, x.y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
};

// N floats from a 16-byte boundary (the vector kernels take tables whose rows and halves start on one)
// as packed pairs.
template <int N, int P>
__device__ __forceinline__ void load_floats(const float* p, uint64_t (&f)[P]) {
  static_assert(N % 2 == 0 && N <= 2 * P, "");
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(p + i));
      f[i / 2] = f2_pack(x.x, x.y);
      f[i / 2 + 1] = f2_pack(x.z, x.w);
    }
  } else {
    const float2 x = __ldg(reinterpret_cast<const float2*>(p));
    f[0] = f2_pack(x.x, x.y);
  }
}

template <int P>
__device__ __forceinline__ void store_codes(uint8_t* p, const uint64_t (&f)[P], const Divisor& d) {
  uint32_t c[P / 2];
#pragma unroll
  for (int i = 0; i < P / 2; ++i) {
    const float2 x = f2_unpack(f[2 * i]), y = f2_unpack(f[2 * i + 1]);
    c[i] = quant_e4m3x2(x.x, x.y, d) | ((uint32_t)quant_e4m3x2(y.x, y.y, d) << 16);
  }
  if constexpr (P == 4) *reinterpret_cast<uint2*>(p) = make_uint2(c[0], c[1]);
  else *reinterpret_cast<uint32_t*>(p) = c[0];
}

// A team of `lanes` lanes (a power of two) serves HPT consecutive heads of one token, queries
// first, then keys, then values.
template <typename T, int V, int HPT>
__global__ void __launch_bounds__(kRopeThreads, HPT == 1 ? 1 : kRopeBlocks) qk_rope_kernel(const __grid_constant__ RopeArgs a, int llanes, int pairs,
                                                               uint32_t groups) {
  pdl_trigger();
  pdl_wait();            // launched as a programmatic dependent: global data from here on
  const int lanes = 1 << llanes;
  const uint32_t team = blockIdx.x * (kRopeThreads >> llanes) + (threadIdx.x >> llanes);   // below 2^32: the host checks
  const int li = threadIdx.x & (lanes - 1);
  const uint32_t tok32 = team / groups;
  const int64_t tok = tok32;
  if (tok >= a.tokens) return;   // whole teams leave; the shuffles below name the team's own lanes
  const int h0 = (int)(team - tok32 * groups) * HPT;
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
    if (has_a) xa[i].template load<true>(src + ea);
    if (has_b) xb[i].template load<true>(src + eb);
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
  constexpr int P = V / 2;
  uint64_t c[P], s[P];
#pragma unroll
  for (int i = 0; i < P; ++i) c[i] = s[i] = 0ull;
  if (pos_ok && active && h0 < a.hq + a.hkv) {
    const float* row = a.cos_sin + pos * a.R;
    if (!a.interleaved) {
      if (rot_a) {
        load_floats<V>(row + ea, c);
        load_floats<V>(row + half + ea, s);
      }
    } else if (rot_b) {                      // the lane's pairs are V consecutive ones
      load_floats<V>(row + (ea >> 1), c);
      load_floats<V>(row + half + (ea >> 1), s);
    } else if (rot_a) {
      load_floats<V / 2>(row + (ea >> 1), c);
      load_floats<V / 2>(row + half + (ea >> 1), s);
    }
  }
  int64_t koff = 0, voff = 0;
  if (slot >= 0) {
    // 32-bit division where the slots allow it
    const int64_t blk = a.num_slots <= 0xffffffffLL ? (int64_t)((uint32_t)slot / (uint32_t)a.bs) : slot / a.bs;
    const int64_t in = slot - blk * a.bs;
    koff = blk * a.k_bs + in * a.hkv * (int64_t)a.D;
    voff = blk * a.v_bs + in * a.hkv * (int64_t)a.D;
  }

#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = h0 + i;
    if (h >= heads) break;
    uint64_t fa[P], fb[P];
#pragma unroll
    for (int e = 0; e < P; ++e) fa[e] = fb[e] = 0ull;
    if (has_a) xa[i].unpack(fa);
    if (has_b) xb[i].unpack(fb);
    const bool is_v = h >= a.hq + a.hkv;
    const bool is_k = !is_v && h >= a.hq;
    if (!is_v) {
      const T* w = reinterpret_cast<const T*>(is_k ? a.k_weight : a.q_weight);
      if (w) {
        uint64_t s2 = 0ull;
#pragma unroll
        for (int e = 0; e < P; ++e) s2 = f2_fma(fb[e], fb[e], f2_fma(fa[e], fa[e], s2));
        const float2 sq = f2_unpack(s2);
        float ss = sq.x + sq.y;
        for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float r = rsqrtf(ss / (float)a.D + a.eps);
        const uint64_t r2 = f2_pack(r, r);
        VecN<T, V> wv;
        uint64_t wf[P];
        if (has_a) {
          wv.load(w + ea);
          wv.unpack(wf);
#pragma unroll
          for (int e = 0; e < P; ++e) fa[e] = f2_mul(f2_mul(fa[e], r2), wf[e]);
        }
        if (has_b) {
          wv.load(w + eb);
          wv.unpack(wf);
#pragma unroll
          for (int e = 0; e < P; ++e) fb[e] = f2_mul(f2_mul(fb[e], r2), wf[e]);
        }
      }
      // Only vectors that rotate: an element past the rotary dim passes, whatever its lane's other elements are.
      if (!a.interleaved) {
        if (rot_a) {
          const uint64_t minus = f2_pack(-1.0f, -1.0f);
#pragma unroll
          for (int e = 0; e < P; ++e) {
            const uint64_t y = fa[e], z = fb[e];
            fa[e] = f2_fma(y, c[e], f2_mul(f2_mul(z, s[e]), minus));
            fb[e] = f2_fma(z, c[e], f2_mul(y, s[e]));
          }
        }
      } else {
        // (y, z) -> (y, z) c + (-z, y) s; pair e of the lane has component e of c and s
        auto turn = [&](uint64_t yz, int e) -> uint64_t {
          const float2 v = f2_unpack(yz), c2 = f2_unpack(c[e >> 1]), s2 = f2_unpack(s[e >> 1]);
          const float ce = e & 1 ? c2.y : c2.x, se = e & 1 ? s2.y : s2.x;
          return f2_fma(yz, f2_pack(ce, ce), f2_mul(f2_pack(-v.y, v.x), f2_pack(se, se)));
        };
        if (rot_a) {
#pragma unroll
          for (int e = 0; e < P; ++e) fa[e] = turn(fa[e], e);
        }
        if (rot_b) {
#pragma unroll
          for (int e = 0; e < P; ++e) fb[e] = turn(fb[e], P + e);
        }
      }
      if (!pos_ok) {
        const float nan = __int_as_float(0x7fc00000);
#pragma unroll
        for (int e = 0; e < P; ++e) fa[e] = fb[e] = f2_pack(nan, nan);
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
        if (has_a) store_codes(dst + ea, fa, d);
        if (has_b) store_codes(dst + eb, fb, d);
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
  int llanes = 0;
  while ((1 << llanes) < pairs) ++llanes;
  // Two heads a team once that still gives every SM its blocks: cos and sin are then loaded once for both
  // and four vector loads are in flight per lane (8192 tokens of 32 + 8 heads of 128, bf16, normalised:
  // 46.5 us, 3.7 TB/s; one head 53.1, four 50.6).
  const int64_t per = kRopeThreads >> llanes;
  const bool many = a.tokens * ((heads + kRopeHeads - 1) / kRopeHeads) >= 148LL * kRopeBlocks * per;
  const int64_t groups = many ? (heads + kRopeHeads - 1) / kRopeHeads : heads;
  const int64_t blocks = (a.tokens * groups + per - 1) / per;
  if (blocks > 0x7fffffffLL || blocks * per > 0xffffffffLL) return cudaErrorInvalidConfiguration;
  if (many) return launch_pdl(qk_rope_kernel<T, V, kRopeHeads>, dim3((unsigned)blocks), dim3(kRopeThreads), 0, st, a, llanes, pairs, (uint32_t)groups);
  return launch_pdl(qk_rope_kernel<T, V, 1>, dim3((unsigned)blocks), dim3(kRopeThreads), 0, st, a, llanes, pairs, (uint32_t)groups);
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
    // cos and sin: rows and their halves on 16 bytes (interleaved V = 4: 8 bytes do, but one rule serves)
    const bool table = (reinterpret_cast<uintptr_t>(a.cos_sin) & 15) == 0 && a.R % 8 == 0;
    const bool ok = table && a.D % v == 0 && a.R % unit == 0 && a.D <= 64 * v && on(a.q) && on(a.k) && on(a.q_out) &&
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
