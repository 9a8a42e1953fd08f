// Causal attention of chunks of new tokens over a paged KV cache.
//
// Request b owns query rows [qo[b], qo[b+1]) and holds seq_lens[b] tokens in the cache, the chunk's
// own among them, so its query i stands at position p = seq_len - q_len + i and sees keys 0..p of
// KV head h / group:
//   out = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m),  s_t = scale log2(e) q.k_t,  m = max_t s_t.
// A row at a negative position sees nothing: its output is 0 and its log-sum-exp -inf.
//
// This file holds the entry point, the kernel for everything that the tcgen05 kernel does not take
// (float32, other head dims) and the merge of partial results.  The kernel here is a flash-attention
// tile: 64 query rows of one KV head's group (tokens x heads packed, so a decoding request's group
// shares each key), four warps of 16 rows, K/V tiles double-buffered in shared memory, products on
// mma.sync with float32 accumulation (16-bit operands, or 3xTF32 for float32: about float32
// accuracy), online softmax in the log2 domain.  e4m3 codes become the query's type on their way
// into shared memory (exactly: both 16-bit types hold every code) and the scales go into the logit
// scale and the output.
// What bounds it: the products (three per float32 one) for chunks, latency for short calls.  2048 new
// tokens of 16384, 32 + 8 heads of 128, bf16: 3.16 ms (163 TFLOP/s), where the tcgen05 kernel takes
// 0.53; five float32 requests of up to 700 tokens, 6 + 2 heads of 64: 21 us.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kvb_common.cuh"
#include "kvb_async.cuh"
#include "mma_sync.cuh"
#include "paged_prefill.cuh"

namespace kvb {

bool paged_prefill_tc_takes(const PagedArgs& a, int q_dtype, int cache_dtype);
int paged_prefill_tcgen05(PagedArgs& a, int q_dtype, int cache_dtype, void* ws, int sms, cudaStream_t st);

namespace {

constexpr int kPpRows = 64;
constexpr int kPpThreads = 128;

// Eight elements of a cache row as eight elements of T at `dst` (shared memory).
template <typename T>
__device__ __forceinline__ void codes_to_smem(uint8_t* dst, uint2 codes) {
  Vec8<T> o;
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t two = ((i < 2 ? codes.x : codes.y) >> (16 * (i & 1))) & 0xffffu;
    const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&hr));
    f[2 * i] = x.x;
    f[2 * i + 1] = x.y;
  }
  o.pack(f);
  o.store(reinterpret_cast<T*>(dst));
}

template <typename T, bool kE4m3, int DP>
__global__ void __launch_bounds__(kPpThreads, 2) paged_prefill_kernel(const __grid_constant__ PagedArgs a) {
  using TR = PfTraits<T>;
  constexpr int BK = TR::kBK;
  constexpr int ES = (int)sizeof(T);
  constexpr int CS = kE4m3 ? 1 : ES;      // bytes of a cache element
  constexpr int kRowB = DP * ES + 16;     // padded row: conflict-free ldmatrix / fragment loads
  constexpr int NT = BK / 8;              // key n-tiles of S
  constexpr int ND = DP / 8;              // d n-tiles of O
  // float16 has few exponents: P is held 2^7 larger there, so that weights down to 2^-21 of the
  // largest keep their full precision.
  constexpr float kUp = std::is_same<T, __half>::value ? 7.0f : 0.0f;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* const qs = smem;
  uint8_t* const ks = qs + kPpRows * kRowB;          // [2][BK] rows
  uint8_t* const vs = ks + 2 * BK * kRowB;           // [2][BK] rows
  __shared__ PgShare share;
  __shared__ int64_t scan[kPpThreads / 32];
  __shared__ int2 page[2][BK];                       // {block, row in it} of a tile's keys; block -1: nothing there
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int D = a.D;
  const PgTiles tiles{kPpRows, BK, a.group};

  // Padding columns [D, DP) of every shared row are zero for the whole kernel (the copies never
  // write them), so they add nothing to Q K^T.
  if (D < DP) {
    const int pad_words = (DP - D) * ES / 4;
    for (int i = tid; i < (kPpRows + 4 * BK) * pad_words; i += kPpThreads) {
      const int r = i / pad_words, c = i - r * pad_words;
      reinterpret_cast<uint32_t*>(smem + r * kRowB + D * ES)[c] = 0u;
    }
  }
  pdl_trigger();
  pdl_wait();            // launched as a programmatic dependent: global data from here on
  pg_share<kPpThreads>(a, tiles, blockIdx.x, gridDim.x, &share, scan, &g_tu_status);
  if (tid == 0) a.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
  const uint32_t qs_a = smem_u32(qs), ks_a = smem_u32(ks), vs_a = smem_u32(vs);

  PgWalk walk(share);
  PgItem it;
  int64_t at = walk.at;
  while (walk.next(a, tiles, it)) {
    const int kl = it.r.kl, rw = it.r.ql * a.group, row0 = it.t * kPpRows, off = it.r.kl - it.r.ql;
    const int64_t kstep = (int64_t)a.hkv * D;         // elements from one token of a block to the next
    const uint8_t* kg = reinterpret_cast<const uint8_t*>(a.k_cache) + (int64_t)it.h * D * CS;
    const uint8_t* vg = reinterpret_cast<const uint8_t*>(a.v_cache) + (int64_t)it.h * D * CS;
    const int32_t* bt = a.block_table + (int64_t)it.b * a.bt_stride;

    auto look_up = [&](int j) {                       // the pages of key tile j
      if (tid < BK) {
        const int key = j * BK + tid;
        int2 e = make_int2(-1, 0);
        if (key < kl) {
          const int blk = key / a.bs;
          const int phys = bt[blk];
          if (phys < 0 || phys >= a.num_blocks) atomicOr(&g_tu_status, kStatusBadPage);
          else e = make_int2(phys, key - blk * a.bs);
        }
        page[j & 1][tid] = e;
      }
    };
    auto load_tile = [&](int j) {                     // keys and values of tile j into buffer j & 1
      const int buf = j & 1;
      constexpr int PC = kE4m3 ? 8 : 16 / ES;         // elements per copy
      const int chunks = D / PC;
      for (int i = tid; i < 2 * BK * chunks; i += kPpThreads) {
        const bool is_v = i >= BK * chunks;
        const int i2 = is_v ? i - BK * chunks : i;
        const int r = i2 / chunks, c = i2 - r * chunks;
        const int2 e = page[buf][r];
        const bool ok = e.x >= 0;
        const uint8_t* src = (is_v ? vg : kg) +
                             (ok ? ((int64_t)e.x * (is_v ? a.v_bs : a.k_bs) + e.y * kstep + c * PC) * CS : 0);
        const uint32_t doff = (uint32_t)((buf * BK + r) * kRowB + c * PC * ES);
        if constexpr (kE4m3) {
          codes_to_smem<T>((is_v ? vs : ks) + doff, ok ? __ldg(reinterpret_cast<const uint2*>(src)) : make_uint2(0u, 0u));
        } else {
          cp_async16((is_v ? vs_a : ks_a) + doff, src, ok);
        }
      }
      cp_async_commit();
    };

    // query rows: row r of the tile is token (row0 + r) / group, head h * group + (row0 + r) % group
    {
      const int chunks = D * ES / 16;
      for (int i = tid; i < kPpRows * chunks; i += kPpThreads) {
        const int r = i / chunks, c = i - r * chunks;
        const int gr = row0 + r;
        const bool ok = gr < rw;
        const int tok = ok ? gr / a.group : 0;
        const int hd = it.h * a.group + (ok ? gr - tok * a.group : 0);
        cp_async16(qs_a + (uint32_t)(r * kRowB + c * 16),
                   reinterpret_cast<const T*>(a.q) + (int64_t)(it.r.q0 + tok) * a.q_ts + (int64_t)hd * D + c * (16 / ES), ok);
      }
      cp_async_commit();
    }
    look_up(it.j0);
    __syncthreads();
    load_tile(it.j0);

    const int r0 = warp * 16;
    const int gr0 = row0 + r0 + g, gr1 = gr0 + 8;      // the thread's two rows
    const int pos0 = gr0 < rw ? off + gr0 / a.group : -1, pos1 = gr1 < rw ? off + gr1 / a.group : -1;
    const int pos_first = row0 + r0 < rw ? off + (row0 + r0) / a.group : -1;
    const bool warp_end = row0 + r0 + 15 >= rw;        // some row of the warp is past the request
    const float sc = a.scale_log2 * (kE4m3 ? __ldg(a.k_scale + it.h) : 1.0f);
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    float o[ND][4];
#pragma unroll
    for (int n = 0; n < ND; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;

    for (int j = it.j0; j < it.j1; ++j) {
      if (j + 1 < it.j1) {
        look_up(j + 1);
        __syncthreads();
        load_tile(j + 1);
        cp_async_wait<1>();
      } else {
        cp_async_wait<0>();
      }
      __syncthreads();
      const int buf = j & 1;
      const uint8_t* kb_s = ks + buf * BK * kRowB;
      const uint8_t* vb_s = vs + buf * BK * kRowB;
      const uint32_t kb_a = ks_a + buf * BK * kRowB, vb_a = vs_a + buf * BK * kRowB;

      // ---- S = Q K^T for this warp's 16 rows and BK keys
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
      if constexpr (TR::k16) {
        const int mat = lane >> 3, rr = lane & 7;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          uint32_t qf[4];
          ldsm_x4(qf, qs_a + (uint32_t)((r0 + (mat & 1) * 8 + rr) * kRowB + (kk * 16 + (mat >> 1) * 8) * 2));
#pragma unroll
          for (int n = 0; n < NT; n += 2) {
            uint32_t bq[4];
            ldsm_x4(bq, kb_a + (uint32_t)((n * 8 + (mat >> 1) * 8 + rr) * kRowB + (kk * 16 + (mat & 1) * 8) * 2));
            mma_k16<TR::kBf>(s[n], qf, bq[0], bq[1]);
            mma_k16<TR::kBf>(s[n + 1], qf, bq[2], bq[3]);
          }
        }
      } else {
        const float* q_r0 = reinterpret_cast<const float*>(qs + (r0 + g) * kRowB) + t4;
        const float* q_r1 = reinterpret_cast<const float*>(qs + (r0 + g + 8) * kRowB) + t4;
#pragma unroll 4
        for (int kk = 0; kk < DP / 8; ++kk) {
          const float af[4] = {q_r0[kk * 8], q_r1[kk * 8], q_r0[kk * 8 + 4], q_r1[kk * 8 + 4]};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float* kr = reinterpret_cast<const float*>(kb_s + (n * 8 + g) * kRowB) + kk * 8 + t4;
            mma_3xtf32(s[n], af, kr[0], kr[4]);
          }
        }
      }

      // ---- scale, causal mask (only where the tile reaches past this warp's first row), online softmax
      const int kbase = j * BK;
      const bool mask = warp_end || kbase + BK - 1 > pos_first;
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = kbase + n * 8 + 2 * t4 + e;
          float v0 = s[n][e] * sc, v1 = s[n][2 + e] * sc;
          if (mask) {
            if (key > pos0) v0 = -INFINITY;
            if (key > pos1) v1 = -INFINITY;
          }
          s[n][e] = v0;
          s[n][2 + e] = v1;
          mx0 = fmaxf(mx0, v0);
          mx1 = fmaxf(mx1, v1);
        }
      }
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
      mx0 = fmaxf(m0, mx0 - kUp);          // m0, m1: the maxima less kUp; P lies in [0, 2^kUp]
      mx1 = fmaxf(m1, mx1 - kUp);
      const float mu0 = mx0 == -INFINITY ? 0.0f : mx0, mu1 = mx1 == -INFINITY ? 0.0f : mx1;   // rows that see nothing yet
      const float al0 = pg_ex2(m0 - mu0), al1 = pg_ex2(m1 - mu1);
      m0 = mx0;
      m1 = mx1;
      float rs0 = 0.0f, rs1 = 0.0f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[n][0] = pg_ex2(s[n][0] - mu0);
        s[n][1] = pg_ex2(s[n][1] - mu0);
        s[n][2] = pg_ex2(s[n][2] - mu1);
        s[n][3] = pg_ex2(s[n][3] - mu1);
        rs0 += s[n][0] + s[n][1];
        rs1 += s[n][2] + s[n][3];
      }
      l0 = l0 * al0 + rs0;
      l1 = l1 * al1 + rs1;
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        o[n][0] *= al0;
        o[n][1] *= al0;
        o[n][2] *= al1;
        o[n][3] *= al1;
      }

      // ---- O += P V
      if constexpr (TR::k16) {
        const int mat = lane >> 3, rr = lane & 7;
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
          const uint32_t pa[4] = {pack16<T>(s[2 * kk][0], s[2 * kk][1]), pack16<T>(s[2 * kk][2], s[2 * kk][3]),
                                  pack16<T>(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                                  pack16<T>(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
          for (int n = 0; n < ND; n += 2) {
            uint32_t bv[4];
            ldsm_x4_t(bv, vb_a + (uint32_t)((kk * 16 + (mat & 1) * 8 + rr) * kRowB + (n + (mat >> 1)) * 8 * 2));
            mma_k16<TR::kBf>(o[n], pa, bv[0], bv[1]);
            if (n + 1 < ND) mma_k16<TR::kBf>(o[n + 1], pa, bv[2], bv[3]);
          }
        }
      } else {
        // A column t <-> key 2t and column t + 4 <-> key 2t + 1 of each 8-key step, so the S
        // accumulator layout is the A fragment as it stands; V's rows are taken in the same order.
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float pa[4] = {s[n][0], s[n][2], s[n][1], s[n][3]};
          const float* v0 = reinterpret_cast<const float*>(vb_s + (n * 8 + 2 * t4) * kRowB) + g;
          const float* v1 = reinterpret_cast<const float*>(vb_s + (n * 8 + 2 * t4 + 1) * kRowB) + g;
#pragma unroll
          for (int nd = 0; nd < ND; ++nd) mma_3xtf32(o[nd], pa, v0[nd * 8], v1[nd * 8]);
        }
      }
      __syncthreads();     // every warp is done with this buffer before the next copy reuses it
    }

    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const float vsc = kE4m3 ? __ldg(a.v_scale + it.h) : 1.0f;   // V codes were used unscaled
    if (it.whole()) {
      const float inv0 = l0 == 0.0f ? 0.0f : vsc / l0, inv1 = l1 == 0.0f ? 0.0f : vsc / l1;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int gr = hf ? gr1 : gr0;
        if (gr >= rw) continue;
        const int tok = gr / a.group, hd = it.h * a.group + (gr - tok * a.group);
        const int64_t orow = (int64_t)(it.r.q0 + tok) * a.hq + hd;
        if (a.lse && t4 == 0) a.lse[orow] = ((hf ? m1 : m0) + log2f(hf ? l1 : l0)) * kPgLn2;
        T* og = reinterpret_cast<T*>(a.out) + orow * D;
        const float inv = hf ? inv1 : inv0;
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const int col = n * 8 + 2 * t4;
          if (col >= D) continue;
          const float x = o[n][2 * hf] * inv, y = o[n][2 * hf + 1] * inv;
          if constexpr (TR::k16) *reinterpret_cast<uint32_t*>(og + col) = pack16<T>(x, y);
          else *reinterpret_cast<float2*>(og + col) = make_float2(x, y);
        }
      }
    } else {
      const int64_t slot = 2 * (int64_t)blockIdx.x + (it.j0 == 0 ? 1 : 0);
      if (it.j0 == 0 && tid == 0)
        a.cut[blockIdx.x] = make_int4(row0, it.b, it.h, pg_cta_of(at + it.n - 1, share.total, share.ctas));
      float* ml = a.part_ml + slot * 2 * kPpRows;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = r0 + g + 8 * hf;
        if (t4 == 0) {
          ml[r] = hf ? m1 : m0;
          ml[kPpRows + r] = hf ? l1 : l0;
        }
        float* po = a.part_o + (slot * kPpRows + r) * D;
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const int col = n * 8 + 2 * t4;
          if (col < D) *reinterpret_cast<float2*>(po + col) = make_float2(o[n][2 * hf] * vsc, o[n][2 * hf + 1] * vsc);
        }
      }
    }
    at += it.j1 - it.j0;
    // (the loop's last barrier has every warp past its reads of the query rows and buffers)
  }
}

// Joins the partial results of the items that were cut: block (c, y) serves the item that CTA c began
// and did not finish, one warp per query row, lanes over the head dimension, parts in unit order.
template <typename T>
__global__ void __launch_bounds__(256) paged_prefill_merge_kernel(const __grid_constant__ PagedArgs a, int rt) {
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x;
  const int4 cut = a.cut[c];
  if (cut.x < 0) return;
  PgRequest r;
  if (!pg_request(a, cut.y, r)) return;
  const int rows = min(rt, r.ql * a.group - cut.x);
  const int lane = threadIdx.x & 31, col = lane * 4;
  const int parts = cut.w - c + 1;
  for (int row = blockIdx.y * 8 + (threadIdx.x >> 5); row < rows; row += gridDim.y * 8) {
    auto slot = [&](int p) -> int64_t { return p == 0 ? 2 * (int64_t)c + 1 : 2 * (int64_t)(c + p); };
    float m = -INFINITY;
    for (int p = lane; p < parts; p += 32) m = fmaxf(m, a.part_ml[slot(p) * 2 * rt + row]);
    m = warp_max(m);
    const float mu = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      const int64_t s = slot(p);
      const float w = pg_ex2(a.part_ml[s * 2 * rt + row] - mu);
      l += w * a.part_ml[(s * 2 + 1) * rt + row];
      if (col < a.D) {
        const float4 x = *reinterpret_cast<const float4*>(a.part_o + (s * rt + row) * a.D + col);
        o.x += w * x.x;
        o.y += w * x.y;
        o.z += w * x.z;
        o.w += w * x.w;
      }
    }
    const int gr = cut.x + row, tok = gr / a.group, hd = cut.z * a.group + (gr - tok * a.group);
    const int64_t orow = (int64_t)(r.q0 + tok) * a.hq + hd;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (a.lse && lane == 0) a.lse[orow] = (m + log2f(l)) * kPgLn2;
    if (col < a.D) {
      T* p = reinterpret_cast<T*>(a.out) + orow * a.D + col;
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      } else {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack16<T>(o.x * inv, o.y * inv), pack16<T>(o.z * inv, o.w * inv));
      }
    }
  }
}

template <typename T, bool kE4m3, int DP>
int launch_paged(const PagedArgs& a, int grid, cudaStream_t st) {
  constexpr int BK = PfTraits<T>::kBK;
  constexpr size_t smem = (size_t)(kPpRows + 4 * BK) * (DP * sizeof(T) + 16);
  auto kern = paged_prefill_kernel<T, kE4m3, DP>;
  // every call: the attribute belongs to the current device's copy of the kernel
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) e = launch_pdl(kern, dim3((unsigned)grid), dim3(kPpThreads), smem, st, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(KVB_E_LAUNCH, "paged_prefill_kernel: %s", cudaGetErrorString(e));
  }
  return check_launch("paged_prefill_kernel");
}

template <typename T, bool kE4m3>
int dispatch_paged(const PagedArgs& a, int grid, cudaStream_t st) {
  if (a.D <= 32) return launch_paged<T, kE4m3, 32>(a, grid, st);
  if (a.D <= 64) return launch_paged<T, kE4m3, 64>(a, grid, st);
  if (a.D <= 96) return launch_paged<T, kE4m3, 96>(a, grid, st);
  return launch_paged<T, kE4m3, 128>(a, grid, st);
}

}  // namespace

int pg_launch_merge(const PagedArgs& a, int dtype, int rt, int ctas, cudaStream_t st) {
  const dim3 grid((unsigned)ctas, (unsigned)(rt >= 64 ? rt / 32 : 1));
  cudaError_t e;
  if (dtype == KVB_BF16) e = launch_pdl(paged_prefill_merge_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, a, rt);
  else if (dtype == KVB_F16) e = launch_pdl(paged_prefill_merge_kernel<__half>, grid, dim3(256), 0, st, a, rt);
  else e = launch_pdl(paged_prefill_merge_kernel<float>, grid, dim3(256), 0, st, a, rt);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(KVB_E_LAUNCH, "paged_prefill_merge_kernel: %s", cudaGetErrorString(e));
  }
  return check_launch("paged_prefill_merge_kernel");
}

}  // namespace kvb

using namespace kvb;

namespace {
int paged_sms() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    sms = 148;
  }
  return sms < kPgMaxCtas / 2 ? sms : kPgMaxCtas / 2;
}
}  // namespace

extern "C" size_t kvb_paged_prefill_attention_workspace_size(int head_dim) {
  if (head_dim <= 0 || head_dim > 128) return 256;
  return std::max(pg_workspace_bytes(kPgMaxCtas, kPpRows, head_dim), pg_workspace_bytes(kPgMaxCtas / 2, 256, head_dim));
}

extern "C" int kvb_paged_prefill_attention_variant(const void* q, int q_dtype, int64_t q_token_stride,
                                                   const void* k_cache, const void* v_cache, int cache_dtype,
                                                   int64_t k_block_stride, int64_t v_block_stride, const float* k_scale,
                                                   const float* v_scale, const int32_t* qo_indptr, const void* seq_lens,
                                                   int seq_lens_dtype, const int32_t* block_table, int64_t bt_stride,
                                                   int batch, int64_t total_q, int num_q_heads, int num_kv_heads,
                                                   int head_dim, int block_size, int64_t num_blocks, int64_t max_seq_len,
                                                   float sm_scale, void* out, float* lse, int variant, void* workspace,
                                                   size_t workspace_bytes, void* stream) {
  if (variant < 0 || variant > 2) return set_error(KVB_E_ARG, "paged_prefill_attention: variant %d", variant);
  if (batch < 0 || total_q < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
      num_blocks < 0 || max_seq_len < 0 || bt_stride < 0)
    return set_error(KVB_E_ARG, "paged_prefill_attention: bad sizes");
  if (!is_float_dtype(q_dtype)) return set_error(KVB_E_DTYPE, "paged_prefill_attention: query dtype %d", q_dtype);
  if (cache_dtype != q_dtype && cache_dtype != KVB_E4M3)
    return set_error(KVB_E_DTYPE, "paged_prefill_attention: the cache holds the query type or e4m3 codes, not dtype %d", cache_dtype);
  if (seq_lens_dtype != KVB_I32 && seq_lens_dtype != KVB_I64) return set_error(KVB_E_DTYPE, "paged_prefill_attention: seq_lens dtype");
  if (num_q_heads % num_kv_heads) return set_error(KVB_E_SHAPE, "paged_prefill_attention: num_q_heads must be a multiple of num_kv_heads");
  if (head_dim % 8 || head_dim > 128)
    return set_error(KVB_E_SHAPE, "paged_prefill_attention: head_dim must be a multiple of 8, at most 128, not %d", head_dim);
  if (batch == 0 || total_q == 0) return KVB_OK;
  const int group = num_q_heads / num_kv_heads;
  if (max_seq_len > bt_stride * block_size)
    return set_error(KVB_E_SHAPE, "paged_prefill_attention: max_seq_len is more than the block table's rows hold");
  if (max_seq_len * group >= (1LL << 30) || total_q * group >= (1LL << 30) || total_q > INT32_MAX)
    return set_error(KVB_E_SHAPE, "paged_prefill_attention: tokens x heads of a KV head's group must stay below 2^30");
  if (!std::isfinite(sm_scale)) return set_error(KVB_E_ARG, "paged_prefill_attention: softmax scale is not finite");
  if (!q || !k_cache || !v_cache || !qo_indptr || !seq_lens || !block_table || !out ||
      (cache_dtype == KVB_E4M3 && (!k_scale || !v_scale)))
    return set_error(KVB_E_ARG, "paged_prefill_attention: null pointer");
  const int es = dtype_size(q_dtype), cs = cache_dtype == KVB_E4M3 ? 1 : es;
  const int64_t block = (int64_t)block_size * num_kv_heads * head_dim;
  if (num_blocks > 1 && (k_block_stride < block || v_block_stride < block))
    return set_error(KVB_E_SHAPE, "paged_prefill_attention: cache blocks overlap");
  const int64_t cal = cs == 1 ? 8 : 16;      // bytes a row of the cache starts on
  if (!aligned16(q) || (q_token_stride * es) % 16 || !aligned16(out) || (reinterpret_cast<uintptr_t>(k_cache) % cal) ||
      (reinterpret_cast<uintptr_t>(v_cache) % cal) || (k_block_stride * cs) % cal || (v_block_stride * cs) % cal)
    return set_error(KVB_E_ALIGN, "paged_prefill_attention: q, its token stride and out 16-byte, caches %d-byte alignment", (int)cal);
  PagedArgs a{};
  a.q = q; a.k_cache = k_cache; a.v_cache = v_cache; a.k_scale = k_scale; a.v_scale = v_scale; a.qo = qo_indptr;
  a.seq_lens = seq_lens; a.block_table = block_table; a.out = out; a.lse = lse; a.q_ts = q_token_stride;
  a.k_bs = k_block_stride; a.v_bs = v_block_stride; a.total_q = total_q; a.num_blocks = num_blocks;
  a.bt_stride = bt_stride; a.max_seq_len = max_seq_len; a.batch = batch; a.hq = num_q_heads; a.hkv = num_kv_heads;
  a.group = group; a.D = head_dim; a.bs = block_size; a.sl64 = seq_lens_dtype == KVB_I64;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  cudaStream_t st = as_stream(stream);
  const int sms = paged_sms();
  const int grid = 2 * sms;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
      workspace_bytes < kvb_paged_prefill_attention_workspace_size(head_dim))
    return set_error(KVB_E_WORKSPACE, "paged_prefill_attention: %zu bytes of workspace, 256-byte aligned, are needed",
                     kvb_paged_prefill_attention_workspace_size(head_dim));
  const bool tc = paged_prefill_tc_takes(a, q_dtype, cache_dtype);
  if (variant == 2 && !tc) return set_error(KVB_E_SHAPE, "paged_prefill_attention: no tcgen05 kernel for this case");
  if (tc && variant != 1) return paged_prefill_tcgen05(a, q_dtype, cache_dtype, workspace, sms, st);
  pg_workspace_layout(a, workspace, grid, kPpRows);
  int rc;
  const bool e4 = cache_dtype == KVB_E4M3;
  if (q_dtype == KVB_BF16) rc = e4 ? dispatch_paged<__nv_bfloat16, true>(a, grid, st) : dispatch_paged<__nv_bfloat16, false>(a, grid, st);
  else if (q_dtype == KVB_F16) rc = e4 ? dispatch_paged<__half, true>(a, grid, st) : dispatch_paged<__half, false>(a, grid, st);
  else rc = e4 ? dispatch_paged<float, true>(a, grid, st) : dispatch_paged<float, false>(a, grid, st);
  if (rc) return rc;
  return pg_launch_merge(a, q_dtype, kPpRows, grid, st);
}

extern "C" int kvb_paged_prefill_attention(const void* q, int q_dtype, int64_t q_token_stride,
                                           const void* k_cache, const void* v_cache, int cache_dtype,
                                           int64_t k_block_stride, int64_t v_block_stride, const float* k_scale,
                                           const float* v_scale, const int32_t* qo_indptr, const void* seq_lens,
                                           int seq_lens_dtype, const int32_t* block_table, int64_t bt_stride,
                                           int batch, int64_t total_q, int num_q_heads, int num_kv_heads,
                                           int head_dim, int block_size, int64_t num_blocks, int64_t max_seq_len,
                                           float sm_scale, void* out, float* lse, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  return kvb_paged_prefill_attention_variant(q, q_dtype, q_token_stride, k_cache, v_cache, cache_dtype, k_block_stride,
                                             v_block_stride, k_scale, v_scale, qo_indptr, seq_lens, seq_lens_dtype,
                                             block_table, bt_stride, batch, total_q, num_q_heads, num_kv_heads, head_dim,
                                             block_size, num_blocks, max_seq_len, sm_scale, out, lse, 0, workspace,
                                             workspace_bytes, stream);
}
