// Causal attention of chunks of new tokens over a paged KV cache on the 5th-generation tensor cores:
// 16-bit queries over a cache of their type or of e4m3 codes, head_dim a multiple of 16 in [64, 128].
// The contract and the mathematics are those of paged_prefill.cu.
//
// One persistent CTA per SM works through its share of (request, KV head, row tile) items
// (paged_prefill.cuh).  The query rows of a KV head's group are packed (row = token x group + head), so
// each key is read once for the whole group.  Two chains run side by side, each with 128 rows (TMEM
// lanes), four softmax warps, its O and two S buffers of 64 keys in tensor memory:
//   S_n = Q K_n^T -> buffer n % 2;  softmax: P_n over S_n;  O += P_n V_n
// with S_{n+1} computed while the softmax of S_n runs:
//   wide items (over 128 rows): chain A has rows 0..127 of the tile, chain B rows 128..255; each goes
//     through both 64-key halves of every K/V tile of 128 keys;
//   deep items (at most 128 rows: decoding, drafts, the last rows of a prompt): both chains have the same
//     rows, A takes the lower half of each K/V tile and B the upper one, and the two results are joined;
//   thin items (at most 16 rows over codes of head_dim 128: one decoded token's group, short drafts) go
//     past the chains: thin_item below.
// Roles: warp 0 issues the TMA loads (boxes of whole page runs gathered through the block table; over codes
// warp 0 those of K and warp 3 those of V); one
// lane each of warps 1 and 2 issues the MMAs of chain A and of chain B (one issuer for both was the
// limit: its 16 MMAs, four commits and four waits a tile took ~2900 cycles, against 1024 of tensor
// time); warp 3 zeroes page tails; warps 4-7 and 8-11 are the softmax groups of A and B; warps 12-15
// gather the query rows and turn e4m3 codes into float16 operands.
// K and V tiles share one ring of shared-memory slots in the order K_0 V_0 K_1 V_1 ...  A page outside
// the cache, and pages past the last token, are loaded from an out-of-range block coordinate, which
// TMA fills with zeros; the rows past the last token inside its page are zeroed in shared memory.
// e4m3: a row of Q is scaled by a power of two that brings its largest element to [1, 2), so float16
// holds it whatever bfloat16's range had; P is float16 too.
// What bounds it: for long chunks two things that have to overlap, the products (S at N = 64 takes 48 cycles
// where 32 would do) and the exponentials (512 cycles for the 128 x 64 scores that a chain's products take
// ~640 for): 2048 new tokens of 16384, 32 + 8 heads of 128, bf16: 530 us, 0.58 of the bf16 rate, tensor pipe
// 53 % and exponentials 59 % of the time.  4 x 512 of 4096 over codes: 185-190 us, those 33 % and 37 %: four
// warps convert every K and V tile in one order.  Decoding over 16-bit caches: HBM (64 sequences of 512 to
// 8192 tokens: 169 us, 5.2 TB/s).  At 128 registers a thread the kernels over codes spill (276 to 312 bytes
// stored), those over 16-bit caches 48.
// Every wait is bounded: by a time limit where one hand-over is waited for, by the limit since the last copy was
// issued where whole items are (a page tail at the end of a share, query rows behind few-row items); on a timeout the roles stop, the producer waits for its own copies,
// the MMA lanes for their MMAs, and the CTA frees its TMEM before exiting.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <cfloat>
#include <mutex>
#include <type_traits>

#include "kvb_common.cuh"
#include "kvb_async.cuh"
#include "mma_sync.cuh"
#include "paged_prefill.cuh"
#include "tcgen05.cuh"

namespace kvb {
namespace {

constexpr int kRows = 128;                 // rows of a chain (TMEM lanes)
constexpr int kKeys = 128;                 // keys per K/V tile
constexpr int kHalf = 64;                  // keys of an S buffer
constexpr int kTile = 2 * kRows;           // rows of a tile
constexpr int kThin = 16;                  // rows of a thin item at most
constexpr int kThreads = 512;
constexpr int kHelpers = 128;              // threads of warps 12-15

template <bool kE4m3, int DC> struct PcLayout {
  static constexpr uint32_t kOp = DC * kChunkBytes;                // one Q, K or V tile of 16-bit operands
  static constexpr uint32_t kRaw = kE4m3 ? kKeys * 64u * DC : 0u;  // one K or V tile of codes
  static constexpr uint32_t kBudget = 224 * 1024;
  static constexpr int kRawSlots = kE4m3 ? 4 : 0;
  static constexpr int kFit = (int)((kBudget - 2 * kOp - kRawSlots * kRaw) / kOp);
  static constexpr int kSlots = kFit < 8 ? kFit : 8;
  static constexpr uint32_t kQ0 = 0, kKv0 = 2 * kOp, kRaw0 = kKv0 + kSlots * kOp;
  static constexpr bool kThinItems = kE4m3 && DC == 2;
  static constexpr size_t kSmem = kRaw0 + (size_t)kRawSlots * kRaw + 1024;
  static_assert(kSlots >= 3, "ring");
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  const uint16_t v = (uint16_t)two;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}

// A wait for the end of whole items, not of one hand-over: it gives up when warp 0 has issued no copy for the limit
// (whose own waits are for one hand-over each), however long the items in between take.
struct Patience {
  volatile uint32_t* copies;     // copies that warp 0 has issued
  volatile int* abort;
  uint64_t t0;
  uint32_t seen;
  __device__ __forceinline__ Patience(volatile uint32_t* c, volatile int* a) : copies(c), abort(a), t0(globaltimer_ns()), seen(*c) {}
  __device__ __forceinline__ bool over() {
    if (*abort) return true;
    const uint32_t now = *copies;
    const uint64_t t = globaltimer_ns();
    if (now != seen) {
      seen = now;
      t0 = t;
    } else if (t - t0 > *(volatile uint64_t*)&g_wait_limit_ns) {
      atomicOr(&g_tu_status, kStatusWaitTimeout);
      return true;
    }
    return false;
  }
};
// Like warp_wait.
__device__ __forceinline__ bool patient_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* copies, volatile int* abort) {
  bool ok = mbar_try_wait(bar, parity);
  if (!ok) {
    Patience p(copies, abort);
    for (uint32_t i = 1; !ok; ++i) {
      ok = mbar_try_wait(bar, parity);
      if (!ok && (i & 255u) == 0 && p.over()) break;
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// What every role derives from an item: key tiles [kt0, kt0 + T) of 128 keys, and the 64-key halves that
// each chain goes through.
struct PcItem {
  int row0;        // first row of the tile in its request
  int rows;        // rows of the tile
  bool wide, thin;
  int kt0, T;
  int TA;          // wide: how many of the tiles chain A uses
  int subs_a, subs_b;   // halves of each chain
  __host__ __device__ __forceinline__ PcItem(const PagedArgs& a, const PgItem& it, bool thin_items) {
    row0 = it.t * kTile;
    rows = min(kTile, it.r.ql * a.group - row0);
    wide = rows > kRows;
    thin = thin_items && rows <= kThin;
    kt0 = it.j0;
    T = it.j1 - it.j0;
    const int x0 = (it.r.kl - it.r.ql) * a.group + row0;        // position x group of the first row
    const int xb = x0 + rows - 1;
    const int seen = xb < 0 ? 0 : xb / a.group;                 // last key that the last row sees
    const bool low = it.j1 * kKeys - kHalf > seen;              // the upper half of the last tile: nobody sees it
    TA = T;
    if (wide) {
      const int xa = x0 + kRows - 1;
      const int seen_a = xa < 0 ? 0 : xa / a.group;
      TA = max(1, min(T, seen_a / kKeys + 1 - kt0));            // (a tile that it sees nothing of keeps the chains in step)
      subs_a = 2 * TA - ((kt0 + TA) * kKeys - kHalf > seen_a ? 1 : 0);
      subs_b = 2 * T - (low ? 1 : 0);
    } else {
      subs_a = T;
      subs_b = T - (low ? 1 : 0);
    }
  }
  __host__ __device__ __forceinline__ int subs(int c) const { return c ? subs_b : subs_a; }
  // tiles that the chain goes through: all, or all but the last
  __host__ __device__ __forceinline__ int tiles(int c) const { return wide ? (c ? T : TA) : subs(c); }
  // tile (of the item) and half of the chain's m-th half
  __device__ __forceinline__ int tile(int m) const { return wide ? m >> 1 : m; }
  __device__ __forceinline__ int half(int c, int m) const { return wide ? m & 1 : c; }
  // whether the chain is done with the tile after its m-th half
  __device__ __forceinline__ bool leaves(int c, int m) const { return !wide || (m & 1) || m + 1 == subs(c); }
};
// Rows of key tile kt past the last token that a box of the tile holds together with tokens.
__device__ __forceinline__ int tail_rows(int kl, int kt, int box) {
  const int end = kl - kt * kKeys, in = end & (box - 1);
  return end > 0 && end < kKeys && in ? box - in : 0;
}

// 8x8 16-bit elements transposed over the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// A thin item, by the eight warps of the softmax groups, each on its own from the ring's tiles as the copies bring
// them: 16 keys of each tile and all of up to 8 rows, or (over 8 rows) 32 keys and half of the rows.
//   S^T = K Q^T (16 keys x 8 rows),  O^T += V^T P^T (head_dim x 8 rows), products of 16 x 8 x 16 in registers:
// K and V are their A operands, straight from the tile (codes turned into float16 on the way: no operand tile is
// written), Q^T and P^T the B operands, and P^T is S^T's fragment transposed.  What a row needs of a head is one
// pass over the keys, so nothing but the bytes counts; the tcgen05 products take 128 rows and two hand-overs a
// tile for the same (a decoding step of 64 sequences of up to 8192 tokens: 226 us with them, 147 like this, 3.0 TB/s;
// 16-bit caches gained nothing, 197 and 201 us: there the bytes count either way).  What bounds it is latency: eight
// warps an SM carry the whole chain of loads, conversions and products (issue slots 29 % used, DRAM 36 %).
template <typename T, class Join>
__device__ __forceinline__ bool thin_item(const PagedArgs& a, const PgItem& it, const PcItem& g, uint8_t* smem, uint64_t* full,
                                          uint64_t* empty, uint32_t u, float* ml_s, Join& join) {
  using L = PcLayout<true, 2>;
  constexpr bool kOutBf = std::is_same<T, __nv_bfloat16>::value;
  constexpr float kUp = 7.0f, kGrow = 8.0f;
  constexpr int NF = L::kRawSlots, D = 128, KS = D / 16;      // KS: 16-element steps of head_dim
  const int tid = threadIdx.x - 128, w = tid >> 5, lane = tid & 31, gq = lane >> 2, t4 = lane & 3;
  const bool split = g.rows > 8;
  const int rb = split ? (w >> 2) * 8 : 0;                   // the warp's first row
  const int kf = split ? (w & 3) * 32 : w * 16, nb = split ? 2 : 1;   // its first key of a tile, blocks of 16
  // Q^T: this lane has row rb + gq, 16 elements from 16 t4 and from 16 (t4 + 4), four a step (the order of the codes of
  // K that the lane reads at once), scaled like the chains' rows
  uint32_t q[KS][2];
  float sc = a.scale_log2;
  {
    const int r = rb + gq, x = g.row0 + r, tok = x / a.group;
    const bool in = r < g.rows;
    const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(it.r.q0 + tok) * a.q_ts + ((int64_t)it.h * a.group + (x - tok * a.group)) * D;
    float mx = 0.0f;
    Vec8<T> v[KS / 2];
#pragma unroll
    for (int j = 0; j < KS / 2; ++j) {
      v[j].w[0] = make_uint4(0u, 0u, 0u, 0u);
      if (in) v[j].load(src + (t4 + 4 * (j >> 1)) * 16 + (j & 1) * 8);
      float f[8];
      v[j].unpack(f);
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(f[e]));
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const int e2 = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 120);
    const float up = __int_as_float((127 - e2) << 23);
#pragma unroll
    for (int j = 0; j < KS / 2; ++j) {
      float f[8];
      v[j].unpack(f);
#pragma unroll
      for (int e = 0; e < 4; ++e) q[2 * j + (e >> 1)][e & 1] = pack2h<false>(f[2 * e] * up, f[2 * e + 1] * up);
    }
    sc *= __ldg(a.k_scale + it.h) * __int_as_float((127 + e2) << 23);
  }
  if (sc == 0.0f) sc = 1e-30f;                               // equal weights
  // rows of this lane's elements of S^T, P^T and O^T: rb + 2 t4 and the next one
  const float sc0 = __shfl_sync(0xffffffffu, sc, t4 * 8), sc1 = __shfl_sync(0xffffffffu, sc, t4 * 8 + 4);
  const int off = it.r.kl - it.r.ql;
  const int pos0 = min(off + (g.row0 + rb + 2 * t4) / a.group, it.r.kl - 1), pos1 = min(off + (g.row0 + rb + 2 * t4 + 1) / a.group, it.r.kl - 1);
  const int pos_min = off + (g.row0 + rb) / a.group;
  // The key of this lane's row of S^T, of a block of 16 (and 8 on): in the order 0 4 1 5 2 6 3 7, and the units of V in
  // the same one, so that the eight lanes of a 16-byte access meet eight units of the swizzled rows.
  const int kq = (gq >> 1) + (gq & 1) * 4;
  float o[KS][4];
#pragma unroll
  for (int j = 0; j < KS; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
  float m0 = -FLT_MAX, m1 = -FLT_MAX, l0 = 0.0f, l1 = 0.0f;  // (-FLT_MAX: nothing seen)
  bool ok = true;
#pragma unroll 1
  for (int i = 0; i < g.T; ++i, u += 2) {
    const int kb = (g.kt0 + i) * kKeys + kf;                 // the warp's first key
    float x[2][4];                                           // keys kq, kq + 8 of a block, rows 2 t4, 2 t4 + 1
    {
      const uint32_t s = u % NF;
      if (!warp_wait(&full[s], (u / NF) & 1)) {
        ok = false;
        break;
      }
      const uint8_t* const tile = smem + L::kRaw0 + s * L::kRaw;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[n][e] = 0.0f;
        if (n >= nb) continue;
        const int k0 = kf + n * 16;
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};               // (two sums: half the chain)
        uint32_t lo[KS], hi[KS];                       // keys kq and kq + 8: the lane's 16-byte units t4 and t4 + 4
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t at = (k0 + kq) * 128 + (((t4 + 4 * j) ^ kq) << 4);
          *reinterpret_cast<uint4*>(lo + 4 * j) = *reinterpret_cast<const uint4*>(tile + at);
          *reinterpret_cast<uint4*>(hi + 4 * j) = *reinterpret_cast<const uint4*>(tile + at + 8 * 128);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint32_t f[4] = {e4m3x2_to_f16x2(lo[ks]), e4m3x2_to_f16x2(hi[ks]), e4m3x2_to_f16x2(lo[ks] >> 16),
                                 e4m3x2_to_f16x2(hi[ks] >> 16)};
          if (ks & 1) mma_k16<false>(y, f, q[ks][0], q[ks][1]);
          else mma_k16<false>(x[n], f, q[ks][0], q[ks][1]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[n][e] = (x[n][e] + y[e]) * (e & 1 ? sc1 : sc0);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
    if (kb + 16 * nb - 1 > pos_min) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (kb + n * 16 + kq + (e >> 1) * 8 > (e & 1 ? pos1 : pos0)) x[n][e] = -INFINITY;
    }
    float b0 = fmaxf(x[0][0], x[0][2]), b1 = fmaxf(x[0][1], x[0][3]);
    if (split) {
      b0 = fmaxf(b0, fmaxf(x[1][0], x[1][2]));
      b1 = fmaxf(b1, fmaxf(x[1][1], x[1][3]));
    }
    // the maxima only move when a score is above one by more than 2^8
    if (__any_sync(0xffffffffu, b0 - kUp > m0 + kGrow || b1 - kUp > m1 + kGrow)) {
#pragma unroll
      for (int k = 4; k <= 16; k <<= 1) {
        b0 = fmaxf(b0, __shfl_xor_sync(0xffffffffu, b0, k));
        b1 = fmaxf(b1, __shfl_xor_sync(0xffffffffu, b1, k));
      }
      const float n0 = b0 - kUp > m0 + kGrow ? b0 - kUp : m0, n1 = b1 - kUp > m1 + kGrow ? b1 - kUp : m1;
      const float f0 = ex2_approx(m0 - n0), f1 = ex2_approx(m1 - n1);
      m0 = n0;
      m1 = n1;
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        o[j][0] *= f0;
        o[j][1] *= f1;
        o[j][2] *= f0;
        o[j][3] *= f1;
      }
    }
    uint32_t p[2][2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (n >= nb) continue;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float p0 = ex2_approx(x[n][2 * e] - m0), p1 = ex2_approx(x[n][2 * e + 1] - m1);
        l0 += p0;
        l1 += p1;
        p[n][e] = transpose8(pack2h<false>(p0, p1));
      }
    }
    const uint32_t s = (u + 1) % NF;
    if (!warp_wait(&full[s], ((u + 1) / NF) & 1)) {
      ok = false;
      break;
    }
    const uint8_t* const tile = smem + L::kRaw0 + s * L::kRaw;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (n >= nb) continue;
      const int k0 = kf + n * 16;
      // V^T: unit kq of keys t4, t4 + 4, t4 + 8 and t4 + 12 (P's 2 t4, 2 t4 + 1 and + 8, + 9); two elements a step
      uint32_t v[4][4];
      const int end = it.r.kl - (g.kt0 + i) * kKeys;       // rows from here on are past the last token: zeros
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = k0 + t4 + 4 * e;
        uint4 y = *reinterpret_cast<const uint4*>(tile + r * 128 + (((kq ^ r) & 7) << 4));
        if (end < kKeys && r >= end) y = make_uint4(0u, 0u, 0u, 0u);
        v[e][0] = y.x;
        v[e][1] = y.y;
        v[e][2] = y.z;
        v[e][3] = y.w;
      }
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const uint32_t lo = __byte_perm(v[0][j >> 1], v[1][j >> 1], j & 1 ? 0x7362 : 0x5140);
        const uint32_t hi = __byte_perm(v[2][j >> 1], v[3][j >> 1], j & 1 ? 0x7362 : 0x5140);
        const uint32_t f[4] = {e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi), e4m3x2_to_f16x2(hi >> 16)};
        mma_k16<false>(o[j], f, p[n][0], p[n][1]);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
  }
  // The warps' results are joined through the second Q tile: O^T as [warp][8 rows][D] with the 16-byte units of a
  // row exchanged by its number.
#pragma unroll
  for (int k = 4; k <= 16; k <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, k);
    l1 += __shfl_xor_sync(0xffffffffu, l1, k);
  }
  ok = join() && ok;                                         // whoever used that tile before is through
  float* const xo = reinterpret_cast<float*>(smem + L::kQ0 + L::kOp);
  if (gq == 0) {
    *reinterpret_cast<float4*>(ml_s + (w * 8 + 2 * t4) * 2) = make_float4(m0, l0, m1, l1);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float* const xr = xo + (w * 8 + 2 * t4 + e) * D;
#pragma unroll
    for (int j = 0; j < KS; j += 2)
      *reinterpret_cast<float4*>(xr + (((kq * 4 + (j >> 1)) ^ t4) << 2)) = make_float4(o[j][e], o[j][e + 2], o[j + 1][e], o[j + 1][e + 2]);
  }
  ok = join() && ok;
  const bool whole = it.whole();
  const float vsc = __ldg(a.v_scale + it.h);
  const int64_t slot = 2 * (int64_t)blockIdx.x + (it.j0 == 0 ? 1 : 0);
  for (int x = tid; ok && x < g.rows * (D / 4); x += 256) {
    const int r = x / (D / 4), d4 = x % (D / 4), w0 = split ? (r >> 3) * 4 : 0, wn = split ? 4 : 8;
    float mj = -FLT_MAX, lj = 0.0f;
    for (int k = 0; k < wn; ++k) mj = fmaxf(mj, ml_s[((w0 + k) * 8 + (r & 7)) * 2]);
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int k = 0; k < wn; ++k) {
      const float2 ml = *reinterpret_cast<const float2*>(ml_s + ((w0 + k) * 8 + (r & 7)) * 2);
      const float4 v = *reinterpret_cast<const float4*>(xo + ((w0 + k) * 8 + (r & 7)) * D + ((d4 ^ ((r >> 1) & 3)) << 2));
      const float f = ex2_approx(ml.x - mj);
      lj += ml.y * f;
      y.x += v.x * f;
      y.y += v.y * f;
      y.z += v.z * f;
      y.w += v.w * f;
    }
    const float fin = whole ? (lj == 0.0f ? 0.0f : vsc / lj) : vsc;
    y = make_float4(y.x * fin, y.y * fin, y.z * fin, y.w * fin);
    if (whole) {
      const int x0 = g.row0 + r, tok = x0 / a.group;
      const int64_t orow = (int64_t)(it.r.q0 + tok) * a.hq + (int64_t)it.h * a.group + (x0 - tok * a.group);
      *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + orow * D + d4 * 4) = make_uint2(pack2h<kOutBf>(y.x, y.y), pack2h<kOutBf>(y.z, y.w));
      if (a.lse && d4 == 0) a.lse[orow] = (mj + log2f(lj)) * kPgLn2;
    } else {
      *reinterpret_cast<float4*>(a.part_o + (slot * kTile + r) * D + d4 * 4) = y;
      if (d4 == 0) {
        a.part_ml[slot * 2 * kTile + r] = mj == -FLT_MAX ? -INFINITY : mj;
        a.part_ml[slot * 2 * kTile + kTile + r] = lj;
      }
    }
  }
  return join() && ok;                                       // before the next item's results overwrite these
}

template <typename T, bool kE4m3, int DC>
__global__ void __launch_bounds__(kThreads, 1) paged_prefill_tc_kernel(const __grid_constant__ CUtensorMap tk,
                                                                       const __grid_constant__ CUtensorMap tv,
                                                                       const __grid_constant__ PagedArgs a, const int box) {
  using L = PcLayout<kE4m3, DC>;
  constexpr bool kBf = !kE4m3 && std::is_same<T, __nv_bfloat16>::value;   // type of the operands
  // float16 has few exponents: P is held 2^7 larger there when the maximum moves, up to 2^15.
  constexpr float kUp = kBf ? 0.0f : 7.0f, kGrow = 8.0f;
  constexpr int NS = L::kSlots, NR = L::kRawSlots;
  constexpr uint32_t kTmemCols = 512;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  __shared__ uint64_t kv_full[NS], kv_empty[NS], tail_full[kE4m3 ? 1 : NS],
      raw_full[kE4m3 ? NR : 1], raw_empty[kE4m3 ? NR : 1], thin_empty[kE4m3 ? NR : 1],
      q_full, q_empty, s_full[4], p_full[4], pv_done[4], mma_done[2], joined,   // s, p, pv: [2 * chain + buffer]
      sc_full[kE4m3 ? 2 : 1], q_seen[kE4m3 ? 2 : 1];   // an item's row scales are there, have been read: by item parity
  __shared__ uint32_t tmem_base_s;
  __shared__ volatile int s_abort;
  __shared__ volatile uint32_t s_copies;         // copies that warp 0 has issued
  __shared__ volatile uint32_t thin_done;        // thin items whose results are joined
  __shared__ PgShare share;
  __shared__ int64_t scan[kThreads / 32];
  __shared__ __align__(16) float join_s[2][kRows];             // [chain][row]: maxima, then sums, at the end of a deep item
  __shared__ int8_t qexp_s[2][kE4m3 ? kTile : 1];   // e of a row's Q scale 2^-e, by item parity

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const PgTiles tiles{kTile, kKeys, a.group};
  // codes: rows of 128, so that the raw tiles have the 128-byte swizzle (make_page_map)
  const bool thin_items = L::kThinItems && a.D == 128;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&kv_full[s], kE4m3 ? 4 : 1);
      mbar_init(&kv_empty[s], 2);            // one arrival for each chain
      if constexpr (!kE4m3) mbar_init(&tail_full[s], 1);
    }
    for (int s = 0; s < NR; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], 4);
    }
    for (int s = 0; s < NR; ++s) mbar_init(&thin_empty[s], 8);
    mbar_init(&q_full, 4);
    mbar_init(&q_empty, 2);
    for (int c = 0; c < 4; ++c) {
      mbar_init(&s_full[c], 1);
      mbar_init(&p_full[c], 4);
      mbar_init(&pv_done[c], 1);
    }
    mbar_init(&mma_done[0], 1);
    mbar_init(&mma_done[1], 1);
    mbar_init(&joined, 8);
    for (int x = 0; x < (kE4m3 ? 2 : 1); ++x) {
      mbar_init(&sc_full[x], 4);
      mbar_init(&q_seen[x], 8);
    }
    s_abort = 0;
    s_copies = 0;
    thin_done = 0;
    fence_mbar_init();
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tv) : "memory");
  }
  pdl_trigger();
  pdl_wait();            // launched as a programmatic dependent: global data from here on
  pg_share<kThreads>(a, tiles, blockIdx.x, gridDim.x, &share, scan, &g_tu_status);
  if (threadIdx.x == 128) a.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);      // (first thread of softmax group A)
  if (share.left == 0) return;
  const int D = a.D;

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  PgWalk walk(share);
  PgItem it;

  if (warp == 0 || (kE4m3 && warp == 3)) {
    // ---------------------------------------------------------------- TMA producer
    // A tile is kKeys / box boxes of `box` keys, each inside one page; lane l serves box l % boxes.
    const int boxes = kKeys / box;
    const int bx = lane & (boxes - 1);
    constexpr int NF = kE4m3 ? NR : NS;                        // ring the copies go to
    uint64_t* const full = kE4m3 ? raw_full : kv_full;
    uint64_t* const empty = kE4m3 ? raw_empty : kv_empty;
    constexpr uint32_t kSlotBytes = kE4m3 ? L::kRaw : L::kOp;
    const uint32_t bytes = kE4m3 ? (uint32_t)(kKeys * D) : kSlotBytes;
    uint32_t u = 0;                                            // copies so far = tiles of the ring used
    uint32_t by_thin = 0, e_par = 0, t_par = 0;                // codes, by slot: whose release to wait for, and its parity
    bool ok = true;
    while (ok && walk.next(a, tiles, it)) {
      const PcItem g(a, it, thin_items);
      const int32_t* bt = a.block_table + (int64_t)it.b * a.bt_stride;
      auto page_of = [&](int kt, int& in) -> int {             // block and row of this lane's box of tile kt
        const int key = kt * kKeys + bx * box;
        in = 0;
        if (key >= it.r.kl) return (int)a.num_blocks;          // past the last token: zeros
        const int blk = key / a.bs;
        in = key - blk * a.bs;
        const int phys = __ldg(bt + blk);
        if (phys < 0 || phys >= a.num_blocks) {
          atomicOr(&g_tu_status, kStatusBadPage);
          return (int)a.num_blocks;
        }
        return phys;
      };
      int in, phys = page_of(g.kt0, in);
      for (int i = 0; i < g.T && ok; ++i) {
        int in_next = 0, phys_next = 0;
        if (i + 1 < g.T) phys_next = page_of(g.kt0 + i + 1, in_next);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++u) {
          if (kE4m3 && kv != (warp == 3)) continue;            // codes: K by warp 0, V by warp 3
          const uint32_t s = u % NF;
          if constexpr (L::kThinItems) {
            const uint32_t bit = 1u << s;
            const bool by = by_thin & bit;
            if (u >= NF) {
              if (!warp_wait(by ? &thin_empty[s] : &empty[s], ((by ? t_par : e_par) >> s) & 1)) s_abort = 1;
              (by ? t_par : e_par) ^= bit;
            }
            by_thin = g.thin ? by_thin | bit : by_thin & ~bit;
          } else {
            if (u >= NF && !warp_wait(&empty[s], ((u / NF) & 1) ^ 1)) s_abort = 1;
          }
          if (__any_sync(0xffffffffu, s_abort)) {
            ok = false;
            break;
          }
          const CUtensorMap* map = kv ? &tv : &tk;
          uint64_t* bar = &full[s];
          // a V tile whose last page has rows past the last token goes through warp 3
          if constexpr (!kE4m3)
            if (kv && tail_rows(it.r.kl, g.kt0 + i, box) > 0) bar = &tail_full[s];
          if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
          if (lane == 0 && warp == 0) s_copies = u + 1;
          __syncwarp();
          // box by box in converged code (issued by the lanes of the boxes instead, each took ~105 cycles)
          for (int x = 0; x < boxes; ++x) {
            const int p = __shfl_sync(0xffffffffu, phys, x), r = __shfl_sync(0xffffffffu, in, x);
            if (elect_one()) {
              if constexpr (kE4m3) {
                const uint32_t pitch = ((uint32_t)(box * D) + 127u) & ~127u;
                tma_load_4d(sbase + L::kRaw0 + s * L::kRaw + x * pitch, map, 0, it.h, r, p, bar);
              } else {
#pragma unroll
                for (int c = 0; c < DC; ++c)
                  tma_load_4d(sbase + L::kKv0 + s * L::kOp + c * kChunkBytes + x * box * 128, map, c * 64, it.h, r, p, bar);
              }
            }
            __syncwarp();
          }
        }
        phys = phys_next;
        in = in_next;
      }
    }
    // every copy this CTA issued has landed before it exits (tails: warp 3 has seen theirs)
    for (uint32_t v = u > NF ? u - NF : 0; v < u; ++v)
      if (!kE4m3 || (v & 1) == (warp == 3)) mbar_wait_bounded(&full[v % NF], (v / NF) & 1);
  } else if (warp <= 2) {
    // ---------------------------------------------------------------- MMA issuers: warp 1 + c, chain c
    {
      const int c = warp - 1;
      const uint32_t tb = tmem + (uint32_t)c * 256u;
      constexpr uint32_t kIdS = idesc_f16(kRows, kHalf, kBf, false);
      const uint32_t id_pv = idesc_f16(kRows, D, kBf, true);
      uint32_t u0 = 0, item = 0;                               // ring position of the item's first tile
      uint32_t n = 0;                                          // halves of the chain whose S has been issued, all items
      bool ok = true;
      while (ok && walk.next(a, tiles, it)) {
        const PcItem g(a, it, thin_items);
        if (g.thin) continue;                                  // (the warps of the softmax groups do it all)
        const int subs = g.subs(c);
        const uint64_t qd = desc_kmajor(sbase + L::kQ0 + (g.wide ? c : 0) * L::kOp);
        auto issue_s = [&](int m) -> bool {
          const uint32_t v = u0 + 2 * g.tile(m), s = v % NS, b = n & 1;
          if (!warp_wait(&kv_full[s], (v / NS) & 1)) return false;
          if (n > 1 && !warp_wait(&pv_done[2 * c + b], ((n >> 1) - 1) & 1)) return false;   // the P it overwrites is used up
          tc_fence_after();
          const uint64_t kd = desc_kmajor(sbase + L::kKv0 + s * L::kOp) + g.half(c, m) * (kHalf * 128 >> 4);
          const bool leaves = g.leaves(c, m), last = m + 1 == subs;
          if (elect_one()) {
            // 16 elements = 32 bytes on in both operands, 64 elements one chunk on
            if (D == 64 * DC) {
#pragma unroll
              for (int ks = 0; ks < 4 * DC; ++ks)
                mma_f16(tb + b * kHalf, qd + (ks >> 2) * (kChunkBytes >> 4) + (ks & 3) * 2,
                        kd + (ks >> 2) * (kChunkBytes >> 4) + (ks & 3) * 2, kIdS, ks > 0);
            } else {
              for (int ks = 0; ks < D / 16; ++ks)
                mma_f16(tb + b * kHalf, qd + (ks >> 2) * (kChunkBytes >> 4) + (ks & 3) * 2,
                        kd + (ks >> 2) * (kChunkBytes >> 4) + (ks & 3) * 2, kIdS, ks > 0);
            }
            mma_commit(&s_full[2 * c + b]);
            if (leaves) mma_commit(&kv_empty[s]);
            if (last) mma_commit(&q_empty);
          }
          __syncwarp();
          ++n;
          return true;
        };
        ok = patient_wait(&q_full, item & 1, &s_copies, &s_abort);
        ++item;
        if (subs == 0 && ok && lane == 0) mbar_arrive(&q_empty);
        const uint32_t n0 = n;
        if (subs > 0) ok = ok && issue_s(0);
        if (subs > 1) ok = ok && issue_s(1);
        for (int m = 0; m < subs && ok; ++m) {
          const uint32_t v = u0 + 2 * g.tile(m) + 1, s = v % NS, b = (n0 + m) & 1;
          ok = warp_wait(&kv_full[s], (v / NS) & 1) && warp_wait(&p_full[2 * c + b], ((n0 + m) >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          // 16 keys: 8 packed columns of P, 16 rows of V
          const uint64_t vd = desc_mnmajor(sbase + L::kKv0 + s * L::kOp, kChunkBytes) + g.half(c, m) * (kHalf * 128 >> 4);
          const bool leaves = g.leaves(c, m);
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < kHalf / 16; ++ks)
              mma_f16_ts(tb + 128u, tb + b * kHalf + (uint32_t)ks * 8u, vd + ks * 128, id_pv, (m | ks) != 0);
            mma_commit(&pv_done[2 * c + b]);
            if (leaves) mma_commit(&kv_empty[s]);
          }
          __syncwarp();
          if (m + 2 < subs) ok = issue_s(m + 2);
        }
        // A tile that only the other chain goes through: seen and passed on all the same.  A wait cannot tell a phase
        // from the one two before, so this warp sees every phase of every slot, and the slot is not filled again before.
        for (int v = 2 * g.tiles(c); v < 2 * g.T && ok; ++v) {
          const uint32_t s = (u0 + v) % NS;
          ok = warp_wait(&kv_full[s], ((u0 + v) / NS) & 1);
          if (ok && lane == 0) mbar_arrive(&kv_empty[s]);
        }
        u0 += 2 * g.T;
        if (__any_sync(0xffffffffu, s_abort)) ok = false;
      }
      if (!ok) s_abort = 1;
      if (elect_one()) mma_commit(&mma_done[c]);              // every MMA issued above has completed before TMEM is freed
      warp_wait(&mma_done[c], 0);
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------------- page tails (16-bit caches)
    // The rows of a V tile past the last token inside its page: zeroed (the weights there are zero, and what the
    // page holds may not be a number), then the tile is passed on.
    if constexpr (!kE4m3) {
      uint32_t u = 0, seen = 0;                                // parity of each slot's tail barrier
      bool ok = true;
      while (ok && walk.next(a, tiles, it)) {
        const PcItem g(a, it, thin_items);
        const int i = it.r.kl / kKeys - g.kt0;                 // the tile with the first row past the last token
        const int rows = i >= 0 && i < g.T ? tail_rows(it.r.kl, g.kt0 + i, box) : 0;
        if (rows > 0) {
          const uint32_t s = (u + 2 * i + 1) % NS;
          if (!patient_wait(&tail_full[s], (seen >> s) & 1, &s_copies, &s_abort)) s_abort = 1;
          seen ^= 1u << s;
          const int end = it.r.kl & (kKeys - 1);
          for (int x = lane; x < rows * 8 * DC; x += 32) {
            const int r = end + x / (8 * DC), q = x % (8 * DC);
            *reinterpret_cast<uint4*>(smem + L::kKv0 + s * L::kOp + (q >> 3) * kChunkBytes + r * 128 + (q & 7) * 16) =
                make_uint4(0u, 0u, 0u, 0u);
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&kv_full[s]);
        }
        u += 2 * g.T;
        if (__any_sync(0xffffffffu, s_abort)) ok = false;
      }
    }
  } else if (warp >= 12) {
    // ---------------------------------------------------------------- helpers: query rows, e4m3 codes to float16
    const int ht = threadIdx.x - 384;                                     // 0 .. 127
    uint32_t u = 0, ur = 0, item = 0, thin = 0;                           // positions in the operand ring and in the raw one
    bool ok = true;
    while (ok && walk.next(a, tiles, it)) {
      const PcItem g(a, it, thin_items);
      if (g.thin) {
        ur += 2 * g.T;
        ++thin;
        continue;
      }
      // The thin items before this one are through: they join their results in the second Q tile, and the raw ring's
      // barriers went on without this warp (a wait cannot tell a phase from the second next).
      if constexpr (L::kThinItems) {
        Patience p(&s_copies, &s_abort);
        while (__any_sync(0xffffffffu, thin_done != thin))
          if (__any_sync(0xffffffffu, p.over())) {
            s_abort = 1;
            break;
          }
        __threadfence_block();
      }
      if (item > 0 && !patient_wait(&q_empty, (item - 1) & 1, &s_copies, &s_abort)) s_abort = 1;
      // S of a short item, and so q_empty, may be done while the softmax still is an item or two back: its row scales
      // stay until it has read them (and have barriers of their own by item parity: a warp that is late cannot tell
      // phase k of one barrier from phase k + 2)
      if constexpr (kE4m3)
        if (item > 1 && !warp_wait(&q_seen[item & 1], ((item >> 1) - 1) & 1)) s_abort = 1;
      if (__any_sync(0xffffffffu, s_abort)) break;
      {
        // Sixteen lanes (eight for D <= 64) take a row: eight elements each, whole rows coalesced.
        constexpr int LPR = 8 * DC;
        const int nrows = g.wide ? kTile : kRows;
        const int q8 = ht % LPR;
        const T* qg = reinterpret_cast<const T*>(a.q) + (int64_t)it.r.q0 * a.q_ts + (int64_t)it.h * a.group * D + q8 * 8;
        const uint32_t dst0 = sbase + L::kQ0 + (q8 >> 3) * kChunkBytes;
        constexpr int RPI = kHelpers / LPR;                                 // rows per pass
        if constexpr (!kE4m3) {
          for (int r = ht / LPR; r < nrows; r += RPI) {
            const int gr = g.row0 + r;
            const bool in = r < g.rows && q8 * 8 < D;
            const int tok = in ? gr / a.group : 0;
            const T* src = in ? qg + (int64_t)tok * a.q_ts + (gr - tok * a.group) * D
                              : reinterpret_cast<const T*>(a.q);
            const uint32_t dst = dst0 + (r >> 7) * L::kOp + (r & 127) * 128 + (((q8 & 7) ^ (r & 7)) << 4);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
          }
          asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
        } else {
          constexpr int U = 4;                                              // rows in flight per thread
          for (int rb = ht / LPR; rb < nrows; rb += U * RPI) {
            Vec8<T> x[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
              const int r = rb + i * RPI, gr = g.row0 + r;
              x[i].w[0] = make_uint4(0u, 0u, 0u, 0u);
              if (r < g.rows && q8 * 8 < D) {
                const int tok = gr / a.group;
                x[i].load(qg + (int64_t)tok * a.q_ts + (gr - tok * a.group) * D);
              }
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
              const int r = rb + i * RPI;
              float f[8];
              x[i].unpack(f);
              float mx = 0.0f;
#pragma unroll
              for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(f[e]));
#pragma unroll
              for (int o = LPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
              // e: the exponent of the row's largest element, within what 2^e and 2^-e have
              const int e2 = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 120);
              const float up = __int_as_float((127 - e2) << 23);
              Vec8<__half> h;
#pragma unroll
              for (int e = 0; e < 8; ++e) f[e] *= up;
              h.pack(f);
              *reinterpret_cast<uint4*>(smem + (dst0 - sbase) + (r >> 7) * L::kOp + (r & 127) * 128 +
                                        (((q8 & 7) ^ (r & 7)) << 4)) = h.w[0];
              if (q8 == 0) qexp_s[item & 1][r] = (int8_t)e2;
            }
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          if constexpr (kE4m3) mbar_arrive(&sc_full[item & 1]);
          mbar_arrive(&q_full);
        }
        ++item;
      }
      if constexpr (kE4m3) {
        const uint32_t pitch = ((uint32_t)(box * D) + 127u) & ~127u;
        const int lbox = __ffs(box) - 1;
        for (int i = 0; i < 2 * g.T && ok; ++i, ++u, ++ur) {
          const uint32_t sr = ur % NR, s = u % NS;
          if (!warp_wait(&raw_full[sr], (ur / NR) & 1)) s_abort = 1;
          if (u >= NS && !warp_wait(&kv_empty[s], ((u / NS) & 1) ^ 1)) s_abort = 1;
          if (__any_sync(0xffffffffu, s_abort)) {
            ok = false;
            break;
          }
          const uint8_t* raw = smem + L::kRaw0 + sr * L::kRaw;
          uint8_t* dst = smem + L::kKv0 + s * L::kOp;
          const int end = it.r.kl - (g.kt0 + (i >> 1)) * kKeys;  // rows from here on are past the last token
          // Thread: eight codes, one 16-byte unit of the operand, of rows r0, r0 + step, ...: a quarter-warp's
          // stores cover a row's eight units, and the swizzle (r & 7) is the thread's own.
          constexpr int UPR = 8 * DC, step = kHelpers / UPR;      // units a row, rows a pass (a multiple of 8)
          const int q = ht % UPR, r0 = ht / UPR;
          const int qb = D == 128 ? ((((q >> 1) ^ r0) & 7) << 4) + (q & 1) * 8 : q * 8;   // of the unit in its row of codes
          uint8_t* const d0 = dst + (q >> 3) * kChunkBytes + r0 * 128 + (((q & 7) ^ (r0 & 7)) << 4);
          auto put = [&](uint8_t* d, uint2 x) {
            *reinterpret_cast<uint4*>(d) =
                make_uint4(e4m3x2_to_f16x2(x.x), e4m3x2_to_f16x2(x.x >> 16), e4m3x2_to_f16x2(x.y), e4m3x2_to_f16x2(x.y >> 16));
          };
          if (D == 64 * DC && end >= kKeys) {                     // whole tiles of whole chunks: rows one after another
            const uint8_t* const r8 = raw + r0 * (64 * DC) + qb;
#pragma unroll
            for (int k = 0; k < kKeys / step; k += 8) {
              uint2 x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = *reinterpret_cast<const uint2*>(r8 + (k + e) * step * 64 * DC);
#pragma unroll
              for (int e = 0; e < 8; ++e) put(d0 + (k + e) * step * 128, x[e]);
            }
          } else if (q * 8 < D) {
            for (int r = r0; r < kKeys; r += step) {
              uint2 x = make_uint2(0u, 0u);
              if (r < end) x = *reinterpret_cast<const uint2*>(raw + (r >> lbox) * pitch + (r & (box - 1)) * D + qb);
              put(d0 + (r - r0) * 128, x);
            }
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&kv_full[s]);
            mbar_arrive(&raw_empty[sr]);
          }
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax (warps 4-7: chain A, 8-11: chain B)
    const int c = (warp - 4) >> 2;
    const int quarter = warp & 3;                          // TMEM lanes this warp may access
    const int row = quarter * 32 + lane;                   // row of the chain = TMEM lane
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_col = tmem + lane_addr + (uint32_t)c * 256u, o_col = s_col + 128u;
    uint32_t n = 0, item = 0;                              // halves of the chain so far; items
    int64_t at = walk.at;                                  // first unit of the item's part
    uint32_t joins = 0, u = 0;                             // u: position in the ring of the copies
    bool ok = true, after_wide = false;                    // after_wide: the item before was a wide one
    auto join = [&]() -> bool {                            // a barrier of the two groups, bounded like every wait
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&joined);
      const bool met = warp_wait(&joined, joins & 1);
      ++joins;
      tc_fence_after();
      return met;
    };
    while (ok && walk.next(a, tiles, it)) {
      const PcItem g(a, it, thin_items);
      if constexpr (L::kThinItems) {
        if (g.thin) {
          // A parity wait cannot tell a phase from the one two before it, so every raw tile of the items before has to
          // have landed for certain.  The chain that goes through an item's last tile knows that of all its tiles; a deep
          // item's groups part from it together, but chain A may leave a wide one without that tile: they meet here.
          if (after_wide) ok = join();
          after_wide = false;
          if (!ok) {
            s_abort = 1;
            break;
          }
          if (!thin_item<T>(a, it, g, smem, raw_full, thin_empty, u, &join_s[0][0], join)) {
            s_abort = 1;
            ok = false;
          }
          if (threadIdx.x == 128) {                          // (behind the last join)
            __threadfence_block();                           // what the joins ordered before this, for who reads the count
            thin_done = thin_done + 1;
            if (!it.whole() && it.j0 == 0) a.cut[blockIdx.x] = make_int4(g.row0, it.b, it.h, pg_cta_of(at + it.n - 1, share.total, share.ctas));
          }
          u += 2 * g.T;
          at += it.j1 - it.j0;
          continue;
        }
      }
      u += 2 * g.T;
      after_wide = g.wide;
      const int trow = (g.wide ? c * kRows : 0) + row;     // row of the tile
      const bool valid = trow < g.rows;
      const bool any_valid = (g.wide ? c * kRows : 0) + quarter * 32 < g.rows;
      const int gr = g.row0 + trow;
      const int off = it.r.kl - it.r.ql;
      const int tok = valid ? gr / a.group : 0;
      const int pos = valid ? off + tok : it.r.kl - 1;     // rows past the request compute on zeros, unseen
      const int pos_min = off + (g.row0 + (g.wide ? c * kRows : 0) + quarter * 32) / a.group;
      float sc = a.scale_log2;
      const int nt = g.subs(c);
      if constexpr (kE4m3) {
        if (!warp_wait(&sc_full[item & 1], (item >> 1) & 1)) s_abort = 1;
        sc *= __ldg(a.k_scale + it.h) * __int_as_float((127 + (int)qexp_s[item & 1][trow]) << 23);
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_seen[item & 1]);
      }
      if (sc == 0.0f) sc = 1e-30f;                         // equal weights; a masked score stays -inf below
      const float hidden = sc >= 0.0f ? -INFINITY : INFINITY;
      const uint64_t sc2 = f2_pack(sc, sc);
      float m = -INFINITY, l = 0.0f;                       // l: the sum of the P so far, at the scale 2^-m
      for (int i = 0; i < nt; ++i, ++n) {
        const uint32_t b = n & 1, s_buf = s_col + b * kHalf;
        if (!warp_wait(&s_full[2 * c + b], (n >> 1) & 1)) {   // warp-uniform
          ok = false;
          break;
        }
        tc_fence_after();
        if (any_valid) {
          const int kb = (g.kt0 + g.tile(i)) * kKeys + g.half(c, i) * kHalf;
          uint32_t r[kHalf], w[kHalf / 2];
          tmem_ld64_async(s_buf, r);
          tmem_ld_wait(r);
          if (kb + kHalf - 1 > pos_min) {                  // some key of the half may pass a row
#pragma unroll
            for (int e = 0; e < kHalf; ++e)
              if (kb + e > pos) r[e] = __float_as_uint(hidden);
          }
          // (two-operand maxima: the three-operand ones took 160 cycles more per 128 scores)
          float x4[4] = {hidden, hidden, hidden, hidden};
          if (sc >= 0.0f) {
#pragma unroll
            for (int e = 0; e < kHalf; ++e) x4[e & 3] = fmaxf(x4[e & 3], __uint_as_float(r[e]));
          } else {
#pragma unroll
            for (int e = 0; e < kHalf; ++e) x4[e & 3] = fminf(x4[e & 3], __uint_as_float(r[e]));
          }
          const float ext = sc >= 0.0f ? fmaxf(fmaxf(x4[0], x4[1]), fmaxf(x4[2], x4[3])) : fminf(fminf(x4[0], x4[1]), fminf(x4[2], x4[3]));
          const float mx = ext * sc - kUp;                 // log2 domain; -inf where the row sees nothing
          // The maximum only moves when it grows by more than 2^8: sum and O carry the same factor, so the
          // result is unchanged, and most halves need no rescaling.
          const bool grow = mx > m + kGrow;
          if (__any_sync(0xffffffffu, grow)) {
            const float alpha = grow ? ex2_approx(m - mx) : 1.0f;
            if (grow) m = mx;
            l *= alpha;
            if (i > 0) {                                   // O *= alpha, once the chain's last PV has completed
              if (!warp_wait(&pv_done[2 * c + (b ^ 1)], ((n - 1) >> 1) & 1)) {
                ok = false;
                break;
              }
              tc_fence_after();
              for (int x = 0; x < (D + 31) / 32; ++x) {
                uint32_t o[32];
                tmem_ld32(o_col + x * 32, o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st32(o_col + x * 32, o);
              }
            }
          }
          const float neg_m = m == -INFINITY ? 0.0f : -m;
          const uint64_t nm2 = f2_pack(neg_m, neg_m);
          uint64_t l2[2] = {0ull, 0ull};
#pragma unroll
          for (int e = 0; e < kHalf; e += 2) {
            const float2 x = f2_unpack(f2_fma(f2_pack(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), sc2, nm2));
            const float p0 = ex2_approx(x.x), p1 = ex2_approx(x.y);
            l2[(e >> 1) & 1] = f2_add(l2[(e >> 1) & 1], f2_pack(p0, p1));
            w[e >> 1] = pack2h<kBf>(p0, p1);
          }
          tmem_st32(s_buf, w);
          const float2 ls = f2_unpack(f2_add(l2[0], l2[1]));
          l += ls.x + ls.y;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * c + b]);
      }
      if (ok && nt > 0) ok = warp_wait(&pv_done[2 * c + ((n - 1) & 1)], ((n - 1) >> 1) & 1);
      tc_fence_after();
      if (!ok) s_abort = 1;
      // ---- the item's result: finished, or a part of it
      float w_own = 1.0f, w_other = 0.0f;
      bool has_other = false;
      if (!g.wide) {
        // exchange through one array: maxima, then (once they have been read) sums
        join_s[c][row] = m;
        ok = join() && ok;
        const float m2 = join_s[c ^ 1][row];
        ok = join() && ok;
        join_s[c][row] = l;
        ok = join() && ok;
        const float l2 = join_s[c ^ 1][row];
        const float mj = fmaxf(m, m2), mu = mj == -INFINITY ? 0.0f : mj;
        w_own = ex2_approx(m - mu);
        w_other = ex2_approx(m2 - mu);
        l = l * w_own + l2 * w_other;
        m = mj;
        has_other = g.subs(c ^ 1) > 0;
      }
      if (ok && any_valid) {
        const float vsc = kE4m3 ? __ldg(a.v_scale + it.h) : 1.0f;
        const bool whole = it.whole();
        const float fin = whole ? (l == 0.0f ? 0.0f : vsc / l) : vsc;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (it.j0 == 0 ? 1 : 0);
        const int64_t orow = (int64_t)(it.r.q0 + tok) * a.hq + it.h * a.group + (gr - tok * a.group);
        T* og = reinterpret_cast<T*>(a.out) + orow * D;
        float* po = a.part_o + (slot * kTile + trow) * D;
        if (valid && (g.wide || c == 0)) {
          if (whole) {
            if (a.lse) a.lse[orow] = (m + log2f(l)) * kPgLn2;
          } else {
            float* ml = a.part_ml + slot * 2 * kTile;
            ml[trow] = m;
            ml[kTile + trow] = l;
          }
        }
        // 32 columns at a time; in a deep item chain A stores the even ones and B the odd ones
        for (int x = g.wide ? 0 : c; x * 32 < D; x += g.wide ? 1 : 2) {
          uint32_t o[32], o2[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = o2[e] = 0u;
          if (nt > 0) tmem_ld32_async(o_col + x * 32, o);
          if (has_other) tmem_ld32_async((o_col ^ 256u) + x * 32, o2);
          tmem_ld_wait(o);
          tmem_ld_wait(o2);
          float f[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            float y = __uint_as_float(o[e]);
            if (!g.wide) y = y * w_own + __uint_as_float(o2[e]) * w_other;
            f[e] = y * fin;
          }
          if (!valid) continue;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (x * 32 + q * 8 >= D) break;
            if (whole) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack2h<std::is_same<T, __nv_bfloat16>::value>(f[8 * q + 2 * e], f[8 * q + 2 * e + 1]);
              *reinterpret_cast<uint4*>(og + x * 32 + q * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
              float4* d4 = reinterpret_cast<float4*>(po + x * 32 + q * 8);
              d4[0] = make_float4(f[8 * q], f[8 * q + 1], f[8 * q + 2], f[8 * q + 3]);
              d4[1] = make_float4(f[8 * q + 4], f[8 * q + 5], f[8 * q + 6], f[8 * q + 7]);
            }
          }
        }
      }
      if (!it.whole() && it.j0 == 0 && threadIdx.x == 128)
        a.cut[blockIdx.x] = make_int4(g.row0, it.b, it.h, pg_cta_of(at + it.n - 1, share.total, share.ctas));
      if (!g.wide) ok = join() && ok;                      // both groups have read both O before either moves on
      if (!ok) s_abort = 1;
      at += it.j1 - it.j0;
      ++item;
    }
    if (!ok) s_abort = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// [blocks, bs, hkv, D] cache: boxes of `box` keys of one page and one head; 16-bit elements 64 at a time
// with the 128-byte swizzle, codes whole rows at a time.
int make_page_map(CUtensorMap* map, const void* base, bool e4m3, bool bf16, const PagedArgs& a, int64_t block_stride, int box) {
  auto fn = encode_tiled();
  if (!fn) return set_error(KVB_E_LAUNCH, "paged_prefill_attention: cuTensorMapEncodeTiled unavailable");
  const cuuint64_t es = e4m3 ? 1 : 2;
  cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)a.hkv, (cuuint64_t)a.bs, (cuuint64_t)a.num_blocks};
  cuuint64_t strides[3] = {(cuuint64_t)a.D * es, (cuuint64_t)a.hkv * a.D * es, (cuuint64_t)block_stride * es};
  cuuint32_t boxes[4] = {e4m3 ? (cuuint32_t)a.D : 64u, 1u, (cuuint32_t)box, 1u};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(map, e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  4, const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  e4m3 && a.D != 128 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, e4m3 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(KVB_E_LAUNCH, "paged_prefill_attention: tensor map failed (%d)", (int)r);
  return KVB_OK;
}

template <typename T, bool kE4m3, int DC>
int launch_pc(const CUtensorMap& mk, const CUtensorMap& mv, const PagedArgs& a, int box, int grid, cudaStream_t st) {
  constexpr size_t smem = PcLayout<kE4m3, DC>::kSmem;
  auto kern = paged_prefill_tc_kernel<T, kE4m3, DC>;
  // every call: the attribute belongs to the current device's copy of the kernel
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) e = launch_pdl(kern, dim3((unsigned)grid), dim3(kThreads), smem, st, mk, mv, a, box);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(KVB_E_LAUNCH, "paged_prefill_tc_kernel: %s", cudaGetErrorString(e));
  }
  return check_launch("paged_prefill_tc_kernel");
}

}  // namespace

// Whether the tcgen05 kernel takes the case: 16-bit queries, head_dim a multiple of 16 in [64, 128], and
// pages that a tile of 128 keys is cut into at most 32 boxes by (a box lies in one page, its rows start on
// the 128-byte grid that TMA wants).  It takes them at every length.  mma.sync kernel / this one, 32 + 8 heads of
// 128, bf16: 2 x 4 of 1000 tokens 17.8 / 16.7 us (over codes 20.3 / 15.4; head_dim 64 14.7 / 15.1), 8 x 1 of
// 500 20.0 / 18.9, 4 x 256 of 256 47.9 / 41.8, 64 x 1 of 4000 433 / 181; one prompt of 64 tokens 10.5 / 16.7.
bool paged_prefill_tc_takes(const PagedArgs& a, int q_dtype, int cache_dtype) {
  const int cs = cache_dtype == KVB_E4M3 ? 1 : 2;
  return (q_dtype == KVB_BF16 || q_dtype == KVB_F16) && a.D % 16 == 0 && a.D >= 64 && a.D <= 128 && a.bs % 4 == 0 &&
         aligned16(a.k_cache) && aligned16(a.v_cache) && (a.k_bs * cs) % 16 == 0 && (a.v_bs * cs) % 16 == 0 &&
         a.num_blocks > 0 && a.num_blocks < INT32_MAX;
}

int paged_prefill_tcgen05(PagedArgs& a, int q_dtype, int cache_dtype, void* ws, int sms, cudaStream_t st) {
  int box = kKeys;
  while (a.bs % box) box >>= 1;
  const bool e4 = cache_dtype == KVB_E4M3, bf = q_dtype == KVB_BF16;
  CUtensorMap mk, mv;
  int rc = make_page_map(&mk, a.k_cache, e4, bf, a, a.k_bs, box);
  if (!rc) rc = make_page_map(&mv, a.v_cache, e4, bf, a, a.v_bs, box);
  if (rc) return rc;
  pg_workspace_layout(a, ws, sms, kTile);
  using B = __nv_bfloat16;
  using H = __half;
  if (a.D <= 64) {
    if (bf) rc = e4 ? launch_pc<B, true, 1>(mk, mv, a, box, sms, st) : launch_pc<B, false, 1>(mk, mv, a, box, sms, st);
    else rc = e4 ? launch_pc<H, true, 1>(mk, mv, a, box, sms, st) : launch_pc<H, false, 1>(mk, mv, a, box, sms, st);
  } else {
    if (bf) rc = e4 ? launch_pc<B, true, 2>(mk, mv, a, box, sms, st) : launch_pc<B, false, 2>(mk, mv, a, box, sms, st);
    else rc = e4 ? launch_pc<H, true, 2>(mk, mv, a, box, sms, st) : launch_pc<H, false, 2>(mk, mv, a, box, sms, st);
  }
  if (rc) return rc;
  return pg_launch_merge(a, q_dtype, kTile, sms, st);
}

}  // namespace kvb

using namespace kvb;

extern "C" int kvb_selftest_paged_item(int q_len, int seq_len, int group, int few_rows, int tile, int unit0, int unit1, int* out) {
  if (!out || q_len <= 0 || seq_len < 0 || group <= 0 || tile < 0 || unit0 < 0 || unit1 <= unit0)
    return set_error(KVB_E_ARG, "selftest_paged_item: bad arguments");
  PagedArgs a{};
  a.group = group;
  const PgTiles tiles{kTile, kKeys, group};
  PgItem it{};
  it.r = PgRequest{0, q_len, seq_len};
  it.t = tile;
  it.j0 = unit0;
  it.j1 = unit1;
  if (tile >= tiles.count(it.r) || unit1 > tiles.units(it.r, tile))
    return set_error(KVB_E_ARG, "selftest_paged_item: no such item");
  const PcItem g(a, it, few_rows != 0);
  const int v[7] = {g.thin ? 0 : g.wide ? 2 : 1, g.rows, g.T, g.tiles(0), g.tiles(1), g.subs(0), g.subs(1)};
  for (int i = 0; i < 7; ++i) out[i] = v[i];
  return KVB_OK;
}

extern "C" int kvb_selftest_paged_units(int q_len, int seq_len, int group, int rows, int keys, int tile, int64_t* out) {
  const PgRequest r{0, q_len, seq_len};
  const PgTiles tiles{rows, keys, group};
  if (!out || q_len <= 0 || seq_len < 0 || group <= 0 || rows <= 0 || keys <= 0 || tile < 0 || tile > tiles.count(r))
    return set_error(KVB_E_ARG, "selftest_paged_units: bad arguments");
  out[0] = tiles.count(r);
  out[1] = tile < tiles.count(r) ? tiles.units(r, tile) : 0;
  out[2] = tiles.before(r, tile);
  return KVB_OK;
}

extern "C" int kvb_selftest_paged_cta_of(int64_t unit, int64_t units, int ctas) {
  return unit < 0 || unit >= units || ctas <= 0 || ctas > units ? -1 : pg_cta_of(unit, units, ctas);
}
