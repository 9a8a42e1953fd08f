// What the paged-prefill kernels share: their arguments, the division of the work over the CTAs and
// the partial results that the merge kernel joins.
//
// A request's chunk of q_len tokens gives q_len * group query rows for each KV head (row r is query
// token r / group, head r % group of the KV head's group), cut into tiles of `rt` rows.  A tile's
// keys, 0 .. the last position of its rows, are cut into units of `bku` keys.  The units of all
// (request, KV head, tile) items, in that order, are dealt out evenly: CTA c of n takes units
// [c W / n, (c + 1) W / n).  So long contexts with few rows, ragged batches and big prompts all give
// every SM the same share, without the host knowing any length.  An item that lies in one CTA is
// finished there; one that is cut leaves a partial result (row maxima, sums and unnormalised
// outputs) in each CTA, and the merge kernel joins them in unit order, so results do not depend on
// timing.
#pragma once

#include "kvb_common.cuh"

namespace kvb {

constexpr unsigned int kStatusBadPage = 2u;      // a block-table entry outside [0, num_blocks)
constexpr unsigned int kStatusBadRequest = 4u;   // a request's lengths outside the tensors
constexpr int kPgMaxCtas = 296;                  // CTAs of one launch at most (sizes the workspace)

struct PagedArgs {
  const void* q;              // [total_q, hq, D], token stride q_ts
  const void* k_cache;        // [num_blocks, bs, hkv, D], block strides k_bs / v_bs (elements)
  const void* v_cache;
  const float* k_scale;       // [hkv] (e4m3 caches) or null
  const float* v_scale;
  const int32_t* qo;          // [batch + 1]
  const void* seq_lens;       // [batch]
  const int32_t* block_table; // [batch, bt_stride]
  void* out;                  // [total_q, hq, D]
  float* lse;                 // [total_q, hq] or null
  float* part_ml;             // [2 * CTAs][2][rt]: row maxima (log2 domain), then sums
  float* part_o;              // [2 * CTAs][rt][D]
  int4* cut;                  // [CTAs]: {first row of the item in its request (-1: none), request, KV head, last CTA}
  int64_t q_ts, k_bs, v_bs, total_q, num_blocks, bt_stride, max_seq_len;
  int batch, hq, hkv, group, D, bs, sl64;
  float scale_log2;           // softmax scale * log2(e)
};

// One request as the division sees it.
struct PgRequest {
  int q0, ql, kl;
};
__device__ __forceinline__ int64_t pg_seq_len(const PagedArgs& a, int b) {
  return a.sl64 ? reinterpret_cast<const int64_t*>(a.seq_lens)[b] : (int64_t)reinterpret_cast<const int32_t*>(a.seq_lens)[b];
}
// Request b; false (and an empty request) when its lengths do not fit the tensors.
__device__ __forceinline__ bool pg_request(const PagedArgs& a, int b, PgRequest& r) {
  const int q0 = a.qo[b], q1 = a.qo[b + 1];
  const int64_t kl = pg_seq_len(a, b);
  r.q0 = q0;
  r.ql = 0;
  r.kl = 0;
  if (q0 < 0 || q1 < q0 || q1 > a.total_q || kl < 0 || kl > a.max_seq_len) return false;
  r.ql = q1 - q0;
  r.kl = (int)kl;
  return true;
}

// sum over t in [0, n) of floor((b + s t) / m), b >= 0, s, m > 0, all numerators below 2^31
// (what s and b hold of whole m's in closed form, then the lattice points below the line counted from the
// other axis, which swaps s and m as Euclid's algorithm does: Graham, Knuth, Patashnik, Concrete
// Mathematics, 2nd ed., section 3.5).
__host__ __device__ __forceinline__ int64_t pg_floor_sum(uint32_t n, uint32_t m, uint32_t s, uint32_t b) {
  int64_t ans = 0;
  while (n > 0) {
    ans += (int64_t)(n - 1) * n / 2 * (s / m) + (int64_t)n * (b / m);
    s %= m;
    b %= m;
    const uint32_t y = s * n + b;
    if (y < m) break;
    n = y / m;
    b = y % m;
    const uint32_t t = m;
    m = s;
    s = t;
  }
  return ans;
}

// Units of tile t of a request with rw = ql * group rows: its last row sees the keys up to position
// floor(x / group), x = (kl - ql) * group + last row, and so x / (group * bku) + 1 units; at least one,
// so that rows that see nothing are written too.
struct PgTiles {
  int rt, bku, group;
  __host__ __device__ __forceinline__ int count(const PgRequest& r) const { return (int)(((int64_t)r.ql * group + rt - 1) / rt); }
  __host__ __device__ __forceinline__ int units(const PgRequest& r, int t) const {
    const int rw = r.ql * group;
    const int last = min((t + 1) * rt, rw) - 1;
    const int x = (r.kl - r.ql) * group + last;
    return x < 0 ? 1 : x / (group * bku) + 1;
  }
  // units of tiles [0, t), t <= count
  __host__ __device__ __forceinline__ int64_t before(const PgRequest& r, int t) const {
    if (t == 0) return 0;
    const int n = count(r);
    int64_t sum = 0;
    int full = t;                                  // tiles of rt rows
    if (t == n) {
      sum = units(r, n - 1);
      --full;
    }
    if (full == 0) return sum;
    sum += full;
    const int x0 = (r.kl - r.ql) * group + rt - 1; // x of tile 0; tile t: x0 + t * rt
    const int skip = x0 >= 0 ? 0 : min(full, (-x0 + rt - 1) / rt);
    if (full > skip)
      sum += pg_floor_sum((uint32_t)(full - skip), (uint32_t)(group * bku), (uint32_t)rt, (uint32_t)(x0 + skip * rt));
    return sum;
  }
};

// This CTA's share: `left` units from unit `j` of tile `t` of KV head `h` of request `b`.
struct PgShare {
  int64_t left;
  int64_t first, total;      // first unit of the share, units in all
  int ctas;                  // CTAs that have a share
  int b, h, t, j;
};

// Fills `s` (shared memory) for CTA `cta` of `grid`.  All NT threads call it; it ends with a barrier.
template <int NT>
__device__ __forceinline__ void pg_share(const PagedArgs& a, const PgTiles& tiles, int cta, int grid, PgShare* s,
                                         int64_t* scan /* NT / 32 */, unsigned int* status) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int NW = NT / 32;
  int64_t mine = 0;                                // requests tid, tid + NT, ...: for the total
  int64_t u_first = 0;                             // units of request tid
  PgRequest r_first{0, 0, 0};
  for (int b = tid; b < a.batch; b += NT) {
    PgRequest r;
    if (!pg_request(a, b, r) && cta == 0) atomicOr(status, kStatusBadRequest);
    const int64_t u = r.ql > 0 ? tiles.before(r, tiles.count(r)) * a.hkv : 0;
    if (b == tid) {
      u_first = u;
      r_first = r;
    }
    mine += u;
  }
  // total over the threads
  int64_t sum = mine;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) scan[warp] = sum;
  if (tid == 0) s->left = 0;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) total += scan[w];
  const int64_t ctas = total < grid ? total : grid;
  const int64_t x0 = ctas > 0 && cta < ctas ? total * cta / ctas : 0, x1 = ctas > 0 && cta < ctas ? total * (cta + 1) / ctas : 0;
  // the request that holds unit x0: exclusive prefixes over the requests, NT at a time
  int64_t carry = 0;
  for (int base = 0; base < a.batch && x1 > x0; base += NT) {
    const int b = base + tid;
    int64_t u = 0;
    PgRequest r{0, 0, 0};
    if (base == 0) {
      u = u_first;
      r = r_first;
    } else if (b < a.batch) {
      pg_request(a, b, r);
      u = r.ql > 0 ? tiles.before(r, tiles.count(r)) * a.hkv : 0;
    }
    int64_t inc = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    __syncthreads();                               // scan[] of the last round has been read
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    int64_t before = carry;
    for (int w = 0; w < warp; ++w) before += scan[w];
    const int64_t pre = before + inc - u;
    if (u > 0 && pre <= x0 && x0 < pre + u) {
      const int64_t per_head = u / a.hkv;
      const int64_t z0 = x0 - pre;
      const int h = (int)(z0 / per_head);
      const int64_t z = z0 - h * per_head;
      int lo = 0, hi = tiles.count(r) - 1;         // the last tile with before(t) <= z
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tiles.before(r, mid) <= z) lo = mid;
        else hi = mid - 1;
      }
      s->b = b;
      s->h = h;
      s->t = lo;
      s->j = (int)(z - tiles.before(r, lo));
      s->left = x1 - x0;
      s->first = x0;
      s->total = total;
      s->ctas = (int)ctas;
    }
    int64_t all = 0;
    for (int w = 0; w < NW; ++w) all += scan[w];
    carry += all;
    if (carry > x0) break;                         // the same for every thread
  }
  __syncthreads();
}

// The item a CTA works on: units [j0, j1) of n of one (request, KV head, tile).
struct PgItem {
  PgRequest r;
  int b, h, t, j0, j1, n;
  __host__ __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == n; }
};
// Walks the items of a share; every role of a CTA walks the same ones on its own.
struct PgWalk {
  int64_t left, at;
  int b, h, t, j;
  PgRequest r;
  __device__ __forceinline__ PgWalk(const PgShare& s) : left(s.left), at(s.first), b(s.b), h(s.h), t(s.t), j(s.j), r{0, 0, 0} {}
  __device__ __forceinline__ bool next(const PagedArgs& a, const PgTiles& tiles, PgItem& it) {
    if (left <= 0) return false;
    if (r.ql == 0) {                               // first item of a request: skip requests without rows
      while (b < a.batch && (!pg_request(a, b, r) || r.ql == 0)) ++b;
      if (b >= a.batch) return false;
    }
    it.r = r;
    it.b = b;
    it.h = h;
    it.t = t;
    it.n = tiles.units(r, t);
    it.j0 = j;
    const int64_t take = min((int64_t)(it.n - j), left);
    it.j1 = j + (int)take;
    left -= take;
    at += take;
    j = 0;
    if (it.j1 == it.n && ++t == tiles.count(r)) {
      t = 0;
      if (++h == a.hkv) {
        h = 0;
        ++b;
        r.ql = 0;
      }
    }
    return true;
  }
};
// CTA that holds unit x.
__host__ __device__ __forceinline__ int pg_cta_of(int64_t x, int64_t total, int ctas) {
  int c = (int)(((x + 1) * ctas - 1) / total);     // floor(total * c / ctas) <= x for this c or the one before
  while (c + 1 < ctas && total * (c + 1) / ctas <= x) ++c;
  while (c > 0 && total * c / ctas > x) --c;
  return c;
}

__device__ __forceinline__ float pg_ex2(float x) {   // 2^x (MUFU.EX2; ex2(-inf) = +0)
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kPgLn2 = 0.6931471805599453f;

// Host side.
inline size_t pg_workspace_bytes(int ctas, int rt, int D) {
  const size_t ml = (size_t)2 * ctas * 2 * rt * 4, o = (size_t)2 * ctas * rt * D * 4, cut = (size_t)ctas * 16;
  return ((cut + 255) & ~size_t(255)) + ((ml + 255) & ~size_t(255)) + o;
}
inline void pg_workspace_layout(PagedArgs& a, void* ws, int ctas, int rt) {
  uint8_t* p = reinterpret_cast<uint8_t*>(ws);
  a.cut = reinterpret_cast<int4*>(p);
  p += ((size_t)ctas * 16 + 255) & ~size_t(255);
  a.part_ml = reinterpret_cast<float*>(p);
  p += ((size_t)2 * ctas * 2 * rt * 4 + 255) & ~size_t(255);
  a.part_o = reinterpret_cast<float*>(p);
}
int pg_launch_merge(const PagedArgs& a, int dtype, int rt, int ctas, cudaStream_t st);

}  // namespace kvb
