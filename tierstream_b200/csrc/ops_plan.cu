// What stands around the products: the grouping of (row, choice) pairs by unit, the joins of per-pair rows, the slope
// times the incoming gradient with its column sums, and the router's selection with its backward pass. All of it moves
// a few bytes per pair or element; every sum has a fixed order, so the same inputs give the same bits.
#include <cfloat>

#include "ops.hpp"

namespace tsb {
namespace ops {
namespace {

constexpr uint32_t kNone = 0xffffffffu;

// ---------------------------------------------------------------------------------------------------------------
// The plan. Counting first: CTA e counts unit e's pairs and resolves its slot. Then CTA e adds up the groups before its
// own (padded rows, tiles) and writes its pairs in ascending order, found by scanning the ids: no atomics,
// so the order never changes. The scan reads the ids once per unit from L2 (256 units x 16,384 pairs: 16 MB); a warp takes
// 512 neighbouring ids a step, 32 a load, and ranks its hits by ballots.
// ---------------------------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024, kPlanEach = 16;  // ids a thread and step

__device__ __forceinline__ int32_t resolve(const Units& u, int32_t e) {
  if (u.abort && *reinterpret_cast<const volatile uint32_t*>(u.abort)) return -1;
  if (u.table) return u.table[e] && u.table[e] % 16 == 0 ? e : -1;
  if (!u.slot_of) return uint32_t(e) < u.n_slots ? e : -1;
  const int32_t s = reinterpret_cast<const volatile int32_t*>(u.slot_of)[(u.unit_base ? *u.unit_base : 0u) + uint32_t(e)];
  return uint32_t(s) < u.n_slots ? s : -1;
}

__device__ __forceinline__ int block_sum(int v, int* red) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) t += red[w];
  return t;
}

__global__ __launch_bounds__(kPlanThreads) void plan_count_kernel(const __grid_constant__ Plan p,
                                                                  const __grid_constant__ Units u,
                                                                  const int32_t* __restrict__ ids) {
  begin_after();
  __shared__ int red[kPlanThreads / 32];
  const int32_t e = blockIdx.x;
  int n = 0;
#pragma unroll 8
  for (uint32_t i = threadIdx.x; i < p.pairs; i += kPlanThreads) n += ids[i] == e;
  for (uint32_t i = blockIdx.x * kPlanThreads + threadIdx.x; i < p.pairs; i += gridDim.x * kPlanThreads)
    p.row_of_pair[i] = -1;  // (until a group takes it)
  n = block_sum(n, red);
  if (threadIdx.x) return;
  const int32_t slot = n ? resolve(u, e) : -1;
  if (n && slot < 0 && u.absent) atomicOr(u.absent, 1u);  // a routed unit that is not there: its rows are left out
  p.cnt[e] = slot < 0 ? 0 : n;
  p.slot[e] = slot < 0 ? 0 : slot;
}

__global__ __launch_bounds__(kPlanThreads) void plan_fill_kernel(const __grid_constant__ Plan p,
                                                                 const int32_t* __restrict__ ids) {
  __shared__ int red[kPlanThreads / 32];
  __shared__ int warp_n[kPlanThreads / 32];
  begin_after();
  const uint32_t e = blockIdx.x;
  int rows = 0, tiles = 0, twice = 0;
  for (uint32_t j = threadIdx.x; j < e; j += kPlanThreads) {
    const int c = p.cnt[j];
    rows += (c + int(p.pad) - 1) / int(p.pad) * int(p.pad);
    tiles += (c + int(p.bm) - 1) / int(p.bm);
    twice += (c + 2 * int(p.bm) - 1) / (2 * int(p.bm));
  }
  rows = block_sum(rows, red);
  tiles = block_sum(tiles, red);
  twice = block_sum(twice, red);
  const int cnt = p.cnt[e];
  const int padded = (cnt + int(p.pad) - 1) / int(p.pad) * int(p.pad), mine = (cnt + int(p.bm) - 1) / int(p.bm),
            mine2 = (mine + 1) / 2;
  if (threadIdx.x == 0) {
    p.off[e] = rows;
    if (e + 1 == p.units) {
      p.head[0] = tiles + mine;
      p.head[1] = rows + padded;
      p.head[2] = twice + mine2;
    }
  }
  for (int i = threadIdx.x; i < mine; i += kPlanThreads) p.tiles[0][tiles + i] = make_int4(p.slot[e], rows, cnt, tiles);
  for (int i = threadIdx.x; i < mine2; i += kPlanThreads) p.tiles[1][twice + i] = make_int4(p.slot[e], rows, cnt, twice);
  if (e + 1 == p.units)
    for (uint32_t i = tiles + mine + threadIdx.x; i < p.max_tiles; i += kPlanThreads) p.tiles[0][i] = make_int4(0, 0, 0, 0);
  for (int i = cnt + threadIdx.x; i < padded; i += kPlanThreads) p.pair_of_row[rows + i] = -1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int done = 0;  // pairs of this unit before the current span of ids
  for (uint32_t i0 = 0; i0 < p.pairs && cnt; i0 += kPlanThreads * kPlanEach) {
    const uint32_t i = i0 + warp * 32 * kPlanEach + lane;
    uint32_t hit[kPlanEach] = {};
    int hits = 0;  // of the warp
    if (i - lane < p.pairs) {
#pragma unroll
      for (int j = 0; j < kPlanEach; ++j) hit[j] = i + 32 * j < p.pairs && ids[i + 32 * j] == int32_t(e);
#pragma unroll
      for (int j = 0; j < kPlanEach; ++j) {
        hit[j] = __ballot_sync(0xffffffffu, hit[j]);
        hits += __popc(hit[j]);
      }
    }
    __syncthreads();
    if (lane == 0) warp_n[warp] = hits;
    __syncthreads();
    int r = rows + done;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w < warp) r += warp_n[w];
      done += warp_n[w];
    }
    if (!hits) continue;
#pragma unroll
    for (int j = 0; j < kPlanEach; ++j) {
      if (!hit[j]) continue;
      if (hit[j] >> lane & 1) {
        const int at = r + __popc(hit[j] & ((1u << lane) - 1));
        p.pair_of_row[at] = int32_t(i + 32 * j);
        p.row_of_pair[i + 32 * j] = at;
      }
      r += __popc(hit[j]);
    }
  }
}

// The same for few pairs in one launch: one CTA, a pair and a unit to a thread.
constexpr int kSmallThreads = 1024;
constexpr uint32_t kSmallPairs = 1024, kSmallUnits = 1024;

__global__ __launch_bounds__(kSmallThreads) void plan_small_kernel(const __grid_constant__ Plan p,
                                                                   const __grid_constant__ Units u,
                                                                   const int32_t* __restrict__ ids) {
  __shared__ int32_t cnt[kSmallUnits], rows[kSmallUnits];
  __shared__ int32_t wr[32], wt[32], wd[32];
  const uint32_t t = threadIdx.x;
  const int lane = t & 31, warp = t >> 5;
  begin_after();
  cnt[t] = 0;
  const int32_t mine = t < p.pairs ? ids[t] : -1;
  __syncthreads();
  const bool valid = uint32_t(mine) < p.units;
  int32_t my_slot = 0;
  if (valid) atomicAdd(&cnt[mine], 1);  // (counts only: their value does not depend on the order)
  __syncthreads();
  if (t < p.units && cnt[t]) {
    const int32_t slot = resolve(u, int32_t(t));
    if (slot < 0) {
      if (u.absent) atomicOr(u.absent, 1u);
      cnt[t] = 0;
    } else {
      my_slot = slot;
    }
  }
  __syncthreads();
  const int c = t < p.units ? cnt[t] : 0;
  const int padded = (c + int(p.pad) - 1) / int(p.pad) * int(p.pad), nt = (c + int(p.bm) - 1) / int(p.bm);
  const int nd = (nt + 1) / 2;
  int r = padded, k = nt, d = nd;  // inclusive scans over the units
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, r, o), b = __shfl_up_sync(0xffffffffu, k, o),
              e = __shfl_up_sync(0xffffffffu, d, o);
    if (lane >= o) r += a, k += b, d += e;
  }
  if (lane == 31) wr[warp] = r, wt[warp] = k, wd[warp] = d;
  __syncthreads();
  for (int w = 0; w < warp; ++w) r += wr[w], k += wt[w], d += wd[w];
  const int first = r - padded;
  rows[t] = first;
  __syncthreads();
  if (t < p.units) {
    p.cnt[t] = c;
    p.off[t] = first;
    p.slot[t] = my_slot;
    if (t + 1 == p.units) p.head[0] = k, p.head[1] = r, p.head[2] = d;
    for (int i = 0; i < nt; ++i) p.tiles[0][k - nt + i] = make_int4(my_slot, first, c, k - nt);
    for (int i = 0; i < nd; ++i) p.tiles[1][d - nd + i] = make_int4(my_slot, first, c, d - nd);
    for (int i = c; i < padded; ++i) p.pair_of_row[first + i] = -1;
  }
  int all = 0;
  for (int w = 0; w < 32; ++w) all += wt[w];
  for (uint32_t i = uint32_t(all) + t; i < p.max_tiles; i += kSmallThreads) p.tiles[0][i] = make_int4(0, 0, 0, 0);
  // warp after warp, its pairs of a unit take the unit's next rows in the lanes' order
  const uint32_t same = __match_any_sync(0xffffffffu, mine);
  const int before = __popc(same & ((1u << lane) - 1));
  const bool takes = valid && cnt[mine];
  int32_t row = -1;
  for (int w = 0; w * 32 < int(p.pairs); ++w) {
    if (warp == w) {
      if (takes) row = rows[mine] + before;
      __syncwarp();
      if (takes && before == 0) rows[mine] += __popc(same);
    }
    __syncthreads();
  }
  if (t < p.pairs) {
    if (row >= 0) p.pair_of_row[row] = int32_t(t);
    p.row_of_pair[t] = row;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Joins: a row's contributions from its choices, added in order in 32 bits and
// rounded once with the residual. V columns a thread; bound by the 32-bit rows' bytes.
// ---------------------------------------------------------------------------------------------------------------
template <class T, int V>
__global__ __launch_bounds__(256) void join_kernel(const int32_t* __restrict__ row_of_pair, const float* __restrict__ src,
                                                   const float* __restrict__ weights, uint32_t top, uint64_t n,
                                                   const T* residual, uint64_t ldr, T* y, uint64_t ldy) {
  begin_after();
  const uint64_t t = blockIdx.x, c = (uint64_t(blockIdx.y) * 256 + threadIdx.x) * V;
  if (c >= n) return;
  float sum[V];
#pragma unroll
  for (int v = 0; v < V; ++v) sum[v] = residual ? to_f(residual[t * ldr + c + v]) : 0.f;
  constexpr uint32_t kAt = 4;  // choices whose loads are in flight together
  for (uint32_t k0 = 0; k0 < top; k0 += kAt) {
    int32_t row[kAt];
    float w[kAt], part[kAt][V];
#pragma unroll
    for (uint32_t j = 0; j < kAt; ++j) {
      row[j] = k0 + j < top ? row_of_pair[t * top + k0 + j] : -1;
      w[j] = weights && row[j] >= 0 ? weights[t * top + k0 + j] : 1.f;
    }
#pragma unroll
    for (uint32_t j = 0; j < kAt; ++j) {
      const float* p = src + uint64_t(row[j] < 0 ? 0 : row[j]) * n + c;
      if (row[j] < 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) part[j][v] = 0.f;
      } else if constexpr (V == 4) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(p));
        part[j][0] = f.x, part[j][1] = f.y, part[j][2] = f.z, part[j][3] = f.w;
      } else {
        part[j][0] = *p;
      }
    }
#pragma unroll
    for (uint32_t j = 0; j < kAt; ++j)
      if (row[j] >= 0)
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] += w[j] * part[j][v];
  }
#pragma unroll
  for (int v = 0; v < V; ++v) y[t * ldy + c + v] = from_f<T>(sum[v]);
}

template <class T, int V>
__global__ __launch_bounds__(256) void join_linear_kernel(int act, const float* __restrict__ src, uint32_t splits,
                                                          uint64_t split_stride, uint64_t n, const T* __restrict__ bias,
                                                          const T* residual, uint64_t ldr, T* y, uint64_t ldy, T* pre,
                                                          uint64_t ldp) {
  begin_after();
  const uint64_t r = blockIdx.x, c = (uint64_t(blockIdx.y) * 256 + threadIdx.x) * V;
  if (c >= n) return;
  float z[V] = {};
  for (uint32_t s = 0; s < splits; ++s) {
    const float* p = src + s * split_stride + r * n + c;
    if constexpr (V == 4) {
      const float4 f = *reinterpret_cast<const float4*>(p);
      z[0] += f.x, z[1] += f.y, z[2] += f.z, z[3] += f.w;
    } else {
      z[0] += *p;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (bias) z[v] += to_f(bias[c + v]);
    if (pre) pre[r * ldp + c + v] = from_f<T>(z[v]);
    y[r * ldy + c + v] = from_f<T>(act_rt(act, z[v]) + (residual ? to_f(residual[r * ldr + c + v]) : 0.f));
  }
}

// a warp adds a pair's sums, lane by lane and then over the lanes
template <class T>
__global__ __launch_bounds__(256) void join_dw_kernel(const int32_t* __restrict__ row_of_pair, uint32_t pairs,
                                                      const float* __restrict__ dwp, uint32_t tiles, T* __restrict__ dw) {
  begin_after();
  const uint32_t i = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= pairs) return;
  const int32_t row = row_of_pair[i];
  float s = 0.f;
  if (row >= 0)
    for (uint32_t j = lane; j < tiles; j += 32) s += dwp[uint64_t(row) * tiles + j];
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) dw[i] = from_f<T>(s);
}

// A warp takes 256 columns of a row, two bytes a lane and load, eight loads in flight: rows that start anywhere are read
// and written in whole sectors all the same.
constexpr uint32_t kCopyCols = 256;
__global__ __launch_bounds__(256) void copies_kernel(const __grid_constant__ Copies j) {
  begin_after();
  const uint64_t stride = uint64_t(gridDim.x) * 8;
  uint64_t at = uint64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  for (int i = 0; i < j.n; ++i) {
    const Copy& c = j.c[i];
    const uint64_t spans = (c.ldd + kCopyCols - 1) / kCopyCols, all = c.rows * spans;
    for (; at < all; at += stride) {
      const uint64_t r = at / spans, k0 = (at - r * spans) * kCopyCols + (threadIdx.x & 31);
      const uint16_t* s = static_cast<const uint16_t*>(c.src) + r * c.ld;
      uint16_t* d = static_cast<uint16_t*>(c.dst) + r * c.ldd;
      uint16_t v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = k0 + 32 * u < c.cols ? s[k0 + 32 * u] : uint16_t(0);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (k0 + 32 * u < c.ldd) d[k0 + 32 * u] = v[u];
    }
    at -= all;  // (the second matrix' spans follow the first's)
  }
}

// ---------------------------------------------------------------------------------------------------------------
// dz = dy act'(pre) (or a copy of dy without an activation), rounded once to the operands' type (the products take
// 16-bit operands), and db from the unrounded values: each CTA sums kDzRows rows of 32 V columns, then 32 threads per
// column add the CTAs' sums, every 32nd in order, and their sums in order.
// ---------------------------------------------------------------------------------------------------------------
constexpr uint32_t kDzRows = 64;

template <class T, int V>
__global__ __launch_bounds__(256) void dz_kernel(int act, const T* __restrict__ dy, uint64_t ldy,
                                                 const T* __restrict__ pre, uint64_t ldp, T* __restrict__ dz,
                                                 uint64_t ldz, uint64_t rows, uint64_t n, float* __restrict__ part) {
  begin_after();
  __shared__ float red[8][32 * V];
  const uint64_t c = (uint64_t(blockIdx.y) * 32 + threadIdx.x) * V;
  const uint64_t r0 = uint64_t(blockIdx.x) * kDzRows, r1 = r0 + kDzRows < rows ? r0 + kDzRows : rows;
  float sum[V] = {};
  if (c < n)
    for (uint64_t r = r0 + threadIdx.y; r < r1; r += 8) {
      T a[V], z[V];
      if constexpr (V == 8) {
        *reinterpret_cast<uint4*>(a) = *reinterpret_cast<const uint4*>(dy + r * ldy + c);
        if (pre) *reinterpret_cast<uint4*>(z) = *reinterpret_cast<const uint4*>(pre + r * ldp + c);
      } else {
        a[0] = dy[r * ldy + c];
        if (pre) z[0] = pre[r * ldp + c];
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float d = to_f(a[v]) * (pre ? slope_rt(act, to_f(z[v])) : 1.f);
        sum[v] += d;
        a[v] = from_f<T>(d);
      }
      if (dz) {
        if constexpr (V == 8) *reinterpret_cast<uint4*>(dz + r * ldz + c) = *reinterpret_cast<uint4*>(a);
        else dz[r * ldz + c] = a[0];
      }
    }
  if (!part) return;
#pragma unroll
  for (int v = 0; v < V; ++v) red[threadIdx.y][threadIdx.x * V + v] = sum[v];
  __syncthreads();
  for (uint32_t j = threadIdx.y * 32 + threadIdx.x; j < 32 * V; j += 256) {
    const uint64_t col = uint64_t(blockIdx.y) * 32 * V + j;
    if (col >= n) continue;
    float s = 0.f;
    for (int w = 0; w < 8; ++w) s += red[w][j];
    part[uint64_t(blockIdx.x) * n + col] = s;
  }
}

template <class T>
__global__ __launch_bounds__(1024) void db_kernel(const float* __restrict__ part, uint32_t chunks, uint64_t n,
                                                  T* __restrict__ db) {
  begin_after();
  __shared__ float red[32][33];
  const uint64_t c = uint64_t(blockIdx.x) * 32 + threadIdx.x;
  float s = 0.f;
  if (c < n)
    for (uint32_t j = threadIdx.y; j < chunks; j += 32) s += part[j * n + c];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y || c >= n) return;
  for (int w = 1; w < 32; ++w) s += red[w][threadIdx.x];
  db[c] = from_f<T>(s);
}

// ---------------------------------------------------------------------------------------------------------------
// The router. A warp holds a row's logits in registers (expert j in lane j % 32) and takes the largest `top` times. Each
// lane has its three largest at hand, so that a choice is one redux over the lanes' largest (a second one finds the lowest
// expert where several are equal); a lane that loses all looks through its logits again, for the three next in order. With
// every lane looking through them for every choice, eight of 256 for 8191 rows took 10.0 us; this way 6.7. Values are words
// in the same order; 0 stands for -inf, a masked expert that is never taken, and NaN; +inf counts as the largest finite
// value. Bound by instructions for long prompts, by the launch for single tokens.
// ---------------------------------------------------------------------------------------------------------------
// (fmaxf drops a NaN; + 0: -0 equals +0)
__device__ __forceinline__ float logit_of(float z) { return fminf(fmaxf(z, -INFINITY), FLT_MAX) + 0.f; }
// finite values as words in the same order above 0, which stands for -inf
__device__ __forceinline__ uint32_t ordered(float z) {
  const uint32_t b = __float_as_uint(z);
  return z == -INFINITY ? 0u : b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t m) { return __uint_as_float(m & 0x80000000u ? m ^ 0x80000000u : ~m); }
// a lane's three largest logits and where they are
struct Three {
  uint32_t m1, m2, m3;
  int i1, i2, i3;
};
// those of `key`, the lower index first among equal ones (AFTER: only what comes behind `last` at index `at` in this order)
template <int V, bool AFTER>
__device__ __forceinline__ Three three_largest(const uint32_t (&key)[V], uint32_t last, int at) {
  Three t{};
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const uint32_t c = !AFTER || key[v] < last || (key[v] == last && v > at) ? key[v] : 0u;
    const bool p1 = c > t.m1, p2 = c > t.m2, p3 = c > t.m3;
    t.i3 = p2 ? t.i2 : p3 ? v : t.i3;
    t.i2 = p1 ? t.i1 : p2 ? v : t.i2;
    t.i1 = p1 ? v : t.i1;
    t.m3 = max(t.m3, min(t.m2, c));
    t.m2 = max(t.m2, min(t.m1, c));
    t.m1 = max(t.m1, c);
  }
  return t;
}
__device__ __forceinline__ float warp_add(float v) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <class T, int V>
__global__ __launch_bounds__(256) void route_kernel(const T* __restrict__ logits, uint64_t ld, uint64_t rows,
                                                    uint32_t experts, uint32_t top, int norm, int32_t* __restrict__ ids,
                                                    float* __restrict__ weights) {
  begin_after();
  const uint64_t row = uint64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const uint32_t lane = threadIdx.x & 31;
  if (row >= rows) return;
  float z[V];
  uint32_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const uint32_t j = lane + 32 * v;
    z[v] = j < experts ? logit_of(to_f(logits[row * ld + j])) : -INFINITY;
    key[v] = ordered(z[v]);
  }
  Three t = three_largest<V, false>(key, 0, 0);
  int have = 3;
  float best = 0.f, mine = 0.f;  // lane i keeps choice i
  int32_t id = -1;
  for (uint32_t i = 0; i < top; ++i) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, t.m1);
    if (!m) break;
    const uint32_t expert = uint32_t(t.i1) * 32 + lane, at = __reduce_min_sync(0xffffffffu, t.m1 == m ? expert : kNone);
    if (i == 0) best = value_of(m);
    if (lane == i) id = int32_t(at), mine = value_of(m);
    const int where = t.i1;
    if (expert == at) t.m1 = t.m2, t.i1 = t.i2, t.m2 = t.m3, t.i2 = t.i3, t.m3 = 0, --have;
    if (have == 0) t = three_largest<V, true>(key, m, where), have = 3;
  }
  const float p = id >= 0 ? expf(mine - best) : 0.f;
  float sum = 0.f;
  if (norm) {
    sum = p;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) sum += z[v] == -INFINITY ? 0.f : expf(z[v] - best);
  }
  sum = warp_add(sum);
  if (lane < top) {
    ids[row * top + lane] = id;
    weights[row * top + lane] = id >= 0 ? p / sum : 0.f;
  }
}

template <class T, class W, int V>
__global__ __launch_bounds__(256) void route_back_kernel(const W* __restrict__ dw, const T* __restrict__ logits,
                                                         uint64_t ld, const int32_t* __restrict__ ids,
                                                         const float* __restrict__ weights, uint64_t rows,
                                                         uint32_t experts, uint32_t top, int norm,
                                                         T* __restrict__ dlogits, uint64_t ldd) {
  begin_after();
  const uint64_t row = uint64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const uint32_t lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int32_t id = lane < top ? ids[row * top + lane] : -1;
  const bool there = uint32_t(id) < experts;
  const float d = there ? to_f(dw[row * top + lane]) : 0.f, w = there ? weights[row * top + lane] : 0.f;
  const float s = warp_add(d * w);  // sum_i dw_i p_i
  float p[V], g[V];
  if (norm) {  // p is the chosen weights and zero elsewhere
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = 0.f;
  } else {
    float m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint32_t j = lane + 32 * v;
      p[v] = j < experts ? logit_of(to_f(logits[row * ld + j])) : -INFINITY;
      m = fmaxf(m, p[v]);
    }
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
    for (int v = 0; v < V; ++v) {
      p[v] = p[v] == -INFINITY ? 0.f : expf(p[v] - m);
      sum += p[v];
    }
    sum = warp_add(sum);
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = sum > 0.f ? p[v] / sum : 0.f;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) g[v] = -s;
  for (uint32_t i = 0; i < top; ++i) {
    const int32_t e = __shfl_sync(0xffffffffu, id, i);
    const float di = __shfl_sync(0xffffffffu, d, i), wi = __shfl_sync(0xffffffffu, w, i);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e == int32_t(lane + 32 * v)) {
        g[v] += di;
        if (norm) p[v] = wi;
      }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const uint32_t j = lane + 32 * v;
    if (j < experts) dlogits[row * ldd + j] = from_f<T>(p[v] * g[v]);
  }
}

template <class F>
void by_experts(uint32_t experts, F&& f) {
  if (experts <= 32) f(std::integral_constant<int, 1>());
  else if (experts <= 64) f(std::integral_constant<int, 2>());
  else if (experts <= 128) f(std::integral_constant<int, 4>());
  else if (experts <= 256) f(std::integral_constant<int, 8>());
  else if (experts <= 512) f(std::integral_constant<int, 16>());
  else f(std::integral_constant<int, 32>());
}
template <class F>
void by_type(int dtype, F&& f) {
  if (dtype == TSB_BF16) f(__nv_bfloat16());
  else if (dtype == TSB_F16) f(__half());
  else f(float());
}

uint64_t aligned(uint64_t n) { return (n + 255) / 256 * 256; }
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

// Plan arrays back to back, each on 256 bytes. A group of c rows has at most c / bm + 1 tiles and pad - 1 padding rows.
Plan plan_at(void* ws, uint32_t units, uint64_t pairs, uint32_t pad, uint32_t bm) {
  Plan p{};
  const uint64_t met = pairs < units ? pairs : units;
  p.units = units;
  p.pairs = uint32_t(pairs);
  p.pad = pad;
  p.bm = bm;
  p.max_rows = uint32_t(pairs + met * (pad - 1));
  p.max_tiles = uint32_t(pairs / bm + met);
  char* c = static_cast<char*>(ws);
  auto take = [&](uint64_t n) {
    int32_t* r = reinterpret_cast<int32_t*>(c);
    c += aligned(n * 4);
    return r;
  };
  p.head = take(3);
  p.cnt = take(units);
  p.off = take(units);
  p.slot = take(units);
  p.pair_of_row = take(p.max_rows);
  p.row_of_pair = take(pairs);
  for (int i = 0; i < 2; ++i) p.tiles[i] = reinterpret_cast<int4*>(take(uint64_t(p.max_tiles) * 4));
  return p;
}
uint64_t plan_bytes(uint32_t units, uint64_t pairs, uint32_t pad, uint32_t bm) {
  const uint64_t met = pairs < units ? pairs : units;
  return aligned(12) + 3 * aligned(uint64_t(units) * 4) + aligned((pairs + met * (pad - 1)) * 4) + aligned(pairs * 4) +
         2 * aligned((pairs / bm + met) * 16);
}

int launch_plan(const Plan& p, const Units& u, const int32_t* ids, cudaStream_t s) {
  if (p.pairs <= kSmallPairs && p.units <= kSmallUnits) {
    return launch(plan_small_kernel, 1, kSmallThreads, 0, 1, s, p, u, ids);
  }
  if (const int e = launch(plan_count_kernel, p.units, kPlanThreads, 0, 1, s, p, u, ids)) return e;
  return launch(plan_fill_kernel, p.units, kPlanThreads, 0, 1, s, p, ids);
}

int launch_join(int dtype, const Plan& p, const float* rows32, const float* weights, uint32_t top, uint64_t rows,
                uint64_t n, const void* residual, uint64_t ldr, void* y, uint64_t ldy, cudaStream_t s) {
  int e = 0;
  by_type(dtype, [&](auto v) {
    using T = decltype(v);
    const T* r = static_cast<const T*>(residual);
    const unsigned v4 = n % 4 == 0 ? 4 : 1;
    e = launch(v4 == 4 ? join_kernel<T, 4> : join_kernel<T, 1>, dim3(unsigned(rows), unsigned(ceil_div(n, 256 * v4))), 256, 0,
               1, s, p.row_of_pair, rows32, weights, top, n, r, ldr, static_cast<T*>(y), ldy);
  });
  return e;
}

int launch_join_linear(int dtype, int act, const float* rows32, uint32_t splits, uint64_t rows, uint64_t n,
                       const void* bias, const void* residual, uint64_t ldr, void* y, uint64_t ldy, void* pre,
                       uint64_t ldp, cudaStream_t s) {
  int e = 0;
  by_type(dtype, [&](auto v) {
    using T = decltype(v);
    const unsigned v4 = n % 4 == 0 ? 4 : 1;
    e = launch(v4 == 4 ? join_linear_kernel<T, 4> : join_linear_kernel<T, 1>,
               dim3(unsigned(rows), unsigned(ceil_div(n, 256 * v4))), 256, 0, 1, s, act, rows32, splits, rows * n, n,
               static_cast<const T*>(bias), static_cast<const T*>(residual), ldr, static_cast<T*>(y), ldy,
               static_cast<T*>(pre), ldp);
  });
  return e;
}

int launch_copies(const Copies& c, cudaStream_t s) {
  uint64_t spans = 0;
  for (int i = 0; i < c.n; ++i) spans += c.c[i].rows * ceil_div(c.c[i].ldd, kCopyCols);
  const uint64_t blocks = ceil_div(spans, 8);
  return launch(copies_kernel, unsigned(blocks < 2368 ? blocks : 2368), 256, 0, 1, s, c);
}

int launch_join_dw(int dtype, const Plan& p, const float* dwp, uint32_t tiles, void* dw, cudaStream_t s) {
  int e = 0;
  by_type(dtype, [&](auto v) {
    using T = decltype(v);
    e = launch(join_dw_kernel<T>, unsigned(ceil_div(p.pairs, 8)), 256, 0, 1, s, p.row_of_pair, p.pairs, dwp, tiles,
               static_cast<T*>(dw));
  });
  return e;
}

uint32_t dz_chunks(uint64_t rows, uint64_t) { return uint32_t(ceil_div(rows, kDzRows)); }

int launch_dz(int dtype, int act, const void* dy, uint64_t ldy, const void* pre, uint64_t ldp, void* dz, uint64_t ldz,
              uint64_t rows, uint64_t n, void* db, float* part, cudaStream_t s) {
  const bool wide = n % 8 == 0 && on16(dy) && ldy % 8 == 0 && (!pre || (on16(pre) && ldp % 8 == 0)) && (!dz || ldz % 8 == 0);
  const uint32_t chunks = dz_chunks(rows, n);
  int e = 0;
  by_type(dtype, [&](auto v) {
    using T = decltype(v);
    const T *a = static_cast<const T*>(dy), *b = act == TSB_ACT_NONE ? nullptr : static_cast<const T*>(pre);
    T* z = static_cast<T*>(dz);
    float* sums = db ? part : nullptr;
    const unsigned each = wide ? 8 : 1;
    e = launch(wide ? dz_kernel<T, 8> : dz_kernel<T, 1>, dim3(chunks, unsigned(ceil_div(n, 32 * each))), dim3(32, 8), 0, 1,
               s, act, a, ldy, b, ldp, z, ldz, rows, n, sums);
    if (!e && db)
      e = launch(db_kernel<T>, unsigned(ceil_div(n, 32)), dim3(32, 32), 0, 1, s, part, chunks, n, static_cast<T*>(db));
  });
  return e;
}

int launch_route(int dtype, const void* logits, uint64_t ld, uint64_t rows, uint32_t experts, uint32_t top, int norm,
                 int32_t* ids, float* weights, cudaStream_t s) {
  int e = 0;
  by_type(dtype, [&](auto v) {
    using T = decltype(v);
    by_experts(experts, [&](auto c) {
      e = launch(route_kernel<T, c.value>, unsigned(ceil_div(rows, 8)), 256, 0, 1, s, static_cast<const T*>(logits), ld, rows,
                 experts, top, norm, ids, weights);
    });
  });
  return e;
}

int launch_route_back(int dtype, int dw_dtype, const void* dw, const void* logits, uint64_t ld, const int32_t* ids,
                      const float* weights, uint64_t rows, uint32_t experts, uint32_t top, int norm, void* dlogits,
                      uint64_t ldd, cudaStream_t s) {
  int e = 0;
  by_type(dtype, [&](auto v) {
    by_type(dw_dtype, [&](auto x) {
      using T = decltype(v);
      using W = decltype(x);
      by_experts(experts, [&](auto c) {
        e = launch(route_back_kernel<T, W, c.value>, unsigned(ceil_div(rows, 8)), 256, 0, 1, s, static_cast<const W*>(dw),
                   static_cast<const T*>(logits), ld, ids, weights, rows, experts, top, norm, static_cast<T*>(dlogits), ldd);
      });
    });
  });
  return e;
}

}  // namespace ops
}  // namespace tsb
