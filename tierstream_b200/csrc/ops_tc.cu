// The products for many rows, on the tensor cores (tcgen05) with both operands staged by TMA.
//
// Persistent CTAs, one per SM, alone on 128-row tiles or in pairs on 256-row tiles (each stages its rows of A and half of
// B, so that a tile's operands cross from L2 once for 256 x 256 sums; a single CTA's 128 x 256 need 96 bytes a clock of the
// 64 an SM gets). One warp keeps TMA loads of 64-wide k slices in flight through a 192 KiB ring (A 16 KiB and half or all
// of B a stage, 128-byte swizzled), one issues tcgen05.mma (32-bit sums in TMEM), and eight warps read finished sums back
// (tcgen05.ld), apply the epilogue of ops.hpp and hand blocks of 32 rows by 64 bytes to TMA stores. The sums are double
// buffered in TMEM: the epilogue of one tile runs under the products of the next. 1369 TFLOP/s at 2047 x 7168 x 4096 in
// fp16, 1509 at 8192^3 (cuBLAS: 1469 and 1652), held by the power cap.
//
// Operands come either with k contiguous (K-major) or with m or n contiguous (MN-major), so that no backward product
// needs a transposed copy. The gate and up products of a tile are one 256-column product (128 columns of each), whose two
// halves of a row meet in the same thread's epilogue; the backward pass adds dy Wd as a third 128-column product, so that
// g, u and dh are never stored. Rows of a group start anywhere; the rows of a tile behind its group's end are computed
// and not stored.
//
// Every wait is bounded (2 s): one that runs out counts in a device word (tsb_ops_timeouts), and the CTA leaves after a
// bounded wait for its copies and products in flight, its TMEM freed.
#include "tc.cuh"

namespace tsb {
namespace ops {
namespace {

constexpr int kRowBytes = 64;  // a store buffer: 32 rows x 64 bytes

__device__ uint32_t g_ops_timeouts;

// kLinDwPart: parts of kLinDw's sum over the rows, each with its own 32-bit rows
enum Mode { kLin, kLinDx, kLinDw, kLinDwPart, kUp, kUpBack, kDown, kDx, kDw };

struct Params {
  Plan plan;
  Product p;         // the epilogue's fields, n, and the groups
  int32_t bn;        // columns of a tile (of each of gate and up)
  int32_t n_tiles;   // tiles along n
  int32_t m_tiles;   // tiles along m when not grouped
  int32_t k_blocks;  // of a segment; with k_rows per unit: from the group
  int32_t vec;       // 16-byte stores are possible: `out` maps are made
  int32_t stages, stage_bytes;
  int32_t pair;      // two CTAs to a tile of 256 rows
  int32_t splits;    // kLinDwPart's parts
};
struct Maps {
  CUtensorMap a[2], b[3], out[3];
};

struct Tile {
  int unit, slot, row0, rows, stored;  // unit: or the part; row0: the group's (of k: the part's) first row; rows: m limit;
                                       // stored: rows to store (padding too)
  int m0, n, kb;
};

// The launch's tiles: groups (or the units' matrices) in unit order, inside each chunks of 2048 rows, inside a chunk the
// column tiles, and the chunk's row tiles innermost, so that tiles running at the same time share a unit's columns from
// L2. What the plan says of a tile is read one tile ahead.
template <int MODE, int CG>
struct Tiles {
  static constexpr bool grouped = MODE == kUp || MODE == kUpBack || MODE == kDown || MODE == kDx;
  int at, end;
  int4 next;  // slot, first row, rows, first tile (of a unit's matrix: first row and rows of its group)
  __device__ __forceinline__ void fetch(const Params& q) {
    if (at >= end) return;
    if (grouped) next = q.plan.tiles[0][at / q.n_tiles];
    if (MODE == kDw) {
      const int unit = at / (q.m_tiles * q.n_tiles);
      next.y = q.plan.off[unit];
      next.z = q.plan.cnt[unit];
    }
  }
  __device__ __forceinline__ Tiles(const Params& q) : at(blockIdx.x / CG), next(make_int4(0, 0, 0, 0)) {
    end = grouped ? q.plan.head[0] * q.n_tiles
                  : q.m_tiles * q.n_tiles * (MODE == kDw ? int(q.plan.units) : MODE == kLinDwPart ? q.splits : 1);
    fetch(q);
  }
  __device__ __forceinline__ bool take(const Params& q, Tile& t) {
    constexpr int kRows = kBM * CG, kChunk = 16 / CG;
    if (at >= end) return false;
    const int4 g = next;
    int local = at, mt = q.m_tiles;
    at += gridDim.x / CG;
    fetch(q);
    t.slot = g.x;
    t.row0 = g.y;
    t.unit = 0;
    t.kb = q.k_blocks;
    if constexpr (grouped) {
      t.rows = g.z;
      t.stored = (g.z + int(q.plan.pad) - 1) / int(q.plan.pad) * int(q.plan.pad);
      mt = (g.z + kRows - 1) / kRows;
      local -= g.w * q.n_tiles;
    } else {
      t.rows = t.stored = int(q.p.m);
      if (MODE == kDw || MODE == kLinDwPart) {
        t.unit = local / (mt * q.n_tiles);
        local -= t.unit * mt * q.n_tiles;
      }
      if (MODE == kDw) t.kb = (g.z + kBK - 1) / kBK;
      if (MODE == kLinDwPart) {
        const int first = int(int64_t(q.k_blocks) * t.unit / q.splits);
        t.kb = int(int64_t(q.k_blocks) * (t.unit + 1) / q.splits) - first;
        t.row0 = first * kBK;
      }
    }
    const int chunk = local / (kChunk * q.n_tiles), in = local - chunk * kChunk * q.n_tiles;
    const int width = min(kChunk, mt - chunk * kChunk);
    t.n = in / width;
    t.m0 = (chunk * kChunk + in - t.n * width) * kRows;
    return true;
  }
};

template <int MODE>
struct Traits {
  static constexpr bool grouped = MODE == kUp || MODE == kUpBack || MODE == kDown || MODE == kDx;
  static constexpr int segs = MODE == kUpBack || MODE == kDx ? 2 : 1;
  static constexpr bool rows_k = MODE == kDw || MODE == kLinDwPart;  // k runs over rows from row0
  static constexpr bool a_mn = MODE == kLinDw || rows_k;
  // the segment whose B is columns of gate, then of up (the last: in the backward pass dh comes first)
  __host__ __device__ static constexpr bool both(int s) { return (MODE == kUp && s == 0) || (MODE == kUpBack && s == 1); }
  // B of segment s with n contiguous
  __host__ __device__ static constexpr bool b_mn(int s) {
    return MODE == kLinDx || MODE == kLinDw || rows_k || MODE == kDx || (MODE == kUpBack && s == 0);
  }
  static constexpr int bufs = MODE == kUpBack ? 1 : 2;
};

// A warp's 32 rows x 64 bytes (thread = row) on their way out: into one of its two buffers in shared memory, 64-byte
// swizzled so that no bank is met twice, and from there by a TMA store that runs while the next block is computed. Blocks
// at an edge that TMA must not cross (the rows behind a group's end, columns of the next tile) and outputs whose rows do
// not start on 16 bytes are written along rows by the lanes instead.
struct Out {
  const CUtensorMap* map;
  int z;  // the unit
  char* buf;
  uint32_t flip;
  bool tma;
};
// E out[rows][cols] from row `y`, column `x` of the map; `p` is its address
template <class E>
__device__ __forceinline__ void store_rows(Out& o, int which, const uint32_t (&v)[16], int64_t x, int64_t y, E* p,
                                           int64_t ld, int rows, int cols, bool whole) {
  const int lane = threadIdx.x & 31;
  constexpr int kPer = 16 / int(sizeof(E));
  char* stage = o.buf + (o.flip & 1u) * (32 * kRowBytes);
  o.flip ^= 1u;
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");  // the store before the last has read
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<uint4*>(stage + lane * kRowBytes + ((i ^ ((lane >> 1) & 3)) * 16)) =
        make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  if (o.tma && whole) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(o.map + which),
                   "r"(int(x)), "r"(int(y)), "r"(o.z), "r"(smem_u32(stage))
                   : "memory");
    }
  } else {
    __syncwarp();
    const int c = (lane & 3) * kPer;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 2);
      const uint4 w = *reinterpret_cast<const uint4*>(stage + r * kRowBytes + (((lane & 3) ^ ((r >> 1) & 3)) * 16));
      if (r >= rows) continue;
      if (o.tma && c + kPer <= cols) {
        *reinterpret_cast<uint4*>(p + r * ld + c) = w;
      } else {
        E e[kPer];
        memcpy(e, &w, 16);
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (c + j < cols) p[r * ld + c + j] = e[j];
      }
    }
    __syncwarp();
  }
  if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");  // (an empty group keeps the count)
}
__device__ __forceinline__ void stores_done() {
  if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  __syncwarp();
}

// 32 elements of a row into registers, `cols` of them inside the matrix
template <class T>
__device__ __forceinline__ void read32(T (&v)[32], const T* p, int cols, bool whole) {
  if (whole) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < cols) v[i] = p[i];
  }
}

// 32 columns of sums, 16 at a time (bn is a multiple of 16: the second half of a last odd block is loaded twice and not
// stored)
__device__ __forceinline__ void sums32(uint32_t base, int c, int bn, float (&v)[2][16]) {
  tmem_ld16(base + c, v[0]);
  tmem_ld16(base + min(c + 16, bn - 16), v[1]);
}

template <class T, int MODE, int ACT>
__device__ __forceinline__ void epilogue(const Params& q, const Tile& t, uint32_t tmem, uint32_t tmem_dh, Out& o, int warp) {
  const Product& p = q.p;
  const int lane = threadIdx.x & 31, quad = warp & 3, half = warp >> 2;
  const uint32_t base = tmem + (uint32_t(quad * 32) << 16);
  const int m = t.m0 + quad * 32;                      // the warp's first row in the group
  const int rows = min(32, t.stored - m);              // (may be <= 0: the loads below stay, they are collective)
  const int64_t n0 = int64_t(t.n) * q.bn;
  const int cols = int(min(int64_t(q.bn), p.n - n0));  // columns of this tile inside the matrix
  const bool zero = MODE == kDw && t.kb == 0;          // a unit without rows: nothing was computed
  // TMA clips at the matrix' edges: a block is whole unless it crosses its group's rows or its tile's columns
  const bool whole_rows = rows == 32 || (!Traits<MODE>::grouped && rows > 0);
  const int64_t y = Traits<MODE>::rows_k ? m : int64_t(t.row0) + m;
  o.z = Traits<MODE>::rows_k ? t.unit : 0;
  if constexpr (MODE == kUp || MODE == kUpBack) {
    float w = 0.f, dw = 0.f;
    if (MODE == kUpBack && lane < rows && m + lane < t.rows) w = p.weights[q.plan.pair_of_row[y + lane]];
    for (int c = half * 32; c < cols; c += 64) {
      uint32_t h[16], d1[16], d2[16];
      float g[2][16], u[2][16], d[2][16];
      sums32(base, c, q.bn, g);
      sums32(base + q.bn, c, q.bn, u);
      if constexpr (MODE == kUpBack) sums32(tmem_dh + (uint32_t(quad * 32) << 16), c, q.bn, d);
      tmem_wait_ld();
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float k0 = act_of<ACT>(g[s][i]), k1 = act_of<ACT>(g[s][i + 1]), u0 = u[s][i], u1 = u[s][i + 1];
          if constexpr (MODE == kUp) {
            h[s * 8 + i / 2] = pack<T>(k0 * u0, k1 * u1);
          } else {
            const float e0 = d[s][i], e1 = d[s][i + 1];
            h[s * 8 + i / 2] = pack<T>(w * k0 * u0, w * k1 * u1);
            d1[s * 8 + i / 2] = pack<T>(w * e0 * u0 * slope_of<ACT>(g[s][i]), w * e1 * u1 * slope_of<ACT>(g[s][i + 1]));
            d2[s * 8 + i / 2] = pack<T>(w * e0 * k0, w * e1 * k1);
            if (c + 16 * s + i < cols) dw += e0 * k0 * u0;
            if (c + 16 * s + i + 1 < cols) dw += e1 * k1 * u1;
          }
        }
      const int64_t at = y * p.ldo + n0 + c;
      const bool whole = whole_rows && c + 32 <= q.bn;
      if constexpr (MODE == kUp) {
        store_rows<T>(o, 0, h, n0 + c, y, static_cast<T*>(p.out) + at, p.ldo, rows, cols - c, whole);
      } else {
        store_rows<T>(o, 0, d1, n0 + c, y, static_cast<T*>(p.dg) + at, p.ldo, rows, cols - c, whole);
        store_rows<T>(o, 1, d2, n0 + c, y, static_cast<T*>(p.du) + at, p.ldo, rows, cols - c, whole);
        if (p.hw) store_rows<T>(o, 2, h, n0 + c, y, static_cast<T*>(p.hw) + at, p.ldo, rows, cols - c, whole);
      }
    }
    if (MODE == kUpBack && p.dwp && lane < rows && m + lane < t.rows) p.dwp[(y + lane) * p.ld_dwp + 2 * t.n + half] = dw;
  } else if constexpr (MODE == kDown || MODE == kDx || MODE == kLinDwPart) {
    float* to = p.rows32 + (MODE == kLinDwPart ? t.unit * p.m + y : y) * p.n + n0;
    for (int c = half * 16; c < cols; c += 32) {
      float v[16];
      tmem_ld16(base + c, v);
      tmem_wait_ld();
      uint32_t b[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) b[i] = __float_as_uint(v[i]);
      store_rows<float>(o, 0, b, n0 + c, y, to + c, p.n, rows, cols - c, whole_rows);
    }
  } else if constexpr (MODE == kLin) {
    const T *bias = static_cast<const T*>(p.bias), *res = static_cast<const T*>(p.residual) + (m + lane) * p.ldr;
    for (int c = half * 32; c < cols; c += 64) {
      const int64_t n = n0 + c;
      const bool inside = q.vec && c + 32 <= cols;
      T b[32] = {}, r[32] = {};
      if (bias) read32(b, bias + n, cols - c, inside);
      if (p.residual && lane < rows) read32(r, res + n, cols - c, inside);
      uint32_t out[16], pre[16];
      float v[2][16];
      sums32(base, c, q.bn, v);
      tmem_wait_ld();
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float z0 = v[s][i] + to_f(b[16 * s + i]), z1 = v[s][i + 1] + to_f(b[16 * s + i + 1]);
          pre[8 * s + i / 2] = pack<T>(z0, z1);
          out[8 * s + i / 2] = pack<T>(act_of<ACT>(z0) + to_f(r[16 * s + i]), act_of<ACT>(z1) + to_f(r[16 * s + i + 1]));
        }
      const bool whole = whole_rows && c + 32 <= q.bn;
      store_rows<T>(o, 0, out, n, y, static_cast<T*>(p.out) + m * p.ldo + n, p.ldo, rows, cols - c, whole);
      if (p.pre) store_rows<T>(o, 1, pre, n, y, static_cast<T*>(p.pre) + m * p.ldp + n, p.ldp, rows, cols - c, whole);
    }
  } else {  // gradients: rounded once
    T* out = static_cast<T*>(p.out) + int64_t(t.unit) * p.out_unit + m * p.ldo + n0;
    for (int c = half * 32; c < cols; c += 64) {
      uint32_t h[16] = {};
      if (!zero) {
        float v[2][16];
        sums32(base, c, q.bn, v);
        tmem_wait_ld();
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 16; i += 2) h[s * 8 + i / 2] = pack<T>(v[s][i], v[s][i + 1]);
      }
      store_rows<T>(o, 0, h, n0 + c, y, out + c, p.ldo, rows, cols - c, whole_rows && c + 32 <= q.bn);
    }
  }
}

template <class T, int MODE, int ACT, int CG>
__global__ __launch_bounds__(kThreads, 1) void tc_kernel(const __grid_constant__ Maps maps,
                                                         const __grid_constant__ Params q) {
  using X = Traits<MODE>;
  const uint32_t stages = uint32_t(q.stages), stage_bytes = uint32_t(q.stage_bytes);
  extern __shared__ char raw[];
  char* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  char* store = smem + kRingBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(store + kEpiWarps * kStoreBytes);
  const uint32_t full = smem_u32(bars), empty = full + 8 * kMaxStages, sums_full = empty + 8 * kMaxStages,
                 sums_empty = sums_full + 16;
  uint32_t* words = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStages + 4);  // [0] TMEM address, [1] a wait ran out
  volatile uint32_t* dead = words + 1;
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0);
  const uint32_t rank = CG == 2 ? cta_rank() : 0;
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < stages; ++s) {
      bar_init(full + 8 * s, 1);
      bar_init(empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      bar_init(sums_full + 8 * b, 1);
      bar_init(sums_empty + 8 * b, CG * kEpiWarps);
    }
    words[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(words))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(words))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
  }
  fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(words);
  begin_after();
  const int half_n = q.bn / CG;              // columns of B that this CTA stages (of a single B)
  const int chunks = (half_n + 63) / 64;     // MN-major B

  if (warp == 0) {  // the loads: each CTA its rows of A and its columns of B, all arriving at the first CTA's barrier
    uint32_t it = 0, st = 0, parity = 1;
    bool ok = true;
    Tile t;
    const uint32_t ring = smem_u32(smem), arrive = CG == 2 ? in_cta(full, 0) : full;
    for (Tiles<MODE, CG> tiles(q); ok && tiles.take(q, t);) {
      t.m0 += int(rank) * kBM;
#pragma unroll
      for (int s = 0; s < X::segs; ++s) {
        const bool pair = X::both(s);
        const uint32_t bytes = kABytes + (X::b_mn(s) ? chunks * 8192 : pair ? q.bn * 128 : half_n * 128);
        const CUtensorMap* ma = &maps.a[MODE == kUpBack ? 1 - s : s];
        const CUtensorMap* mb = &maps.b[MODE == kUpBack && s == 0 ? 2 : pair ? rank : s];
        const int z = X::grouped ? t.slot : 0, n0 = t.n * q.bn + (pair ? 0 : int(rank) * half_n);
        const int m0 = X::a_mn ? t.m0 : t.row0 + t.m0;
        int k0 = 0, krow = X::rows_k ? t.row0 : 0;
        for (int kb = 0; kb < t.kb; ++kb, k0 += kBK, krow += kBK) {
          ok = bar_wait(empty + 8 * st, parity, dead);
          if (!ok) break;
          const uint32_t sa = ring + st * stage_bytes, sb = sa + kABytes, bar = arrive + 8 * st;
          if (elect()) {
            if (rank == 0) bar_expect(bar, CG * bytes);
            if constexpr (X::a_mn) {
              tma_load<CG>(sa, ma, m0, krow, 0, bar);
              tma_load<CG>(sa + 8192, ma, m0 + 64, krow, 0, bar);
            } else {
              tma_load<CG>(sa, ma, k0, m0, 0, bar);
            }
            if (X::b_mn(s)) {
              for (int c = 0; c < chunks; ++c) tma_load<CG>(sb + c * 8192, mb, n0 + 64 * c, krow, z, bar);
            } else {
              tma_load<CG>(sb, mb, k0, n0, z, bar);
            }
          }
          ++it;
          if (++st == stages) st = 0, parity ^= 1;
        }
        if (!ok) break;
      }
    }
    if (!ok)  // leave no copy in flight behind
      for (uint32_t j = it > stages ? it - stages : 0; j < it; ++j) {
        volatile uint32_t none = 0;
        (void)bar_wait((rank == 0 ? full : empty) + 8 * (j % stages), (j / stages) & 1, &none);
      }
  } else if (warp == 1 && rank == 0) {  // the products, for both CTAs
    uint32_t it = 0, nt = 0, st = 0, parity = 0;
    bool ok = true;
    Tile t;
    const uint64_t ring_a = desc(smem_u32(smem), X::a_mn);
    constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    for (Tiles<MODE, CG> tiles(q); ok && tiles.take(q, t); ++nt) {
      const int buf = nt % X::bufs;
#pragma unroll
      for (int s = 0; s < X::segs; ++s) {
        // (dh of tile nt goes where tile nt - 2 had its own: read before tile nt - 1's gate and up could start)
        if (s == X::segs - 1 || !(MODE == kUpBack)) {
          ok = ok && bar_wait(sums_empty + 8 * buf, ((nt / X::bufs) & 1) ^ 1, dead);
          if (!ok) break;
        }
        fence_after();
        const int n = X::both(s) ? 2 * q.bn : q.bn;
        const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | (uint32_t(X::a_mn) << 15) |
                               (uint32_t(X::b_mn(s)) << 16) | (uint32_t(n >> 3) << 17) |
                               (uint32_t(CG * kBM >> 4) << 24);
        const uint32_t d = tmem + (MODE == kUpBack && s == 0 ? 256 + 128 * (nt & 1) : buf * 256);
        const bool fresh = !(MODE == kDx && s == 1);  // dx: both segments add into the same sums
        const uint64_t ring_b = desc(smem_u32(smem) + kABytes, X::b_mn(s));
        for (int kb = 0; kb < t.kb; ++kb) {
          ok = bar_wait(full + 8 * st, parity, dead);
          if (!ok) break;
          fence_after();
          const uint64_t da = ring_a + st * (stage_bytes >> 4), db = ring_b + st * (stage_bytes >> 4);
          if (elect()) {
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k)
              mma<CG>(d, da + uint64_t((X::a_mn ? 2048 : 32) * k >> 4), db + uint64_t((X::b_mn(s) ? 2048 : 32) * k >> 4),
                      idesc, !(fresh && kb == 0 && k == 0));
            commit<CG>(empty + 8 * st);
          }
          ++it;
          if (++st == stages) st = 0, parity ^= 1;
        }
        if (!ok) break;
      }
      if (ok && elect()) commit<CG>(sums_full + 8 * buf);
    }
    if (!ok && it) {  // the products already issued read shared memory and TMEM: let them end
      volatile uint32_t none = 0;
      (void)bar_wait(empty + 8 * ((it - 1) % stages), ((it - 1) / stages) & 1, &none);
    }
  } else if (warp >= 4) {  // the epilogue
    uint32_t nt = 0;
    Tile t;
    Out out{maps.out, 0, store + (warp - 4) * kStoreBytes, 0, q.vec != 0};
    for (Tiles<MODE, CG> tiles(q); tiles.take(q, t); ++nt) {
      t.m0 += int(rank) * kBM;
      const int buf = nt % X::bufs;
      if (!bar_wait(sums_full + 8 * buf, (nt / X::bufs) & 1, dead)) break;
      __syncwarp();
      fence_after();
      epilogue<T, MODE, ACT>(q, t, tmem + buf * 256, tmem + 256 + 128 * (nt & 1), out, warp - 4);
      fence_before();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) {
        if constexpr (CG == 2) bar_arrive_cluster(in_cta(sums_empty + 8 * buf, 0));
        else bar_arrive(sums_empty + 8 * buf);
      }
    }
    stores_done();
  }
  fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // neither CTA's memory goes while the other's copies, products or arrivals use it
  fence_after();
  if (warp == 1) {
    __syncwarp();
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    if ((threadIdx.x & 31) == 0 && *dead) atomicAdd(&g_ops_timeouts, 1u);
  }
}

// rows of grouped buffers: row r is source row pair_of_row[r] / top, padding rows are zeros
struct Gather {
  const uint4* src[2];
  uint4* dst[2];
  uint64_t ld16[2];
};
__global__ __launch_bounds__(256) void gather_kernel(const __grid_constant__ Plan plan, uint32_t top, uint32_t n16,
                                                     const __grid_constant__ Gather g) {
  begin_after();
  const uint32_t r = blockIdx.x;
  const uint4* src = g.src[blockIdx.y];
  uint4* dst = g.dst[blockIdx.y];
  if (int32_t(r) >= plan.head[1]) return;
  const int32_t pair = plan.pair_of_row[r];
  const uint4* s = src + uint64_t(pair < 0 ? 0 : uint32_t(pair) / top) * g.ld16[blockIdx.y];
  for (uint32_t c = threadIdx.x; c < n16; c += 256)
    dst[uint64_t(r) * n16 + c] = pair < 0 ? make_uint4(0, 0, 0, 0) : s[c];
}

template <class T, int MODE, int ACT, int CG>
int go_pair(const Maps& maps, const Params& q, int grid, cudaStream_t s) {
  static std::atomic<uint64_t> devices{0};
  const auto kernel = tc_kernel<T, MODE, ACT, CG>;
  if (const int e = allow_smem(reinterpret_cast<const void*>(kernel), devices)) return e;
  return launch(kernel, unsigned(grid * CG), kThreads, kSmemBytes, CG, s, maps, q);
}
template <class T, int MODE, int ACT>
int go(const Maps& maps, const Params& q, int grid, cudaStream_t s) {
  if constexpr (Traits<MODE>::grouped) return go_pair<T, MODE, ACT, 2>(maps, q, grid, s);
  else return q.pair ? go_pair<T, MODE, ACT, 2>(maps, q, grid, s) : go_pair<T, MODE, ACT, 1>(maps, q, grid, s);
}
template <class T, int MODE>
int go_act(int act, const Maps& maps, const Params& q, int grid, cudaStream_t s) {
  switch (act) {
    case TSB_ACT_SILU: return go<T, MODE, TSB_ACT_SILU>(maps, q, grid, s);
    case TSB_ACT_GELU: return go<T, MODE, TSB_ACT_GELU>(maps, q, grid, s);
    case TSB_ACT_GELU_TANH: return go<T, MODE, TSB_ACT_GELU_TANH>(maps, q, grid, s);
    case TSB_ACT_RELU: return go<T, MODE, TSB_ACT_RELU>(maps, q, grid, s);
  }
  return go<T, MODE, TSB_ACT_NONE>(maps, q, grid, s);
}
template <int MODE>
int go_type(int dtype, int act, const Maps& maps, const Params& q, int grid, cudaStream_t s) {
  if constexpr (MODE == kLin || MODE == kUp || MODE == kUpBack)
    return dtype == TSB_BF16 ? go_act<__nv_bfloat16, MODE>(act, maps, q, grid, s)
                             : go_act<__half, MODE>(act, maps, q, grid, s);
  else
    return dtype == TSB_BF16 ? go<__nv_bfloat16, MODE, 0>(maps, q, grid, s) : go<__half, MODE, 0>(maps, q, grid, s);
}

struct Shape {  // one operand as memory: [slots][rows][cols] with cols contiguous
  const void* p;
  uint64_t cols, rows, ld, slots, slot_bytes;
};
bool fits(const Shape& s) {
  return on16(s.p) && s.ld % 8 == 0 && s.slot_bytes % 16 == 0 && s.slot_bytes < (uint64_t(1) << 40) && s.cols >= 1;
}

}  // namespace

// Columns a tile: of the multiples of 16 (32 for a pair) up to 256, the one whose last wave of tiles wastes least. A tile
// costs its columns plus about 32 (the narrower tile re-reads A for fewer products). Under the power cap the widths lie
// close: 2047 x 7168 x 4096 on 74 pairs takes 95 us at 160 (five waves, the choice), 94 at 224, 96 at 256 and 102 at 128;
// 4096^3 102 at 192 (the choice), 107 at 160; 8192 x 8192 x 4096 366 at 256 (the choice), 406 at 160.
int tc_columns(int64_t m, int64_t n, int sms) {
  const int cg = m > kBM ? 2 : 1, step = 16 * cg;
  const uint64_t m_tiles = ceil_div(uint64_t(m), uint64_t(kBM * cg));
  int best = step;
  int64_t cost = INT64_MAX;
  for (int bn = 256; bn >= step; bn -= step) {
    const int64_t waves = int64_t(ceil_div(m_tiles * ceil_div(uint64_t(n), uint64_t(bn)), uint64_t(sms / cg)));
    const int64_t c = waves * (bn + 32);
    if (c < cost) cost = c, best = bn;
  }
  return best;
}

// one of the two strides is 1, the other a multiple of 8 elements
bool tc_fits(const Operand& o) {
  return on16(o.p) && (o.s_i == 1 || o.s_k == 1) && (o.s_k == 1 ? o.s_i : o.s_k) % 8 == 0 && (o.s_i != 1 || o.s_k != 1);
}

int launch_gather(const Plan& plan, uint32_t top, uint64_t n, const void* src, uint64_t ld, void* dst, const void* src2,
                  uint64_t ld2, void* dst2, cudaStream_t s) {
  const Gather g{{static_cast<const uint4*>(src), static_cast<const uint4*>(src2)},
                 {static_cast<uint4*>(dst), static_cast<uint4*>(dst2)},
                 {ld / 8, ld2 / 8}};
  return launch(gather_kernel, dim3(plan.max_rows, src2 ? 2 : 1), 256, 0, 1, s, plan, top, uint32_t(n / 8), g);
}

int launch_tc(int dtype, const Product& p, int splits, int columns, const Plan* plan, const Units* u, cudaStream_t s) {
  if (!encoder()) return int(cudaErrorNotSupported);
  const int sms = sm_count();
  if (!sms) return int(cudaErrorInvalidDevice);
  Params q{};
  q.p = p;
  if (plan) q.plan = *plan;
  const bool a_mn = p.a[0].s_k != 1;
  Mode mode;
  if (p.epi == kEpiLinear) mode = kLin;
  else if (p.epi == kEpiUp) mode = kUp;
  else if (p.epi == kEpiUpBack) mode = kUpBack;
  else if (p.epi == kEpiRows32) mode = !p.grouped ? kLinDwPart : p.segs == 2 ? kDx : kDown;
  else mode = p.per_unit ? kDw : (a_mn ? kLinDw : kLinDx);
  // Pairs of CTAs share a 256-row tile when there are rows for it: each stages half of B, so a tile's operands cross from
  // L2 once for 256 x 256 sums instead of 128 x 256 (the SM's 64 bytes a clock from L2 bound the single CTA).
  q.pair = p.grouped || p.m > kBM;
  const int cg = q.pair ? 2 : 1;
  q.k_blocks = int(ceil_div(uint64_t(p.k), kBK));
  q.m_tiles = p.grouped ? 0 : int(ceil_div(uint64_t(p.m), uint64_t(cg * kBM)));
  q.splits = splits;
  const int64_t m_tiles = p.grouped ? plan->max_tiles : int64_t(q.m_tiles) * (p.per_unit ? int64_t(plan->units) : splits);
  const bool narrow = mode == kUp || mode == kUpBack;
  q.bn = p.grouped || p.per_unit ? (narrow ? 128 : 256) : columns;
  const int64_t step = 16 * cg;  // a product's columns: whole 16 for one CTA, 32 for a pair
  if (q.bn > (p.n + step - 1) / step * step) q.bn = int((p.n + step - 1) / step * step);
  q.n_tiles = int(ceil_div(uint64_t(p.n), uint64_t(q.bn)));
  q.vec = p.epi == kEpiRows32   ? p.n % 4 == 0
          : p.epi == kEpiUpBack ? on16(p.dg) && on16(p.du) && on16(p.hw) && p.ldo % 8 == 0
                                : on16(p.out) && p.ldo % 8 == 0 && p.out_unit % 8 == 0 && on16(p.bias) &&
                                      on16(p.residual) && p.ldr % 8 == 0 && on16(p.pre) && p.ldp % 8 == 0;
  Maps maps;
  std::memset(&maps, 0, sizeof maps);
  auto shape = [&](const Operand& o, int64_t n_i, int64_t n_k) {
    Shape r{};
    const bool k_inner = o.s_k == 1;
    r.cols = uint64_t(k_inner ? n_k : n_i);
    r.rows = uint64_t(k_inner ? n_i : n_k);
    r.ld = uint64_t(k_inner ? o.s_i : o.s_k);
    r.slots = 1;
    r.p = o.p;
    if (o.part >= 0) {
      r.p = u->part[o.part];
      r.slots = u->n_slots;
      r.slot_bytes = u->stride[o.part];
    }
    return r;
  };
  for (int i = 0; i < p.segs; ++i) {
    // A's maps: one per k loop (gate and up share theirs)
    const int64_t rows = p.grouped ? plan->max_rows : p.m, ks = p.per_unit ? plan->max_rows : p.k;
    const Shape a = shape(p.a[i], rows, ks), b = shape(p.b[i], p.n, ks);
    if (!fits(a) || !fits(b)) return int(cudaErrorInvalidValue);
    const int ia = narrow ? (i == 2 ? 1 : 0) : i;
    if (!make_map(&maps.a[ia], dtype, a.p, a.cols, a.rows, a.ld, a.slots, a.slot_bytes, a_mn ? 64 : kBM) ||
        !make_map(&maps.b[i], dtype, b.p, b.cols, b.rows, b.ld, b.slots, b.slot_bytes,
                  p.b[i].s_k == 1 ? uint32_t(narrow ? q.bn : q.bn / cg) : 64))
      return int(cudaErrorInvalidValue);
  }
  if (q.vec) {  // where the results go, by TMA
    const uint64_t rows = uint64_t(p.grouped ? plan->max_rows : p.m), n = uint64_t(p.n);
    void* const outs[3] = {p.epi == kEpiRows32 ? p.rows32 : p.epi == kEpiUpBack ? p.dg : p.out,
                           p.epi == kEpiUpBack ? p.du : p.pre, p.hw};
    const uint64_t lds[3] = {uint64_t(p.epi == kEpiRows32 ? p.n : p.ldo), uint64_t(p.epi == kEpiUpBack ? p.ldo : p.ldp),
                             uint64_t(p.ldo)};
    const uint64_t slots = p.per_unit ? plan->units : uint64_t(splits);
    const uint64_t slot_bytes = p.per_unit ? uint64_t(p.out_unit) * 2 : rows * n * 4;
    for (int i = 0; i < 3; ++i)
      if (outs[i] && !make_map(&maps.out[i], p.epi == kEpiRows32 ? TSB_F32 : dtype, outs[i], n, rows, lds[i], slots,
                               slot_bytes, 32, true))
        return int(cudaErrorInvalidValue);
  }
  // as many stages as the ring holds: narrow tiles are bound by the loads' latency
  const int b_cols = narrow ? q.bn : q.bn / cg;
  q.stage_bytes = kABytes + int(ceil_div(uint64_t(b_cols), 64)) * 8192;
  q.stages = kRingBytes / q.stage_bytes < kMaxStages ? kRingBytes / q.stage_bytes : kMaxStages;
  const int64_t tiles = m_tiles * q.n_tiles;
  if (tiles >= (int64_t(1) << 30)) return int(cudaErrorInvalidValue);
  const int grid = int(tiles < sms / cg ? tiles : sms / cg);
  switch (mode) {
    case kLin: return go_type<kLin>(dtype, p.act, maps, q, grid, s);
    case kLinDx: return go_type<kLinDx>(dtype, 0, maps, q, grid, s);
    case kLinDw: return go_type<kLinDw>(dtype, 0, maps, q, grid, s);
    case kLinDwPart: return go_type<kLinDwPart>(dtype, 0, maps, q, grid, s);
    case kUp: return go_type<kUp>(dtype, p.act, maps, q, grid, s);
    case kUpBack: return go_type<kUpBack>(dtype, p.act, maps, q, grid, s);
    case kDown: return go_type<kDown>(dtype, 0, maps, q, grid, s);
    case kDx: return go_type<kDx>(dtype, 0, maps, q, grid, s);
    case kDw: return go_type<kDw>(dtype, 0, maps, q, grid, s);
  }
  return int(cudaErrorInvalidValue);
}

int ops_take_timeouts(uint32_t* out) {
  uint32_t v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_ops_timeouts, sizeof v);
  if (e == cudaSuccess && v) {
    const uint32_t zero = 0;
    e = cudaMemcpyToSymbol(g_ops_timeouts, &zero, sizeof zero);
  }
  *out = v;
  return int(e);
}

}  // namespace ops
}  // namespace tsb
