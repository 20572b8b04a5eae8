// The feed-forward block's products on the tensor cores for groups of any length: the unit's matrix supplies the rows of
// the tensor core's tile and the group's rows its columns.
//
// A group's length is known on the device only and is rarely a multiple of 128; as columns a group takes a multiple of 32
// of them, evenly cut (270 rows: three tiles of 96), where as rows it would take whole tiles of 128 or 256. A pair of CTAs
// works on 256 rows of the matrix, 128 each, and each stages half of the group's rows, so that shared memory, which bounds
// small tiles (each staged byte is written and read through the same 128 bytes a clock), moves 88 KB a slice of k for 256
// gate and 256 up rows by 128 rows of x, where single CTAs with the group as rows moved 192 KB.
//
// The rest is as in ops_tc.cu: persistent pairs, a ring of TMA stages, one warp issuing tcgen05.mma, sums in TMEM double
// buffered, eight epilogue warps, TMA stores. Gate and up of a feature lie in the same TMEM lane, 128 columns apart; in
// the backward pass dh comes third and alternates between two column ranges. A lane of the epilogue holds a feature, its
// registers the group's rows; results are transposed through the warp's store buffers.
#include "tc.cuh"

namespace tsb {
namespace ops {
namespace {

__device__ uint32_t g_group_timeouts;

// kLin, kLinDx: one matrix (k contiguous, or its rows contiguous) and host-known rows, as a single group
enum Mode { kUp, kUpBack, kDown, kDx, kLin, kLinDx };

struct Params {
  Plan plan;
  Product p;
  int32_t bm;        // the group's rows a tile at most
  int32_t list;      // which of the plan's tile lists has them
  int32_t f_tiles;   // tiles of 256 rows of the matrix
  int32_t k_blocks;  // of a segment
  int32_t rows;      // kLin, kLinDx: rows of x
  int32_t splits;    // parts of the sum over k, each with its own 32-bit rows
  int32_t split_rows;  // rows of a split's 32-bit rows
  int32_t vec;       // `out` maps are made
  int32_t stages, stage_bytes;
};
struct Maps {
  CUtensorMap a[3], b[2], out[3];
};

struct Tile {
  int slot, row0;        // row0: the tile's first grouped row
  int rows, cols;        // rows of the group to store, and the products' columns (a multiple of 32)
  int f0;
  int split, kb0, kb1;   // its slices of k, over all segments
};

// The launch's tiles: groups in unit order, inside a group chunks of up to 8 tiles of its rows, inside a chunk the matrix'
// tiles, the chunk's row tiles innermost, so that tiles running at the same time share a unit's matrix rows from L2. What
// the plan says of a tile is read one tile ahead.
template <int MODE>
struct Tiles {
  static constexpr bool dense = MODE == kLin || MODE == kLinDx;
  static constexpr bool split = MODE != kUp && MODE != kUpBack;
  int at, end;
  int4 next;
  __device__ __forceinline__ void fetch(const Params& q) {
    if (at < end && !dense) next = q.plan.tiles[q.list][(split ? at / q.splits : at) / q.f_tiles];
  }
  __device__ __forceinline__ Tiles(const Params& q) : at(blockIdx.x / 2), next(make_int4(0, 0, q.rows, 0)) {
    end = (dense ? (q.rows + q.bm - 1) / q.bm : q.plan.head[2 * q.list]) * q.f_tiles * q.splits;
    fetch(q);
  }
  __device__ __forceinline__ bool take(const Params& q, Tile& t) {
    constexpr int kChunk = 8;
    if (at >= end) return false;
    const int4 g = next;
    int L = at;
    at += gridDim.x / 2;
    fetch(q);
    const int all = (MODE == kDx ? 2 : 1) * q.k_blocks;
    t.split = 0, t.kb0 = 0, t.kb1 = all;
    if (split && q.splits > 1) {
      t.split = L % q.splits;
      L /= q.splits;
      t.kb0 = all * t.split / q.splits;
      t.kb1 = all * (t.split + 1) / q.splits;
    }
    const int cnt = dense ? g.z : (g.z + int(q.plan.pad) - 1) / int(q.plan.pad) * int(q.plan.pad);  // padding rows too
    const int tiles = (cnt + q.bm - 1) / q.bm, local = L - g.w * q.f_tiles;
    const int size = ((cnt + tiles - 1) / tiles + 31) & ~31;
    const int chunk = local / (kChunk * q.f_tiles), in = local - chunk * kChunk * q.f_tiles;
    const int width = min(kChunk, tiles - chunk * kChunk);
    const int f = in / width, m0 = (chunk * kChunk + in - f * width) * size;
    t.slot = g.x;
    t.f0 = f * 2 * kBM;
    t.row0 = g.y + m0;
    t.rows = min(size, cnt - m0);
    t.cols = (t.rows + 31) & ~31;
    return true;
  }
};

template <int MODE>
struct Traits {
  static constexpr int segs = MODE == kUpBack ? 2 : 1;  // sums of their own (dx's two matrices add into one)
  static constexpr int bufs = MODE == kUpBack ? 1 : 2;
  __host__ __device__ static constexpr bool both(int s) { return (MODE == kUp && s == 0) || (MODE == kUpBack && s == 1); }
  // the matrix with its rows (of the tile) contiguous
  __host__ __device__ static constexpr bool a_mn(int s) { return MODE == kDx || MODE == kLinDx || (MODE == kUpBack && s == 0); }
  __host__ __device__ static constexpr int a_map(int s) {
    return MODE == kDown || (MODE == kUpBack && s == 0) ? 2 : 0;
  }
  __host__ __device__ static constexpr int b_map(int s) { return MODE == kUpBack ? 1 - s : 0; }
};

// A warp's buffer of rows of the group by its 32 features, on its way out (see ops_tc.cu): 32 rows of 16-bit values, or 16
// of 32-bit ones.
struct Out {
  const CUtensorMap* map;
  char* buf;
  uint32_t flip;
  bool tma;
};
__device__ __forceinline__ char* out_begin(Out& o) {
  char* b = o.buf + (o.flip & 1u) * 2048;
  o.flip ^= 1u;
  if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
  __syncwarp();
  return b;
}
// where lane (feature) `lane` of row r goes: 64-byte rows of 16-bit, 128-byte rows of 32-bit values, swizzled as the maps
template <class E>
__device__ __forceinline__ uint32_t out_at(int r, int lane) {
  if constexpr (sizeof(E) == 2) return uint32_t(r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) * 16) + (lane & 7) * 2);
  else return uint32_t(r * 128 + (((lane >> 2) ^ (r & 7)) * 16) + (lane & 3) * 4);
}
template <class E>
__device__ __forceinline__ void out_end(Out& o, char* b, int which, int x, int y, int z, E* p, int64_t ld, int rows,
                                        int cols) {
  constexpr int kRows = 64 / int(sizeof(E));
  const int lane = threadIdx.x & 31;
  if (o.tma && rows >= kRows && cols > 0) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0)
      asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(o.map + which),
                   "r"(x), "r"(y), "r"(z), "r"(smem_u32(b))
                   : "memory");
  } else {
    __syncwarp();
    for (int r = 0; r < min(rows, kRows); ++r)
      if (lane < cols) p[r * ld + lane] = *reinterpret_cast<const E*>(b + out_at<E>(r, lane));
    __syncwarp();
  }
  if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// 32 values of 32 lanes to the sum over lanes of value `lane`: halves are exchanged five times
__device__ __forceinline__ float lane_sums(float (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const bool hi = lane & o;
      const float send = hi ? v[i] : v[i + o], keep = hi ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  return v[0];
}

template <class T, int MODE, int ACT>
__device__ __forceinline__ void epilogue(const Params& q, const Tile& t, uint32_t tmem, uint32_t tmem_dh, uint32_t rank,
                                         Out& o, int warp) {
  const Product& p = q.p;
  const int lane = threadIdx.x & 31, quad = warp & 3, half = warp >> 2;
  const uint32_t lanes = uint32_t(quad * 32) << 16;
  const int f = t.f0 + int(rank) * kBM + quad * 32;
  const int cols = int(min(int64_t(32), p.n - f));  // features of this warp inside the matrix (may be <= 0)
  if constexpr (MODE == kUp || MODE == kUpBack) {
    for (int c = half * 32; c < t.cols; c += 64) {
      float g[2][16], u[2][16], d[2][16];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        tmem_ld16(tmem + lanes + c + 16 * s, g[s]);
        tmem_ld16(tmem + lanes + 128 + c + 16 * s, u[s]);
        if constexpr (MODE == kUpBack) tmem_ld16(tmem_dh + lanes + c + 16 * s, d[s]);
      }
      const int rows = min(32, t.rows - c);
      const int y = t.row0 + c;
      float w = 0.f;  // of row c + lane
      if (MODE == kUpBack && lane < rows) {
        const int32_t pair = q.plan.pair_of_row[y + lane];
        w = pair < 0 ? 0.f : p.weights[pair];
      }
      tmem_wait_ld();
      const int64_t at = int64_t(y) * p.ldo + f;
      if constexpr (MODE == kUp) {
        char* b = out_begin(o);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            *reinterpret_cast<T*>(b + out_at<T>(16 * s + i, lane)) = from_f<T>(act_of<ACT>(g[s][i]) * u[s][i]);
        out_end<T>(o, b, 0, f, y, 0, static_cast<T*>(p.out) + at, p.ldo, rows, cols);
      } else {
        float dw[32];
        char* b = out_begin(o);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int r = 16 * s + i;
            const float wr = __shfl_sync(0xffffffffu, w, r), k = act_of<ACT>(g[s][i]), dh = d[s][i];
            dw[r] = dh * k * u[s][i];
            *reinterpret_cast<T*>(b + out_at<T>(r, lane)) = from_f<T>(wr * dh * u[s][i] * slope_of<ACT>(g[s][i]));
            d[s][i] = wr * dh * k;
            g[s][i] = wr * k * u[s][i];
          }
        out_end<T>(o, b, 0, f, y, 0, static_cast<T*>(p.dg) + at, p.ldo, rows, cols);
        b = out_begin(o);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 16; ++i) *reinterpret_cast<T*>(b + out_at<T>(16 * s + i, lane)) = from_f<T>(d[s][i]);
        out_end<T>(o, b, 1, f, y, 0, static_cast<T*>(p.du) + at, p.ldo, rows, cols);
        if (p.hw) {
          b = out_begin(o);
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 16; ++i) *reinterpret_cast<T*>(b + out_at<T>(16 * s + i, lane)) = from_f<T>(g[s][i]);
          out_end<T>(o, b, 2, f, y, 0, static_cast<T*>(p.hw) + at, p.ldo, rows, cols);
        }
        if (p.dwp) {  // features outside the matrix have u = 0
          const float sum = lane_sums(dw);
          if (lane < rows) p.dwp[int64_t(y + lane) * p.ld_dwp + f / 32] = sum;
        }
      }
    }
  } else {
    for (int c = half * 16; c < t.cols; c += 32) {
      float v[16];
      tmem_ld16(tmem + lanes + c, v);
      tmem_wait_ld();
      char* b = out_begin(o);
#pragma unroll
      for (int i = 0; i < 16; ++i) *reinterpret_cast<float*>(b + out_at<float>(i, lane)) = v[i];
      const int y = t.row0 + c;
      out_end<float>(o, b, 0, f, y, t.split, p.rows32 + (int64_t(t.split) * q.split_rows + y) * p.n + f, p.n, t.rows - c,
                     cols);
    }
  }
}

template <class T, int MODE, int ACT>
__global__ __launch_bounds__(kThreads, 1) void group_kernel(const __grid_constant__ Maps maps,
                                                            const __grid_constant__ Params q) {
  using X = Traits<MODE>;
  extern __shared__ char raw[];
  char* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  char* store = smem + kRingBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(store + kEpiWarps * kStoreBytes);
  const uint32_t full = smem_u32(bars), empty = full + 8 * kMaxStages, sums_full = empty + 8 * kMaxStages,
                 sums_empty = sums_full + 16;
  uint32_t* words = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStages + 4);
  volatile uint32_t* dead = words + 1;
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0);
  const uint32_t rank = cta_rank(), stages = uint32_t(q.stages), stage_bytes = uint32_t(q.stage_bytes);
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < stages; ++s) {
      bar_init(full + 8 * s, 1);
      bar_init(empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      bar_init(sums_full + 8 * b, 1);
      bar_init(sums_empty + 8 * b, 2 * kEpiWarps);
    }
    words[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(words)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  cluster_sync();
  fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(words);
  begin_after();

  if (warp == 0) {  // the loads: 128 rows of the matrix and half of the group's rows, arriving at the first CTA's barrier
    uint32_t it = 0, st = 0, parity = 1;
    bool ok = true;
    Tile t;
    const uint32_t ring = smem_u32(smem), arrive = in_cta(full, 0);
    for (Tiles<MODE> tiles(q); ok && tiles.take(q, t);) {
      const int boxes = t.cols / 32;  // of 16 rows
      const int r0 = t.row0 + int(rank) * (t.cols / 2), f0 = t.f0 + int(rank) * kBM;
#pragma unroll
      for (int s = 0; s < X::segs; ++s) {
        constexpr int kA = kABytes;
        const int a_bytes = X::both(s) ? 2 * kA : kA;
        const uint32_t bytes = uint32_t(a_bytes + boxes * 2048);
        const CUtensorMap *ma = &maps.a[X::a_map(s)], *mb = &maps.b[X::b_map(s)];
        int k0 = t.kb0 * kBK;
        for (int kb = t.kb0; kb < t.kb1; ++kb, k0 += kBK) {
          if (MODE == kDx && kb >= q.k_blocks && mb == maps.b)  // on to up's matrix and du
            ma = maps.a + 1, mb = maps.b + 1, k0 -= q.k_blocks * kBK;
          ok = bar_wait(empty + 8 * st, parity, dead);
          if (!ok) break;
          const uint32_t sa = ring + st * stage_bytes, sb = sa + a_bytes, bar = arrive + 8 * st;
          if (elect()) {
            if (rank == 0) bar_expect(bar, 2 * bytes);
            if (X::a_mn(s)) {
              tma_load<2>(sa, ma, f0, k0, t.slot, bar);
              tma_load<2>(sa + 8192, ma, f0 + 64, k0, t.slot, bar);
            } else {
              tma_load<2>(sa, ma, k0, f0, t.slot, bar);
              if (X::both(s)) tma_load<2>(sa + kA, &maps.a[1], k0, f0, t.slot, bar);
            }
            for (int b = 0; b < boxes; ++b) tma_load<2>(sb + b * 2048, mb, k0, r0 + 16 * b, 0, bar);
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
    constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t ring = smem_u32(smem);
    for (Tiles<MODE> tiles(q); ok && tiles.take(q, t); ++nt) {
      const int buf = nt % X::bufs;
#pragma unroll
      for (int s = 0; s < X::segs; ++s) {
        // (dh of tile nt goes where tile nt - 2 had its own: read before tile nt - 1's gate and up could start)
        if (MODE != kUpBack || s == 1) {
          ok = ok && bar_wait(sums_empty + 8 * buf, ((nt / X::bufs) & 1) ^ 1, dead);
          if (!ok) break;
        }
        fence_after();
        const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | (uint32_t(X::a_mn(s)) << 15) |
                               (uint32_t(t.cols >> 3) << 17) | (uint32_t(2 * kBM >> 4) << 24);
        const uint32_t d = tmem + (MODE == kUpBack && s == 0 ? 256 + 128 * (nt & 1) : buf * 256);
        const uint64_t ring_a = desc(ring, X::a_mn(s)), ring_a2 = desc(ring + kABytes, false),
                       ring_b = desc(ring + (X::both(s) ? 2 : 1) * kABytes, false);
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          ok = bar_wait(full + 8 * st, parity, dead);
          if (!ok) break;
          fence_after();
          const uint32_t at = st * (stage_bytes >> 4);
          if (elect()) {
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) {
              const bool add = kb > t.kb0 || k > 0;
              mma<2>(d, ring_a + at + uint64_t((X::a_mn(s) ? 2048 : 32) * k >> 4), ring_b + at + uint64_t(32 * k >> 4),
                     idesc, add);
              if (X::both(s)) mma<2>(d + 128, ring_a2 + at + uint64_t(32 * k >> 4), ring_b + at + uint64_t(32 * k >> 4),
                                     idesc, add);
            }
            commit<2>(empty + 8 * st);
          }
          ++it;
          if (++st == stages) st = 0, parity ^= 1;
        }
        if (!ok) break;
      }
      if (ok && elect()) commit<2>(sums_full + 8 * buf);
    }
    if (!ok && it) {  // the products already issued read shared memory and TMEM: let them end
      volatile uint32_t none = 0;
      (void)bar_wait(empty + 8 * ((it - 1) % stages), ((it - 1) / stages) & 1, &none);
    }
  } else if (warp >= 4) {  // the epilogue
    uint32_t nt = 0;
    Tile t;
    Out out{maps.out, store + (warp - 4) * kStoreBytes, 0, q.vec != 0};
    for (Tiles<MODE> tiles(q); tiles.take(q, t); ++nt) {
      const int buf = nt % X::bufs;
      if (!bar_wait(sums_full + 8 * buf, (nt / X::bufs) & 1, dead)) break;
      __syncwarp();
      fence_after();
      epilogue<T, MODE, ACT>(q, t, tmem + buf * 256, tmem + 256 + 128 * (nt & 1), rank, out, warp - 4);
      fence_before();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) bar_arrive_cluster(in_cta(sums_empty + 8 * buf, 0));
    }
    if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA's memory goes while the other's copies, products or arrivals use it
  fence_after();
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    if ((threadIdx.x & 31) == 0 && *dead) atomicAdd(&g_group_timeouts, 1u);
  }
}

template <class T, int MODE, int ACT>
int go(const Maps& maps, const Params& q, int pairs, cudaStream_t s) {
  static std::atomic<uint64_t> devices{0};
  const auto kernel = group_kernel<T, MODE, ACT>;
  if (const int e = allow_smem(reinterpret_cast<const void*>(kernel), devices)) return e;
  return launch(kernel, unsigned(pairs * 2), kThreads, kSmemBytes, 2, s, maps, q);
}
template <class T, int MODE>
int go_act(int act, const Maps& maps, const Params& q, int pairs, cudaStream_t s) {
  switch (act) {
    case TSB_ACT_SILU: return go<T, MODE, TSB_ACT_SILU>(maps, q, pairs, s);
    case TSB_ACT_GELU: return go<T, MODE, TSB_ACT_GELU>(maps, q, pairs, s);
    case TSB_ACT_GELU_TANH: return go<T, MODE, TSB_ACT_GELU_TANH>(maps, q, pairs, s);
    case TSB_ACT_RELU: return go<T, MODE, TSB_ACT_RELU>(maps, q, pairs, s);
  }
  return go<T, MODE, TSB_ACT_NONE>(maps, q, pairs, s);
}
template <class T>
int go_mode(Mode mode, int act, const Maps& maps, const Params& q, int pairs, cudaStream_t s) {
  switch (mode) {
    case kUp: return go_act<T, kUp>(act, maps, q, pairs, s);
    case kUpBack: return go_act<T, kUpBack>(act, maps, q, pairs, s);
    case kDown: return go<T, kDown, 0>(maps, q, pairs, s);
    case kDx: return go<T, kDx, 0>(maps, q, pairs, s);
    case kLin: return go<T, kLin, 0>(maps, q, pairs, s);
    case kLinDx: return go<T, kLinDx, 0>(maps, q, pairs, s);
  }
  return int(cudaErrorInvalidValue);
}

}  // namespace

int launch_group(int dtype, const Product& p, int splits, const Plan* plan, const Units* u, cudaStream_t s) {
  if (!encoder()) return int(cudaErrorNotSupported);
  const int sms = sm_count();
  if (!sms) return int(cudaErrorInvalidDevice);
  Params q{};
  q.p = p;
  const bool rows32 = p.epi == kEpiRows32;
  Mode mode;
  if (!plan) mode = p.b[0].s_k == 1 ? kLin : kLinDx;
  else mode = p.epi == kEpiUp ? kUp : p.epi == kEpiUpBack ? kUpBack : p.segs == 2 ? kDx : kDown;
  // gate and up (and dh) share TMEM: 128 columns each; one product's sums take 256
  q.list = rows32 ? 1 : 0;
  q.bm = int(kGroupRows << q.list);
  if (plan) q.plan = *plan;
  q.rows = int(p.m);
  q.splits = splits;
  q.split_rows = plan ? int(plan->max_rows) : int(p.m);
  q.f_tiles = int(ceil_div(uint64_t(p.n), 2 * kBM));
  q.k_blocks = int(ceil_div(uint64_t(p.k), kBK));
  q.vec = rows32 ? p.n % 4 == 0 : mode == kUp ? on16(p.out) && p.ldo % 8 == 0
                                              : on16(p.dg) && on16(p.du) && on16(p.hw) && p.ldo % 8 == 0;
  Maps maps;
  std::memset(&maps, 0, sizeof maps);
  for (int i = 0; i < p.segs; ++i) {
    const Operand &b = p.a[i], &a = p.b[i];  // (the group's rows are the products' second operand here)
    const bool k_inner = a.s_k == 1;
    const int part = a.part < 0 ? 0 : a.part;
    if (!make_map(&maps.a[part], dtype, plan ? u->part[part] : a.p, uint64_t(k_inner ? p.k : p.n),
                  uint64_t(k_inner ? p.n : p.k), uint64_t(k_inner ? a.s_i : a.s_k), plan ? u->n_slots : 1,
                  plan ? u->stride[part] : 0, k_inner ? kBM : 64) ||
        !make_map(&maps.b[mode == kUpBack ? i / 2 : mode == kDx ? i : 0], dtype, b.p, uint64_t(p.k),
                  uint64_t(q.split_rows), uint64_t(b.s_i), 1, 0, 16))
      return int(cudaErrorInvalidValue);
  }
  if (q.vec) {
    void* const outs[3] = {rows32 ? p.rows32 : mode == kUp ? p.out : p.dg, p.du, p.hw};
    for (int i = 0; i < 3; ++i)
      if (outs[i] && !make_map(&maps.out[i], rows32 ? TSB_F32 : dtype, outs[i], uint64_t(p.n), uint64_t(q.split_rows),
                               uint64_t(rows32 ? p.n : p.ldo), uint64_t(splits), uint64_t(q.split_rows) * uint64_t(p.n) * 4,
                               rows32 ? 16 : 32, !rows32))
        return int(cudaErrorInvalidValue);
  }
  q.stage_bytes = q.list == 0 ? 2 * kABytes + 8192 : 2 * kABytes;
  q.stages = kRingBytes / q.stage_bytes;
  const int64_t tiles = (plan ? int64_t(plan->max_tiles) : int64_t(ceil_div(uint64_t(p.m), uint64_t(q.bm)))) * q.f_tiles * splits;
  if (tiles >= (int64_t(1) << 30)) return int(cudaErrorInvalidValue);
  const int pairs = int(tiles < sms / 2 ? tiles : sms / 2);
  return dtype == TSB_BF16 ? go_mode<__nv_bfloat16>(mode, p.act, maps, q, pairs, s)
                           : go_mode<__half>(mode, p.act, maps, q, pairs, s);
}

int group_take_timeouts(uint32_t* out) {
  uint32_t v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_group_timeouts, sizeof v);
  if (e == cudaSuccess && v) {
    const uint32_t zero = 0;
    e = cudaMemcpyToSymbol(g_group_timeouts, &zero, sizeof zero);
  }
  *out = v;
  return int(e);
}

}  // namespace ops
}  // namespace tsb
