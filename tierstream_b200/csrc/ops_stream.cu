// The products for few rows: y[r][n] = sum_k x[r][k] w[n][k] with at most 8 rows of a group at a time, so the weights'
// bytes bound it and the design is about keeping them in flight.
//
// The weights never touch shared memory. A warp's 16 x 64 block of weights is two 32-byte loads a lane, taken as mma
// fragments as they come: the order of k inside a sum is free, so lane (q, t) holds elements 16 t .. 16 t + 15 of its rows
// and of the x rows alike, and words 2 j and 2 j + 1 of each feed the j-th m16n8k16. Whole 128-byte lines of eight rows
// per load and the 256-byte L2 hint matter: with 16-byte loads (64 bytes of a row each) one token through two 352 MB
// units took 167 us, with these 115 us (90 % of the measured copy rate over both products). The eight rows of x (the n
// side of the mma) come through L1, which they fit. For gate and up the 16 rows are 8 of each, so that both halves of a
// result end in the same CTA. (More rows of x a tile, with more rows of w a warp to pay for them, lost to the tensor
// cores' own path at every size tried: 143 us against 35 us for 24 rows of 8192 x 8192.)
//
// Between the block's two products act(g) u is kept as two 16-bit values, its rounding and what that left out, which both
// meet the down matrix' fragments: the weights' loads stay the bound, and the middle is as good as 32 bits.
//
// A CTA of four warps owns 16 rows of w (8 of gate and up) and splits k over its warps, a cluster of up to 8 CTAs splits
// it further when there are few rows of w; the sums are added in a fixed order through (distributed) shared memory.
#include "ops.hpp"

namespace tsb {
namespace ops {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kStep = 64, kUnroll = 2, kSpan = kStep * kUnroll;
enum Mode { kLin, kUp, kDown };

struct Params {
  Plan plan;
  Units units;
  Product p;
  const void* x;
  const void* w;
  int64_t ldx, ldw;
  int32_t top;  // kUp: row r of the group is row pair / top of x
  int32_t splits;
};

// sixteen 16-bit values
struct Words {
  uint32_t w[8];
};
// WIDE: rows start on 32 bytes and hold whole sixteens; else on 16 bytes, and `left` elements of the row remain
template <bool WIDE>
__device__ __forceinline__ Words load_weights(const void* p, int64_t left) {
  Words v{};
  if (left <= 0) return v;
  if constexpr (WIDE) {
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]),
                   "=r"(v.w[7])
                 : "l"(p));
  } else {
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3])
                 : "l"(p));
    if (left > 8)
      asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
                   : "l"(static_cast<const char*>(p) + 16));
  }
  return v;
}
template <bool WIDE>
__device__ __forceinline__ Words load_x(const void* p, int64_t left) {
  Words v{};
  if (left > 0) *reinterpret_cast<uint4*>(v.w) = *static_cast<const uint4*>(p);
  if (left > (WIDE ? 0 : 8)) *reinterpret_cast<uint4*>(v.w + 4) = static_cast<const uint4*>(p)[1];
  return v;
}
template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_float(const float* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(uint32_t(__cvta_generic_to_shared(p))), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

template <class T, int MODE, bool WIDE>
__global__ __launch_bounds__(kThreads) void stream_kernel(const __grid_constant__ Params q) {
  constexpr int kHalf = 8, kRows = MODE == kUp ? kHalf : 2 * kHalf, kTok = kStreamTile;
  __shared__ float red[kWarps][2 * kHalf][kTok + 1];
  __shared__ float sum[2 * kHalf][kTok + 1];
  begin_after();
  const Product& p = q.p;
  const uint32_t rank = blockIdx.x % uint32_t(q.splits);
  const int64_t n0 = int64_t(blockIdx.x / uint32_t(q.splits)) * kRows;
  int32_t row0 = int32_t(blockIdx.y) * kTok;
  int rows;
  const T *w0, *w1;  // of each pair of 8-row blocks; w1's rows are up's, or the next 8 MT rows of w
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  int64_t ldw;
  if constexpr (MODE == kLin) {
    rows = int(min(int64_t(kTok), p.m - row0));
    ldw = q.ldw;
    w0 = static_cast<const T*>(q.w);
    w1 = w0 + kHalf * ldw;
  } else {
    const int4 info = q.plan.tiles[0][blockIdx.y];
    rows = min(kTok, info.z - (int(blockIdx.y) - info.w) * kTok);
    if (!info.z) return;  // (every CTA of the cluster leaves)
    row0 = info.y + (int(blockIdx.y) - info.w) * kTok;
    ldw = p.k;
    w0 = reinterpret_cast<const T*>(unit_part(q.units, MODE == kUp ? 0 : 2, info.x));
    w1 = MODE == kUp ? reinterpret_cast<const T*>(unit_part(q.units, 1, info.x)) : w0 + kHalf * ldw;
  }
  w0 += (n0 + g) * ldw + 16 * t;
  w1 += (n0 + g) * ldw + 16 * t;
  const bool in0 = n0 + g < p.n, in1 = MODE == kUp ? in0 : n0 + kHalf + g < p.n, inx = g < rows;
  int64_t src = inx ? row0 + g : row0;
  if constexpr (MODE == kUp) src = q.plan.pair_of_row[src] / q.top;
  const T* xr = static_cast<const T*>(q.x) + src * q.ldx + 16 * t;
  float acc[4] = {};
  for (int64_t k0 = (int64_t(rank) * kWarps + warp) * kSpan; k0 < p.k; k0 += int64_t(q.splits) * kWarps * kSpan) {
    Words a[kUnroll], b[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t k = k0 + u * kStep, left = p.k - k - 16 * t;
      a[u] = load_weights<WIDE>(w0 + k, in0 ? left : 0);
      b[u] = load_weights<WIDE>(w1 + k, in1 ? left : 0);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t k = k0 + u * kStep, left = p.k - k - 16 * t;
#pragma unroll
      for (int part = 0; part < (MODE == kDown ? 2 : 1); ++part) {
        const Words x = load_x<WIDE>(xr + k + part * p.k, inx ? left : 0);
#pragma unroll
        for (int h = 0; h < 4; ++h)
          mma16816<T>(acc, a[u].w[2 * h], b[u].w[2 * h], a[u].w[2 * h + 1], b[u].w[2 * h + 1], x.w[2 * h],
                      x.w[2 * h + 1]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) red[warp][g + kHalf * (e >> 1)][2 * t + (e & 1)] = acc[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * kHalf * kTok; i += kThreads) {
    const int c = i % (2 * kHalf), r = i / (2 * kHalf);
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += red[w][c][r];
    sum[c][r] = s;
  }
  if (q.splits > 1) {
    cluster_sync();
    if (rank == 0)
      for (int i = threadIdx.x; i < 2 * kHalf * kTok; i += kThreads) {
        const int c = i % (2 * kHalf), r = i / (2 * kHalf);
        float s = sum[c][r];
        for (int o = 1; o < q.splits; ++o) s += peer_float(&sum[c][r], uint32_t(o));
        sum[c][r] = s;
      }
    cluster_sync();  // the other CTAs' sums stay until they are read
    if (rank) return;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * kTok; i += kThreads) {
    const int c = i % kRows, r = i / kRows;
    const int64_t n = n0 + c;
    if (r >= rows || n >= p.n) continue;
    const float z0 = sum[c][r];
    if constexpr (MODE == kUp) {
      T* out = static_cast<T*>(p.out) + (int64_t(row0) + r) * p.ldo + n;
      const float h = act_rt(p.act, z0) * sum[c + kHalf][r];
      const T hi = from_f<T>(h);
      const float lo = h - to_f(hi);
      out[0] = hi;
      out[p.n] = from_f<T>(lo - lo == 0.f ? lo : 0.f);  // (nothing is left out of an infinity or a NaN)
    } else if constexpr (MODE == kDown) {
      p.rows32[(int64_t(row0) + r) * p.n + n] = z0;
    } else {
      const int64_t m = int64_t(row0) + r;
      const float z = z0 + (p.bias ? to_f(static_cast<const T*>(p.bias)[n]) : 0.f);
      if (p.pre) static_cast<T*>(p.pre)[m * p.ldp + n] = from_f<T>(z);
      float y = act_rt(p.act, z);
      if (p.residual) y += to_f(static_cast<const T*>(p.residual)[m * p.ldr + n]);
      static_cast<T*>(p.out)[m * p.ldo + n] = from_f<T>(y);
    }
  }
}

template <class T, int MODE>
int go(bool wide, const Params& q, dim3 grid, cudaStream_t s) {
  return launch(wide ? stream_kernel<T, MODE, true> : stream_kernel<T, MODE, false>, grid, kThreads, 0, q.splits, s,
                q);
}

// CTAs of a cluster that split k: enough that the GPU's 148 SMs hold about six CTAs each, as long as a warp keeps a span
// of k (linear_logits-like 128 x 4096 for one row: 8 splits).
int splits_for(int64_t ctas, int64_t k) {
  int s = 1;
  while (s < 8 && ctas * s < 888 && k > int64_t(s) * kWarps * kSpan) s *= 2;
  return s;
}

}  // namespace

int launch_stream(int dtype, const Product& p, uint32_t top, const Plan* plan, const Units* u,
                  cudaStream_t s) {
  Params q{};
  q.p = p;
  q.x = p.a[0].p;
  q.ldx = p.a[0].s_i;
  q.top = int32_t(top);
  const Mode mode = p.epi == kEpiLinear ? kLin : p.epi == kEpiUp ? kUp : kDown;
  int64_t m_tiles = 0;
  if (mode == kLin) {
    q.w = p.b[0].p;
    q.ldw = p.b[0].s_i;
    m_tiles = int64_t(ceil_div(uint64_t(p.m), kStreamTile));
  } else {
    q.plan = *plan;
    q.units = *u;
    m_tiles = plan->max_tiles;
  }
  const int64_t n_tiles = int64_t(ceil_div(uint64_t(p.n), uint64_t(mode == kUp ? 8 : 16)));
  // 32-byte loads: the rows of w on 32 bytes
  auto on32 = [](const void* v, uint64_t stride) { return ((reinterpret_cast<uintptr_t>(v) | stride) & 31u) == 0; };
  bool wide = p.k % 16 == 0;
  if (mode == kLin) wide = wide && on32(q.w, uint64_t(q.ldw) * 2);
  else if (u->table) wide = false;
  else
    for (int i = mode == kUp ? 0 : 2; i < (mode == kUp ? 2 : 3); ++i) wide = wide && on32(u->part[i], u->stride[i]);
  q.splits = splits_for(m_tiles * n_tiles, p.k);
  const dim3 grid(unsigned(n_tiles * q.splits), unsigned(m_tiles));
  if (dtype == TSB_BF16)
    return mode == kLin ? go<__nv_bfloat16, kLin>(wide, q, grid, s)
           : mode == kUp ? go<__nv_bfloat16, kUp>(wide, q, grid, s)
                         : go<__nv_bfloat16, kDown>(wide, q, grid, s);
  return mode == kLin ? go<__half, kLin>(wide, q, grid, s)
         : mode == kUp ? go<__half, kUp>(wide, q, grid, s)
                       : go<__half, kDown>(wide, q, grid, s);
}

}  // namespace ops
}  // namespace tsb
