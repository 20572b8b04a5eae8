// The products for few rows: y[r][n] = sum_k x[r][k] w[n][k] with at most 8 NT rows of a group at a time, so the weights'
// bytes bound it and the design is about keeping them in flight.
//
// The weights never touch shared memory. A warp's 16 x 32 block of weights is two 16-byte loads a lane, taken as mma
// fragments as they come: the order of k inside a sum is free, so lane (q, t) holds elements 8 t .. 8 t + 7 of its rows
// and of the x rows alike, and words 2 j and 2 j + 1 of each feed the j-th m16n8k16. Eight such loads are in flight per
// lane before the first is used. The rows of x (the n side of the mma, 8 a tile) come through L1, which they fit.
// For gate and up the 16 rows are 8 of each, so that both halves of a result end in the same CTA.
//
// A CTA of four warps owns 16 rows of w (8 of gate and up) and splits k over its warps, a cluster of up to 8 CTAs splits
// it further when there are few rows of w; the sums are added in a fixed order through (distributed) shared memory.
#include "ops.hpp"

namespace tsb {
namespace ops {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kStep = 32, kUnroll = 4, kSpan = kStep * kUnroll;
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

__device__ __forceinline__ uint4 load_weights(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
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
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
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

template <class T, int MODE, int NT>
__global__ __launch_bounds__(kThreads) void stream_kernel(const __grid_constant__ Params q) {
  constexpr int kRows = MODE == kUp ? 8 : 16, kTok = 8 * NT;
  __shared__ float red[kWarps][16][kTok + 1];
  __shared__ float sum[16][kTok + 1];
  const Product& p = q.p;
  const uint32_t rank = blockIdx.x % uint32_t(q.splits);
  const int64_t n0 = int64_t(blockIdx.x / uint32_t(q.splits)) * kRows;
  int32_t unit = 0, row0 = int32_t(blockIdx.y) * kTok;
  int rows;
  const T *w0, *w1;  // the lane's two rows of w
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const bool in0 = n0 + g < p.n, in1 = MODE == kUp ? in0 : n0 + g + 8 < p.n;
  int64_t ldw;
  if constexpr (MODE == kLin) {
    rows = int(min(int64_t(kTok), p.m - row0));
    ldw = q.ldw;
    w0 = static_cast<const T*>(q.w);
    w1 = w0 + 8 * ldw;
  } else {
    const int4 info = q.plan.tile_info[blockIdx.y];  // slot, first row, rows, unit
    rows = info.z;
    if (rows <= 0) return;  // (every CTA of the cluster leaves)
    row0 = info.y;
    unit = info.w;
    ldw = p.k;
    w0 = reinterpret_cast<const T*>(unit_part(q.units, MODE == kUp ? 0 : 2, unit, info.x));
    w1 = MODE == kUp ? reinterpret_cast<const T*>(unit_part(q.units, 1, unit, info.x)) : w0 + 8 * ldw;
  }
  w0 += (n0 + g) * ldw + 8 * t;
  w1 += (n0 + g) * ldw + 8 * t;
  const T* xr[NT];
  bool inx[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = 8 * j + g;
    inx[j] = r < rows;
    int64_t src = inx[j] ? row0 + r : row0;
    if constexpr (MODE == kUp) src = q.plan.pair_of_row[src] / q.top;
    xr[j] = static_cast<const T*>(q.x) + src * q.ldx + 8 * t;
  }
  float acc[NT][4] = {};
  for (int64_t k0 = (int64_t(rank) * kWarps + warp) * kSpan; k0 < p.k; k0 += int64_t(q.splits) * kWarps * kSpan) {
    uint4 a[kUnroll], b[kUnroll];
    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t k = k0 + u * kStep;
      const bool in = k + 8 * t < p.k;  // (k is a multiple of 8)
      a[u] = in && in0 ? load_weights(w0 + k) : zero;
      b[u] = in && in1 ? load_weights(w1 + k) : zero;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t k = k0 + u * kStep;
      const bool in = k + 8 * t < p.k;
      uint4 x[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) x[j] = in && inx[j] ? *reinterpret_cast<const uint4*>(xr[j] + k) : zero;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          mma16816<T>(acc[j], word(a[u], 2 * h), word(b[u], 2 * h), word(a[u], 2 * h + 1), word(b[u], 2 * h + 1),
                      word(x[j], 2 * h), word(x[j], 2 * h + 1));
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[warp][g + 8 * (i >> 1)][8 * j + 2 * t + (i & 1)] = acc[j][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * kTok; i += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += red[w][i % 16][i / 16];
    sum[i % 16][i / 16] = s;
  }
  if (q.splits > 1) {
    cluster_sync();
    if (rank == 0)
      for (int i = threadIdx.x; i < 16 * kTok; i += kThreads) {
        float s = sum[i % 16][i / 16];
        for (int r = 1; r < q.splits; ++r) s += peer_float(&sum[i % 16][i / 16], uint32_t(r));
        sum[i % 16][i / 16] = s;
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
      static_cast<T*>(p.out)[(int64_t(row0) + r) * p.ldo + n] = from_f<T>(act_rt(p.act, z0) * sum[c + 8][r]);
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

template <class T, int MODE, int NT>
int go(const Params& q, dim3 grid, cudaStream_t s) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = dim3(kThreads);
  c.stream = s;
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeClusterDimension;
  a[0].val.clusterDim.x = unsigned(q.splits);
  a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
  c.attrs = a;
  c.numAttrs = 1;
  return int(cudaLaunchKernelEx(&c, stream_kernel<T, MODE, NT>, q));
}
template <class T, int MODE>
int go_rows(int nt, const Params& q, dim3 grid, cudaStream_t s) {
  return nt == 1 ? go<T, MODE, 1>(q, grid, s) : nt == 2 ? go<T, MODE, 2>(q, grid, s) : go<T, MODE, 4>(q, grid, s);
}

// CTAs of a cluster that split k: enough that the GPU's 148 SMs hold about six CTAs each, as long as a warp keeps a span
// of k (linear_logits-like 128 x 4096 for one row: 8 splits).
int splits_for(int64_t ctas, int64_t k) {
  int s = 1;
  while (s < 8 && ctas * s < 888 && k > int64_t(s) * kWarps * kSpan) s *= 2;
  return s;
}

}  // namespace

int launch_stream(int dtype, const Product& p, uint32_t rows_a_tile, uint32_t top, const Plan* plan, const Units* u,
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
    m_tiles = int64_t(ceil_div(uint64_t(p.m), rows_a_tile));
  } else {
    q.plan = *plan;
    q.units = *u;
    m_tiles = plan->max_tiles;
  }
  const int64_t n_tiles = int64_t(ceil_div(uint64_t(p.n), mode == kUp ? 8 : 16));
  q.splits = splits_for(m_tiles * n_tiles, p.k);
  const dim3 grid(unsigned(n_tiles * q.splits), unsigned(m_tiles));
  const int nt = int(rows_a_tile / 8);
  if (dtype == TSB_BF16)
    return mode == kLin ? go_rows<__nv_bfloat16, kLin>(nt, q, grid, s)
           : mode == kUp ? go_rows<__nv_bfloat16, kUp>(nt, q, grid, s)
                         : go_rows<__nv_bfloat16, kDown>(nt, q, grid, s);
  return mode == kLin ? go_rows<__half, kLin>(nt, q, grid, s)
         : mode == kUp ? go_rows<__half, kUp>(nt, q, grid, s)
                       : go_rows<__half, kDown>(nt, q, grid, s);
}

}  // namespace ops
}  // namespace tsb
