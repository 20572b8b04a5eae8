// The feed-forward block's products for every size, stride and alignment: C[m][n] = sum_k A[m][k] B[n][k] with up to three
// operand pairs and three accumulators, rows gathered through the plan, the matrices of a unit found through its slot, and
// the epilogues of ops.hpp. One CTA of four warps computes a 64 x 64 tile from 32-wide slices of k staged in shared memory
// by element loads along whichever index is contiguous; the products run on mma.sync with 32-bit sums. The element loads
// bound it (8.6 TFLOP/s for a prompt of 2047 rows over 128 units): it serves what the other kernels refuse, units whose
// rows do not start on 16 bytes and gradients of units found by address.
#include "ops.hpp"

namespace tsb {
namespace ops {
namespace {

constexpr int kThreads = 128, kBK = 32, kLd = kBK + 8;  // 80-byte rows: the fragments' 32-bit reads meet no bank twice

template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

struct Group {
  int32_t unit, slot, row0;  // row0: the group's first grouped row
  int64_t rows;
};

// 64 x 32 elements of an operand into registers: lanes along the contiguous index.
template <class T>
__device__ __forceinline__ void fetch(const Operand& o, const T* p, int64_t i0, int64_t n_i, int64_t k0, int64_t n_k,
                                      int32_t row0, T (&v)[16]) {
  const bool along_k = o.s_k == 1;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int e = threadIdx.x + j * kThreads;
    const int64_t i = i0 + (along_k ? e / kBK : e % 64), k = k0 + (along_k ? e % kBK : e / 64);
    v[j] = from_f<T>(0.f);
    if (i < n_i && k < n_k) {
      int64_t gi = i, gk = k;
      bool there = true;
      if (o.map) {
        const int32_t r = o.map[row0 + (o.map_k ? k : i)];
        there = r >= 0;
        (o.map_k ? gk : gi) = r / o.div;
      } else if (o.part < 0) {
        (o.map_k ? gk : gi) += row0;  // a grouped buffer
      }
      if (there) v[j] = p[gi * o.s_i + gk * o.s_k];
    }
  }
}
template <class T>
__device__ __forceinline__ void put(const Operand& o, const T (&v)[16], T* s) {
  const bool along_k = o.s_k == 1;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int e = threadIdx.x + j * kThreads;
    s[(along_k ? e / kBK : e % 64) * kLd + (along_k ? e % kBK : e / 64)] = v[j];
  }
}

template <class T, int NACC>
__global__ __launch_bounds__(kThreads) void tile_kernel(const __grid_constant__ Product p,
                                                        const __grid_constant__ Plan plan,
                                                        const __grid_constant__ Units units) {
  __shared__ __align__(16) T sa[64 * kLd];
  __shared__ __align__(16) T sb[64 * kLd];
  __shared__ float red[2][64];
  begin_after();
  Group g{};
  int64_t m0 = int64_t(blockIdx.x) * 64;
  if (p.grouped) {
    const int4 i = plan.tiles[0][blockIdx.x];
    if (!i.z) return;
    g.slot = i.x;
    g.row0 = i.y;
    g.rows = i.z;
    m0 = int64_t(int(blockIdx.x) - i.w) * 64;
  } else {  // a matrix per unit
    g.unit = blockIdx.z;
    g.rows = plan.cnt[g.unit];
    g.row0 = plan.off[g.unit];
    g.slot = plan.slot[g.unit];
  }
  const int64_t n0 = int64_t(blockIdx.y) * 64;
  const int64_t n_m = p.grouped ? g.rows : p.m, n_k = p.k_rows ? g.rows : p.k;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane >> 2, t = lane & 3;
  const int wm = (warp & 1) * 32, wn = (warp >> 1) * 32;
  float acc[NACC][2][4][4] = {};
  for (int s = 0; s < p.segs; ++s) {
    const Operand &oa = p.a[s], &ob = p.b[s];
    const T* pa = static_cast<const T*>(oa.p);
    const T* pb = ob.part >= 0 ? reinterpret_cast<const T*>(unit_part(units, ob.part, g.slot))
                               : static_cast<const T*>(ob.p);
    const int which = p.acc[s];
    for (int64_t k0 = 0; k0 < n_k; k0 += kBK) {
      T va[16], vb[16];
      fetch(oa, pa, m0, n_m, k0, n_k, g.row0, va);
      fetch(ob, pb, n0, p.n, k0, n_k, g.row0, vb);
      __syncthreads();
      put(oa, va, sa);
      put(ob, vb, sb);
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < kBK; kk += 16) {
        uint32_t fa[2][4], fb[4][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            fa[i][r] = *reinterpret_cast<const uint32_t*>(sa + (wm + i * 16 + q + (r & 1) * 8) * kLd + kk + 2 * t +
                                                          (r >> 1) * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            fb[j][r] = *reinterpret_cast<const uint32_t*>(sb + (wn + j * 8 + q) * kLd + kk + 2 * t + r * 8);
#pragma unroll
        for (int c = 0; c < NACC; ++c)
          if (c == which) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) mma16816<T>(acc[c][i][j], fa[i], fb[j]);
          }
      }
    }
  }
  // lane (q, t) holds rows q and q + 8, columns 2 t and 2 t + 1 of each 16 x 8 block
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t m = m0 + wm + i * 16 + q + h * 8;
      const bool in = m < n_m;
      float w = 0.f, dw = 0.f;
      if (p.epi == kEpiUpBack && in) w = p.weights[plan.pair_of_row[g.row0 + m]];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int64_t n = n0 + wn + j * 8 + 2 * t + c;
          const float a0 = acc[0][i][j][2 * h + c];
          if (!in || n >= p.n) continue;
          if (p.epi == kEpiStore) {
            static_cast<T*>(p.out)[g.unit * p.out_unit + m * p.ldo + n] = from_f<T>(a0);
          } else if (p.epi == kEpiRows32) {
            p.rows32[(g.row0 + m) * p.n + n] = a0;
          } else if constexpr (NACC >= 2) {
            const float a1 = acc[1][i][j][2 * h + c];
            if (p.epi == kEpiUp) {
              static_cast<T*>(p.out)[(g.row0 + m) * p.ldo + n] = from_f<T>(act_rt(p.act, a0) * a1);
            } else if constexpr (NACC >= 3) {
              const float dh = acc[2][i][j][2 * h + c], k = act_rt(p.act, a0);
              const int64_t at = (g.row0 + m) * p.ldo + n;
              static_cast<T*>(p.dg)[at] = from_f<T>(w * dh * a1 * slope_rt(p.act, a0));
              static_cast<T*>(p.du)[at] = from_f<T>(w * dh * k);
              if (p.hw) static_cast<T*>(p.hw)[at] = from_f<T>(w * k * a1);
              dw += dh * k * a1;
            }
          }
        }
      if (NACC >= 3 && p.epi == kEpiUpBack && p.dwp) {
        dw += __shfl_xor_sync(0xffffffffu, dw, 1);
        dw += __shfl_xor_sync(0xffffffffu, dw, 2);
        if (t == 0) red[wn >> 5][wm + i * 16 + q + h * 8] = dw;
      }
    }
  if (NACC >= 3 && p.epi == kEpiUpBack && p.dwp) {
    __syncthreads();
    const int64_t m = m0 + threadIdx.x;
    if (threadIdx.x < 64 && m < n_m)
      p.dwp[(g.row0 + m) * p.ld_dwp + blockIdx.y] = red[0][threadIdx.x] + red[1][threadIdx.x];
  }
}

template <class T>
int go(const Product& p, const Plan& plan, const Units& u, cudaStream_t s) {
  // unit tiles of `plan.bm` rows are walked as 64-row tiles: the plan handed here was made with bm = 64
  const dim3 grid(p.grouped ? plan.max_tiles : unsigned(ceil_div(p.m, 64)), unsigned(ceil_div(p.n, 64)),
                  p.per_unit ? plan.units : 1);
  int accs = 1;
  for (int i = 0; i < p.segs; ++i) accs = p.acc[i] + 1 > accs ? p.acc[i] + 1 : accs;
  return launch(accs == 1 ? tile_kernel<T, 1> : accs == 2 ? tile_kernel<T, 2> : tile_kernel<T, 3>, grid, kThreads, 0, 1,
                s, p, plan, u);
}

}  // namespace

int launch_tile(int dtype, const Product& p, const Plan& plan, const Units& units, cudaStream_t s) {
  return dtype == TSB_BF16 ? go<__nv_bfloat16>(p, plan, units, s) : go<__half>(p, plan, units, s);
}

}  // namespace ops
}  // namespace tsb
