// The operators an engine runs beside the streamed units: the matrix product with its epilogue, the router's selection
// and the gated feed-forward block of the units in their slots. Internal types shared by the entry points (ops_api.cu)
// and the kernels: ops_plan.cu (grouping, joins, routing), ops_tile.cu (every size and alignment), ops_stream.cu (few
// rows: the weights' bytes bound it) and ops_tc.cu (many rows: the tensor cores bound it).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "tierstream/tsb.h"

namespace tsb {
namespace ops {

// Where the units' matrices live: part p of unit u at base[p] + slot x stride[p] (slot_of[first + u], or u), or at
// table[u] + offset[p]. part 0 gate [ffn][hidden], 1 up [ffn][hidden], 2 down [hidden][ffn], rows back to back.
struct Units {
  const int32_t* slot_of;
  const uint32_t* unit_base;  // device word added to the unit's index in slot_of (NULL: 0)
  const uint64_t* table;
  const uint32_t* abort;
  uint32_t* absent;
  uint32_t n_units, n_slots;
  const char* part[3];
  uint64_t stride[3];
};

// The (row, choice) pairs grouped by unit, built on the device by launch_plan: unit e's pairs, in ascending order, are
// rows [off[e], off[e] + cnt[e]) of every grouped buffer; rows up to the next multiple of `pad` have no pair (-1).
struct Plan {
  int32_t* head;  // [0] tiles of `bm` rows, [1] grouped rows (padding included), [2] tiles of 2 `bm` rows
  int32_t* cnt;
  int32_t* off;
  int32_t* slot;
  int32_t* pair_of_row;
  int32_t* row_of_pair;
  // per tile of `bm` and of 2 `bm` rows, group by group: the unit's slot, the group's first row, its rows, and its first
  // tile; behind the last tile of `bm` rows, up to max_tiles, zeros
  int4* tiles[2];
  uint32_t units, pairs, max_rows, max_tiles, pad, bm;
};

__host__ __device__ inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

#ifdef __CUDACC__
// The operators' kernels overlap their launches with what precedes them on the stream: each lets its successor start at
// once (the successor's blocks then wait here, set up, while this one drains) and touches global memory only once all
// that was before it has ended. A chain saves 1 to 2 us a launch.
__device__ __forceinline__ void begin_after() {
  asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
}

// Launches `kernel`, which begins with begin_after(), on `s`.
template <class... P, class... A>
int launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t s, A... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = smem;
  c.stream = s;
  cudaLaunchAttribute a[2];
  c.attrs = a;
  if (cluster > 1) {
    a[c.numAttrs].id = cudaLaunchAttributeClusterDimension;
    a[c.numAttrs].val.clusterDim.x = unsigned(cluster);
    a[c.numAttrs].val.clusterDim.y = a[c.numAttrs].val.clusterDim.z = 1;
    ++c.numAttrs;
  }
  a[c.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[c.numAttrs].val.programmaticStreamSerializationAllowed = 1;
  ++c.numAttrs;
  return int(cudaLaunchKernelEx(&c, kernel, P(args)...));
}

// (units found by address have their index for a slot)
__device__ __forceinline__ const char* unit_part(const Units& u, int p, int32_t slot) {
  return u.table ? reinterpret_cast<const char*>(u.table[slot]) + u.stride[p] : u.part[p] + uint64_t(slot) * u.stride[p];
}

// Activations and their slopes in 32 bits. The exponentials and quotients are the fast intrinsics, off by a few 2^-22 of
// the value where the results are rounded to 2^-9 or 2^-12; (1 + tanh q) / 2 is the logistic of 2 q.
__device__ __forceinline__ float logistic(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }
constexpr float kGelu1 = 1.5957691216057308f, kGelu3 = 0.071354816272600250f;  // 2 sqrt(2 / pi), and times 0.044715
// The normal distribution's integral up to z by Abramowitz and Stegun's 7.1.26, off by at most 7.5e-8 (32-bit
// (1 + erf) / 2 is off by 6e-8); `e` is exp(-z^2 / 2), which its slope needs too.
__device__ __forceinline__ float normal_upto(float z, float e) {
  const float t = __fdividef(1.f, 1.f + 0.23164189f * fabsf(z));  // 0.3275911 / sqrt 2
  const float tail = 0.5f * e * t *
                     (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  return z < 0.f ? tail : 1.f - tail;
}
template <int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == TSB_ACT_SILU) return z * logistic(z);
  if constexpr (ACT == TSB_ACT_GELU) return z * normal_upto(z, __expf(-0.5f * z * z));
  if constexpr (ACT == TSB_ACT_GELU_TANH) return z * logistic(z * (kGelu1 + kGelu3 * z * z));
  if constexpr (ACT == TSB_ACT_RELU) return z < 0.f ? 0.f : z;  // (a NaN stays one)
  return z;
}
template <int ACT>
__device__ __forceinline__ float slope_of(float z) {
  if constexpr (ACT == TSB_ACT_SILU) {
    const float p = logistic(z);
    return p * (1.f + z * (1.f - p));
  }
  if constexpr (ACT == TSB_ACT_GELU) {
    const float e = __expf(-0.5f * z * z);
    return normal_upto(z, e) + z * e * 0.39894228040143268f;
  }
  if constexpr (ACT == TSB_ACT_GELU_TANH) {
    const float p = logistic(z * (kGelu1 + kGelu3 * z * z));
    const float r = p * (1.f - p);  // (0 far out, where the factors beside it pass 32 bits)
    return r > 0.f ? p + z * r * (kGelu1 + 3.f * kGelu3 * z * z) : p;
  }
  if constexpr (ACT == TSB_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  return 1.f;
}
__device__ __forceinline__ float act_rt(int act, float z) {
  switch (act) {
    case TSB_ACT_SILU: return act_of<TSB_ACT_SILU>(z);
    case TSB_ACT_GELU: return act_of<TSB_ACT_GELU>(z);
    case TSB_ACT_GELU_TANH: return act_of<TSB_ACT_GELU_TANH>(z);
    case TSB_ACT_RELU: return act_of<TSB_ACT_RELU>(z);
  }
  return z;
}
__device__ __forceinline__ float slope_rt(int act, float z) {
  switch (act) {
    case TSB_ACT_SILU: return slope_of<TSB_ACT_SILU>(z);
    case TSB_ACT_GELU: return slope_of<TSB_ACT_GELU>(z);
    case TSB_ACT_GELU_TANH: return slope_of<TSB_ACT_GELU_TANH>(z);
    case TSB_ACT_RELU: return slope_of<TSB_ACT_RELU>(z);
  }
  return 1.f;
}

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
#endif

// What a product writes. Sums are held in 32 bits up to here; each store below rounds once.
enum Epi {
  kEpiLinear,   // z = acc + bias; pre = z; out = act(z) + residual (aligned operands only)
  kEpiStore,    // out = acc (a gradient), per unit at out + e x out_unit
  kEpiRows32,   // rows32[row][n] = acc in 32 bits (joined later)
  kEpiUp,       // out[row][n] = act(acc0) x acc1
  kEpiUpBack,   // from g = acc0, u = acc1, dh = acc2 and the pair's weight w: dg, du, hw = w x h, and per row the sum
                // of dh x h over this tile's columns into dwp[row][tile]
};

// One operand of a product: element (i, k) at p + i x s_i + k x s_k elements. map: rows are gathered, row r of the
// grouped buffer being row map[r] / div of p (-1: zeros); the gathered index is i, or k with map_k.
struct Operand {
  const void* p;
  int64_t s_i, s_k;
  const int32_t* map;
  int32_t div, map_k;
  int32_t part;  // >= 0: p is part `part` of the group's unit
};

struct Product {
  Operand a[3], b[3];
  int32_t acc[3];  // which accumulator segment s adds to
  int32_t segs;
  // m runs over the rows of a group (grouped) or over `m` (a matrix per unit, or one matrix); n over `n`; k over `k`, or
  // over the group's rows (k_rows)
  int64_t m, n, k;
  int32_t grouped, per_unit, k_rows;
  Epi epi;
  int32_t act;
  void* out;
  int64_t ldo, out_unit;
  const void* bias;
  const void* residual;
  int64_t ldr;
  void* pre;
  int64_t ldp;
  float* rows32;
  void* dg;
  void* du;
  void* hw;
  float* dwp;
  int64_t ld_dwp;
  const float* weights;
};

// ops_plan.cu
uint64_t plan_bytes(uint32_t units, uint64_t pairs, uint32_t pad, uint32_t bm);
Plan plan_at(void* ws, uint32_t units, uint64_t pairs, uint32_t pad, uint32_t bm);
int launch_plan(const Plan& p, const Units& u, const int32_t* ids, cudaStream_t s);
// y[t] = residual[t] + sum over k of w[t][k] x rows32[row_of_pair[t top + k]]
int launch_join(int dtype, const Plan& p, const float* rows32, const float* weights, uint32_t top, uint64_t rows,
                uint64_t n, const void* residual, uint64_t ldr, void* y, uint64_t ldy, cudaStream_t s);
// y = act(sum over the splits of rows32 + bias) + residual, pre the sum itself
int launch_join_linear(int dtype, int act, const float* rows32, uint32_t splits, uint64_t rows, uint64_t n,
                       const void* bias, const void* residual, uint64_t ldr, void* y, uint64_t ldy, void* pre,
                       uint64_t ldp, cudaStream_t s);
// dweights[pair] = sum over tiles of dwp[row][tile]
int launch_join_dw(int dtype, const Plan& p, const float* dwp, uint32_t tiles, void* dw, cudaStream_t s);
int launch_route(int dtype, const void* logits, uint64_t ld, uint64_t rows, uint32_t experts, uint32_t top, int norm,
                 int32_t* ids, float* weights, cudaStream_t s);
int launch_route_back(int dtype, int dw_dtype, const void* dw, const void* logits, uint64_t ld, const int32_t* ids,
                      const float* weights, uint64_t rows, uint32_t experts, uint32_t top, int norm, void* dlogits,
                      uint64_t ldd, cudaStream_t s);
// Copies of matrices whose rows do not start on 16 bytes to rows that do, the columns up to ldd filled with zeros.
struct Copy {
  const void* src;
  void* dst;
  uint64_t ld, ldd, rows, cols;
};
struct Copies {
  Copy c[2];
  int n;
};
int launch_copies(const Copies& c, cudaStream_t s);
// dz = dy x act'(pre) (act none: not written) and, with db, its column sums; part: [chunks][n] floats
uint32_t dz_chunks(uint64_t rows, uint64_t n);
int launch_dz(int dtype, int act, const void* dy, uint64_t ldy, const void* pre, uint64_t ldp, void* dz, uint64_t ldz,
              uint64_t rows, uint64_t n, void* db, float* part, cudaStream_t s);

// ops_tile.cu: the feed-forward block's products at any size, stride and alignment
constexpr uint32_t kTileM = 64, kTileN = 64;
int launch_tile(int dtype, const Product& p, const Plan& plan, const Units& units, cudaStream_t s);


// ops_stream.cu: products of few rows, in tiles of 8 (the plan's bm). Rows of x and w start on 16 bytes and k
// is a multiple of 8; gathered rows are read where they are (top: the pairs a row has).
constexpr uint32_t kStreamTile = 8;
int launch_stream(int dtype, const Product& p, uint32_t top, const Plan* plan, const Units* units, cudaStream_t s);

// ops_tc.cu: products of many rows on tcgen05; grouped ones take tiles of kTcRows rows (the plan's bm). tc_fits: TMA can
// read the operand. Gathered operands are gathered first: launch_gather copies n columns of every grouped row (n a
// multiple of 8), of a second source too unless src2 is NULL.
constexpr uint32_t kTcRows = 256;
bool tc_fits(const Operand& o);
int tc_columns(int64_t m, int64_t n, int sms);
int launch_gather(const Plan& plan, uint32_t top, uint64_t n, const void* src, uint64_t ld, void* dst, const void* src2,
                  uint64_t ld2, void* dst2, cudaStream_t s);
// columns: of a plain product's tiles. kEpiRows32 of a plain product whose k runs over rows: parts of the sum, as in
// launch_group.
int launch_tc(int dtype, const Product& p, int splits, int columns, const Plan* plan, const Units* units, cudaStream_t s);
int ops_take_timeouts(uint32_t* out);

// ops_group.cu: the grouped products with the unit's matrix as rows, for groups of any length (the plan's bm kGroupRows)
constexpr uint32_t kGroupRows = 128;
// plan NULL: one matrix p.b[0] and p.m rows of p.a[0]. kEpiRows32 may split the sum over k: split j's rows at rows32 +
// j x rows x n (rows: the plan's max_rows, or p.m).
int launch_group(int dtype, const Product& p, int splits, const Plan* plan, const Units* units, cudaStream_t s);
int group_take_timeouts(uint32_t* out);

}  // namespace ops
}  // namespace tsb
