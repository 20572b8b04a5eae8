// The entry points of the operators (include/tierstream/tsb.h): argument checks, the workspace's layout and the choice
// of kernels.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <string>

#include "errors.hpp"
#include "ops.hpp"

namespace tsb {
const char* set_error(const std::string& msg);
}

namespace {

using namespace tsb::ops;

template <class F>
ss_status run(F&& f) {
  try {
    f();
    return SS_OK;
  } catch (const tsb::Error& e) {
    tsb::set_error(e.what());
    return e.status();
  } catch (const std::exception& e) {
    tsb::set_error(e.what());
    return SS_E_BACKEND;
  }
}
void need(bool ok, const char* fn, const char* what) {
  if (!ok) tsb::fail(SS_E_INVALID, std::string(fn) + ": " + what);
}
// pointers on whole elements of `size` bytes (NULL is)
void need_elements(const char* fn, std::initializer_list<const void*> pointers, uintptr_t size) {
  uintptr_t all = 0;
  for (const void* p : pointers) all |= reinterpret_cast<uintptr_t>(p);
  need((all & (size - 1)) == 0, fn, "a pointer is not on a whole element");
}
void ck(int e, const char* fn, const char* what) {
  if (e == 0) return;
  (void)cudaGetLastError();
  tsb::fail(SS_E_BACKEND, std::string(fn) + ": " + what + ": " + cudaGetErrorString(cudaError_t(e)));
}

constexpr uint64_t kMaxDim = uint64_t(1) << 20, kMaxRows = uint64_t(1) << 28;

// The workspace handed out front to back, every piece on 256 bytes.
struct Arena {
  char* base;
  uint64_t used = 0;
  void* take(uint64_t bytes) {
    char* p = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
};
void need_workspace(const char* fn, const void* ws, uint64_t have, uint64_t want) {
  need(!want || (ws && have >= want), fn, "the workspace is smaller than the call's _workspace says");
  need(!want || (reinterpret_cast<uintptr_t>(ws) & 255u) == 0, fn, "the workspace must be 256-byte aligned");
}

Operand dense(const void* p, int64_t s_i, int64_t s_k, int map_k = 0) { return {p, s_i, s_k, nullptr, 1, map_k, -1}; }
Operand gathered(const void* p, int64_t s_i, int64_t s_k, const Plan& plan, uint32_t top, int map_k = 0) {
  return {p, s_i, s_k, plan.pair_of_row, int32_t(top), map_k, -1};
}
Operand of_unit(int part, int64_t s_i, int64_t s_k) { return {nullptr, s_i, s_k, nullptr, 1, 0, part}; }

// Where the kernel that streams the weights (8 rows a tile) beats the tensor cores' own path, whose 128-row tiles are
// mostly empty then: a plain product of at most 8 rows (32 us against 58 at 6 x 8192 x 8192, 34 against 48 at 8 x 4096 x
// 14336, where the other's 128 column tiles cannot keep enough bytes in flight), and the feed-forward block with at most
// two rows for each unit that may be met (730 us against 767 at two of 64 units of 88 MB, 327 against 362 at one of 8 of
// 352 MB, 663 against 644 at two of 128 of 38 MB; at four 800 against 750 there). A small block too, whose units are read
// again for every 8 rows, from L2: it saves the tensor cores' path its gathered copy and the start of its kernels (11 us
// against 18 at 37 rows for each of 3 units of 0.2 MB, 14 against 21 at 12 of 2 of 2.2 MB, 23 against 36 at 11 of 6 of
// 5.1 MB, 43 MB read again; 30 against 24 at 142 of 7 of 0.6 MB, 76 MB; 36 against 25 at 32 of 16 of 3.1 MB, 200 MB).
constexpr uint64_t kStreamRows = kStreamTile, kStreamEach = 2;
constexpr double kStreamAgain = 48e6;

// How a plain product runs. The times are fits, in us, to what the kernels took a 64-wide slice of k on this GPU (148 SMs):
// 0.10 + 0.0012 columns for a pair of CTAs (0.254 measured at 128 columns, 0.405 at 256; 0.2 at least), 0.17 + 0.00098
// columns for a single one, about 6 for a launch's start and end, 3 for the join's, which reads 32-bit rows at 6 TB/s.
struct How {
  enum Kind { kStream, kTc, kGroup } kind;
  int splits, columns;
};
constexpr int kSms = 148;
double slice_us(double columns) { return columns < 84 ? 0.2 : 0.10 + 0.0012 * columns; }

// The gradient of a matrix, a sum over rows: with few tiles the rows are split so that the parts fill the GPU's CTAs
// once to four times (200 x 1024 over 32768 rows: 142 us whole, 26 in parts).
How how_rows(const Product& p) {
  const int cg = p.m > 128 ? 2 : 1;
  const uint64_t kb = ceil_div(uint64_t(p.k), 64), m_tiles = ceil_div(uint64_t(p.m), uint64_t(128 * cg));
  const auto us = [&](int bn, uint64_t s) {
    const uint64_t waves = ceil_div(m_tiles * ceil_div(uint64_t(p.n), uint64_t(bn)) * s, uint64_t(kSms / cg));
    return double(waves * ceil_div(kb, s)) * (cg == 2 ? slice_us(bn) : 0.17 + 0.00098 * bn);
  };
  How best{How::kTc, 1, tc_columns(p.m, p.n, kSms)};
  double least = us(best.columns, 1);
  for (int bn = 64; bn <= 256; bn += 64) {
    const uint64_t tiles = m_tiles * ceil_div(uint64_t(p.n), uint64_t(bn));
    for (uint64_t w = 1; w <= 4; ++w) {
      const uint64_t s = std::min<uint64_t>(w * uint64_t(kSms / cg) / tiles, 32);
      if (s < 2 || s * 4 > kb) continue;
      const double t = us(bn, s) + 3 + double(s) * double(p.m) * double(p.n) * 8 / 6e6;
      if (t < least) least = t, best = {How::kTc, int(s), bn};
    }
  }
  return best;
}

How how(const Product& p) {
  const bool forward = p.epi == kEpiLinear;
  if (forward && uint64_t(p.m) <= kStreamRows) return {How::kStream, 1, 0};
  if (p.a[0].s_k != 1) return how_rows(p);
  const double kb = double(ceil_div(uint64_t(p.k), 64)), bytes = 2.0 * double(p.n) * double(p.k) / 6.5e6;
  // the matrix as columns, in the columns a tile that launch_tc would take
  const int cg = p.m > 128 ? 2 : 1;
  const int bn = tc_columns(p.m, p.n, kSms);
  const uint64_t tc_tiles = ceil_div(uint64_t(p.m), 128 * cg) * ceil_div(uint64_t(p.n), uint64_t(bn));
  const double waves = double(ceil_div(tc_tiles, uint64_t(kSms / cg)));
  const double tc = 6 + std::max(bytes, waves * kb * (cg == 2 ? slice_us(bn) : 0.17 + 0.00098 * bn));
  // the matrix as rows, k split
  const uint64_t tiles = ceil_div(uint64_t(p.m), 2 * kGroupRows);
  const double cols = double((ceil_div(uint64_t(p.m), tiles) + 31) / 32 * 32);
  How best{How::kTc, 1, bn};
  double least = tc;
  for (int s = 1; s <= 8 && s * 4 <= kb; ++s) {
    const double w = double(ceil_div(tiles * ceil_div(uint64_t(p.n), 256) * s, kSms / 2));
    const double us = 9 + std::max(bytes, w * std::ceil(kb / s) * slice_us(cols)) + s * double(p.m) * double(p.n) * 8 / 6e6;
    if (us < least) least = us, best = {How::kGroup, s, 0};
  }
  return best;
}

uint64_t product_bytes(const Product& p) {
  const How h = how(p);
  return h.kind == How::kGroup || h.splits > 1 ? uint64_t(h.splits) * uint64_t(p.m) * uint64_t(p.n) * 4 : 0;
}
int product(int dtype, const Product& p, float* rows32, cudaStream_t s) {
  const How h = how(p);
  if (h.kind == How::kStream) return launch_stream(dtype, p, 1, nullptr, nullptr, s);
  if (h.kind == How::kTc && h.splits == 1) return launch_tc(dtype, p, 1, h.columns, nullptr, nullptr, s);
  Product r = p;
  r.epi = kEpiRows32;
  r.rows32 = rows32;
  if (const int e = h.kind == How::kTc ? launch_tc(dtype, r, h.splits, h.columns, nullptr, nullptr, s)
                                       : launch_group(dtype, r, h.splits, nullptr, nullptr, s))
    return e;
  return launch_join_linear(dtype, p.act, rows32, uint32_t(h.splits), uint64_t(p.m), uint64_t(p.n), p.bias, p.residual,
                            uint64_t(p.ldr), p.out, uint64_t(p.ldo), p.pre, uint64_t(p.ldp), s);
}

// An operand, [rows][cols] in memory, whose rows do not start on 16 bytes (or, `whole`, do not hold whole eights) is copied
// into the workspace first: the fast kernels read it from there.
void align(Operand& o, uint64_t rows, uint64_t cols, bool whole, Arena& w, Copies& copies) {
  if (tc_fits(o) && !(whole && cols % 8)) return;
  const uint64_t ld = o.s_k == 1 ? uint64_t(o.s_i) : uint64_t(o.s_k), ldd = (cols + 7) / 8 * 8;
  const bool k_inner = !o.map_k && o.s_k == 1;
  void* dst = w.take(rows * ldd * 2);
  copies.c[copies.n++] = {o.p, dst, ld, ldd, rows, cols};
  o.p = dst;
  (k_inner ? o.s_i : o.s_k) = int64_t(ldd);
}

// ---- linear ----
void check_linear(const tsb_linear_args* a) {
  const char* fn = "tsb_linear";
  need(a && a->struct_size >= sizeof *a, fn, "null or short argument struct");
  need(a->dtype == TSB_BF16 || a->dtype == TSB_F16, fn, "dtype must be TSB_BF16 or TSB_F16");
  need(a->act <= TSB_ACT_RELU, fn, "unknown activation");
  need(a->n >= 1 && a->k >= 1 && a->n <= kMaxDim && a->k <= kMaxDim, fn, "n and k must be in [1, 2^20]");
  need(a->rows < kMaxRows, fn, "rows must be below 2^28");
  if (!a->rows) return;
  need(a->x && a->w && a->y, fn, "null argument");
  need_elements(fn, {a->x, a->w, a->bias, a->residual, a->y, a->pre}, 2);
  need(a->ldx >= a->k && a->ldw >= a->k && a->ldy >= a->n && (!a->residual || a->ldr >= a->n) &&
           (!a->pre || a->ldp >= a->n),
       fn, "a leading dimension is shorter than its row");
}

struct LinearSpace {
  Product p;
  Copies copies;
  float* rows32;
  uint64_t bytes;
};
LinearSpace linear_space(const tsb_linear_args* a) {
  Arena w{static_cast<char*>(a->workspace)};
  LinearSpace r{};
  Product& p = r.p;
  p.segs = 1;
  p.a[0] = dense(a->x, int64_t(a->ldx), 1);
  p.b[0] = dense(a->w, int64_t(a->ldw), 1);
  p.m = int64_t(a->rows), p.n = int64_t(a->n), p.k = int64_t(a->k);
  const bool few = a->rows <= kStreamRows;  // (streamed rows are read in whole eights)
  align(p.a[0], a->rows, a->k, few, w, r.copies);
  align(p.b[0], a->n, a->k, few, w, r.copies);
  if (few) p.k = (p.k + 7) / 8 * 8;
  p.epi = kEpiLinear;
  p.act = int(a->act);
  p.out = a->y, p.ldo = int64_t(a->ldy);
  p.bias = a->bias;
  p.residual = a->residual, p.ldr = int64_t(a->ldr);
  p.pre = a->pre, p.ldp = int64_t(a->ldp);
  r.rows32 = static_cast<float*>(w.take(product_bytes(p)));
  r.bytes = w.used;
  return r;
}

void linear(const tsb_linear_args* a) {
  const char* fn = "tsb_linear";
  check_linear(a);
  if (!a->rows) return;
  const LinearSpace w = linear_space(a);
  need_workspace(fn, a->workspace, a->workspace_bytes, w.bytes);
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  if (w.copies.n) ck(launch_copies(w.copies, s), fn, "aligned copies");
  ck(product(int(a->dtype), w.p, w.rows32, s), fn, "launch");
}

void check_linear_back(const tsb_linear_grad_args* a) {
  const char* fn = "tsb_linear_backward";
  need(a && a->struct_size >= sizeof *a, fn, "null or short argument struct");
  need(a->dtype == TSB_BF16 || a->dtype == TSB_F16, fn, "dtype must be TSB_BF16 or TSB_F16");
  need(a->act <= TSB_ACT_RELU, fn, "unknown activation");
  need(a->n >= 1 && a->k >= 1 && a->n <= kMaxDim && a->k <= kMaxDim, fn, "n and k must be in [1, 2^20]");
  need(a->rows < kMaxRows, fn, "rows must be below 2^28");
  need(!a->dw || a->lddw >= a->k, fn, "a leading dimension is shorter than its row");
  need_elements(fn, {a->dy, a->x, a->w, a->act == TSB_ACT_NONE ? nullptr : a->pre, a->dx, a->dw, a->db}, 2);
  if (!a->rows) return;
  need(a->dy && (!a->dx || a->w) && (!a->dw || a->x), fn, "null argument");
  need(a->act == TSB_ACT_NONE || a->pre, fn, "an activation's slope needs pre");
  need(a->lddy >= a->n && (!a->dx || (a->ldw >= a->k && a->lddx >= a->k)) && (!a->dw || a->ldx >= a->k) &&
           (a->act == TSB_ACT_NONE || a->ldp >= a->n),
       fn, "a leading dimension is shorter than its row");
}

struct LinearBackSpace {
  void* dz;  // NULL: dy itself
  uint64_t ldz;
  Copies copies;
  Product dx, dw;
  float *part, *rows32, *dw32;
  uint64_t bytes;
};
LinearBackSpace linear_back_space(const tsb_linear_grad_args* a) {
  Arena w{static_cast<char*>(a->workspace)};
  LinearBackSpace r{};
  if (!a->rows || (!a->dx && !a->dw && !a->db)) return r;
  const void* dz = a->dy;
  r.ldz = a->lddy;
  // dz: the slope times dy, or a copy of dy whose rows start on 16 bytes
  if (a->act != TSB_ACT_NONE || ((a->dx || a->dw) && !tc_fits(dense(a->dy, int64_t(a->lddy), 1)))) {
    r.ldz = (a->n + 7) / 8 * 8;
    dz = r.dz = w.take(a->rows * r.ldz * 2);
  }
  if (a->db) r.part = static_cast<float*>(w.take(uint64_t(dz_chunks(a->rows, a->n)) * a->n * 4));
  if (a->dx) {
    Product& p = r.dx;
    p.segs = 1;
    p.a[0] = dense(dz, int64_t(r.ldz), 1);
    p.b[0] = dense(a->w, 1, int64_t(a->ldw), 1);
    align(p.b[0], a->n, a->k, false, w, r.copies);
    p.m = int64_t(a->rows), p.n = int64_t(a->k), p.k = int64_t(a->n);
    p.epi = kEpiStore;
    p.out = a->dx, p.ldo = int64_t(a->lddx);
    r.rows32 = static_cast<float*>(w.take(product_bytes(p)));
  }
  if (a->dw) {
    Product& p = r.dw;
    p.segs = 1;
    p.a[0] = dense(dz, 1, int64_t(r.ldz), 1);
    p.b[0] = dense(a->x, 1, int64_t(a->ldx), 1);
    align(p.b[0], a->rows, a->k, false, w, r.copies);
    p.m = int64_t(a->n), p.n = int64_t(a->k), p.k = int64_t(a->rows);
    p.epi = kEpiStore;
    p.out = a->dw, p.ldo = int64_t(a->lddw);
    r.dw32 = static_cast<float*>(w.take(product_bytes(p)));
  }
  r.bytes = w.used;
  return r;
}

void linear_back(const tsb_linear_grad_args* a) {
  const char* fn = "tsb_linear_backward";
  check_linear_back(a);
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  if (!a->rows) {
    if (a->dw) ck(int(cudaMemset2DAsync(a->dw, a->lddw * 2, 0, a->k * 2, a->n, s)), fn, "dw");
    if (a->db) ck(int(cudaMemsetAsync(a->db, 0, a->n * 2, s)), fn, "db");
    return;
  }
  if (!a->dx && !a->dw && !a->db) return;
  const LinearBackSpace w = linear_back_space(a);
  need_workspace(fn, a->workspace, a->workspace_bytes, w.bytes);
  if (w.copies.n) ck(launch_copies(w.copies, s), fn, "aligned copies");
  if (w.dz || a->db)
    ck(launch_dz(int(a->dtype), int(a->act), a->dy, a->lddy, a->pre, a->ldp, w.dz, w.ldz, a->rows, a->n, a->db, w.part, s),
       fn, "slope");
  if (a->dx) ck(product(int(a->dtype), w.dx, w.rows32, s), fn, "dx");
  if (a->dw) ck(product(int(a->dtype), w.dw, w.dw32, s), fn, "dw");
}

// ---- the gated feed-forward block ----
Units units_of(const tsb_units* u) {
  Units r{};
  r.slot_of = u->slot_of;
  r.unit_base = u->unit_base;
  r.table = u->table;
  r.abort = u->abort;
  r.absent = u->absent_err;
  r.n_units = u->n_units;
  r.n_slots = u->n_slots;
  for (int i = 0; i < 3; ++i) {
    r.part[i] = static_cast<const char*>(u->part[i]);
    r.stride[i] = u->stride[i];
  }
  return r;
}

template <class A>
void check_ffn_shape(const A* a, const char* fn) {
  need(a && a->struct_size >= sizeof *a, fn, "null or short argument struct");
  need(a->dtype == TSB_BF16 || a->dtype == TSB_F16, fn, "dtype must be TSB_BF16 or TSB_F16");
  need(a->act <= TSB_ACT_RELU, fn, "unknown activation");
  need(a->hidden >= 1 && a->ffn >= 1 && a->hidden <= kMaxDim && a->ffn <= kMaxDim, fn,
       "hidden and ffn must be in [1, 2^20]");
  need(a->top >= 1 && a->top <= 64, fn, "top must be in [1, 64]");
  need(a->rows <= kMaxRows / a->top, fn, "rows x top must be at most 2^28");
  const tsb_units* u = a->units;
  need(u && u->struct_size >= sizeof *u, fn, "null or short units struct");
  need(u->n_units >= 1 && u->n_units <= 65535, fn, "n_units must be in [1, 65535]");
  need(u->table || (u->part[0] && u->part[1] && u->part[2] && u->n_slots >= 1), fn, "no parts and no table");
  if (!u->table) need_elements(fn, {u->part[0], u->part[1], u->part[2]}, 2);
  need_elements(fn, {u->slot_of, u->unit_base, u->abort, u->absent_err, a->ids, a->weights}, 4);
  need_elements(fn, {u->table}, 8);
  need(u->stride[0] % 2 == 0 && u->stride[1] % 2 == 0 && u->stride[2] % 2 == 0, fn,
       "the parts' strides must be whole elements");
}

// Whether every row of the block's matrices starts on 16 bytes (a unit found by address: its slots are 256-byte aligned,
// so its matrices' offsets decide).
bool ffn_rows16(const tsb_units* u, uint64_t hidden, uint64_t ffn, const void* x, uint64_t ldx, const void* dy,
            uint64_t lddy) {
  auto on16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  if (hidden % 8 || ffn % 8 || !on16(x) || ldx % 8 || !on16(dy) || lddy % 8) return false;
  for (int i = 0; i < 3; ++i)
    if ((!u->table && !on16(u->part[i])) || u->stride[i] % 16 || u->stride[i] >= (uint64_t(1) << 40)) return false;
  return true;
}

// On the tensor cores' own path a unit's matrix supplies the rows and the group's rows the columns, except for groups so
// long that whole 256-row tiles waste little of them.
uint32_t tc_tile(uint64_t each) { return each >= 4 * kTcRows ? kTcRows : kGroupRows; }
int launch_grouped(int dtype, const Product& p, const Plan* plan, const Units* u, cudaStream_t s) {
  return p.grouped && plan->bm == kGroupRows ? launch_group(dtype, p, 1, plan, u, s) : launch_tc(dtype, p, 1, 0, plan, u, s);
}

struct FfnSpace {
  Plan plan;
  bool tc, stream;
  void* xs;
  void* h;
  int64_t ldh;
  float* rows32;
  uint64_t bytes;
};
FfnSpace ffn_space(const tsb_ffn_args* a) {
  Arena w{static_cast<char*>(a->workspace)};
  FfnSpace r{};
  const uint64_t pairs = a->rows * a->top;
  // few rows for each unit that may be met, or units by address, which TMA cannot find: the weights are streamed
  const uint64_t each = ceil_div(pairs, pairs < a->units->n_units ? pairs : a->units->n_units);
  const double again = double(pairs) / kStreamTile * 6 * double(a->hidden) * double(a->ffn);
  r.stream = (each <= kStreamEach || again <= kStreamAgain || a->units->table) &&
             pairs / kStreamTile + a->units->n_units <= 65535 &&  // (a grid's y)
             ffn_rows16(a->units, a->hidden, a->ffn, a->x, a->ldx, nullptr, 0);
  r.tc = !r.stream && !a->units->table && ffn_rows16(a->units, a->hidden, a->ffn, a->x, a->ldx, nullptr, 0);
  const uint32_t bm = r.stream ? kStreamTile : r.tc ? tc_tile(each) : kTileM;
  r.plan = plan_at(w.take(plan_bytes(a->units->n_units, pairs, 1, bm)), a->units->n_units, pairs, 1, bm);
  if (r.tc) r.xs = w.take(uint64_t(r.plan.max_rows) * a->hidden * 2);
  // (streamed, the middle is two 16-bit values)
  r.ldh = int64_t(a->ffn) * (r.stream ? 2 : 1);
  r.h = w.take(uint64_t(r.plan.max_rows) * uint64_t(r.ldh) * 2);
  r.rows32 = static_cast<float*>(w.take(uint64_t(r.plan.max_rows) * a->hidden * 4));
  r.bytes = w.used;
  return r;
}

void check_ffn(const tsb_ffn_args* a) {
  const char* fn = "tsb_ffn";
  check_ffn_shape(a, fn);
  if (!a->rows) return;
  need(a->x && a->ids && a->weights && a->y, fn, "null argument");
  need_elements(fn, {a->x, a->residual, a->y}, 2);
  need(a->ldx >= a->hidden && a->ldy >= a->hidden && (!a->residual || a->ldr >= a->hidden), fn,
       "a leading dimension is shorter than its row");
}

void ffn(const tsb_ffn_args* a) {
  const char* fn = "tsb_ffn";
  check_ffn(a);
  if (!a->rows) return;
  const FfnSpace w = ffn_space(a);
  need_workspace(fn, a->workspace, a->workspace_bytes, w.bytes);
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  const Units u = units_of(a->units);
  const int64_t d = int64_t(a->hidden), f = int64_t(a->ffn);
  ck(launch_plan(w.plan, u, a->ids, s), fn, "plan");
  Product p{};
  p.grouped = 1;
  p.segs = 2;
  p.a[0] = p.a[1] = gathered(a->x, int64_t(a->ldx), 1, w.plan, a->top);
  p.b[0] = of_unit(0, d, 1);
  p.b[1] = of_unit(1, d, 1);
  p.acc[1] = 1;
  p.n = f, p.k = d;
  p.epi = kEpiUp;
  p.act = int(a->act);
  p.out = w.h, p.ldo = w.ldh;
  const auto go = [&](const Product& pr) {
    return w.stream ? launch_stream(int(a->dtype), pr, a->top, &w.plan, &u, s)
           : w.tc   ? launch_grouped(int(a->dtype), pr, &w.plan, &u, s)
                    : launch_tile(int(a->dtype), pr, w.plan, u, s);
  };
  if (w.tc) {
    ck(launch_gather(w.plan, a->top, a->hidden, a->x, a->ldx, w.xs, nullptr, 0, nullptr, s), fn, "gather");
    p.a[0] = p.a[1] = dense(w.xs, d, 1);
  }
  ck(go(p), fn, "gate and up");
  Product q{};
  q.grouped = 1;
  q.segs = 1;
  q.a[0] = dense(w.h, w.ldh, 1);
  q.b[0] = of_unit(2, f, 1);
  q.n = d, q.k = f;
  q.epi = kEpiRows32;
  q.rows32 = w.rows32;
  ck(go(q), fn, "down");
  ck(launch_join(int(a->dtype), w.plan, w.rows32, a->weights, a->top, a->rows, a->hidden, a->residual, a->ldr, a->y,
                 a->ldy, s),
     fn, "join");
}

struct FfnBackSpace {
  Plan plan;
  bool tc;
  void *xs, *dys, *dg, *du, *hw;
  float *dwp, *rows32;
  uint32_t dw_tiles;
  uint64_t bytes;
};
FfnBackSpace ffn_back_space(const tsb_ffn_grad_args* a) {
  Arena w{static_cast<char*>(a->workspace)};
  FfnBackSpace r{};
  const uint64_t pairs = a->rows * a->top;
  r.tc = !a->units->table && ffn_rows16(a->units, a->hidden, a->ffn, a->x, a->ldx, a->dy, a->lddy);
  // (sums over a group's rows run in slices of 64 on the tensor cores: zero rows fill the last one)
  const uint64_t each = ceil_div(pairs, pairs < a->units->n_units ? pairs : a->units->n_units);
  const uint32_t bm = r.tc ? tc_tile(each) : kTileM, pad = r.tc && a->dgate ? 64 : 1;
  r.plan = plan_at(w.take(plan_bytes(a->units->n_units, pairs, pad, bm)), a->units->n_units, pairs, pad, bm);
  if (r.tc) {
    r.xs = w.take(uint64_t(r.plan.max_rows) * a->hidden * 2);
    r.dys = w.take(uint64_t(r.plan.max_rows) * a->hidden * 2);
  }
  r.dg = w.take(uint64_t(r.plan.max_rows) * a->ffn * 2);
  r.du = w.take(uint64_t(r.plan.max_rows) * a->ffn * 2);
  if (a->dgate) r.hw = w.take(uint64_t(r.plan.max_rows) * a->ffn * 2);
  r.dw_tiles = !r.tc               ? uint32_t(ceil_div(a->ffn, kTileN))
               : bm == kGroupRows ? 8 * uint32_t(ceil_div(a->ffn, 256))
                                  : 2 * uint32_t(ceil_div(a->ffn, 128));
  if (a->dweights) r.dwp = static_cast<float*>(w.take(uint64_t(r.plan.max_rows) * r.dw_tiles * 4));
  if (a->dx) r.rows32 = static_cast<float*>(w.take(uint64_t(r.plan.max_rows) * a->hidden * 4));
  r.bytes = w.used;
  return r;
}

void check_ffn_back(const tsb_ffn_grad_args* a) {
  const char* fn = "tsb_ffn_backward";
  check_ffn_shape(a, fn);
  need((a->dgate && a->dup && a->ddown) || (!a->dgate && !a->dup && !a->ddown), fn,
       "dgate, dup and ddown go together");
  if (!a->rows) return;
  need(a->dy && a->x && a->ids && a->weights, fn, "null argument");
  need_elements(fn, {a->dy, a->x, a->dx, a->dweights, a->dgate, a->dup, a->ddown}, 2);
  need(a->ldx >= a->hidden && a->lddy >= a->hidden && (!a->dx || a->lddx >= a->hidden), fn,
       "a leading dimension is shorter than its row");
}

void ffn_back(const tsb_ffn_grad_args* a) {
  const char* fn = "tsb_ffn_backward";
  check_ffn_back(a);
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  const int64_t d = int64_t(a->hidden), f = int64_t(a->ffn);
  if (!a->rows) {
    for (void* g : {a->dgate, a->dup, a->ddown})
      if (g) ck(int(cudaMemsetAsync(g, 0, uint64_t(a->units->n_units) * a->hidden * a->ffn * 2, s)), fn, "zeros");
    return;
  }
  if (!a->dx && !a->dweights && !a->dgate) return;
  const FfnBackSpace w = ffn_back_space(a);
  need_workspace(fn, a->workspace, a->workspace_bytes, w.bytes);
  const Units u = units_of(a->units);
  const int dt = int(a->dtype);
  ck(launch_plan(w.plan, u, a->ids, s), fn, "plan");
  const auto go = [&](const Product& pr) {
    return w.tc ? launch_grouped(dt, pr, &w.plan, &u, s) : launch_tile(dt, pr, w.plan, u, s);
  };
  Operand x_rows = gathered(a->x, int64_t(a->ldx), 1, w.plan, a->top),
          dy_rows = gathered(a->dy, int64_t(a->lddy), 1, w.plan, a->top),
          x_sum = gathered(a->x, 1, int64_t(a->ldx), w.plan, a->top, 1),
          dy_sum = gathered(a->dy, 1, int64_t(a->lddy), w.plan, a->top, 1);
  if (w.tc) {
    ck(launch_gather(w.plan, a->top, a->hidden, a->x, a->ldx, w.xs, a->dy, a->lddy, w.dys, s), fn, "gather");
    x_rows = dense(w.xs, d, 1);
    dy_rows = dense(w.dys, d, 1);
    x_sum = dense(w.xs, 1, d, 1);
    dy_sum = dense(w.dys, 1, d, 1);
  }
  {
    Product p{};
    p.grouped = 1;
    p.segs = 3;
    p.a[0] = p.a[1] = x_rows;
    p.a[2] = dy_rows;
    p.b[0] = of_unit(0, d, 1);
    p.b[1] = of_unit(1, d, 1);
    p.b[2] = of_unit(2, 1, f);
    p.acc[1] = 1, p.acc[2] = 2;
    p.n = f, p.k = d;
    p.epi = kEpiUpBack;
    p.act = int(a->act);
    p.dg = w.dg, p.du = w.du, p.hw = w.hw, p.ldo = f;
    p.dwp = w.dwp, p.ld_dwp = w.dw_tiles;
    p.weights = a->weights;
    ck(go(p), fn, "gate, up and dh");
  }
  if (a->dweights) ck(launch_join_dw(dt, w.plan, w.dwp, w.dw_tiles, a->dweights, s), fn, "dweights");
  if (a->dx) {
    Product p{};
    p.grouped = 1;
    p.segs = 2;
    p.a[0] = dense(w.dg, f, 1);
    p.a[1] = dense(w.du, f, 1);
    p.b[0] = of_unit(0, 1, d);
    p.b[1] = of_unit(1, 1, d);
    p.n = d, p.k = f;
    p.epi = kEpiRows32;
    p.rows32 = w.rows32;
    ck(go(p), fn, "dx");
    ck(launch_join(dt, w.plan, w.rows32, nullptr, a->top, a->rows, a->hidden, nullptr, 0, a->dx, a->lddx, s), fn,
       "join");
  }
  if (a->dgate) {
    Product p{};
    p.per_unit = 1;
    p.k_rows = 1;
    p.segs = 1;
    p.epi = kEpiStore;
    p.out_unit = d * f;
    p.m = f, p.n = d, p.ldo = d;
    p.b[0] = x_sum;
    p.a[0] = dense(w.dg, 1, f, 1);
    p.out = a->dgate;
    ck(go(p), fn, "dgate");
    p.a[0] = dense(w.du, 1, f, 1);
    p.out = a->dup;
    ck(go(p), fn, "dup");
    p.m = d, p.n = f, p.ldo = f;
    p.a[0] = dy_sum;
    p.b[0] = dense(w.hw, 1, f, 1);
    p.out = a->ddown;
    ck(go(p), fn, "ddown");
  }
}

template <class A, class F>
uint64_t bytes_of(const A* a, void (*check)(const A*), F&& space) {
  try {
    check(a);
    return a->rows ? space(a).bytes : 0;
  } catch (const std::exception&) {
    return 0;
  }
}

}  // namespace

extern "C" {

uint64_t tsb_linear_workspace(const tsb_linear_args* a) {
  return bytes_of(a, check_linear, linear_space);
}
ss_status tsb_linear(const tsb_linear_args* a) {
  return run([&] { linear(a); });
}
uint64_t tsb_linear_backward_workspace(const tsb_linear_grad_args* a) {
  return bytes_of(a, check_linear_back, linear_back_space);
}
ss_status tsb_linear_backward(const tsb_linear_grad_args* a) {
  return run([&] { linear_back(a); });
}

ss_status tsb_route(uint32_t dtype, const void* logits, uint64_t ld, uint64_t rows, uint32_t experts, uint32_t top,
                    int norm, int32_t* ids, float* weights, void* stream) {
  return run([&] {
    const char* fn = "tsb_route";
    need(dtype <= TSB_F32, fn, "dtype must be TSB_BF16, TSB_F16 or TSB_F32");
    need(experts >= 1 && experts <= 1024, fn, "experts must be in [1, 1024]");
    need(top >= 1 && top <= 32 && top <= experts, fn, "top must be in [1, 32] and at most experts");
    need(rows < kMaxRows, fn, "rows must be below 2^28");
    if (!rows) return;
    need(logits && ids && weights, fn, "null argument");
    need_elements(fn, {logits}, dtype == TSB_F32 ? 4 : 2);
    need_elements(fn, {ids, weights}, 4);
    need(ld >= experts, fn, "a leading dimension is shorter than its row");
    ck(launch_route(int(dtype), logits, ld, rows, experts, top, norm, ids, weights, static_cast<cudaStream_t>(stream)),
       fn, "launch");
  });
}
ss_status tsb_route_backward(uint32_t dtype, uint32_t dw_dtype, const void* dweights, const void* logits, uint64_t ld,
                             const int32_t* ids, const float* weights, uint64_t rows, uint32_t experts, uint32_t top,
                             int norm, void* dlogits, uint64_t ldd, void* stream) {
  return run([&] {
    const char* fn = "tsb_route_backward";
    need(dtype <= TSB_F32 && dw_dtype <= TSB_F32, fn, "dtypes must be TSB_BF16, TSB_F16 or TSB_F32");
    need(experts >= 1 && experts <= 1024, fn, "experts must be in [1, 1024]");
    need(top >= 1 && top <= 32 && top <= experts, fn, "top must be in [1, 32] and at most experts");
    need(rows < kMaxRows, fn, "rows must be below 2^28");
    if (!rows) return;
    need(dweights && (norm || logits) && ids && weights && dlogits, fn, "null argument");
    need_elements(fn, {norm ? nullptr : logits, dlogits}, dtype == TSB_F32 ? 4 : 2);
    need_elements(fn, {dweights}, dw_dtype == TSB_F32 ? 4 : 2);
    need_elements(fn, {ids, weights}, 4);
    need((norm || ld >= experts) && ldd >= experts, fn, "a leading dimension is shorter than its row");
    ck(launch_route_back(int(dtype), int(dw_dtype), dweights, logits, ld, ids, weights, rows, experts, top, norm,
                         dlogits, ldd, static_cast<cudaStream_t>(stream)),
       fn, "launch");
  });
}

ss_status tsb_units_from_view(const ss_dg_device_view* v, uint32_t g, uint32_t n_units, uint64_t matrix_bytes,
                              tsb_units* out) {
  return run([&] {
    const char* fn = "tsb_units_from_view";
    need(v && out, fn, "null argument");
    need(v->struct_size >= offsetof(ss_dg_device_view, absent_err), fn, "short view");
    need(g < v->n_gated, fn, "no such gated layer");
    need(v->n_parts >= 3, fn, "a unit needs the parts gate, up and down");
    *out = tsb_units{};
    out->struct_size = sizeof *out;
    out->n_units = n_units;
    out->n_slots = v->slots;
    out->slot_of = v->slot_of;
    out->unit_base = v->unit_base + g;
    out->abort = v->abort;
    out->absent_err = v->struct_size >= sizeof *v ? v->absent_err : nullptr;
    for (int i = 0; i < 3; ++i) {
      need(v->parts[i].bytes >= matrix_bytes, fn, "a part is smaller than its matrix");
      out->part[i] = v->parts[i].base;
      out->stride[i] = v->parts[i].stride;
    }
  });
}

uint64_t tsb_ffn_workspace(const tsb_ffn_args* a) { return bytes_of(a, check_ffn, ffn_space); }
ss_status tsb_ffn(const tsb_ffn_args* a) {
  return run([&] { ffn(a); });
}
uint64_t tsb_ffn_backward_workspace(const tsb_ffn_grad_args* a) {
  return bytes_of(a, check_ffn_back, ffn_back_space);
}
ss_status tsb_ffn_backward(const tsb_ffn_grad_args* a) {
  return run([&] { ffn_back(a); });
}

int tsb_ops_timeouts(void) {
  uint32_t v = 0, w = 0;
  const int a = ops_take_timeouts(&v), b = group_take_timeouts(&w);
  return a == 0 && b == 0 ? int(v + w) : -1;
}

}  // extern "C"
