// The gradient of a layer's activation and bias, and dropout, for gfx950: plain or quantised in
// the one pass that computes them.  The entry points are fp64emu_act_f8_backward and
// fp64emu_dropout_f8.

#include "f8_act.h"
#include "f8_common.h"
#include "f8_drop.h"
#include "f8_sums.h"

namespace {

struct ActGradArgs {
  const void *dy, *h;
  int64_t M, N, ld_dy, ld_h;
  int64_t blocks;                            // of 128 along a row
  int per;                                   // rows of a thread (rows kernel)
  void* dh;
  int64_t ld_dh;
  float* part;                               // sums over the rows of a group: [groups][N], or null
  Out8 rows, cols;
};

// A group's column sums from those of its threads' rows: thread t has columns 8 (t % 16) on.
struct ColumnRoom { float v[4][kBlk]; };

__device__ __forceinline__ void emit_sums(const float (&mine)[8], int cols, float* to, ColumnRoom& room) {
  const int cl = threadIdx.x & 15, wave = threadIdx.x >> 6;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float s = mine[j];
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if ((threadIdx.x & 48) == 0) room.v[wave][8 * cl + j] = s;
  }
  __syncthreads();
  const int c = threadIdx.x;
  if (c < cols && c < kBlk) to[c] = (room.v[0][c] + room.v[1][c]) + (room.v[2][c] + room.v[3][c]);
}

// One work group per 128 x 128 tile, for columns: dh in both orientations and its sums over the
// tile's rows from one reading.  Bound by its bytes: 8192 x 8192 bfloat16 with gelu_tanh and the bias's
// gradient 91 to 97 us, 4.2 to 4.5 TB/s of the copy's 5.2, with relu 90, gelu 96; the sums and their last kernel take 4 of them.
// (Its vector units are busy for 77% of it.)
// A kernel for each activation: with the choice in it, it spilled 250 registers and took 137.
template <int kT, int kAct>
__global__ void __launch_bounds__(kThreads, kT == FP64EMU_F32 ? 2 : 4) act_grad_tile_kernel(ActGradArgs a) {
  __shared__ TileLds lds;
  __shared__ ColumnRoom room;
  const uint32_t blocks = (uint32_t)a.blocks;
  const int64_t kb = blockIdx.x % blocks, mb = blockIdx.x / blocks;
  const int64_t row0 = mb * kBlk, col0 = kb * kBlk;
  const TilePlace t = tile_place(row0, col0, a.M, a.N);
  Held<FP64EMU_F32> d;
  {
    Held<kT> dy, h;
    int64_t row = row0 + 8 * t.rg;
    const int64_t col = col0 + 8 * t.cl;
#pragma unroll
    for (int p = 0; p < 8; ++p, ++row) {
      dy.load(p, a.dy, row * a.ld_dy + col, t.valid(p));
      if (kAct) h.load(p, a.h, row * a.ld_h + col, t.valid(p));
    }
#pragma unroll
    for (int p = 0; p < 8; ++p) {
#pragma unroll
      for (int j = 0; j < 8; ++j) d.v[p][j] = activated_back<kAct>(h.at(p, j), dy.at(p, j));
      __builtin_amdgcn_sched_barrier(0);     // (a row's temporaries at a time)
    }
  }
  if (a.part) {
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s[j] = d.v[0][j];
#pragma unroll
      for (int p = 1; p < 8; ++p) s[j] += d.v[p][j];
    }
    emit_sums(s, t.cols, a.part + mb * a.N + col0, room);
  }
  if (a.rows.q) emit_rows<FP64EMU_E4M3>(d, t, row0, col0, kb, a.rows);
  emit_cols<FP64EMU_E4M3>(d, t, row0, col0, mb, a.cols, lds);
}

// Without columns: a work group has 16 x per rows of one block of 128 columns, a row's block on 16
// lanes, 16 rows at a time.  8192 x 8192 plain 93 us (4.3 TB/s); 333 x 777 4.1 and the last sums' 2.5, where
// two launches take the host 6.
template <int kT, int kAct>
__global__ void __launch_bounds__(kThreads) act_grad_rows_kernel(ActGradArgs a) {
  __shared__ ColumnRoom room;
  const uint32_t blocks = (uint32_t)a.blocks;
  const int64_t kb = blockIdx.x % blocks, strip = blockIdx.x / blocks;
  Unit u;
  u.cl = threadIdx.x & 15;
  u.kb = kb;
  u.col = kb * kBlk + 8 * u.cl;
  u.valid = (int)(a.N - u.col < 8 ? a.N - u.col : 8);
  u.row = strip * a.per * 16 + (threadIdx.x >> 4);
  float s[8] = {};
  for (int i = 0; i < a.per && u.row < a.M; ++i, u.row += 16) {
    Held<kT> dy, h;
    dy.load(0, a.dy, u.row * a.ld_dy + u.col, u.valid);
    if (kAct) h.load(0, a.h, u.row * a.ld_h + u.col, u.valid);
    Held<FP64EMU_F32> d;
#pragma unroll
    for (int j = 0; j < 8; ++j) d.v[0][j] = activated_back<kAct>(h.at(0, j), dy.at(0, j));
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] += d.v[0][j];
    if (a.dh) store8<kT>(a.dh, u.row * a.ld_dh + u.col, u.valid, d.v[0]);
    if (a.rows.q) emit_unit<FP64EMU_E4M3>(d, u, u.col, u.kb, a.rows);
  }
  if (a.part) emit_sums(s, (int)(a.N - kb * kBlk < kBlk ? a.N - kb * kBlk : kBlk), a.part + strip * a.N + kb * kBlk, room);
}

struct DropArgs {
  const void* x;
  const int64_t* rng;
  int64_t M, K, ldx;
  int64_t blocks;
  uint32_t threshold;
  void* y;
  int64_t ldy;
  Out8 rows, cols;
};

template <int kT>
__device__ __forceinline__ void dropped(const Held<kT>& x, int p, const Drop& drop, uint64_t chunk, float (&y)[8]) {
  const Kept kept(drop, chunk);
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = kept.at(j) ? x.at(p, j) * drop.scale : 0.0f;
}

// A block of a row on 16 lanes.  8192 x 8192 bfloat16 plain 43 us (6.2 TB/s, more than the copy's 5.2), in 8 bits 47: the
// generator's twenty wide products for eight elements hide behind the memory.
template <int kT>
__global__ void __launch_bounds__(kThreads) dropout_rows_kernel(DropArgs a) {
  const Drop drop = drop_of(a.threshold, a.rng);
  const int64_t units = a.M * a.blocks, chunks = (a.K + 7) / 8;
  for (int64_t i = blockIdx.x * 16 + (threadIdx.x >> 4); i < units; i += gridDim.x * 16) {
    const Unit u = unit_at(i, a.blocks, a.K);
    Held<kT> x;
    Held<FP64EMU_F32> y;
    x.load(0, a.x, u.row * a.ldx + u.col, u.valid);
    dropped(x, 0, drop, (uint64_t)(u.row * chunks + u.col / 8), y.v[0]);
    if (a.y) store8<kT>(a.y, u.row * a.ldy + u.col, u.valid, y.v[0]);
    if (a.rows.q) emit_unit<FP64EMU_E4M3>(y, u, u.col, u.kb, a.rows);
  }
}

// Both ways by tiles of 128 x 128: 8192 x 8192 bfloat16 58 to 62 us, 4.4 to 4.7 TB/s, as the quantiser's 60.
template <int kT>
__global__ void __launch_bounds__(kThreads, kT == FP64EMU_F32 ? 3 : 4) dropout_tile_kernel(DropArgs a) {
  __shared__ TileLds lds;
  const uint32_t blocks = (uint32_t)a.blocks;
  const int64_t kb = blockIdx.x % blocks, mb = blockIdx.x / blocks;
  const int64_t row0 = mb * kBlk, col0 = kb * kBlk;
  const TilePlace t = tile_place(row0, col0, a.M, a.K);
  const Drop drop = drop_of(a.threshold, a.rng);
  const int64_t chunks = (a.K + 7) / 8, row = row0 + 8 * t.rg, col = col0 + 8 * t.cl;
  Held<FP64EMU_F32> y;
  {
    Held<kT> x;
#pragma unroll
    for (int p = 0; p < 8; ++p) x.load(p, a.x, (row + p) * a.ldx + col, t.valid(p));
#pragma unroll
    for (int p = 0; p < 8; ++p) dropped(x, p, drop, (uint64_t)((row + p) * chunks + col / 8), y.v[p]);
  }
  if (a.rows.q) emit_rows<FP64EMU_E4M3>(y, t, row0, col0, kb, a.rows);
  emit_cols<FP64EMU_E4M3>(y, t, row0, col0, mb, a.cols, lds);
}

// ---------------------------------------------------------------------------
// Host side.

constexpr int64_t kMaxGroups = (1ll << 31) / kThreads;

// Rows of a thread of act_grad_rows_kernel: one until the launch has 2048 work groups, then as many as
// keep it there, up to 16, so that few parts are left of the column sums.
int rows_per(int64_t M, int64_t blocks) {
  int per = 1;
  while (per < 16 && (M + 16 * per - 1) / (16 * per) * blocks > 2048) per *= 2;
  return per;
}

int64_t act_groups(int64_t M, int64_t N, bool cols) {
  const int64_t blocks = (N + kBlk - 1) / kBlk, tall = cols ? kBlk : 16 * rows_per(M, blocks);
  return (M + tall - 1) / tall;
}

int check_two(const fp64emu_f8_t* rows, const fp64emu_f8_t* cols) {
  for (const fp64emu_f8_t* f : {rows, cols})
    if (f && (f->fmt != FP64EMU_E4M3 || f->tiles)) return invalid("outputs are e4m3 with scales by rows");
  return FP64EMU_OK;
}

}  // namespace

extern "C" {

size_t fp64emu_act_f8_backward_workspace(int64_t M, int64_t N, int cols) {
  if (M <= 0 || N <= 0 || N >= 1ll << 31) return 0;
  const int64_t groups = act_groups(M, N, cols != 0);
  return groups > 1 ? 4 * (size_t)(groups * N) : 0;
}

int fp64emu_act_f8_backward(const void* dy, const void* h, int dtype, int act, int64_t M, int64_t N, int64_t ld_dy,
                            int64_t ld_h, void* dh, int64_t ld_dh, const fp64emu_f8_t* rows, const fp64emu_f8_t* cols,
                            float* dbias, void* workspace, size_t workspace_bytes, fp64emu_stream_t stream) {
  if (M < 0 || N < 0) return invalid("shapes must be non-negative");
  if (N >= 1ll << 31) return invalid("shapes must be below 2^31 columns");
  if (!known_dtype(dtype)) return invalid("dtype must be FP64EMU_F32, FP64EMU_BF16 or FP64EMU_F16");
  if (!known_act(act)) return invalid("act must be one of FP64EMU_ACT_*");
  if (int st = check_two(rows, cols)) return st;
  if (N == 0) return FP64EMU_OK;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Sums sums{};
  sums.out[0] = dbias;
  sums.D = N;
  if (M == 0) return launch_sums(sums, dbias ? 1 : 0, s);      // a sum of nothing
  if (!dh && !rows && !cols && !dbias) return invalid("no output asked for");
  if (!dy || (act && !h)) return invalid("null operand pointer");
  if (ld_dy < N || (act && ld_h < N) || (dh && ld_dh < N)) return invalid("rows are shorter than N");
  if (cols && dh) return invalid("columns come without dh in its plain form");
  ActGradArgs a{};
  if (int st = out8(rows, N, &a.rows)) return st;
  if (int st = out8(cols, M, &a.cols)) return st;
  a.dy = dy;
  a.h = h;
  a.M = M;
  a.N = N;
  a.ld_dy = ld_dy;
  a.ld_h = ld_h;
  a.blocks = (N + kBlk - 1) / kBlk;
  a.per = rows_per(M, a.blocks);
  a.dh = dh;
  a.ld_dh = ld_dh;
  sums.groups = act_groups(M, N, cols != nullptr);
  if (sums.groups > kMaxGroups / a.blocks) return invalid("operand too large for one launch");
  if (dbias) {
    const size_t need = fp64emu_act_f8_backward_workspace(M, N, cols != nullptr);
    if (need && (!workspace || workspace_bytes < need))
      return fp64emu_fail(FP64EMU_EWORKSPACE, "workspace too small: see fp64emu_act_f8_backward_workspace");
    if (need && !multiple(workspace, 4)) return invalid("workspace must be 4-byte aligned");
    a.part = sums.groups > 1 ? static_cast<float*>(workspace) : dbias;
    sums.part[0] = a.part;
  }
  const unsigned groups = (unsigned)(sums.groups * a.blocks);
  with_act(act, [&](auto which) {
    constexpr int kAct = decltype(which)::value;
#define FP64EMU_ACT_GRAD(T)                                                   \
  case T:                                                                     \
    if (cols) act_grad_tile_kernel<T, kAct><<<groups, kThreads, 0, s>>>(a);   \
    else act_grad_rows_kernel<T, kAct><<<groups, kThreads, 0, s>>>(a);        \
    break;
    switch (dtype) {
      FP64EMU_ACT_GRAD(FP64EMU_F32)
      FP64EMU_ACT_GRAD(FP64EMU_BF16)
      FP64EMU_ACT_GRAD(FP64EMU_F16)
    }
#undef FP64EMU_ACT_GRAD
  });
  if (int st = check_hip(hipGetLastError(), "act_f8_backward launch")) return st;
  return launch_sums(sums, dbias && sums.groups > 1 ? 1 : 0, s);
}

int fp64emu_dropout_f8(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, int drop, const int64_t* rng, void* y,
                       int64_t ldy, const fp64emu_f8_t* rows, const fp64emu_f8_t* cols, fp64emu_stream_t stream) {
  if (M < 0 || K < 0) return invalid("shapes must be non-negative");
  if (!known_dtype(dtype)) return invalid("dtype must be FP64EMU_F32, FP64EMU_BF16 or FP64EMU_F16");
  if (drop < 0 || drop > 65535) return invalid("drop must be in 0 .. 65535");
  if (drop && !rng) return invalid("drop needs rng");
  if (int st = check_two(rows, cols)) return st;
  if (M == 0 || K == 0) return FP64EMU_OK;
  if (!y && !rows && !cols) return invalid("no output asked for");
  if (!x) return invalid("null operand pointer");
  if (ldx < K || (y && ldy < K)) return invalid("rows are shorter than K");
  if (cols && y) return invalid("columns come without y in its plain form");
  DropArgs a{};
  if (int st = out8(rows, K, &a.rows)) return st;
  if (int st = out8(cols, M, &a.cols)) return st;
  a.x = x;
  a.rng = rng;
  a.M = M;
  a.K = K;
  a.ldx = ldx;
  a.blocks = (K + kBlk - 1) / kBlk;
  a.threshold = (uint32_t)drop;
  a.y = y;
  a.ldy = ldy;
  const int64_t mblocks = (M + kBlk - 1) / kBlk;
  if (mblocks > kMaxGroups / a.blocks) return invalid("operand too large for one launch");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const unsigned groups = (unsigned)(mblocks * a.blocks), few = unit_groups(M, a.blocks);
#define FP64EMU_DROP(T)                                                 \
  case T:                                                               \
    if (cols) dropout_tile_kernel<T><<<groups, kThreads, 0, s>>>(a);    \
    else dropout_rows_kernel<T><<<few, kThreads, 0, s>>>(a);            \
    break;
  switch (dtype) {
    FP64EMU_DROP(FP64EMU_F32)
    FP64EMU_DROP(FP64EMU_BF16)
    FP64EMU_DROP(FP64EMU_F16)
  }
#undef FP64EMU_DROP
  return check_hip(hipGetLastError(), "dropout_f8 launch");
}

}  // extern "C"
