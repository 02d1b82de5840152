// Operands in 8-bit floating point with one float32 scale per block of 128,
// for gfx950: the quantiser, products of such operands on the f8 matrix
// instructions, and the gated activation whose checkpoint is held so.  The
// entry points are those of include/fp64emu.h (fp64emu_*_f8*).
//
// A block with a = max(largest magnitude, 2^-110) has the scale s = a / F and
// the codes q = rne8(x ((1 / a) F)), F the format's largest value.  The floor
// keeps 1 / a finite for a block of zeros; the product exceeds F by at most three
// float32 roundings, which the conversion rounds back to F.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>
#include <utility>

#include "fp64emu.h"
#include "status.h"

namespace {

constexpr int kThreads = 256;
constexpr int kBlk = 128;                         // elements that share a scale
constexpr uint32_t kTinyBits = 0x08800000;        // 2^-110
constexpr int64_t kMaxGridZ = 65535;

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef unsigned int v2u __attribute__((ext_vector_type(2)));
typedef unsigned short v8s __attribute__((ext_vector_type(8)));

__host__ __device__ constexpr float top_of(int fmt) { return fmt == FP64EMU_E4M3 ? 448.0f : 57344.0f; }

// ---------------------------------------------------------------------------
// Values in and codes out, eight at a time.  Rows start anywhere: accesses of
// eight elements are unaligned ones (the hardware splits those that need it),
// and only a row's last, partial eight go element by element.

__device__ __forceinline__ float bf16_value(unsigned short h) {
  return __builtin_bit_cast(float, (uint32_t)h << 16);
}
__device__ __forceinline__ unsigned short bf16_round(float f) {   // nearest even; NaN stays NaN
  return __builtin_bit_cast(unsigned short, (__bf16)f);
}

template <int kT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (kT == FP64EMU_F32) return static_cast<const float*>(p)[i];
  if constexpr (kT == FP64EMU_BF16) return bf16_value(static_cast<const unsigned short*>(p)[i]);
  return (float)static_cast<const _Float16*>(p)[i];
}
template <int kT>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if constexpr (kT == FP64EMU_F32) static_cast<float*>(p)[i] = v;
  if constexpr (kT == FP64EMU_BF16) static_cast<unsigned short*>(p)[i] = bf16_round(v);
  if constexpr (kT == FP64EMU_F16) static_cast<_Float16*>(p)[i] = (_Float16)v;
}

template <int kT>
__device__ __forceinline__ void store8(void* p, int64_t i, int valid, const float (&v)[8]) {
  if (valid >= 8) {
    if constexpr (kT == FP64EMU_F32) {
      __builtin_memcpy(static_cast<float*>(p) + i, v, 32);
    } else {
      v8s a;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        a[j] = kT == FP64EMU_BF16 ? bf16_round(v[j])
                                  : __builtin_bit_cast(unsigned short, (_Float16)v[j]);
      __builtin_memcpy(static_cast<unsigned short*>(p) + i, &a, 16);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (j < valid) store1<kT>(p, i + j, v[j]);
}

template <int kFmt>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int v = 0;
  if constexpr (kFmt == FP64EMU_E4M3) {
    v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, v, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
  } else {
    v = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, v, false);
    v = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, v, true);
  }
  return (uint32_t)v;
}

// The values of four codes.
template <int kFmt>
__device__ __forceinline__ void values4(uint32_t w, float* v) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  v2f lo, hi;
  if constexpr (kFmt == FP64EMU_E4M3) {
    lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  } else {
    lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false);
    hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true);
  }
  v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
}

// Eight codes, the first `valid` of them.
__device__ __forceinline__ void put8(uint8_t* q, int valid, v2u w) {
  if (valid >= 8) {
    typedef v2u v2u_any __attribute__((aligned(1)));
    __builtin_nontemporal_store(w, reinterpret_cast<v2u_any*>(q));
    return;
  }
  uint64_t v = (uint64_t)w[1] << 32 | w[0];
#pragma unroll 1
  for (int j = 0; j < valid; ++j, v >>= 8) q[j] = (uint8_t)v;
}
__device__ __forceinline__ v2u get8(const uint8_t* q, int valid) {
  v2u w = {0u, 0u};
  if (valid >= 8) {
    __builtin_memcpy(&w, q, 8);
    return w;
  }
  uint64_t v = 0;
#pragma unroll 1
  for (int j = valid - 1; j >= 0; --j) v = v << 8 | q[j];
  return v2u{(uint32_t)v, (uint32_t)(v >> 32)};
}

// Magnitudes are compared as integers: for floats with the sign cleared that
// is the order of their values, with NaN above infinity, so that one NaN in a
// block becomes its maximum.
__device__ __forceinline__ uint32_t mag(float f) { return __builtin_bit_cast(uint32_t, f) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
typedef unsigned short v2s __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t umax16(uint32_t a, uint32_t b) {   // of each half
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2s, a),
                                                                __builtin_bit_cast(v2s, b)));
}

// Eight rows of eight elements of x as they came, in a thread's registers.
// Column magnitudes come as kWords words of the values' own width (two to a
// word in 16 bits), so that their joining takes half the steps there.
template <int kT>
struct Held {
  static constexpr int kWords = 4;
  v4u w[8];
  __device__ __forceinline__ void load(int p, const void* x, int64_t i, int valid) {
    const unsigned short* q = static_cast<const unsigned short*>(x) + i;
    if (valid >= 8) {
      __builtin_memcpy(&w[p], q, 16);
      return;
    }
    uint64_t lo = 0, hi = 0;
#pragma unroll 1
    for (int j = valid - 1; j >= 0; --j) {
      hi = hi << 16 | lo >> 48;
      lo = lo << 16 | q[j];
    }
    w[p] = v4u{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  }
  // Makes the compiler unpack the words again instead of keeping 64 floats beside
  // them from one use to the next (bfloat16: 59 registers, not 120, in the quantiser both
  // ways, 127, not 234, in the activation).
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int p = 0; p < 8; ++p) asm volatile("" : "+v"(w[p]));
  }
  static __device__ __forceinline__ float value(uint32_t h) {
    return kT == FP64EMU_BF16 ? bf16_value((unsigned short)h)
                              : (float)__builtin_bit_cast(_Float16, (unsigned short)h);
  }
  __device__ __forceinline__ float at(int p, int j) const { return value(w[p][j >> 1] >> (16 * (j & 1))); }
  static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return umax16(a, b); }
  // The magnitude of column j in the words' column word, as a float's bits.
  static __device__ __forceinline__ uint32_t bits(uint32_t word, int j) {
    return __builtin_bit_cast(uint32_t, value(word >> (16 * (j & 1)) & 0xffffu));
  }
  __device__ __forceinline__ uint32_t row_mag(int p) const {
    uint32_t m = 0;
#pragma unroll
    for (int d = 0; d < 4; ++d) m = umax16(m, w[p][d] & 0x7fff7fffu);
    return __builtin_bit_cast(uint32_t, value(umax(m & 0xffffu, m >> 16)));
  }
  __device__ __forceinline__ uint32_t col_word(int d) const {
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p) m = umax16(m, w[p][d] & 0x7fff7fffu);
    return m;
  }
};

template <>
struct Held<FP64EMU_F32> {
  static constexpr int kWords = 8;
  float v[8][8];
  __device__ __forceinline__ void load(int p, const void* x, int64_t i, int valid) {
    const float* q = static_cast<const float*>(x) + i;
    if (valid >= 8) {
      __builtin_memcpy(v[p], q, 32);
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[p][j] = j < valid ? q[j] : 0.0f;
  }
  __device__ __forceinline__ void again() {}
  __device__ __forceinline__ float at(int p, int j) const { return v[p][j]; }
  static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return umax(a, b); }
  static __device__ __forceinline__ uint32_t bits(uint32_t word, int) { return word; }
  __device__ __forceinline__ uint32_t row_mag(int p) const {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = umax(m, mag(v[p][j]));
    return m;
  }
  __device__ __forceinline__ uint32_t col_word(int d) const {
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p) m = umax(m, mag(v[p][d]));
    return m;
  }
};

// The maximum over the 16 lanes of a DPP row, in all of them.
__device__ __forceinline__ uint32_t row16_max(uint32_t m) {
  m = umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x128, 0xf, 0xf, false));   // row_ror:8
  m = umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x124, 0xf, 0xf, false));
  m = umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x122, 0xf, 0xf, false));
  return umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x121, 0xf, 0xf, false));
}
// Lane kLane of each DPP row, in all of the row.
template <int kLane>
__device__ __forceinline__ float row16_lane(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x150 + kLane,
                                                              0xf, 0xf, false));   // row_newbcast
}
template <class Fn, int... kP>
__device__ __forceinline__ void each_row(const Fn& fn, std::integer_sequence<int, kP...>) {
  (fn(std::integral_constant<int, kP>{}), ...);
}
__device__ __forceinline__ float amax_of(uint32_t m) { return __builtin_bit_cast(float, umax(m, kTinyBits)); }

// F / a as (1 / a) F, both rounded.  1 / a: the hardware's reciprocal (within one
// ulp) and one Newton step, y + y (1 - a y) with fused multiply-adds, which rounds
// correctly (checked for all 2^23 significands; the exponent does not matter
// while 1 / a is normal); a division (ten instructions and more) past that.
template <int kFmt>
__device__ __forceinline__ float inverse_scale(float a) {
  float y;
  if (a <= 0x1p125f) {
    y = __builtin_amdgcn_rcpf(a);
    y = fmaf(fmaf(-a, y, 1.0f), y, y);
  } else {
    y = 1.0f / a;
  }
  return y * top_of(kFmt);
}
// a / F, rounded once: F is a constant, the quotient's first guess off by an ulp at
// most, the remainder a - F q exact (a >= 2^-110), so the correction rounds correctly.
template <int kFmt>
__device__ __forceinline__ float scale_of(float a) {
  constexpr float inv = 1.0f / top_of(kFmt);
  const float q = a * inv;
  return a < __builtin_inff() ? fmaf(fmaf(-top_of(kFmt), q, a), inv, q) : a;
}

// One quantised output as the kernels take it (an fp64emu_f8_t for one member
// at a time); q null: not asked for.
struct Out8 {
  uint8_t* q;
  float* s;
  int64_t ld, stride, s_row, s_block, s_stride;
};

__device__ __forceinline__ void member(Out8& o, int64_t b) {
  o.q += b * o.stride;
  o.s += b * o.s_stride;
}

// ---------------------------------------------------------------------------
// A 128 x 128 tile in the registers of 256 threads: thread t holds rows
// 8 (t / 16) .. + 7 and columns 8 (t % 16) .. + 7.  A row's block is then 16
// lanes of one DPP row, so its maximum takes four DPP steps; a column's is
// spread over the 16 row groups: two lane exchanges and one pass through LDS.
// The transposed codes go through LDS too, in 8-byte chunks (one thread's 8 rows
// of a column) whose place in the column's 128 bytes is xored with the column
// group, so that neither the writes (16 column groups of one row group) nor the
// reads (16 chunks of one column) collide.
struct TileLds {
  uint32_t colmax[4][kBlk];
  uint8_t codes[kBlk * kBlk];
};

struct TilePlace {
  int rg, cl;                // row and column group of the thread
  int rows, cols;            // valid rows and columns of the tile
  __device__ __forceinline__ int valid(int p) const { return 8 * rg + p < rows ? cols - 8 * cl : 0; }
};

__device__ __forceinline__ TilePlace tile_place(int64_t row0, int64_t col0, int64_t M, int64_t K) {
  return {(int)threadIdx.x >> 4, (int)threadIdx.x & 15, (int)(M - row0 < kBlk ? M - row0 : kBlk),
          (int)(K - col0 < kBlk ? K - col0 : kBlk)};
}

template <int kFmt, class H>
__device__ __forceinline__ v2u row_codes(const H& v, int p, float r) {
  return v2u{codes4<kFmt>(v.at(p, 0) * r, v.at(p, 1) * r, v.at(p, 2) * r, v.at(p, 3) * r),
             codes4<kFmt>(v.at(p, 4) * r, v.at(p, 5) * r, v.at(p, 6) * r, v.at(p, 7) * r)};
}

// The rows' blocks of a tile at row0, block kb of the output.
template <int kFmt, class H>
__device__ __forceinline__ void emit_rows(const H& v, const TilePlace& t, int64_t row0, int64_t col0,
                                          int64_t kb, const Out8& o) {
  uint8_t* q = o.q + (row0 + 8 * t.rg) * o.ld + col0 + 8 * t.cl;
  float mine = 0.0f;         // lane cl < 8 of the row group writes row cl's scale
#pragma unroll
  for (int p = 0; p < 8; ++p, q += o.ld) {
    const float a = amax_of(row16_max(v.row_mag(p)));
    mine = t.cl == p ? a : mine;
    put8(q, t.valid(p), row_codes<kFmt>(v, p, inverse_scale<kFmt>(a)));
  }
  if (t.cl < 8 && 8 * t.rg + t.cl < t.rows)
    o.s[(row0 + 8 * t.rg + t.cl) * o.s_row + kb * o.s_block] = scale_of<kFmt>(mine);
}

// The columns' codes: q row (col0 + column), byte row0 + row.  r[j]: F / a of
// this thread's column j.
template <int kFmt, class H>
__device__ __forceinline__ void emit_transposed(const H& v, const float (&r)[8], const TilePlace& t,
                                                int64_t row0, int64_t col0, const Out8& o, TileLds& lds) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const v2u w = {codes4<kFmt>(v.at(0, j) * r[j], v.at(1, j) * r[j], v.at(2, j) * r[j], v.at(3, j) * r[j]),
                   codes4<kFmt>(v.at(4, j) * r[j], v.at(5, j) * r[j], v.at(6, j) * r[j], v.at(7, j) * r[j])};
    *reinterpret_cast<v2u*>(lds.codes + (8 * t.cl + j) * kBlk + 8 * (t.rg ^ t.cl)) = w;
  }
  __syncthreads();
  const int chunk = t.cl, left = t.rows - 8 * chunk;       // 16 lanes: one column's 128 bytes
  uint8_t* q = o.q + (col0 + t.rg) * o.ld + row0 + 8 * chunk;
#pragma unroll
  for (int p = 0; p < 8; ++p, q += 16 * o.ld) {
    const int c = p * 16 + t.rg;
    const v2u w = *reinterpret_cast<const v2u*>(lds.codes + c * kBlk + 8 * (chunk ^ (c >> 3)));
    if (c < t.cols) put8(q, left, w);
  }
}

template <int kFmt, class H>
__device__ __forceinline__ void emit_cols(const H& v, const TilePlace& t, int64_t row0, int64_t col0,
                                          int64_t mb, const Out8& o, TileLds& lds) {
  constexpr int kW = H::kWords, kPer = 8 / kW;               // columns per word
#pragma unroll
  for (int d = 0; d < kW; ++d) {
    uint32_t m = v.col_word(d);
    m = H::join(m, (uint32_t)__shfl_xor((int)m, 16));
    m = H::join(m, (uint32_t)__shfl_xor((int)m, 32));
    if ((t.rg & 3) == 0) lds.colmax[t.rg >> 2][kW * t.cl + d] = m;
  }
  __syncthreads();
  auto joined = [&](int word) {
    return H::join(H::join(lds.colmax[0][word], lds.colmax[1][word]),
                   H::join(lds.colmax[2][word], lds.colmax[3][word]));
  };
  float r[8];
#pragma unroll
  for (int d = 0; d < kW; ++d) {
    const uint32_t m = joined(kW * t.cl + d);
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      r[kPer * d + e] = inverse_scale<kFmt>(amax_of(H::bits(m, e)));
  }
  const int c = threadIdx.x;
  if (c < t.cols)
    o.s[(col0 + c) * o.s_row + mb * o.s_block] = scale_of<kFmt>(amax_of(H::bits(joined(c / kPer), c % kPer)));
  emit_transposed<kFmt>(v, r, t, row0, col0, o, lds);
}

// One scale for the whole tile, both orientations.
template <int kFmt, class H>
__device__ __forceinline__ void emit_tile(const H& v, const TilePlace& t, int64_t row0, int64_t col0,
                                          const Out8& rows, const Out8& cols, TileLds& lds) {
  uint32_t m = 0;
#pragma unroll
  for (int p = 0; p < 8; ++p) m = umax(m, v.row_mag(p));
  m = row16_max(m);
  m = umax(m, (uint32_t)__shfl_xor((int)m, 16));
  m = umax(m, (uint32_t)__shfl_xor((int)m, 32));
  if ((threadIdx.x & 63) == 0) lds.colmax[threadIdx.x >> 6][0] = m;
  __syncthreads();
  const float a = amax_of(umax(umax(lds.colmax[0][0], lds.colmax[1][0]),
                               umax(lds.colmax[2][0], lds.colmax[3][0])));
  const float r = inverse_scale<kFmt>(a), s = scale_of<kFmt>(a);
  const int64_t mb = row0 / kBlk, kb = col0 / kBlk;
  if (rows.q) {
    if (threadIdx.x == 0) rows.s[mb * rows.s_row + kb * rows.s_block] = s;
    uint8_t* q = rows.q + (row0 + 8 * t.rg) * rows.ld + col0 + 8 * t.cl;
#pragma unroll
    for (int p = 0; p < 8; ++p, q += rows.ld) put8(q, t.valid(p), row_codes<kFmt>(v, p, r));
  }
  if (cols.q) {
    if (threadIdx.x == 0) cols.s[kb * cols.s_row + mb * cols.s_block] = s;
    const float rr[8] = {r, r, r, r, r, r, r, r};
    emit_transposed<kFmt>(v, rr, t, row0, col0, cols, lds);
  }
}

// ---------------------------------------------------------------------------
// Quantiser.
struct QuantArgs {
  const void* x;
  int64_t batch0, M, K, ldx, stride_x;                     // batch0: member of blockIdx.z = 0
  int64_t kblocks;
  Out8 rows, cols;
};

enum { kRows = 1, kCols = 2, kTiles = 4 };                 // what a call asks for

// One work group per 128 x 128 tile (blocks along K fastest: a row of tiles
// reads whole rows of x), every value read once.  Bound by its bytes: 8192 x 8192
// bfloat16 into rows and columns 60 us, 4.6 TB/s where a large copy reaches 5.2.
// A float32 2049 x 4097 into tiles both ways 15 us against 10 at that rate: 561
// groups, two or three to a CU, all reading first and all writing last.
template <int kT, int kFmt, int kForm>
__global__ void __launch_bounds__(kThreads, kT == FP64EMU_F32 ? 3 : 4) quant_tile_kernel(QuantArgs g) {
  __shared__ TileLds lds;
  const uint32_t kblocks = (uint32_t)g.kblocks;
  const int64_t kb = blockIdx.x % kblocks, mb = blockIdx.x / kblocks;
  const int64_t row0 = mb * kBlk, col0 = kb * kBlk;
  const TilePlace t = tile_place(row0, col0, g.M, g.K);
  const int64_t b = g.batch0 + blockIdx.z;
  if (g.rows.q) member(g.rows, b);
  if (g.cols.q) member(g.cols, b);
  Held<kT> v;
  int64_t i = b * g.stride_x + (row0 + 8 * t.rg) * g.ldx + col0 + 8 * t.cl;
#pragma unroll
  for (int p = 0; p < 8; ++p, i += g.ldx) v.load(p, g.x, i, t.valid(p));
  if constexpr (kForm & kTiles) {
    emit_tile<kFmt>(v, t, row0, col0, g.rows, g.cols, lds);
  } else {
    if constexpr (kForm & kRows) {
      emit_rows<kFmt>(v, t, row0, col0, kb, g.rows);
      v.again();
    }
    emit_cols<kFmt>(v, t, row0, col0, mb, g.cols, lds);
  }
}

// Rows only: 16 lanes per block, so that one token's blocks spread over work groups
// instead of filling 1 row in 128 of a tile.  1 x 8192: 2.3 us, one memory round trip
// and a launch.
struct Unit {
  int64_t row, kb, col;      // block kb of a row; the lane's first column
  int cl, valid;
};
// Unit i of `rows` rows of `blocks` blocks of a matrix of K columns.
__device__ __forceinline__ Unit unit_at(int64_t i, int64_t blocks, int64_t K) {
  Unit u;
  u.row = (uint64_t)i >> 31 ? i / blocks : (int64_t)((uint32_t)i / (uint32_t)blocks);
  u.kb = i - u.row * blocks;
  u.cl = threadIdx.x & 15;
  u.col = u.kb * kBlk + 8 * u.cl;
  u.valid = (int)(K - u.col < 8 ? K - u.col : 8);
  return u;
}
// A unit's codes and scale from a lane's eight values.
template <int kFmt, class H>
__device__ __forceinline__ void emit_unit(const H& v, const Unit& u, int64_t col, int64_t kb, const Out8& o) {
  const float a = amax_of(row16_max(v.row_mag(0)));
  put8(o.q + u.row * o.ld + col, u.valid, row_codes<kFmt>(v, 0, inverse_scale<kFmt>(a)));
  if (u.cl == 0) o.s[u.row * o.s_row + kb * o.s_block] = scale_of<kFmt>(a);
}

template <int kT, int kFmt>
__global__ void __launch_bounds__(kThreads) quant_rows_kernel(QuantArgs g) {
  const int64_t b = g.batch0 + blockIdx.z, units = g.M * g.kblocks;
  Out8 o = g.rows;
  member(o, b);
  for (int64_t i = blockIdx.x * 16 + (threadIdx.x >> 4); i < units; i += gridDim.x * 16) {
    const Unit u = unit_at(i, g.kblocks, g.K);
    Held<kT> v;
    v.load(0, g.x, b * g.stride_x + u.row * g.ldx + u.col, u.valid);
    emit_unit<kFmt>(v, u, u.col, u.kb, o);
  }
}

// ---------------------------------------------------------------------------
// Gated activation.  1 / (1 + e^-g): e^-g = 2^(-g log2 e) with the product's
// rounding error carried into the result (as a relative term, ln 2 times the
// error), so that large |g| keeps float32 accuracy with the hardware's 2^x.
__device__ __forceinline__ float sigmoid(float g) {
  constexpr float kL = 1.44269502f, kLlo = 1.92596303e-8f;      // log2 e = kL + kLlo
  const float t = -g * kL;
  const float lo = fmaf(-g, kL, -t) - g * kLlo;
  float e = __builtin_amdgcn_exp2f(t);
  // Outside the normal range of 2^t the term is left out: there it would be inf - inf.
  if (fabsf(t) < 126.0f) e = fmaf(e, lo * 0.693147182f, e);
  return __builtin_amdgcn_rcpf(1.0f + e);                       // within one ulp
}

struct SwigluArgs {
  const void* h;
  int64_t M, F, ldh;
  int64_t fblocks;
  void* y;
  int64_t ldy;
  Out8 keep, rows, cols;
};

// One work group per 128 x 128 tile of y.  Bound by its bytes: 8192 x 4096 with the
// checkpoint and y both ways 61 us, 4.5 TB/s of the copy's 5.2.
template <int kT>
__global__ void __launch_bounds__(kThreads) swiglu_kernel(SwigluArgs a) {
  constexpr int kF = FP64EMU_E4M3;
  __shared__ TileLds lds;
  const uint32_t fblocks = (uint32_t)a.fblocks;
  const int64_t fb = blockIdx.x % fblocks, mb = blockIdx.x / fblocks;
  const int64_t row0 = mb * kBlk, col0 = fb * kBlk;
  const TilePlace t = tile_place(row0, col0, a.M, a.F);
  Held<FP64EMU_F32> y;
  {
    Held<kT> g, u;
    int64_t i = (row0 + 8 * t.rg) * a.ldh + col0 + 8 * t.cl;
#pragma unroll
    for (int p = 0; p < 8; ++p, i += a.ldh) {
      g.load(p, a.h, i, t.valid(p));
      u.load(p, a.h, i + a.F, t.valid(p));
    }
    if (a.keep.q) {
      emit_rows<kF>(g, t, row0, col0, fb, a.keep);
      emit_rows<kF>(u, t, row0, a.F + col0, a.fblocks + fb, a.keep);
      g.again();
      u.again();
    }
#pragma unroll
    for (int p = 0; p < 8; ++p)
#pragma unroll
      for (int j = 0; j < 8; ++j) y.v[p][j] = g.at(p, j) * sigmoid(g.at(p, j)) * u.at(p, j);
  }
  if (a.y) {
#pragma unroll
    for (int p = 0; p < 8; ++p)
      store8<kT>(a.y, (row0 + 8 * t.rg + p) * a.ldy + col0 + 8 * t.cl, t.valid(p), y.v[p]);
  }
  if (a.rows.q) emit_rows<kF>(y, t, row0, col0, fb, a.rows);
  if (a.cols.q) emit_cols<kF>(y, t, row0, col0, mb, a.cols, lds);
}

// Without columns to write: a block of a row on 16 lanes.  1 x 4096: 2.3 us, where a
// tile's work group took 6.4.
template <int kT>
__global__ void __launch_bounds__(kThreads) swiglu_rows_kernel(SwigluArgs a) {
  constexpr int kF = FP64EMU_E4M3;
  const int64_t units = a.M * a.fblocks;
  for (int64_t i = blockIdx.x * 16 + (threadIdx.x >> 4); i < units; i += gridDim.x * 16) {
    const Unit t = unit_at(i, a.fblocks, a.F);
    Held<kT> g, u;
    g.load(0, a.h, t.row * a.ldh + t.col, t.valid);
    u.load(0, a.h, t.row * a.ldh + a.F + t.col, t.valid);
    if (a.keep.q) {
      emit_unit<kF>(g, t, t.col, t.kb, a.keep);
      emit_unit<kF>(u, t, a.F + t.col, a.fblocks + t.kb, a.keep);
    }
    Held<FP64EMU_F32> y;
#pragma unroll
    for (int j = 0; j < 8; ++j) y.v[0][j] = g.at(0, j) * sigmoid(g.at(0, j)) * u.at(0, j);
    if (a.y) store8<kT>(a.y, t.row * a.ldy + t.col, t.valid, y.v[0]);
    if (a.rows.q) emit_unit<kF>(y, t, t.col, t.kb, a.rows);
  }
}

struct SwigluGradArgs {
  const void* dy;
  int64_t M, F, ldy;
  int64_t fblocks, tiles;
  Out8 keep;                 // read
  void* dh;
  int64_t ldh;
  Out8 rows, cols;
};

// Two work groups per 128 x 128 tile of dy, one for dg's tile and one for du's
// (which needs no u): both tiles' values at once took 256 registers and 110 us
// at 8192 x 4096, where this takes half of them.  The two are eight groups apart,
// on one XCD, whose L2 then has what both read.  8192 x 4096 both ways 73 us, 3.7 TB/s:
// 65 with the sigmoid left out and 50 without the columns, so the transposed
// codes' way through LDS and their stores hold it most.
template <int kT, int kO>
__global__ void __launch_bounds__(kThreads, kT == FP64EMU_F32 ? 2 : 4) swiglu_grad_kernel(SwigluGradArgs a) {
  constexpr int kF = FP64EMU_E4M3;
  __shared__ TileLds lds;
  const bool up = blockIdx.x & 8;                            // du's half
  const uint32_t tile = (blockIdx.x >> 4) * 8 + (blockIdx.x & 7), fblocks = (uint32_t)a.fblocks;
  if (tile >= a.tiles) return;
  const int64_t fb = tile % fblocks, mb = tile / fblocks;
  const int64_t row0 = mb * kBlk, col0 = fb * kBlk;
  const TilePlace t = tile_place(row0, col0, a.M, a.F);
  // Lane cl of a row group has row cl % 8's scale, of g in the lower eight lanes
  // and of u in the upper ones: broadcast within the DPP row where it is used.
  float scales = 0.0f;
  if (8 * t.rg + (t.cl & 7) < t.rows)
    scales = a.keep.s[(row0 + 8 * t.rg + (t.cl & 7)) * a.keep.s_row +
                      (t.cl < 8 ? fb : a.fblocks + fb) * a.keep.s_block];
  Held<FP64EMU_F32> d;
  {
    Held<kT> dy;
    v2u g[8], u[8];
    int64_t i = (row0 + 8 * t.rg) * a.ldy + col0 + 8 * t.cl;
    const uint8_t* q = a.keep.q + (row0 + 8 * t.rg) * a.keep.ld + col0 + 8 * t.cl;
#pragma unroll
    for (int p = 0; p < 8; ++p, i += a.ldy, q += a.keep.ld) {
      const int valid = t.valid(p);
      dy.load(p, a.dy, i, valid);
      g[p] = get8(q, valid);
      u[p] = get8(q + a.F, up ? 0 : valid);
    }
    auto row = [&](auto P) {
      constexpr int p = decltype(P)::value;
      const float sg = row16_lane<p>(scales), su = row16_lane<8 + p>(scales);
      float gv[8], uv[8];
      values4<kF>(g[p][0], gv);
      values4<kF>(g[p][1], gv + 4);
      values4<kF>(u[p][0], uv);
      values4<kF>(u[p][1], uv + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = gv[j] * sg, s = sigmoid(x), ds = dy.at(p, j) * s;
        d.v[p][j] = up ? ds * x : ds * (uv[j] * su) * fmaf(x, 1.0f - s, 1.0f);
      }
    };
    each_row(row, std::make_integer_sequence<int, 8>{});
  }
  const int64_t at = up ? a.F : 0, block = up ? a.fblocks : 0;
  if (a.dh) {
#pragma unroll
    for (int p = 0; p < 8; ++p)
      store8<kO>(a.dh, (row0 + 8 * t.rg + p) * a.ldh + at + col0 + 8 * t.cl, t.valid(p), d.v[p]);
  }
  if (a.rows.q) emit_rows<kF>(d, t, row0, at + col0, block + fb, a.rows);
  if (a.cols.q) emit_cols<kF>(d, t, row0, at + col0, mb, a.cols, lds);
}

// Without columns to write: a block of a row on 16 lanes, both halves.  333 x 777:
// 3.9 us, where tiles took 11.3.
template <int kT, int kO>
__global__ void __launch_bounds__(kThreads) swiglu_grad_rows_kernel(SwigluGradArgs a) {
  constexpr int kF = FP64EMU_E4M3;
  const int64_t units = a.M * a.fblocks;
  for (int64_t i = blockIdx.x * 16 + (threadIdx.x >> 4); i < units; i += gridDim.x * 16) {
    const Unit t = unit_at(i, a.fblocks, a.F);
    Held<kT> dy;
    dy.load(0, a.dy, t.row * a.ldy + t.col, t.valid);
    const uint8_t* q = a.keep.q + t.row * a.keep.ld + t.col;
    const v2u g = get8(q, t.valid), u = get8(q + a.F, t.valid);
    const float* s = a.keep.s + t.row * a.keep.s_row;
    const float sg = s[t.kb * a.keep.s_block], su = s[(a.fblocks + t.kb) * a.keep.s_block];
    Held<FP64EMU_F32> dg, du;
    float gv[8], uv[8];
    values4<kF>(g[0], gv);
    values4<kF>(g[1], gv + 4);
    values4<kF>(u[0], uv);
    values4<kF>(u[1], uv + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = gv[j] * sg, sig = sigmoid(x), ds = dy.at(0, j) * sig;
      du.v[0][j] = ds * x;
      dg.v[0][j] = ds * (uv[j] * su) * fmaf(x, 1.0f - sig, 1.0f);
    }
    if (a.dh) {
      store8<kO>(a.dh, t.row * a.ldh + t.col, t.valid, dg.v[0]);
      store8<kO>(a.dh, t.row * a.ldh + a.F + t.col, t.valid, du.v[0]);
    }
    if (a.rows.q) {
      emit_unit<kF>(dg, t, t.col, t.kb, a.rows);
      emit_unit<kF>(du, t, a.F + t.col, a.fblocks + t.kb, a.rows);
    }
  }
}

// ---------------------------------------------------------------------------
// Products.  out^T = B A^T on v_mfma_f32_16x16x128_f8f6f4: one instruction
// covers one block of 128 along K, so its float32 result is scaled by
// sA sB and added to the running sums, which stay in float32 registers.  B's
// rows are the instruction's first operand: lane l then holds output column
// (token) l % 16 and four successive n, so that a tile scale of B and a row
// scale of A make one factor per lane, and the four values are one store.
//
// Operand order: lane l holds 32 bytes of row l % 16, at k = 32 (l / 16).
// Which k those are to the instruction does not matter as long as A and B
// agree, since every k of a block has the same scales.

struct MmArgs {
  const uint8_t *A, *B;
  const float *sA, *sB;
  void* out;
  float* part;                       // partial sums [splits, batch, M, N] if splits > 1
  int64_t lda, ldb, strideA, strideB;
  int64_t sA_row, sA_blk, sA_str, sB_row, sB_blk, sB_str;
  int64_t ldo, stride_o;
  int64_t K;
  int M, N, batch;
  int nkb, splits, kb_per_split;     // blocks along K: of all, and of one split
  int tiles_m, tiles_n;
  int dtype, accumulate;
  int b_tiles;                       // B's scales by tiles
  int vec_o;                         // out's rows start at multiples of 4 elements
};

typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));

// A block's sum has to come out where the scales' own product leaves float32's range (2^-80 by
// 2^-70, or 2^70 by 2^60 beside codes of zero).
//
// Split scales, for any: 2^x and s / 2^x, x the exponent kept to -110 .. 100.  The matrix
// instructions take 2^x with the codes, exactly, and the block's sum meets only the
// product of the two remainders, 1 to 4 for scales in that range.  In that range of x every
// code's value is a normal bfloat16, and what goes beyond it (zero, denormal, infinite
// scales) stays in the remainder.
struct Split { float power, rest; };
__device__ __forceinline__ Split split_scale(float s) {
  const uint32_t e =
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_fmed3f(fabsf(s), 0x1p-110f, 0x1p100f)) & 0x7f800000u;
  return {__builtin_bit_cast(float, e), s * __builtin_bit_cast(float, 0x7f000000u - e)};
}

// One frame, for scales whose product is below 2^24: the sums are kept at 2^40 times their size.
// A block's sum is at most 2^39 (128 products of two e5m2 codes), so a product of scales that is denormal
// at that size belongs to a result that is denormal at its own, and 2^24 blocks of at most 2^64 2^39
// stay finite.  Both scales below 2^12 will do, too.
constexpr float kFrame = 0x1p40f, kFrameTop = 0x1p64f;       // of the products of scales, at 2^40 times
constexpr float kFrameTopA = 0x1p52f, kFrameTopB = 0x1p12f;  // of A's scales, at 2^40 times, and of B's

// A fragment as the block's sum takes it.  Its 32 codes as they are, for one
// v_mfma_f32_16x16x128_f8f6f4; or as bfloat16, which holds both formats'
// values, for four v_mfma_f32_16x16x32_bf16.  The former aligns the products of
// neighbouring k to the largest before it adds them and keeps about 13 bits below
// it (measured: of 2^16 + 2^(16 - d) at adjacent k the second is lost from d = 14
// on; at k eight apart it is kept to float32's own 23): typically 2e-5 to 4e-5 of
// a block's sum in norm, at most eight products' 2^-13 each, 2^-10 of the sum of magnitudes.
// Beside the rounding of a bfloat16 result (1.6e-3) that is nothing, beside a float16 one's
// (2.1e-4) one per cent more error, and far above a float32 one's; where blocks cancel
// it is relative to them and not to the result.  The latter rounds as float32 sums do (1e-8
// there), at half the rate and the conversions' cost.  So: the first for
// 16-bit outputs of large products, the second for float32 ones, and where the
// product waits for memory anyway.  A caller who needs the second asks for float32.
// `power`: 2^x of the lane's row, if the scales are split.
template <bool kExact, int kFmt>
struct Frag {
  v8i c;
  int x;                             // the exponent as the instruction has it: 2^(x - 127)
  __device__ __forceinline__ explicit Frag(const v8i& codes) : c(codes) {}
  __device__ __forceinline__ Frag(const v8i& codes, float power)
      : c(codes), x(__builtin_bit_cast(int, power) >> 23) {}
  __device__ __forceinline__ Frag() {}
};
template <int kFmt>
struct Frag<true, kFmt> {
  v8b c[4];
  __device__ __forceinline__ Frag() {}
  __device__ __forceinline__ explicit Frag(const v8i& codes) : Frag(codes, 1.0f) {}
  __device__ __forceinline__ Frag(const v8i& codes, float power) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v2b w[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = (uint32_t)codes[2 * j + h];
        if constexpr (kFmt == FP64EMU_E4M3) {
          w[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, power, false);
          w[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, power, true);
        } else {
          w[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(x, power, false);
          w[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(x, power, true);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) c[j][i] = w[i >> 1][i & 1];
    }
  }
};

template <bool kSplit, bool kExact, int kFB, int kFA>
__device__ __forceinline__ v4f block_sum(const Frag<kExact, kFB>& b, const Frag<kExact, kFA>& a) {
  v4f p = {0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (kExact) {
#pragma unroll
    for (int j = 0; j < 4; ++j) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.c[j], a.c[j], p, 0, 0, 0);
  } else if constexpr (kSplit) {
    p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.c, a.c, p, kFB, kFA, 0, b.x, 0, a.x);
  } else {
    p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.c, a.c, p, kFB, kFA, 0, 0, 0, 0);
  }
  return p;
}

__device__ __forceinline__ v8i join(const v4i& a, const v4i& b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// 16 bytes of a row at k, those past K as zero codes (whatever the memory
// holds there, if it is memory at all).  Any alignment.  A row's last, partial 16
// are its last 16 bytes moved down.
__device__ __forceinline__ v4i load16_masked(const uint8_t* row, int64_t k, int64_t K) {
  if (k + 16 <= K) {
    v4i v;
    __builtin_memcpy(&v, row + k, 16);
    return v;
  }
  uint64_t w[2] = {0, 0};
  if (k < K && K >= 16) {
    __builtin_memcpy(w, row + K - 16, 16);
    const int drop = 8 * (int)(k + 16 - K);                  // bits, 8 .. 120
    if (drop < 64) {
      w[0] = w[0] >> drop | w[1] << (64 - drop);
      w[1] >>= drop;
    } else {
      w[0] = w[1] >> (drop - 64);
      w[1] = 0;
    }
  } else if (k < K) {
#pragma unroll 1
    for (int64_t j = K - 1; j >= k; --j) {
      w[1] = w[1] << 8 | w[0] >> 56;
      w[0] = w[0] << 8 | row[j];
    }
  }
  return v4i{(int)w[0], (int)(w[0] >> 32), (int)w[1], (int)(w[1] >> 32)};
}

// Four successive outputs (m, n .. n + 3).
__device__ __forceinline__ void store_out(const MmArgs& g, int64_t b, int64_t m, int64_t n, v4f v) {
  const int valid = (int)(g.N - n < 4 ? g.N - n : 4);
  const int64_t i = b * g.stride_o + m * g.ldo + n;
  if (g.vec_o && valid == 4) {
    if (g.dtype == FP64EMU_F32) {
      v4f* o = reinterpret_cast<v4f*>(static_cast<float*>(g.out) + i);
      if (g.accumulate) v += *o;
      *o = v;
    } else {
      typedef unsigned short v4s __attribute__((ext_vector_type(4)));
      v4s* o = reinterpret_cast<v4s*>(static_cast<unsigned short*>(g.out) + i);
      const bool bf = g.dtype == FP64EMU_BF16;
      if (g.accumulate) {
        const v4s w = *o;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] += bf ? bf16_value(w[j]) : (float)__builtin_bit_cast(_Float16, (unsigned short)w[j]);
      }
      v4s r;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        r[j] = bf ? bf16_round(v[j]) : __builtin_bit_cast(unsigned short, (_Float16)v[j]);
      *o = r;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j >= valid) break;
    float x = v[j];
    if (g.dtype == FP64EMU_F32) {
      if (g.accumulate) x += load1<FP64EMU_F32>(g.out, i + j);
      store1<FP64EMU_F32>(g.out, i + j, x);
    } else if (g.dtype == FP64EMU_BF16) {
      if (g.accumulate) x += load1<FP64EMU_BF16>(g.out, i + j);
      store1<FP64EMU_BF16>(g.out, i + j, x);
    } else {
      if (g.accumulate) x += load1<FP64EMU_F16>(g.out, i + j);
      store1<FP64EMU_F16>(g.out, i + j, x);
    }
  }
}

// The partial sums of one split instead of an output.
__device__ __forceinline__ void store_part(const MmArgs& g, int split, int64_t b, int64_t m, int64_t n, v4f v) {
  float* o = g.part + (((int64_t)split * g.batch + b) * g.M + m) * g.N + n;
  const int64_t left = g.N - n;
  if (left >= 4 && (g.N & 3) == 0) {
    *reinterpret_cast<v4f*>(o) = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) o[j] = v[j];
}

// Sum of the splits' partial sums, in their order.
__global__ void __launch_bounds__(kThreads) sum_parts_kernel(MmArgs g) {
  const int64_t row_quads = (g.N + 3) / 4, total = (int64_t)g.batch * g.M * row_quads;
  const int64_t step = (int64_t)gridDim.x * kThreads;
  const int splits = g.splits;
  g.splits = 1;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += step) {
    const int64_t bm = i / row_quads, n = (i - bm * row_quads) * 4;
    const float* p = g.part + bm * g.N + n;
    const int64_t one = (int64_t)g.batch * g.M * g.N, left = g.N - n;
    v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (left >= 4 && (g.N & 3) == 0) {
      for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const v4f*>(p + s * one);
    } else {
      for (int s = 0; s < splits; ++s)
        for (int j = 0; j < 4; ++j)
          if (j < left) v[j] += p[s * one + j];
    }
    store_out(g, bm / g.M, bm % g.M, n, v);
  }
}

// s_waitcnt: at most `vm` vector-memory operations outstanding, LDS done.
template <int vm>
__device__ __forceinline__ void wait_vm_lgkm0() {
  static_assert(vm >= 0 && vm < 64, "vmcnt field");
  __builtin_amdgcn_s_waitcnt((vm & 15) | (7 << 4) | (0 << 8) | ((vm >> 4) << 14));
}
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xc07f); }   // LDS done
// Barrier without the fences of __syncthreads(), which would drain the copies in flight.
__device__ __forceinline__ void barrier_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

typedef __attribute__((address_space(3))) uint8_t lds_u8;

// A buffer resource over `bytes` bytes at a work-group-uniform p.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_src(const void* p, uint32_t bytes) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0,
                                           __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}

// Tiles of kBM x kBN outputs, kWM x kWN waves of (kBM / kWM) x (kBN / kWN).
//
// 8192^3 to bfloat16 on 256 x 256 tiles: 467-471 us, 2.3 PFLOP/s, where the library's f8
// product with one scale for each matrix takes 354-357.  What it is made of, by leaving
// parts out on the same inputs: matrix instructions and scaling FMAs on registers 348 us
// (294 on zeros, so the power limit; the matrix units' own cycles come to 253 at 2.07 GHz), with
// the LDS reads 354, with the copies 460.  Without its stores it took 429 where it took 466
// with them, before whole non-temporal lines gave 12 to 14 of those back.  The wait for
// the copies costs 6, the barrier nothing measurable.
// The FMAs hide behind the matrix instructions up to four vector instructions each;
// scales by rows on both sides take eight (8192^3 546 us).
//
// Exact products on 128 x 256 tiles: 4096 x 4096 x 8192, scales by rows on both sides, 264 us
// (1.0 PFLOP/s), by tiles 245; the library's bfloat16 product reaches 1.6.  Bound by vector
// instructions: 128 conversions, 64 FMAs and 64 products of scales a wave and block for 64 matrix
// instructions, which hide one each.  Converting once per work group instead, through
// LDS, left too few registers to hide its phases: 325 us, where registers took 248.
//
// A stage holds one block of K: kBN rows of B and kBM rows of A of 128 bytes
// each, then their scales.  A lane's fragment is 16-byte chunks l / 16 and
// l / 16 + 4 of row l % 16.  LDS serves a 16-byte read of 64 lanes sixteen at a time
// over its 256 bytes of banks, lanes 0-3, 12-15 and 20-27 first, 4-11, 16-19 and 28-31
// next; chunk c of row r lies at place c ^ (r / 2 % 8) of the row's eight, which gives
// each such sixteen sixteen places (c ^ r % 8 with chunks 2 (l / 16) and + 1 met twice in
// each and took 5.0e7 of 1.06e8 LDS cycles; now 1.6e6 of 6.2e7, the epilogue's).  The copies write LDS in lane order: the lane
// that owns a place fetches the chunk that belongs there.
template <int kBM_, int kBN_, int kWM_, int kWN_>
struct MmShape {
  static constexpr int kBM = kBM_, kBN = kBN_, kWM = kWM_, kWN = kWN_;
  static constexpr int kWaves = kWM * kWN, kT = 64 * kWaves;
  static constexpr int kTM = kBM / kWM / 16, kTN = kBN / kWN / 16;   // 16 x 16 tiles per wave
  static constexpr int kCopB = kBN / 8 / kWaves, kCopA = kBM / 8 / kWaves;   // copies per wave
  static constexpr int kOffA = kBN * kBlk, kOffS = (kBN + kBM) * kBlk;
  static constexpr int kStage = kOffS + 4 * (kBN + kBM);
  static_assert(kTM == 4, "four tiles a row");
  static_assert(kT >= kBM + kBN && kBN % 64 == 0 && kBM % 64 == 0, "one scale per thread and stage");
  static_assert(2 * kStage <= 160 * 1024, "two stages in LDS");
};

// Four successive elements at p, of which `valid` exist: to and from T[4].
template <class T>
__device__ __forceinline__ void put4(T* p, int valid, const T (&w)[4]) {
  if (valid >= 4) {
    __builtin_memcpy(p, w, sizeof(w));
    return;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < valid) p[j] = w[j];
}
template <class T>
__device__ __forceinline__ void get4(const T* p, int valid, T (&w)[4]) {
  if (valid >= 4) {
    __builtin_memcpy(w, p, sizeof(w));
    return;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j) w[j] = j < valid ? p[j] : T{};
}

// An item's partial sums (kForm 0), or what it adds to bfloat16 (1) or float16 (2)
// outputs, from the accumulators, a row of tiles at a time.
template <class S, int kForm>
__device__ __forceinline__ void store_rows(const v4f (&acc)[S::kTN][S::kTM], void* out, int64_t ld, int rows,
                                           int cols) {
  using T = std::conditional_t<kForm == 0, float, unsigned short>;
  T* p = static_cast<T*>(out);
#pragma unroll
  for (int y = 0; y < S::kTM; ++y, p += 16 * ld) {
    if (y * 16 < rows) {
      T old[S::kTN][4];
      if constexpr (kForm != 0) {
#pragma unroll
        for (int x = 0; x < S::kTN; ++x) get4(p + x * 16, cols - x * 16, old[x]);
      }
#pragma unroll
      for (int x = 0; x < S::kTN; ++x) {
        T w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = acc[x][y][i];
          if constexpr (kForm == 0)
            w[i] = v;
          else if constexpr (kForm == 1)
            w[i] = bf16_round(v + bf16_value(old[x][i]));
          else
            w[i] = __builtin_bit_cast(unsigned short, (_Float16)(v + (float)__builtin_bit_cast(_Float16, old[x][i])));
        }
        put4(p + x * 16, cols - x * 16, w);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// From (m, n) on, a lane's first output.
template <class S, bool kExact>
__device__ __forceinline__ void store_tile(const MmArgs& g, int64_t m, int64_t n, int b, int split,
                                           const v4f (&acc)[S::kTN][S::kTM]) {
  const int rows = (int)(g.M - m), cols = (int)(g.N - n);
  const int64_t at = b * g.stride_o + m * g.ldo + n;
  if (kExact || g.splits > 1)          // (whole float32 sums take the way through LDS)
    store_rows<S, 0>(acc, g.part + (((int64_t)split * g.batch + b) * g.M + m) * g.N + n, g.N, rows, cols);
  else if (g.dtype == FP64EMU_BF16)
    store_rows<S, 1>(acc, static_cast<unsigned short*>(g.out) + at, g.ldo, rows, cols);
  else
    store_rows<S, 2>(acc, static_cast<unsigned short*>(g.out) + at, g.ldo, rows, cols);
}

// 16 bytes anywhere, not kept in the caches: what nothing here reads again.
__device__ __forceinline__ void store16_past(void* p, const void* w) {
  typedef v4u v4u_any __attribute__((aligned(2)));
  v4u v;
  __builtin_memcpy(&v, w, 16);
  __builtin_nontemporal_store(v, static_cast<v4u_any*>(p));
}

template <class S, bool kExact, int kFA, int kFB, bool kRowB>
__device__ __forceinline__ void mm_tile(const MmArgs& g) {
  // The two stages, or the waves' rows of out.
  constexpr int kOut = S::kWaves * S::kTM * 16 * (S::kTN * 16 * (kExact ? 4 : 2) + 16);
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kOut > 2 * S::kStage ? kOut : 2 * S::kStage];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave % S::kWM, wn = wave / S::kWM;

  // Work item: member and split, then the tile.  Work group i runs on XCD i % 8:
  // each XCD takes a contiguous run of tiles, in panels of 8 tile rows, so that
  // its 32 CUs share operand panels in its L2.
  const int tiles = g.tiles_m * g.tiles_n;
  int item;
  {
    const int total = (int)gridDim.x, x = (int)blockIdx.x & 7, i = (int)blockIdx.x >> 3;
    const int q = total >> 3, r = total & 7;
    item = x * q + (x < r ? x : r) + i;
  }
  const int outer = item / tiles;
  item -= outer * tiles;
  const int b = outer % g.batch, split = outer / g.batch;
  constexpr int kPanel = 8;
  const int per = kPanel * g.tiles_n, panel = item / per, left = g.tiles_m - panel * kPanel;
  const int high = left < kPanel ? left : kPanel, in = item - panel * per;
  const int tm = panel * kPanel + in % high, tn = in / high;
  const int64_t m0 = (int64_t)tm * S::kBM, n0 = (int64_t)tn * S::kBN;
  const int rowsA = (int)(g.M - m0 < S::kBM ? g.M - m0 : S::kBM);
  const int rowsB = (int)(g.N - n0 < S::kBN ? g.N - n0 : S::kBN);
  const int kb0 = split * g.kb_per_split;
  const int kb1 = kb0 + g.kb_per_split < g.nkb ? kb0 + g.kb_per_split : g.nkb;
  const int nk = kb1 - kb0;

  const uint8_t* A = g.A + b * g.strideA + m0 * g.lda;
  const uint8_t* B = g.B + b * g.strideB + n0 * g.ldb;
  // Up to the end of the last row's last 16 bytes (rows are 16-byte aligned here).
  const int64_t K16 = (g.K + 15) & ~(int64_t)15;
  const __amdgpu_buffer_rsrc_t srcA = buffer_src(A, (uint32_t)((rowsA - 1) * g.lda + K16));
  const __amdgpu_buffer_rsrc_t srcB = buffer_src(B, (uint32_t)((rowsB - 1) * g.ldb + K16));
  const int chunk = ((lane & 7) ^ ((wave & 1) * 4 + (lane >> 4))) * 16;   // of rows 8 (2 i + wave % 2) + lane / 8
  uint32_t offA[S::kCopA], offB[S::kCopB];       // rows past the end repeat the last one
#pragma unroll
  for (int i = 0; i < S::kCopB; ++i) {
    const int r = (i * S::kWaves + wave) * 8 + (lane >> 3);
    offB[i] = (uint32_t)((r < rowsB ? r : rowsB - 1) * g.ldb + chunk);
  }
#pragma unroll
  for (int i = 0; i < S::kCopA; ++i) {
    const int r = (i * S::kWaves + wave) * 8 + (lane >> 3);
    offA[i] = (uint32_t)((r < rowsA ? r : rowsA - 1) * g.lda + chunk);
  }
  // Thread t < kBN: the scale of B's row t; else of A's row t - kBN (whole waves of either).
  const float* sp;
  const bool forB = wave * 64 < S::kBN;
  const int64_t sblk = forB ? g.sB_blk : g.sA_blk;
  {
    const int t = threadIdx.x;
    if (forB) {
      const int64_t r = n0 + (t < rowsB ? t : rowsB - 1);
      sp = g.sB + b * g.sB_str + (kRowB ? r : r / kBlk) * g.sB_row;
    } else {
      const int64_t r = t - S::kBN < rowsA ? t - S::kBN : rowsA - 1;
      sp = g.sA + b * g.sA_str + (m0 + r) * g.sA_row;
    }
    sp += kb0 * sblk;
  }

  // Block kb into stage st.  The block's offset is part of each lane's where it
  // ends past K, so that the resource's bound covers it.
  constexpr int kAll = S::kCopA + S::kCopB;
  auto copy = [&](int kb, int st, int c) {
    lds_u8* stage = (lds_u8*)lds + st * S::kStage;
    if (c < S::kCopB)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(srcB, stage + (c * S::kWaves + wave) * 1024, 16,
                                               (int)(offB[c] + (uint32_t)kb * kBlk), 0, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(srcA, stage + S::kOffA + ((c - S::kCopB) * S::kWaves + wave) * 1024, 16,
                                               (int)(offA[c - S::kCopB] + (uint32_t)kb * kBlk), 0, 0, 0);
  };
  auto copy_scales = [&](int st) {
    if (wave * 64 >= S::kBN + S::kBM) return;
    __builtin_amdgcn_global_load_lds(sp, (lds_u8*)lds + st * S::kStage + S::kOffS + wave * 256, 4, 0, 0);
    sp += sblk;
  };
  constexpr int kParts = 4, kPer = (kAll + kParts - 1) / kParts;
  auto issue = [&](int kb, int st, int part) {
#pragma unroll
    for (int c = 0; c < kAll; ++c)
      if (c / kPer == part) copy(kb, st, c);
    if (part == 0) copy_scales(st);
  };

  // Codes past K in a stage become zeros (the memory there is padding or
  // another row): thread t has row t of the stage, B's rows first.
  const int tail = (int)(g.K & (kBlk - 1));
  auto clear_tail = [&](int st) {
    uint8_t* row = lds + st * S::kStage + threadIdx.x * kBlk;
    for (int c = (int)threadIdx.x < S::kBN + S::kBM ? tail >> 4 : 8; c < 8; ++c) {
      v4i* w = reinterpret_cast<v4i*>(row + ((c ^ ((threadIdx.x >> 1) & 7)) << 4));
      v4i v = *w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int left = tail - 16 * c - 4 * j;             // bytes of this word before K
        v[j] = left >= 4 ? v[j] : left <= 0 ? 0 : v[j] & (int)((1u << (8 * left)) - 1);
      }
      *w = v;
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);                       // lgkmcnt(0)
    barrier_lds();
  };

  v4f acc[S::kTN][S::kTM];
#pragma unroll
  for (int x = 0; x < S::kTN; ++x)
#pragma unroll
    for (int y = 0; y < S::kTM; ++y) acc[x][y] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  const int fr = lane & 15, fg = lane >> 4;
  const int slot = (fg ^ (fr >> 1)) * 16;                    // chunk fg; chunk fg + 4 is at slot ^ 64
  const int fragB = (wn * S::kTN * 16 + fr) * kBlk, fragA = S::kOffA + (wm * S::kTM * 16 + fr) * kBlk;
  auto frag = [&](const uint8_t* stage, int base) {
    return join(*reinterpret_cast<const v4i*>(stage + base + slot),
                *reinterpret_cast<const v4i*>(stage + base + (slot ^ 64)));
  };
  Frag<kExact, kFA> fa[S::kTM];
  v8i fb;
  float sa[S::kTM];
  auto scale = [&](const uint8_t* stage, int row) { return reinterpret_cast<const float*>(stage + S::kOffS)[row]; };
  const int rowA = S::kBN + wm * S::kTM * 16 + fr, rowB = wn * S::kTN * 16;
  auto scale_a = [&](const uint8_t* stage, int y) {
    return scale(stage, rowA + y * 16) * (kRowB ? kFrame : kFrame * scale(stage, rowB));
  };
  auto scale_b = [&](const uint8_t* stage, int x) {
    return *reinterpret_cast<const v4f*>(stage + S::kOffS + 4 * (rowB + x * 16 + 4 * fg));
  };
  // Whether the wave's scales of the block fit the frame (not where one is NaN); far: its largest of B.
  auto far_b = [&](const uint8_t* stage) {
    float f = 0.0f;
    for (int r = 0; kRowB && r < S::kTN * 16; r += 64) f += fabsf(scale(stage, rowB + r + lane));
    return f;
  };
  float far = 0.0f;
  auto fits = [&] {
    const float a = fabsf(sa[0]) + fabsf(sa[1]) + fabsf(sa[2]) + fabsf(sa[3]);
    const bool in = kRowB ? a < kFrameTopA && far < kFrameTopB : a < kFrameTop;
    return __builtin_amdgcn_ballot_w64(!in) == 0;
  };
  // acc[x][y] += the scaled block sum p.
  auto add = [&](int x, int y, const v4f& p, const v4f& sb) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc[x][y][i] = fmaf(p[i], kRowB ? sa[y] * sb[i] : sa[y], acc[x][y][i]);
    // Here, and not wherever the compiler finds room: it moved all of a block's
    // sums behind its last tile, with every p kept until then.
    asm volatile("" : "+v"(acc[x][y]));
  };

  // One barrier per block, before its last row of tiles: when a wave has B's last
  // fragment of stage i & 1 in registers and its copies of block i + 1 (issued a
  // whole block earlier) have landed, it waits for the others; the stage is then
  // free for block i + 2 and the next one is whole, and the last row's matrix
  // instructions cover the reads of the next block's fragments, each of A's as
  // its register comes free.  Row x of tiles issues its matrix instructions
  // while row x - 1's sums are scaled and B's next fragment is on its way; the
  // scheduling barriers keep the compiler from reading the fragments ahead (which
  // spilled 75 registers).
  for (int part = 0; part < kParts; ++part) issue(kb0, 0, part);
  wait_vm_lgkm0<0>();
  if (nk > 1) issue(kb0 + 1, 1, 0);
  barrier_lds();
  if (tail && nk == 1 && kb1 == g.nkb) clear_tail(0);
  fb = frag(lds, fragB);
#pragma unroll
  for (int y = 0; y < S::kTM; ++y) {
    fa[y] = Frag<kExact, kFA>(frag(lds, fragA + y * 16 * kBlk));
    sa[y] = scale_a(lds, y);
  }
  far = far_b(lds);
  // Block i in the frame, or with split scales, whose A comes from the stage again.
  auto block = [&](auto split, int i) {
    constexpr bool kSplit = decltype(split)::value;
    const uint8_t* stage = lds + (i & 1) * S::kStage;
    const uint8_t* after = lds + ((i + 1) & 1) * S::kStage;
    v4f p[2][S::kTM], sb[2];
    float sa_next[S::kTM], power_b = 1.0f;
    constexpr int kLast = S::kTN - 1;
    if constexpr (kSplit) {
      const Split one = split_scale(scale(stage, rowB));       // of a tile of B
      power_b = one.power;
#pragma unroll
      for (int y = 0; y < S::kTM; ++y) {
        const Split a = split_scale(scale(stage, rowA + y * 16));
        fa[y] = Frag<kExact, kFA>(frag(stage, fragA + y * 16 * kBlk), a.power);
        sa[y] = kRowB ? a.rest : a.rest * one.rest;
      }
    }
    auto refill = [&](int y) {
      if constexpr (kSplit) return;
      fa[y] = Frag<kExact, kFA>(frag(after, fragA + y * 16 * kBlk));
      sa_next[y] = scale_a(after, y);
    };
#pragma unroll
    for (int x = 0; x < S::kTN; ++x) {
      v8i next;
      if constexpr (kRowB) sb[x & 1] = scale_b(stage, x);
      if constexpr (kRowB && kSplit) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sb[x & 1][e] = split_scale(sb[x & 1][e]).rest;
        power_b = split_scale(scale(stage, rowB + x * 16 + fr)).power;
      }
      if (x == kLast) {
        wait_vm_lgkm0<0>();
        barrier_lds();
        if (i + 2 < nk) issue(kb0 + i + 2, i & 1, 0);
        if (tail && i + 2 == nk && kb1 == g.nkb) clear_tail((i + 1) & 1);
        next = frag(after, fragB);                           // (past the last block: unused)
        if constexpr (!kSplit) far = far_b(after);
      } else {
        next = frag(stage, fragB + (x + 1) * 16 * kBlk);
      }
      if (x + 1 < kParts && i + 1 < nk) issue(kb0 + i + 1, (i + 1) & 1, x + 1);
      Frag<kExact, kFB> fbx;
      if constexpr (kSplit) fbx = Frag<kExact, kFB>(fb, power_b);
      else fbx = Frag<kExact, kFB>(fb);
      // Step s of four: a quarter of K of every tile (bfloat16; a tile's own four follow
      // each other four instructions apart, not back to back), or tile s.
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if constexpr (kExact) {
#pragma unroll
          for (int y = 0; y < S::kTM; ++y)
            p[x & 1][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                fbx.c[s], fa[y].c[s], s == 0 ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : p[x & 1][y], 0, 0, 0);
        } else {
          p[x & 1][s] = block_sum<kSplit, kExact, kFB, kFA>(fbx, fa[s]);
        }
        if (x == kLast && !kExact) refill(s);
        if (x > 0) add(x - 1, s, p[(x - 1) & 1][s], sb[(x - 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (x == kLast && kExact) {
#pragma unroll
        for (int y = 0; y < S::kTM; ++y) refill(y);
      }
      fb = next;
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int y = 0; y < S::kTM; ++y) {
      add(kLast, y, p[kLast & 1][y], sb[kLast & 1]);
      if constexpr (!kSplit) sa[y] = sa_next[y];
    }
  };
  // A wave that meets larger scales takes its sums out of the frame and stays with split ones:
  // with them for every block, 8192^3 took 9% longer to bfloat16 and 6% to float32, mostly for the
  // instructions' scale operands' own issue slots; the frame's check and its end take 1 and 2%.
  int done = 0;
  for (; done < nk && fits(); ++done) block(std::false_type{}, done);
#pragma unroll
  for (int x = 0; x < S::kTN; ++x)
#pragma unroll
    for (int y = 0; y < S::kTM; ++y) acc[x][y] *= 1.0f / kFrame;
  for (; done < nk; ++done) block(std::true_type{}, done);

  if (g.splits > 1 || (!kExact && g.accumulate)) {
    store_tile<S, kExact>(g, m0 + wm * S::kTM * 16 + fr, n0 + wn * S::kTN * 16 + 4 * fg, b, split, acc);
    return;
  }
  // Through LDS, so that a store writes whole lines of out past the caches: 8192 x
  // 8192 x 1024 took 104 us with the four values of a lane stored as they lie (8 or 16
  // bytes of a row), 108 us with whole lines, 89 us with whole lines and non-temporal
  // stores.  Each wave has its own room: its rows of out, 16 bytes apart beyond
  // their length so that neither side meets a bank twice.
  using T = std::conditional_t<kExact, float, unsigned short>;
  constexpr int kRow = S::kTN * 16 * (int)sizeof(T) + 16, kEach = 16 / (int)sizeof(T);
  constexpr int kLanes = S::kTN * 16 / kEach;                  // lanes of one row
  barrier_lds();                                             // every wave is done with the stages
  uint8_t* room = lds + wave * (S::kTM * 16 * kRow);
#pragma unroll
  for (int y = 0; y < S::kTM; ++y)
#pragma unroll
    for (int x = 0; x < S::kTN; ++x) {
      T w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kExact) w[i] = acc[x][y][i];
        else w[i] = g.dtype == FP64EMU_BF16 ? bf16_round(acc[x][y][i])
                                            : __builtin_bit_cast(unsigned short, (_Float16)acc[x][y][i]);
      }
      __builtin_memcpy(__builtin_assume_aligned(room + (y * 16 + fr) * kRow + (x * 16 + 4 * fg) * sizeof(T),
                                                4 * sizeof(T)), w, 4 * sizeof(T));
    }
  // Other lanes of the wave read these rows: not before they are written, whatever the
  // compiler can tell of the addresses (the LDS itself keeps a wave's order).
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const int64_t n = n0 + wn * S::kTN * 16 + (lane % kLanes) * kEach;
  const int valid = (int)(g.N - n < kEach ? g.N - n : kEach);
  int64_t m = m0 + wm * S::kTM * 16 + lane / kLanes;
  T* to = static_cast<T*>(g.out) + b * g.stride_o + m * g.ldo + n;
  const uint8_t* from = room + (lane / kLanes) * kRow + (lane % kLanes) * 16;
  constexpr int kRows = 64 / kLanes;                         // rows of one store
  // What out holds, read whole before the first store: one by one, each store's
  // rows would wait for memory (16 times a tile).
  constexpr int kSteps = kExact ? S::kTM * 16 / kRows : 1;
  T old[kSteps][kEach];
  if constexpr (kExact) {
    if (g.accumulate) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const T* q = to + (int64_t)i * kRows * g.ldo;
        if (m + i * kRows >= g.M) break;
        if (valid == kEach) {
          __builtin_memcpy(old[i], q, 16);
        } else {
#pragma unroll
          for (int j = 0; j < kEach - 1; ++j) old[i][j] = j < valid ? q[j] : T{};
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < S::kTM * 16 / kRows; ++i, m += kRows, to += kRows * g.ldo) {
    T w[kEach];
    __builtin_memcpy(w, __builtin_assume_aligned(from + i * kRows * kRow, 16), 16);
    if (m >= g.M) continue;
    if constexpr (kExact) {
      if (g.accumulate) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) w[j] += old[i][j];
      }
    }
    if (valid == kEach) {
      store16_past(to, w);
    } else {
#pragma unroll
      for (int j = 0; j < kEach - 1; ++j)
        if (j < valid) to[j] = w[j];
    }
  }
}

template <class S, bool kExact, int kFA, int kFB, bool kRowB>
__global__ void __launch_bounds__(S::kT, 2) mm_tile_kernel(MmArgs g) {
  mm_tile<S, kExact, kFA, kFB, kRowB>(g);
}

// Rows of any alignment into rows of a multiple of 16 bytes, 16 bytes a thread.
__global__ void __launch_bounds__(kThreads) pack_rows_kernel(const uint8_t* q, int64_t ld, int64_t stride,
                                                             uint8_t* to, int64_t rows, int64_t total,
                                                             int64_t K) {
  const int64_t chunks = (K + 15) / 16, step = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total * chunks; i += step) {
    const int64_t r = i / chunks, c = i - r * chunks, b = r / rows;
    const v4i v = load16_masked(q + b * stride + (r - b * rows) * ld, c * 16, K);
    *reinterpret_cast<v4i*>(to + i * 16) = v;
  }
}

// Few rows of A: the product reads B once and little else.  A work group has
// kTN x 16 rows of B and all waves on them, wave w at blocks w, w + kFewWaves,
// ... of K; fragments come straight from memory (lane l's 32 bytes are the
// instruction's operand as they lie in the row), and the waves' sums meet in LDS.
// All of an iteration's operands and scales are loaded before the first is used (one
// token through 8192 x 8192: 14.9 us without that fence, 13.1 with it).  Bound by B's
// bytes there, at 5.1 TB/s; by the latency of its few iterations where the product is
// small (333 x 501 x 777: 6.4 us, 11.2 on 128 x 128 tiles).
constexpr int kFewWaves = 8;

template <int kTM, int kTN, int kU, int kFA, int kFB, bool kRowB>
__global__ void __launch_bounds__(64 * kFewWaves) mm_few_kernel(MmArgs g) {
  __shared__ v4f red[kFewWaves][kTN * kTM][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const int tiles = g.tiles_m * g.tiles_n;
  const int outer = blockIdx.x / tiles, item = blockIdx.x - outer * tiles;
  const int b = outer % g.batch, split = outer / g.batch;
  const int64_t m0 = (int64_t)(item / g.tiles_n) * (16 * kTM), n0 = (int64_t)(item % g.tiles_n) * (16 * kTN);
  const int kb0 = split * g.kb_per_split;
  const int kb1 = kb0 + g.kb_per_split < g.nkb ? kb0 + g.kb_per_split : g.nkb;

  const uint8_t *pa[kTM], *pb[kTN];
  const float *sa[kTM], *sb[kTN][kRowB ? 5 : 1];             // rows 4 fg + i of the outputs, then the fragment's row fr
#pragma unroll
  for (int y = 0; y < kTM; ++y) {
    const int64_t m = m0 + y * 16 + fr < g.M ? m0 + y * 16 + fr : g.M - 1;
    pa[y] = g.A + b * g.strideA + m * g.lda;
    sa[y] = g.sA + b * g.sA_str + m * g.sA_row;
  }
#pragma unroll
  for (int x = 0; x < kTN; ++x) {
    const int64_t n = n0 + x * 16 + fr < g.N ? n0 + x * 16 + fr : g.N - 1;
    pb[x] = g.B + b * g.strideB + n * g.ldb;
#pragma unroll
    for (int i = 0; i < (kRowB ? 5 : 1); ++i) {
      const int64_t r = n0 + x * 16 + (!kRowB ? 0 : i < 4 ? 4 * fg + i : fr);
      sb[x][i] = g.sB + b * g.sB_str + (kRowB ? (r < g.N ? r : g.N - 1) : r / kBlk) * g.sB_row;
    }
  }

  v4f acc[kTN][kTM];
#pragma unroll
  for (int x = 0; x < kTN; ++x)
#pragma unroll
    for (int y = 0; y < kTM; ++y) acc[x][y] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  auto frag = [&](const uint8_t* row, int kb) {
    const int64_t k = (int64_t)kb * kBlk + 32 * fg;
    return join(load16_masked(row, k, g.K), load16_masked(row, k + 16, g.K));
  };
  auto whole = [&](const uint8_t* row, int kb) {
    v8i v;
    __builtin_memcpy(&v, row + (int64_t)kb * kBlk + 32 * fg, 32);
    return v;
  };
  // A block's operands as they are loaded, all of them before the first is used.
  struct Block {
    v8i b[kTN], a[kTM];
    float sa[kTM], sb[kTN][kRowB ? 5 : 1];
  };
  auto scales = [&](Block& o, int kb) {
#pragma unroll
    for (int y = 0; y < kTM; ++y) o.sa[y] = sa[y][kb * g.sA_blk];
#pragma unroll
    for (int x = 0; x < kTN; ++x)
#pragma unroll
      for (int i = 0; i < (kRowB ? 5 : 1); ++i) o.sb[x][i] = sb[x][i][kb * g.sB_blk];
  };
  auto step = [&](const Block& o) {
    Frag<true, kFA> fa[kTM];
    float ra[kTM];
#pragma unroll
    for (int y = 0; y < kTM; ++y) {
      const Split sc = split_scale(o.sa[y]);
      ra[y] = sc.rest;
      fa[y] = Frag<true, kFA>(o.a[y], sc.power);
    }
#pragma unroll
    for (int x = 0; x < kTN; ++x) {
      float rb[kRowB ? 4 : 1];
#pragma unroll
      for (int i = 0; i < (kRowB ? 4 : 1); ++i) rb[i] = split_scale(o.sb[x][i]).rest;
      const Frag<true, kFB> fb(o.b[x], split_scale(o.sb[x][kRowB ? 4 : 0]).power);
#pragma unroll
      for (int y = 0; y < kTM; ++y) {
        const v4f p = block_sum<true, true, kFB, kFA>(fb, fa[y]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[x][y][i] = fmaf(p[i], ra[y] * rb[kRowB ? i : 0], acc[x][y][i]);
      }
    }
  };

  const int full = (int)(g.K / kBlk) < kb1 ? (int)(g.K / kBlk) : kb1;    // blocks before it are whole
  int kb = kb0 + wave;
  for (; kb + (kU - 1) * kFewWaves < full; kb += kU * kFewWaves) {
    Block o[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
#pragma unroll
      for (int x = 0; x < kTN; ++x) o[u].b[x] = whole(pb[x], kb + u * kFewWaves);
#pragma unroll
      for (int y = 0; y < kTM; ++y) o[u].a[y] = whole(pa[y], kb + u * kFewWaves);
      scales(o[u], kb + u * kFewWaves);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < kU; ++u) step(o[u]);
  }
  for (; kb < kb1; kb += kFewWaves) {
    Block o;
#pragma unroll
    for (int x = 0; x < kTN; ++x) o.b[x] = frag(pb[x], kb);
#pragma unroll
    for (int y = 0; y < kTM; ++y) o.a[y] = frag(pa[y], kb);
    scales(o, kb);
    step(o);
  }

#pragma unroll
  for (int x = 0; x < kTN; ++x)
#pragma unroll
    for (int y = 0; y < kTM; ++y) red[wave][x * kTM + y][lane] = acc[x][y];
  __syncthreads();
  for (int t = wave; t < kTN * kTM; t += kFewWaves) {
    v4f v = red[0][t][lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) v += red[w][t][lane];
    const int64_t m = m0 + (t % kTM) * 16 + fr, n = n0 + (t / kTM) * 16 + 4 * fg;
    if (m >= g.M || n >= g.N) continue;
    if (g.splits > 1) store_part(g, split, b, m, n, v);
    else store_out(g, b, m, n, v);
  }
}

// ---------------------------------------------------------------------------
// Host side.

using Tile256 = MmShape<256, 256, 4, 2>;
using TileWide = MmShape<128, 256, 2, 4>;
using Tile128 = MmShape<128, 128, 2, 2>;

enum { kFew = 0, kSquare128 = 1, kSquare256 = 2, kWide = 3 };   // forms of a product

struct MmPlan {
  int form;
  int tile_m, tile_n;
  int64_t tiles_m, tiles_n;
  int splits, kb_per_split;
};

constexpr int kCUs = 256;

// A form's time in microseconds, launch included: `groups` work groups of `steps`
// blocks of K each, `reach` the operands' bytes as often as the eight XCDs' L2 fetch them.
// A work group's blocks take this long with one group to a CU, longer where the groups of
// all CUs share the caches' rate or two share a CU; few rows are also held by what they
// fetch (8192 x 64 x 8192 to float32: 37 us, the 128 x 128 tiles with eight splits 28).
// Fitted to 32 shapes of 1 to 8192 rows and columns and 512 to 100000 deep, to bfloat16
// and to float32, in the forms and splits that suit each: of those 64 runs 63 come within
// 5% of their fastest and the last, 1024^3 to bfloat16, within 10%.  Of 54 runs on 27
// other shapes, which served only to choose between equally good constants, 47 come
// within 5%, six within 14%, and 300 x 300 x 256 to bfloat16 takes 6.6 us where few rows take
// 3.9, as 16-bit products of at most 256 deep with more than 32 rows do.  Weights that do not
// stay in the caches were not among them, and it is off there: 1 x 28672 x 8192 takes 128 x 128
// tiles with two splits, 54 us, few rows 40; 1 x 128256 x 4096 108, 88.
// Both sides: 512 x 512 x 4096 in few rows with two splits 12.5 us, on 128 x 128 tiles with
// four 16.8; 2048^3 on 128 x 128 tiles 19.4, 256 x 256 27.7; 3000^3 42.5 the other way, 58.0.
double mm_time(int form, int tile_m, bool exact, double groups, double steps, double reach) {
  const double share = std::min(groups, (double)kCUs) / kCUs;
  switch (form) {
    case kFew: {               // eight waves, a block each
      const double per = tile_m == 16 ? 0.7 : tile_m == 32 ? 1.2 : 2.6;
      const double rounds = std::ceil(groups / (tile_m == 16 ? 2 * kCUs : kCUs));
      return 2.5 + std::max(rounds * (1.0 + per * std::ceil(steps / 8)), reach / 5e6);
    }
    case kSquare128: {         // two groups to a CU, the last round's perhaps one
      const double one = exact ? 1.37 : 0.98, two = exact ? 1.86 : 1.12;
      const double full = std::floor(groups / (2 * kCUs)), rest = groups - full * 2 * kCUs;
      return 2.5 + full * (1.5 + two * steps) + (rest > 0 ? 1.5 + (rest <= kCUs ? one : two) * steps : 0.0);
    }
    case kSquare256:
      return 1.0 + std::ceil(groups / kCUs) * (5.0 + (1.3 + 0.4 * share) * steps);
    default:
      return 2.0 + std::ceil(groups / kCUs) * (5.0 + 1.75 * steps);
  }
}

constexpr int64_t kMaxGroups = (1ll << 31) / kThreads;    // work items of one launch stay below 2^31
// Rows of operands that the tile kernels copy: a tile's 256 within 32-bit offsets, those of the last,
// partial block included.
constexpr int64_t kMaxTileRow = (1ll << 32) / 256 - kBlk;

// The form and the number of K splits that take least by mm_time, of those that one launch
// holds (splits = 0: none); a split adds a launch and its partial sums' way to memory and back.
MmPlan plan_mm(int64_t batch, int64_t M, int64_t N, int64_t K, int dtype) {
  const bool exact = dtype == FP64EMU_F32;
  const int64_t nkb = (K + kBlk - 1) / kBlk;
  MmPlan best{};
  double least = 1e300;
  auto consider = [&](int form, int tm, int tn) {
    const int64_t tiles_m = (M + tm - 1) / tm, tiles_n = (N + tn - 1) / tn;
    if (form != kFew && (K + 15) / 16 * 16 >= kMaxTileRow) return;
    const double reach = (double)batch * (double)K * ((double)M * (double)std::min<int64_t>(tiles_n, 8) +
                                                      (double)N * (double)std::min<int64_t>(tiles_m, 8));
    for (int64_t s = 1; s <= 32; s *= 2) {
      if (s > 1 && nkb < 2 * s) break;
      if (tiles_m > kMaxGroups / 2 / tiles_n / batch / s) break;
      const int64_t per = (nkb + s - 1) / s;
      double t = mm_time(form, tm, exact, (double)(batch * tiles_m * tiles_n) * (double)s, (double)per, reach);
      if (s > 1) t += 1.5 + 0.25 * (double)s + 7.0 * (double)s * (double)(batch * M) * (double)N / 4e6;
      if (t >= least) continue;
      least = t;
      best = MmPlan{form, tm, tn, tiles_m, tiles_n, per > 0 ? (int)((nkb + per - 1) / per) : 1, (int)per};
    }
  };
  if (M <= 16) consider(kFew, 16, 16);
  else if (M <= 32) consider(kFew, 32, 32);
  else consider(kFew, 64, 32);
  consider(kSquare128, 128, 128);
  if (exact) consider(kWide, 128, 256);
  else consider(kSquare256, 256, 256);
  return best;
}

int check_hip(hipError_t e, const char* what) {
  if (e == hipSuccess) return FP64EMU_OK;
  return fp64emu_fail(FP64EMU_EHIP, std::string(what) + ": " + hipGetErrorString(e));
}

int invalid(const char* msg) { return fp64emu_fail(FP64EMU_EINVAL, msg); }

bool multiple(const void* p, int64_t of) { return reinterpret_cast<uintptr_t>(p) % of == 0; }

int size_of(int dtype) { return dtype == FP64EMU_F32 ? 4 : 2; }

bool known_dtype(int d) { return d == FP64EMU_F32 || d == FP64EMU_BF16 || d == FP64EMU_F16; }
bool known_fmt(int f) { return f == FP64EMU_E4M3 || f == FP64EMU_E5M2; }

// A quantised output of `rows` x `depth` codes, or NULL.
int out8(const fp64emu_f8_t* f, int64_t depth, Out8* o) {
  *o = Out8{};
  if (!f) return FP64EMU_OK;
  if (!f->q || !f->s) return invalid("null 8-bit operand");
  if (!known_fmt(f->fmt)) return invalid("fmt must be FP64EMU_E4M3 or FP64EMU_E5M2");
  if (f->ld < depth) return invalid("8-bit rows are shorter than their depth");
  *o = Out8{f->q, f->s, f->ld, f->stride, f->s_row, f->s_block, f->s_stride};
  return FP64EMU_OK;
}

// Work groups for a matrix's blocks of rows, 16 each.
unsigned unit_groups(int64_t rows, int64_t blocks) {
  return (unsigned)std::min<int64_t>((rows * blocks + 15) / 16, 1 << 20);
}

template <int kT, int kFmt>
int launch_quant(QuantArgs g, int64_t batch, int64_t mblocks, bool tiles, hipStream_t s) {
  for (; g.batch0 < batch; g.batch0 += kMaxGridZ) {
    const unsigned z = (unsigned)std::min(batch - g.batch0, kMaxGridZ);
    const dim3 grid((unsigned)(mblocks * g.kblocks), 1, z);
    if (tiles) {
      quant_tile_kernel<kT, kFmt, kTiles><<<grid, kThreads, 0, s>>>(g);
    } else if (!g.cols.q) {
      quant_rows_kernel<kT, kFmt><<<dim3(unit_groups(g.M, g.kblocks), 1, z), kThreads, 0, s>>>(g);
    } else if (!g.rows.q) {
      quant_tile_kernel<kT, kFmt, kCols><<<grid, kThreads, 0, s>>>(g);
    } else {
      quant_tile_kernel<kT, kFmt, kRows | kCols><<<grid, kThreads, 0, s>>>(g);
    }
    if (int st = check_hip(hipGetLastError(), "quant_f8 launch")) return st;
  }
  return FP64EMU_OK;
}

template <class S, bool kExact, int kFA, int kFB>
void launch_tile(const MmArgs& g, unsigned groups, hipStream_t s) {
  if (g.b_tiles) mm_tile_kernel<S, kExact, kFA, kFB, false><<<groups, S::kT, 0, s>>>(g);
  else mm_tile_kernel<S, kExact, kFA, kFB, true><<<groups, S::kT, 0, s>>>(g);
}

template <int kTM, int kTN, int kU, int kFA, int kFB>
void launch_few(const MmArgs& g, unsigned groups, hipStream_t s) {
  if (g.b_tiles) mm_few_kernel<kTM, kTN, kU, kFA, kFB, false><<<groups, 64 * kFewWaves, 0, s>>>(g);
  else mm_few_kernel<kTM, kTN, kU, kFA, kFB, true><<<groups, 64 * kFewWaves, 0, s>>>(g);
}

template <int kFA, int kFB>
void launch_mm(const MmArgs& g, const MmPlan& p, unsigned groups, hipStream_t s) {
  const bool exact = g.dtype == FP64EMU_F32;
  if (p.form == kSquare256) launch_tile<Tile256, false, kFA, kFB>(g, groups, s);
  else if (p.form == kWide) launch_tile<TileWide, true, kFA, kFB>(g, groups, s);
  else if (p.form == kSquare128 && exact) launch_tile<Tile128, true, kFA, kFB>(g, groups, s);
  else if (p.form == kSquare128) launch_tile<Tile128, false, kFA, kFB>(g, groups, s);
  else if (p.tile_m == 16) launch_few<1, 1, 4, kFA, kFB>(g, groups, s);
  else if (p.tile_m == 32) launch_few<2, 2, 1, kFA, kFB>(g, groups, s);
  else launch_few<4, 2, 1, kFA, kFB>(g, groups, s);
}

// Whether the tile kernels can copy an operand's rows as they lie.
bool copyable(const fp64emu_f8_t& f) {
  return multiple(f.q, 16) && f.ld % 16 == 0 && f.stride % 16 == 0 && f.ld < kMaxTileRow;
}

// Partial sums, then the rows of A and of B that are laid out again.
struct MmRoom { size_t parts, A, B; };

MmRoom mm_room(const fp64emu_mm_f8_t* p, const MmPlan& plan) {
  MmRoom r{};
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  if (plan.splits > 1) r.parts = up((size_t)plan.splits * 4 * (size_t)(p->batch * p->M * p->N));
  const size_t ld = (size_t)((p->K + 15) / 16 * 16);
  if (plan.form != kFew && !copyable(p->A)) r.A = up((size_t)(p->batch * p->M) * ld);
  if (plan.form != kFew && !copyable(p->B)) r.B = up((size_t)(p->batch * p->N) * ld);
  return r;
}

void pack(const fp64emu_f8_t& f, int64_t batch, int64_t rows, int64_t K, uint8_t* to, hipStream_t s) {
  const int64_t work = batch * rows * ((K + 15) / 16);
  const unsigned groups = (unsigned)std::min<int64_t>((work + kThreads - 1) / kThreads, 65536);
  pack_rows_kernel<<<groups, kThreads, 0, s>>>(f.q, f.ld, f.stride, to, rows, batch * rows, K);
}

int check_mm(const fp64emu_mm_f8_t* p) {
  if (!p) return invalid("product must not be NULL");
  if (p->batch < 0 || p->M < 0 || p->N < 0 || p->K < 0) return invalid("shapes must be non-negative");
  if (p->M >= (1ll << 31) - 256 || p->N >= (1ll << 31) - 256 || p->batch >= (1ll << 31) ||
      p->K >= (1ll << 31) - kBlk)
    return invalid("shapes must be below 2^31");
  if (!known_dtype(p->dtype)) return invalid("dtype must be FP64EMU_F32, FP64EMU_BF16 or FP64EMU_F16");
  if (!known_fmt(p->A.fmt) || !known_fmt(p->B.fmt))
    return invalid("fmt must be FP64EMU_E4M3 or FP64EMU_E5M2");
  if (p->A.tiles) return invalid("A's scales are by rows");
  return FP64EMU_OK;
}

}  // namespace

extern "C" {

int fp64emu_quant_f8(const void* x, int dtype, int64_t batch, int64_t M, int64_t K, int64_t ldx,
                     int64_t stride_x, const fp64emu_f8_t* rows, const fp64emu_f8_t* cols,
                     fp64emu_stream_t stream) {
  if (batch < 0 || M < 0 || K < 0) return invalid("shapes must be non-negative");
  if (!known_dtype(dtype)) return invalid("dtype must be FP64EMU_F32, FP64EMU_BF16 or FP64EMU_F16");
  if (!rows && !cols) return invalid("no output asked for");
  if (rows && cols && (rows->tiles != cols->tiles || rows->fmt != cols->fmt))
    return invalid("rows and cols must agree in fmt and tiles");
  if (batch == 0 || M == 0 || K == 0) return FP64EMU_OK;
  if (!x) return invalid("null operand pointer");
  if (ldx < K) return invalid("rows of x are shorter than K");
  QuantArgs g{};
  if (int st = out8(rows, K, &g.rows)) return st;
  if (int st = out8(cols, M, &g.cols)) return st;
  const int64_t mblocks = (M + kBlk - 1) / kBlk;
  g.x = x;
  g.M = M;
  g.K = K;
  g.ldx = ldx;
  g.stride_x = stride_x;
  g.kblocks = (K + kBlk - 1) / kBlk;
  const bool tiles = (rows ? rows : cols)->tiles != 0;
  if (mblocks > kMaxGroups / g.kblocks) return invalid("operand too large for one launch");
  const int fmt = (rows ? rows : cols)->fmt;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define FP64EMU_QUANT(T)                                                             \
  case T:                                                                            \
    return fmt == FP64EMU_E4M3 ? launch_quant<T, FP64EMU_E4M3>(g, batch, mblocks, tiles, s)        \
                               : launch_quant<T, FP64EMU_E5M2>(g, batch, mblocks, tiles, s);
  switch (dtype) {
    FP64EMU_QUANT(FP64EMU_F32)
    FP64EMU_QUANT(FP64EMU_BF16)
    FP64EMU_QUANT(FP64EMU_F16)
  }
#undef FP64EMU_QUANT
  return invalid("dtype");
}

size_t fp64emu_mm_f8_workspace(const fp64emu_mm_f8_t* p) {
  if (check_mm(p) || p->batch * p->M == 0 || p->N == 0 || p->K == 0) return 0;
  const MmPlan plan = plan_mm(p->batch, p->M, p->N, p->K, p->dtype);
  if (plan.splits == 0) return 0;
  const MmRoom r = mm_room(p, plan);
  return r.parts + r.A + r.B;
}

int fp64emu_mm_f8_plan(const fp64emu_mm_f8_t* p, fp64emu_mm_f8_plan_t* out) {
  if (!out) return invalid("plan must not be NULL");
  *out = fp64emu_mm_f8_plan_t{};
  if (int st = check_mm(p)) return st;
  if (p->batch * p->M == 0 || p->N == 0 || p->K == 0) return FP64EMU_OK;
  const MmPlan plan = plan_mm(p->batch, p->M, p->N, p->K, p->dtype);
  if (plan.splits == 0) return invalid("product too large for one launch");
  const bool tiles = plan.form != kFew;
  *out = {plan.tile_m, plan.tile_n, plan.splits, !tiles || p->dtype == FP64EMU_F32, tiles && !copyable(p->A),
          tiles && !copyable(p->B)};
  return FP64EMU_OK;
}

int fp64emu_mm_f8(const fp64emu_mm_f8_t* p, void* workspace, size_t workspace_bytes,
                  fp64emu_stream_t stream) {
  if (int st = check_mm(p)) return st;
  if (p->batch == 0 || p->M == 0 || p->N == 0) return FP64EMU_OK;
  if (!p->out) return invalid("null operand pointer");
  if (p->ldo < p->N) return invalid("rows of out are shorter than N");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  MmArgs g{};
  g.out = p->out;
  g.ldo = p->ldo;
  g.stride_o = p->stride_o;
  g.dtype = p->dtype;
  g.accumulate = p->accumulate != 0;
  g.M = (int)p->M;
  g.N = (int)p->N;
  g.K = p->K;
  g.batch = (int)p->batch;
  const int quad = 4 * size_of(p->dtype);
  g.vec_o = multiple(p->out, quad) && p->ldo % 4 == 0 && p->stride_o % 4 == 0;
  if (p->K == 0) {
    // An empty sum: zeros, or out as it is.
    if (g.accumulate) return FP64EMU_OK;
    g.splits = 0;
  } else {
    if (!p->A.q || !p->A.s || !p->B.q || !p->B.s) return invalid("null 8-bit operand");
    if (p->A.ld < p->K || p->B.ld < p->K) return invalid("8-bit rows are shorter than their depth");
  }
  const int64_t quads = p->batch * p->M * ((p->N + 3) / 4);
  const unsigned sum_groups = (unsigned)std::min<int64_t>((quads + kThreads - 1) / kThreads, 65536);
  if (p->K == 0) {
    sum_parts_kernel<<<sum_groups, kThreads, 0, s>>>(g);
    return check_hip(hipGetLastError(), "mm_f8 launch");
  }
  const MmPlan plan = plan_mm(p->batch, p->M, p->N, p->K, p->dtype);
  if (plan.splits == 0) return invalid("product too large for one launch");
  const MmRoom room = mm_room(p, plan);
  const size_t need = room.parts + room.A + room.B;
  if (need && (!workspace || workspace_bytes < need))
    return fp64emu_fail(FP64EMU_EWORKSPACE, "workspace too small: see fp64emu_mm_f8_workspace");
  if (need && !multiple(workspace, 16)) return invalid("workspace must be 16-byte aligned");
  g.A = p->A.q;
  g.B = p->B.q;
  g.sA = p->A.s;
  g.sB = p->B.s;
  g.lda = p->A.ld;
  g.ldb = p->B.ld;
  g.strideA = p->A.stride;
  g.strideB = p->B.stride;
  g.sA_row = p->A.s_row;
  g.sA_blk = p->A.s_block;
  g.sA_str = p->A.s_stride;
  g.sB_row = p->B.s_row;
  g.sB_blk = p->B.s_block;
  g.sB_str = p->B.s_stride;
  g.part = static_cast<float*>(workspace);
  g.nkb = (int)((p->K + kBlk - 1) / kBlk);
  g.splits = plan.splits;
  g.kb_per_split = plan.kb_per_split;
  g.tiles_m = (int)plan.tiles_m;
  g.tiles_n = (int)plan.tiles_n;
  g.b_tiles = p->B.tiles != 0;
  const unsigned groups = (unsigned)(plan.tiles_m * plan.tiles_n * p->batch * plan.splits);
  const int64_t K16 = (p->K + 15) / 16 * 16;
  if (room.A) {
    uint8_t* to = static_cast<uint8_t*>(workspace) + room.parts;
    pack(p->A, p->batch, p->M, p->K, to, s);
    g.A = to;
    g.lda = K16;
    g.strideA = p->M * K16;
  }
  if (room.B) {
    uint8_t* to = static_cast<uint8_t*>(workspace) + room.parts + room.A;
    pack(p->B, p->batch, p->N, p->K, to, s);
    g.B = to;
    g.ldb = K16;
    g.strideB = p->N * K16;
  }
  if (p->A.fmt == FP64EMU_E4M3) {
    if (p->B.fmt == FP64EMU_E4M3) launch_mm<FP64EMU_E4M3, FP64EMU_E4M3>(g, plan, groups, s);
    else launch_mm<FP64EMU_E4M3, FP64EMU_E5M2>(g, plan, groups, s);
  } else {
    if (p->B.fmt == FP64EMU_E4M3) launch_mm<FP64EMU_E5M2, FP64EMU_E4M3>(g, plan, groups, s);
    else launch_mm<FP64EMU_E5M2, FP64EMU_E5M2>(g, plan, groups, s);
  }
  if (int st = check_hip(hipGetLastError(), "mm_f8 launch")) return st;
  if (plan.splits > 1) {
    sum_parts_kernel<<<sum_groups, kThreads, 0, s>>>(g);
    return check_hip(hipGetLastError(), "mm_f8 launch");
  }
  return FP64EMU_OK;
}

int fp64emu_swiglu_f8(const void* h, int dtype, int64_t M, int64_t F, int64_t ldh, void* y, int64_t ldy,
                      const fp64emu_f8_t* keep, const fp64emu_f8_t* rows, const fp64emu_f8_t* cols,
                      fp64emu_stream_t stream) {
  if (M < 0 || F < 0) return invalid("shapes must be non-negative");
  if (!known_dtype(dtype)) return invalid("dtype must be FP64EMU_F32, FP64EMU_BF16 or FP64EMU_F16");
  for (const fp64emu_f8_t* f : {keep, rows, cols})
    if (f && (f->fmt != FP64EMU_E4M3 || f->tiles)) return invalid("outputs are e4m3 with scales by rows");
  if (M == 0 || F == 0) return FP64EMU_OK;
  if (!y && !keep && !rows && !cols) return invalid("no output asked for");
  if (!h) return invalid("null operand pointer");
  if (ldh < 2 * F || (y && ldy < F)) return invalid("rows are shorter than their width");
  SwigluArgs a{};
  if (int st = out8(keep, 2 * F, &a.keep)) return st;
  if (int st = out8(rows, F, &a.rows)) return st;
  if (int st = out8(cols, M, &a.cols)) return st;
  a.h = h;
  a.M = M;
  a.F = F;
  a.ldh = ldh;
  a.fblocks = (F + kBlk - 1) / kBlk;
  a.y = y;
  a.ldy = ldy;
  const int64_t mblocks = (M + kBlk - 1) / kBlk;
  if (mblocks > kMaxGroups / a.fblocks) return invalid("operand too large for one launch");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const unsigned groups = (unsigned)(mblocks * a.fblocks);
  const unsigned few = unit_groups(M, a.fblocks);
#define FP64EMU_SWIGLU(T)                                            \
  case T:                                                            \
    if (cols) swiglu_kernel<T><<<groups, kThreads, 0, s>>>(a);       \
    else swiglu_rows_kernel<T><<<few, kThreads, 0, s>>>(a);          \
    break;
  switch (dtype) {
    FP64EMU_SWIGLU(FP64EMU_F32)
    FP64EMU_SWIGLU(FP64EMU_BF16)
    FP64EMU_SWIGLU(FP64EMU_F16)
  }
#undef FP64EMU_SWIGLU
  return check_hip(hipGetLastError(), "swiglu_f8 launch");
}

int fp64emu_swiglu_f8_backward(const void* dy, int dtype, int64_t M, int64_t F, int64_t ldy,
                               const fp64emu_f8_t* keep, void* dh, int out_dtype, int64_t ldh,
                               const fp64emu_f8_t* rows, const fp64emu_f8_t* cols,
                               fp64emu_stream_t stream) {
  if (M < 0 || F < 0) return invalid("shapes must be non-negative");
  if (!known_dtype(dtype) || !known_dtype(out_dtype))
    return invalid("dtype must be FP64EMU_F32, FP64EMU_BF16 or FP64EMU_F16");
  if (out_dtype != dtype && out_dtype != FP64EMU_F32)
    return invalid("out_dtype must be dy's or FP64EMU_F32");
  if (!keep) return invalid("null 8-bit operand");
  for (const fp64emu_f8_t* f : {keep, rows, cols})
    if (f && (f->fmt != FP64EMU_E4M3 || f->tiles)) return invalid("operands are e4m3 with scales by rows");
  if ((rows || cols) && F % kBlk) return invalid("quantised gradients need F as a multiple of 128");
  if (M == 0 || F == 0) return FP64EMU_OK;
  if (!dh && !rows && !cols) return invalid("no output asked for");
  if (!dy) return invalid("null operand pointer");
  if (ldy < F || (dh && ldh < 2 * F)) return invalid("rows are shorter than their width");
  SwigluGradArgs a{};
  if (int st = out8(keep, 2 * F, &a.keep)) return st;
  if (int st = out8(rows, 2 * F, &a.rows)) return st;
  if (int st = out8(cols, M, &a.cols)) return st;
  a.dy = dy;
  a.M = M;
  a.F = F;
  a.ldy = ldy;
  a.fblocks = (F + kBlk - 1) / kBlk;
  a.dh = dh;
  a.ldh = ldh;
  const int64_t mblocks = (M + kBlk - 1) / kBlk;
  if (mblocks > kMaxGroups / 4 / a.fblocks) return invalid("operand too large for one launch");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  a.tiles = mblocks * a.fblocks;
  const unsigned groups = (unsigned)((a.tiles + 7) / 8 * 16);
  const unsigned few = unit_groups(M, a.fblocks);
#define FP64EMU_GRAD(T, O)                                              \
  if (dtype == T && out_dtype == O) {                                   \
    if (cols) swiglu_grad_kernel<T, O><<<groups, kThreads, 0, s>>>(a);  \
    else swiglu_grad_rows_kernel<T, O><<<few, kThreads, 0, s>>>(a);     \
  }
  FP64EMU_GRAD(FP64EMU_F32, FP64EMU_F32)
  FP64EMU_GRAD(FP64EMU_BF16, FP64EMU_BF16)
  FP64EMU_GRAD(FP64EMU_F16, FP64EMU_F16)
  FP64EMU_GRAD(FP64EMU_BF16, FP64EMU_F32)
  FP64EMU_GRAD(FP64EMU_F16, FP64EMU_F32)
#undef FP64EMU_GRAD
  return check_hip(hipGetLastError(), "swiglu_f8 launch");
}

}  // extern "C"
