// What the sources of the 8-bit operators share, for gfx950: values in and codes
// out, the scale of a block, matrices of 128 x 128 tiles and of rows quantised from
// registers, the sigmoid, and the checks of their C entry points.
//
// A block with a = max(largest magnitude, 2^-110) has the scale s = a / F and
// the codes q = rne8(x ((1 / a) F)), F the format's largest value.  The floor
// keeps 1 / a finite for a block of zeros; the product exceeds F by at most three
// float32 roundings, which the conversion rounds back to F.
#pragma once
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

// A block of a row on 16 lanes, eight elements each.
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

// ---------------------------------------------------------------------------
// 1 / (1 + e^-g): e^-g = 2^(-g log2 e) with the product's
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

// ---------------------------------------------------------------------------
// Host side.

inline int check_hip(hipError_t e, const char* what) {
  if (e == hipSuccess) return FP64EMU_OK;
  return fp64emu_fail(FP64EMU_EHIP, std::string(what) + ": " + hipGetErrorString(e));
}

inline int invalid(const char* msg) { return fp64emu_fail(FP64EMU_EINVAL, msg); }

inline bool multiple(const void* p, int64_t of) { return reinterpret_cast<uintptr_t>(p) % of == 0; }

inline int size_of(int dtype) { return dtype == FP64EMU_F32 ? 4 : 2; }

inline bool known_dtype(int d) { return d == FP64EMU_F32 || d == FP64EMU_BF16 || d == FP64EMU_F16; }
inline bool known_fmt(int f) { return f == FP64EMU_E4M3 || f == FP64EMU_E5M2; }

// A quantised output of `rows` x `depth` codes, or NULL.
inline int out8(const fp64emu_f8_t* f, int64_t depth, Out8* o) {
  *o = Out8{};
  if (!f) return FP64EMU_OK;
  if (!f->q || !f->s) return invalid("null 8-bit operand");
  if (!known_fmt(f->fmt)) return invalid("fmt must be FP64EMU_E4M3 or FP64EMU_E5M2");
  if (f->ld < depth) return invalid("8-bit rows are shorter than their depth");
  *o = Out8{f->q, f->s, f->ld, f->stride, f->s_row, f->s_block, f->s_stride};
  return FP64EMU_OK;
}

// Work groups for a matrix's blocks of rows, 16 each.
inline unsigned unit_groups(int64_t rows, int64_t blocks) {
  return (unsigned)std::min<int64_t>((rows * blocks + 15) / 16, 1 << 20);
}

}  // namespace
