// Norms before and after a block, fused with the block's gate, dropout and residual, for
// gfx950: the residual stream's next value and its norm, plain or as the next product's
// 8-bit operand, and the gradient of both.  The entry points are fp64emu_norm_f8*.
//
// With i(v) = (mean(v^2) + eps)^-1/2 over a row of D elements:
//
//   z = y i(y) post,  v = scale r + gate drop(z),  x = v i(v) w
//
// (z = y without post, v = r without y.)  v is rounded once, where it is stored as the
// new stream; x is taken from the unrounded one.

#include "f8_common.h"
#include "f8_drop.h"
#include "f8_sums.h"

namespace {

struct NormArgs {
  const void *r, *y, *gate, *w, *post;
  const int64_t* rng;
  int64_t M, D, ld_r, ld_y, ld_gate;         // ld_gate 0: one gate for all rows
  int64_t blocks;                            // of 128 along a row
  int w_type, post_type, gate_type;
  uint32_t threshold;
  float scale, eps, over_d;                  // over_d: 1 / D
  void* out;                                 // the new stream
  void* x;
  int64_t ld_out, ld_x;
  float* stats;                              // i(v), then i(y), M each
  Out8 rows, cols;
};

struct NormGradArgs {
  const void *dx, *dr;
  int64_t ld_dx, ld_dr;
  void *dr_out, *dy, *dgates;
  int64_t ld_dr_out, ld_dy, ld_dgates;
  int wide;                                  // dgates is float32
  float *dw, *dpost, *dgate;                 // [D], or a group's part of them, [groups][D] each
  float* back;                               // rows of any length: a row's, as GradRow has it
};

// Eight elements of a row as they came.  A launch's kernels load whole ones of all their operands behind one
// branch and the last, partial ones of a row behind another, element by element: a branch for each operand
// took 60 registers of addresses and masks more.
template <int kT>
struct Eight {
  v4u w;
  __device__ __forceinline__ void whole(const void* p, int64_t i) {
    __builtin_memcpy(&w, static_cast<const unsigned short*>(p) + i, 16);
  }
  __device__ __forceinline__ void part(const void* p, int64_t i, int valid) {
    const unsigned short* q = static_cast<const unsigned short*>(p) + i;
    uint64_t lo = 0, hi = 0;
#pragma unroll 1
    for (int j = valid - 1; j >= 0; --j) {
      hi = hi << 16 | lo >> 48;
      lo = lo << 16 | q[j];
    }
    w = v4u{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  }
  __device__ __forceinline__ void zero() { w = v4u{0u, 0u, 0u, 0u}; }
  __device__ __forceinline__ float at(int j) const {
    const uint32_t h = w[j >> 1] >> (16 * (j & 1));
    return kT == FP64EMU_BF16 ? bf16_value((unsigned short)h) : (float)__builtin_bit_cast(_Float16, (unsigned short)h);
  }
  // Makes the compiler unpack element j on from here on, and not before: it unpacked all elements of a row's
  // operands at once and kept them.
  __device__ __forceinline__ void from_here(int j) { asm volatile("" : "+v"(w[j >> 1])); }
};
template <>
struct Eight<FP64EMU_F32> {
  v4f v[2];
  __device__ __forceinline__ void whole(const void* p, int64_t i) {
    __builtin_memcpy(v, static_cast<const float*>(p) + i, 32);
  }
  __device__ __forceinline__ void part(const void* p, int64_t i, int valid) {
    const float* q = static_cast<const float*>(p) + i;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j >> 2][j & 3] = j < valid ? q[j] : 0.0f;
  }
  __device__ __forceinline__ void zero() { v[0] = v[1] = v4f{0.0f, 0.0f, 0.0f, 0.0f}; }
  __device__ __forceinline__ float at(int j) const { return v[j >> 2][j & 3]; }
  __device__ __forceinline__ void from_here(int) {}
};

// Eight elements from i on, those past `valid` as zeros.
template <int kT>
__device__ __forceinline__ void load8(const void* p, int64_t i, int valid, float (&v)[8]) {
  Eight<kT> e;
  if (valid >= 8) e.whole(p, i);
  else e.part(p, i, valid);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = e.at(j);
}
// Eight elements of a weight of any type, as they came (ones without one): loaded first, told apart where
// they are used.  With the type's branch around load and conversion a kernel waited for each weight before it
// asked for the next (8192 x 4096 rows 54 us, 51 without).
struct EightAny {
  v4u a, b;
  __device__ __forceinline__ void load(int type, const void* p, int64_t i, int valid) {
    a = b = v4u{0u, 0u, 0u, 0u};
    if (!p || valid <= 0) return;
    if (valid < 8) {
      if (type == FP64EMU_F32) {
        const uint32_t* q = static_cast<const uint32_t*>(p) + i;
#pragma unroll
        for (int j = 0; j < 7; ++j)
          if (j < valid) (j < 4 ? a : b)[j & 3] = q[j];
      } else {
        const unsigned short* q = static_cast<const unsigned short*>(p) + i;
#pragma unroll
        for (int j = 0; j < 7; ++j)
          if (j < valid) a[j >> 1] |= (uint32_t)q[j] << (16 * (j & 1));
      }
    } else if (type == FP64EMU_F32) {
      __builtin_memcpy(&a, static_cast<const float*>(p) + i, 16);
      __builtin_memcpy(&b, static_cast<const float*>(p) + i + 4, 16);
    } else {
      __builtin_memcpy(&a, static_cast<const unsigned short*>(p) + i, 16);
    }
  }
  __device__ __forceinline__ void values(int type, const void* p, float (&v)[8]) const {
    if (!p) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 1.0f;
    } else if (type == FP64EMU_F32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __builtin_bit_cast(float, j < 4 ? a[j & 3] : b[j & 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t h = a[j >> 1] >> (16 * (j & 1));
        v[j] = type == FP64EMU_BF16 ? bf16_value((unsigned short)h) : (float)__builtin_bit_cast(_Float16, (unsigned short)h);
      }
    }
  }
};
__device__ __forceinline__ void load8_any(int type, const void* p, int64_t i, int valid, float (&v)[8]) {
  EightAny e;
  e.load(type, p, i, valid);
  e.values(type, p, v);
}

template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ float dpp(float v) {         // 0 in the rows that are masked out
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, kRowMask, 0xf, false));
}
template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ double dpp(double v) {
  v2u w = __builtin_bit_cast(v2u, v);
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[i], kCtrl, kRowMask, 0xf, false);
  return __builtin_bit_cast(double, w);
}
__device__ __forceinline__ float from_lane(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ double from_lane(double v, int lane) {
  v2u w = __builtin_bit_cast(v2u, v);
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = (uint32_t)__builtin_amdgcn_readlane((int)w[i], lane);
  return __builtin_bit_cast(double, w);
}
// The sum over the 16 lanes of a DPP row, the same bits in all of them; T: float or double.
template <class T>
__device__ __forceinline__ T row16_sum(T v) {
  v += dpp<0x128>(v);                        // row_ror:8
  v += dpp<0x124>(v);
  v += dpp<0x122>(v);
  return v + dpp<0x121>(v);
}
// Over a wave, scalar: on vector instructions alone, where lane exchanges go through the LDS unit.
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
  v = row16_sum(v);
  v += dpp<0x142, 0xa>(v);                   // row_bcast:15: rows 1 and 3 add the row before
  v += dpp<0x143, 0xc>(v);                   // row_bcast:31: rows 2 and 3 add the half before
  return from_lane(v, 63);
}
// Of two values over a wave, scalar: a in the lower 32 lanes and b in the upper ones from the first step on, which
// takes half the steps of one after the other.
__device__ __forceinline__ void wave_sums(double& a, double& b) {
  v2u x = __builtin_bit_cast(v2u, a), y = __builtin_bit_cast(v2u, b);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto r = __builtin_amdgcn_permlane32_swap(x[i], y[i], false, false);
    x[i] = r[0];                             // a's lower lanes, b's lower lanes
    y[i] = r[1];                             // a's upper lanes, b's upper lanes
  }
  double v = row16_sum(__builtin_bit_cast(double, x) + __builtin_bit_cast(double, y));
  v += dpp<0x142, 0xa>(v);
  a = from_lane(v, 31);
  b = from_lane(v, 63);
}

// How a launch lays rows on threads: kT threads a row, eight elements each (so 16 neighbouring
// lanes hold a block of 128), work groups of 256 threads or one row.
template <int kT_>
struct RowShape {
  static constexpr int kT = kT_, kGroup = kT > kThreads ? kT : kThreads, kRows = kGroup / kT;
  // Which of the group's rows a thread has: the same for a wave, where it is, so that addresses of rows are scalar.
  static __device__ __forceinline__ int sub() {
    if constexpr (kRows == 1) return 0;
    const int s = threadIdx.x / kT;
    return kT >= 64 ? __builtin_amdgcn_readfirstlane(s) : s;
  }
  // Row m of a matrix of rows of ld elements of T.  Scalar where a wave has one row: the compiler kept
  // a pointer for each operand in vector registers from row to row.
  template <int kType>
  static __device__ __forceinline__ uint8_t* row(const void* p, int64_t m, int64_t ld) {
    uint64_t a = reinterpret_cast<uint64_t>(p) + (uint64_t)(m * ld) * (kType == FP64EMU_F32 ? 4 : 2);
    if constexpr (kT >= 64) {
      const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
      a = (uint64_t)hi << 32 | lo;
    }
    return reinterpret_cast<uint8_t*>(a);
  }
};

// Sums over the threads of a row, in all of them; `turn` alternates from call to call, so that one
// barrier is enough.
template <int kT, int kN, int kGroup, class T = float>
struct RowSum {
  static constexpr int kWaves = kT / 64;
  struct alignas(16) Room { T v[2][kN][kGroup / 64]; };
  static __device__ __forceinline__ void run(T (&v)[kN], Room& room, int& turn) {
    if constexpr (sizeof(T) == 8 && kT >= 64) {
      static_assert(kN == 3, "the gradient's sums");
      v[0] = wave_sum((float)v[0]);          // (nothing is taken off the first of them)
      wave_sums(v[1], v[2]);
    } else {
#pragma unroll
      for (int n = 0; n < kN; ++n) v[n] = kT >= 64 ? wave_sum(v[n]) : row16_sum(v[n]);
    }
    if constexpr (kT > 64) {
      const int wave = threadIdx.x >> 6, first = wave / kWaves * kWaves;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int n = 0; n < kN; ++n) room.v[turn][n][wave] = v[n];
      }
      __syncthreads();
      if constexpr (sizeof(T) == 8) {
        // A DPP row for each sum, a lane for each wave's part of it: in each thread the parts would take 48 registers.
        static_assert(kN <= 4 && kWaves <= 16, "a wave has them all");
        const int lane = threadIdx.x & 63, n = lane >> 4, w = lane & 15;
        T s = n < kN && w < kWaves ? room.v[turn][n < kN ? n : 0][first + (w < kWaves ? w : 0)] : T{};
        s = row16_sum(s);
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = from_lane(s, 16 * i);
        turn ^= 1;
        return;
      }
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        T s = room.v[turn][n][first];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) s += room.v[turn][n][first + w];
        v[n] = s;
      }
      turn ^= 1;
    }
  }
};

// The hardware's 1 / sqrt, within one ulp, and a Newton step.
__device__ __forceinline__ float inverse_rms(float squares, const NormArgs& g) {
  const float m = fmaf(squares, g.over_d, g.eps), y = __builtin_amdgcn_rsqf(m);
  return m < __builtin_inff() ? fmaf(y * 0.5f, fmaf(-m * y, y, 1.0f), y) : y;      // (past that inf 0)
}

// v of eight elements from those of r and y; kept(j): whether element j stays.
template <class Kept>
__device__ __forceinline__ void joined(const NormArgs& g, const Drop& drop, const Kept& kept, float iy, const float (&y)[8],
                                       const float (&post)[8], const float (&gate)[8], float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float z = g.post ? y[j] * iy * post[j] : y[j];
    v[j] = g.scale * v[j] + gate[j] * (kept(j) ? z * drop.scale : 0.0f);
  }
}

template <int kR, int kY>
__device__ __forceinline__ void emit_norm(const NormArgs& g, int64_t m, int64_t col, int valid, float iv,
                                          const float (&v)[8], const float (&w)[8]) {
  Held<FP64EMU_F32> x;
#pragma unroll
  for (int j = 0; j < 8; ++j) x.v[0][j] = v[j] * iv * w[j];
  if (g.x) store8<kY>(g.x, m * g.ld_x + col, valid, x.v[0]);
  if (g.rows.q) {
    // (All 16 lanes of a block come here or none: those past the row hold zeros.)
    const float a = amax_of(row16_max(x.row_mag(0)));
    put8(g.rows.q + m * g.rows.ld + col, valid, row_codes<FP64EMU_E4M3>(x, 0, inverse_scale<FP64EMU_E4M3>(a)));
    const int64_t kb = col / kBlk;
    if ((threadIdx.x & 15) == 0 && valid > 0) g.rows.s[m * g.rows.s_row + kb * g.rows.s_block] = scale_of<FP64EMU_E4M3>(a);
  }
}

// Rows whose values stay in registers from the first sum to the last store.  A work group takes
// rows blockIdx.x kRows + .., gridDim.x kRows apart, the weights in registers throughout and the next
// row's values on their way.  Bound by its bytes: 8192 x 4096 bfloat16 with y, post and gate 50 us in 8 bits
// (4.75 TB/s), 46 plain (5.8, more than the copy's 5.2); its vector units are busy for 62% of it, with the generator, which adds
// 6% to its cycles, for 66%.  (Sixteen elements a thread: as fast, and one row of 8192 5.6 us where this takes 4.4.)
template <int kR, int kY, class S>
__global__ void __launch_bounds__(S::kGroup) norm_rows_kernel(NormArgs g) {
  constexpr int kT = S::kT;
  using Sum = RowSum<kT, 1, S::kGroup>;
  __shared__ typename Sum::Room room;
  const int t = threadIdx.x % kT, sub = S::sub();
  const Drop drop = drop_of(g.y ? g.threshold : 0, g.rng);
  const int64_t row_chunks = (g.D + 7) / 8;
  const int col = 8 * t, left = (int)g.D - col, valid = left < 0 ? 0 : left < 8 ? left : 8;
  int turn = 0;
  Eight<kR> r;
  Eight<kY> y, gates;
  auto fetch = [&](int64_t m) {
    const uint8_t* pr = S::template row<kR>(g.r, m, g.ld_r);
    const uint8_t* py = S::template row<kY>(g.y, m, g.ld_y);
    const uint8_t* pg = S::template row<kY>(g.gate, m, g.ld_gate);
    const int n = m < g.M ? valid : 0;
    y.zero();
    gates.zero();
    if (n == 8) {
      r.whole(pr, col);
      if (g.y) y.whole(py, col);
      if (g.ld_gate) gates.whole(pg, col);
    } else {
      r.part(pr, col, n);
      if (g.y) y.part(py, col, n);
      if (g.ld_gate) gates.part(pg, col, n);
    }
  };
  const int64_t step = (int64_t)gridDim.x * S::kRows;
  int64_t m = (int64_t)blockIdx.x * S::kRows + sub;
  fetch(m);
  float w[8], post[8], gate[8];
  {
    EightAny ew, ep, eg;
    ep.load(g.post_type, g.post, col, valid);
    eg.load(g.gate_type, g.ld_gate == 0 ? g.gate : nullptr, col, valid);
    ew.load(g.w_type, g.w, col, valid);
    ep.values(g.post_type, g.post, post);
    eg.values(g.gate_type, g.gate, gate);
    ew.values(g.w_type, g.w, w);
  }
  for (int64_t first = (int64_t)blockIdx.x * S::kRows; first < g.M; first += step, m += step) {
    Eight<kR> ro = r;
    Eight<kY> yo = y, go = gates;
    fetch(m + step);
    // (The generator works while the row is on its way.)
    const Kept kept(drop, (uint64_t)(m * row_chunks + t));
    float v[8], yv[8], iy = 1.0f;
    if (g.post) {
      float s[1] = {0.0f};
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] = fmaf(yo.at(j), yo.at(j), s[0]);
      Sum::run(s, room, turn);
      iy = inverse_rms(s[0], g);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j % 2 == 0) {
        ro.from_here(j);
        yo.from_here(j);
      }
      v[j] = ro.at(j);
      yv[j] = yo.at(j);
      if (g.ld_gate) gate[j] = go.at(j);
    }
    if (g.y) {
      joined(g, drop, [&](int j) { return kept.at(j); }, iy, yv, post, gate, v);
      if (g.out && m < g.M) store8<kR>(S::template row<kR>(g.out, m, g.ld_out), col, valid, v);
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < 8; ++j) s[0] = fmaf(v[j], v[j], s[0]);
    Sum::run(s, room, turn);
    const float iv = inverse_rms(s[0], g);
    if (m < g.M) {
      if (g.stats && t == 0) {
        g.stats[m] = iv;
        if (g.post) g.stats[g.M + m] = iy;
      }
      emit_norm<kR, kY>(g, m, col, valid, iv, v, w);
    }
  }
}

// Eight elements of v again from memory, for rows that do not stay in registers.
template <int kR, int kY>
__device__ __forceinline__ void joined_at(const NormArgs& g, const Drop& drop, int64_t m, int64_t col, int valid,
                                          float iy, float (&v)[8]) {
  load8<kR>(g.r, m * g.ld_r + col, valid, v);
  if (!g.y) return;
  float y[8], post[8], gate[8];
  load8<kY>(g.y, m * g.ld_y + col, valid, y);
  load8_any(g.post_type, g.post, col, valid, post);
  load8_any(g.gate_type, g.gate, m * g.ld_gate + col, valid, gate);
  const Kept kept(drop, (uint64_t)(m * ((g.D + 7) / 8) + col / 8));
  joined(g, drop, [&](int j) { return kept.at(j); }, iy, y, post, gate, v);
}

// Rows of any length, a row to a work group of 1024, read once for each sum and once for x: past
// the registers' 8192 elements a row's second and third reading come from L2 (8192 x 16384 bfloat16 with y and post
// fetches 546 MB, r and y once being 537).  435 us by rows, 2.2 TB/s: it unpacks and joins every element three times, and its vector
// units are busy for 64% of that.
constexpr int kLong = 1024;

template <int kR, int kY>
__global__ void __launch_bounds__(kLong) norm_long_kernel(NormArgs g) {
  using Sum = RowSum<kLong, 1, kLong>;
  __shared__ typename Sum::Room room;
  const Drop drop = drop_of(g.y ? g.threshold : 0, g.rng);
  int turn = 0;
  auto each = [&](auto fn) {
    // (Whole blocks of 128 of the last round, so that emit_norm's 16 lanes are there together.)
    for (int64_t col = 8 * threadIdx.x; col < g.blocks * kBlk; col += 8 * kLong) {
      const int64_t left = g.D - col;
      fn(col, left < 0 ? 0 : left < 8 ? (int)left : 8);
    }
  };
  for (int64_t m = blockIdx.x; m < g.M; m += gridDim.x) {
    float iy = 1.0f;
    if (g.post) {
      float s[1] = {0.0f};
      each([&](int64_t col, int valid) {
        float y[8];
        load8<kY>(g.y, m * g.ld_y + col, valid, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0] = fmaf(y[j], y[j], s[0]);
      });
      Sum::run(s, room, turn);
      iy = inverse_rms(s[0], g);
    }
    float s[1] = {0.0f};
    each([&](int64_t col, int valid) {
      float v[8];
      joined_at<kR, kY>(g, drop, m, col, valid, iy, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] = fmaf(v[j], v[j], s[0]);
    });
    Sum::run(s, room, turn);
    const float iv = inverse_rms(s[0], g);
    if (g.stats && threadIdx.x == 0) {
      g.stats[m] = iv;
      if (g.post) g.stats[g.M + m] = iy;
    }
    if (!g.out && !g.x && !g.rows.q) continue;
    each([&](int64_t col, int valid) {
      float v[8], w[8];
      joined_at<kR, kY>(g, drop, m, col, valid, iy, v);
      load8_any(g.w_type, g.w, col, valid, w);
      // (r may be the new stream itself: its last reading is above.)
      if (g.out) store8<kR>(g.out, m * g.ld_out + col, valid, v);
      emit_norm<kR, kY>(g, m, col, valid, iv, v, w);
    });
  }
}

// x's columns by tiles of 128 x 128, once the rows' statistics are there.  The rows' kernel writes everything
// else: it waits for its sums, and the stores cost it little (with the statistics alone from that kernel and all outputs
// from this one 8192 x 4096 both ways took 3% more).  Bound by its bytes: r and y again and a byte a value, 41 to 47 us there,
// 3.6 to 4 TB/s, of 91 both ways and 82 to 85 without the generator, which adds 14% to this kernel's cycles.
template <int kR, int kY>
__global__ void __launch_bounds__(kThreads, kR == FP64EMU_F32 ? 2 : 3) norm_tile_kernel(NormArgs g) {
  __shared__ TileLds lds;
  const uint32_t blocks = (uint32_t)g.blocks;
  const int64_t kb = blockIdx.x % blocks, mb = blockIdx.x / blocks;
  const int64_t row0 = mb * kBlk, col0 = kb * kBlk, row = row0 + 8 * ((int)threadIdx.x >> 4);
  const TilePlace t = tile_place(row0, col0, g.M, g.D);
  const int64_t col = col0 + 8 * t.cl;
  const Drop drop = drop_of(g.y ? g.threshold : 0, g.rng);
  const int n = t.valid(0) > 0 ? (t.valid(0) < 8 ? t.valid(0) : 8) : 0;
  // Lane cl of a row group has row cl % 8's statistics, i(v) in the lower eight lanes and i(y) in the
  // upper ones: broadcast within the DPP row where they are used.
  float stat = 0.0f;
  if (8 * t.rg + (t.cl & 7) < t.rows && (t.cl < 8 || g.post)) stat = g.stats[(t.cl < 8 ? 0 : g.M) + row + (t.cl & 7)];
  Held<FP64EMU_F32> x;
  {
    Held<kR> r;
    Held<kY> y;
    // The weights before the rows: behind them the tile took 7 us more of 40.
    float w[8], post[8], gate[8];
    EightAny ew, ep, eg;
    ew.load(g.w_type, g.w, col, n);
    ep.load(g.post_type, g.post, col, n);
    eg.load(g.gate_type, g.ld_gate == 0 ? g.gate : nullptr, col, n);
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      r.load(p, g.r, (row + p) * g.ld_r + col, t.valid(p));
      if (g.y) y.load(p, g.y, (row + p) * g.ld_y + col, t.valid(p));
    }
    ew.values(g.w_type, g.w, w);
    ep.values(g.post_type, g.post, post);
    eg.values(g.gate_type, g.gate, gate);
    // The generator works while the rows are on their way: a byte of a mask for each row.
    uint32_t mask[2] = {~0u, ~0u};
    if (drop.threshold) {
      const uint64_t chunk = (uint64_t)(row * ((g.D + 7) / 8) + col / 8);
      mask[0] = mask[1] = 0;
#pragma unroll
      for (int p = 0; p < 8; ++p) mask[p >> 2] |= kept_of(drop, chunk + p * ((g.D + 7) / 8)) << (8 * (p & 3));
    }
    asm volatile("" : "+v"(mask[0]), "+v"(mask[1]));
    auto each = [&](auto P) {
      constexpr int p = decltype(P)::value;
      const float iv = row16_lane<p>(stat), iy = row16_lane<8 + p>(stat);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = r.at(p, j);
      if (g.y) {
        float yv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) yv[j] = y.at(p, j);
        if (g.ld_gate) load8<kY>(g.gate, (row + p) * g.ld_gate + col, t.valid(p), gate);
        joined(g, drop, [&](int j) { return (mask[p >> 2] >> (8 * (p & 3) + j) & 1) != 0; }, iy, yv, post, gate, v);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) x.v[p][j] = v[j] * iv * w[j];
    };
    each_row(each, std::make_integer_sequence<int, 8>{});
  }
  emit_cols<FP64EMU_E4M3>(x, t, row0, col0, mb, g.cols, lds);
}

// ---------------------------------------------------------------------------
// Gradient.  With vh = v i(v), yh = y i(y) and k drop's factor of an element:
//
//   t = dr + i(v) (dx w - vh c1),                     c1 = mean(dx w vh)     t: v's gradient
//   dz = t gate k,  dy = i(y) (dz post - yh c2),      c2 = mean(dz post yh)
//   dw = sum dx vh,  dpost = sum dz yh,  dgate = sum t k yh post    over the rows
//
// and scale t is r's gradient.  c2 is linear in c1: with e = dr + i(v) dx w and q = gate k post y, it is
// i(y) (mean(q e) - i(v)^2 c1 mean(q v)), so that one joint sum of three gives both and a row takes
// one barrier.  Where the stream is mostly the branch's output and dx lies along it, the two cancel: the threads'
// sums are then joined, and subtracted, in 64 bits, which leaves dy as far from the formula as a second pass over what is
// left would (joined in 32 bits, 2.4 to 2.7 times as far).  v is the stream as it is stored.

// The three sums of eight elements: of (dx w) v, and with k what remains of gate and drop (0 where dropped),
// q = k post y, of q e and of q v.  The rows' own factors i(v) and i(y) join them at their ends.
template <bool kPost>
struct GradSums {
  static constexpr int kN = kPost ? 3 : 1;
  using Joint = std::conditional_t<kPost, double, float>;      // what the threads' sums are joined in
  static __device__ __forceinline__ void add(float v, float dx, float dr, float w, float iv, float kept_gate, float post,
                                             float y, float (&s)[kN]) {
    const float gw = dx * w;
    s[0] = fmaf(gw, v, s[0]);
    if constexpr (kPost) {
      const float q = kept_gate * post * y, e = fmaf(iv, gw, dr);
      s[1] = fmaf(q, e, s[1]);
      s[2] = fmaf(q, v, s[2]);
    }
  }
};

// A row's factors once its sums are there: t = dr + iv dx w - back v; dy = iy dz post - c2 y.
struct GradRow { float iv, iy, back, c2; };

template <bool kPost>
__device__ __forceinline__ GradRow grad_row(const typename GradSums<kPost>::Joint (&s)[GradSums<kPost>::kN], float iv, float iy,
                                            float over_d) {
  GradRow r{iv, iy, 0.0f, 0.0f};
  const float c1 = (float)s[0] * iv * over_d;                  // mean(dx w vh)
  r.back = iv * iv * c1;
  // mean(dz post yh) is i(y) (s1 - back s2) / D, of the same rounded back that t takes
  if constexpr (kPost) r.c2 = iy * iy * (iy * ((float)fma(-(double)r.back, s[2], s[1]) * over_d));
  return r;
}
// A row's sums over its threads from a thread's own.
template <class Sum, bool kPost>
__device__ __forceinline__ GradRow joined_row(const float (&mine)[GradSums<kPost>::kN], typename Sum::Room& room, int& turn, float iv,
                                              float iy, float over_d) {
  typename GradSums<kPost>::Joint s[GradSums<kPost>::kN];
#pragma unroll
  for (int i = 0; i < GradSums<kPost>::kN; ++i) s[i] = mine[i];
  Sum::run(s, room, turn);
  return grad_row<kPost>(s, iv, iy, over_d);
}

struct GradOut { float t, dy, dz, z, dgate; };

// An element's gradients: kept_scale is drop's factor, 0 where dropped.
template <bool kPost>
__device__ __forceinline__ GradOut grad_of(const GradRow& r, float v, float dx, float dr, float w, float kept_scale,
                                           float gate, float post, float y) {
  GradOut o;
  o.t = fmaf(-r.back, v, fmaf(r.iv, dx * w, dr));
  const float u = o.t * kept_scale;
  o.dz = u * gate;
  if constexpr (kPost) {
    o.z = y * r.iy;                                            // (yh)
    o.dy = fmaf(-r.c2, y, r.iy * (o.dz * post));
    o.dgate = u * (o.z * post);
  } else {
    o.z = kept_scale != 0.0f ? y : 0.0f;                       // (whatever a dropped y was)
    o.dy = o.dz;
    o.dgate = u * o.z;
  }
  return o;
}

// Eight elements of a gate's gradient for each row, in y's type or float32.
template <int kY>
__device__ __forceinline__ void put_gates(const NormGradArgs& d, int64_t m, int64_t col, int valid, const float (&v)[8]) {
  if (kY == FP64EMU_F32 || d.wide) store8<FP64EMU_F32>(d.dgates, m * d.ld_dgates + col, valid, v);
  else store8<kY>(d.dgates, m * d.ld_dgates + col, valid, v);
}

// A group's sums over its rows into its part of [groups][D] (or the result itself, with one group).
template <class S, class Column>
__device__ __forceinline__ void join_rows(const float (&sum)[8], const Column& of, float* part, int64_t D, float* lds) {
  constexpr int kT = S::kT;
  const int t = threadIdx.x % kT, sub = threadIdx.x / kT;
  float* to = part + (int64_t)blockIdx.x * D;
  if constexpr (S::kRows == 1) {
    if (of.in) store8<FP64EMU_F32>(to, of.col, 8, sum);
  } else {
    __syncthreads();                         // (whatever the room held before)
#pragma unroll
    for (int j = 0; j < 8; ++j) lds[j * S::kGroup + threadIdx.x] = sum[j];
    __syncthreads();
    if (sub == 0) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = lds[j * S::kGroup + t];
#pragma unroll
        for (int i = 1; i < S::kRows; ++i) v[j] += lds[j * S::kGroup + i * kT + t];
      }
      if (of.in) store8<FP64EMU_F32>(to, of.col, 8, v);
    }
  }
}

// Rows in registers, as norm_rows_kernel, but kC times eight elements a thread (element 8 (c kT + t) on) for rows past 4096:
// 1024 threads a row leave 128 registers each, which the sums over the rows, kept a column to a thread,
// do not fit.  A row's values stay as they came and are worked out again after its sums; with one
// chunk the next row's are on their way meanwhile.  A row's last, partial eight elements are its last eight: what the
// thread beside has of them comes out the same from both and counts once in the sums (with loads and stores
// of parts the kernel took 195 registers).  8192 x 4096 bfloat16 with everything 90 to 97 us, the last sums' 5 among
// them: 4.2 to 4.5 TB/s of the copy's 5.2; two work groups of 512 on a CU share its vector units, which are busy for 65% of
// that time, and each waits for its row's one barrier.  kPost: y has a norm; without it y may be absent, too.  kGates: a gate
// for each row, whose values and gradient do not fit 128 registers as the rest does.
template <int kR, int kY, class S, int kC, bool kPost, bool kGates>
__global__ void __launch_bounds__(S::kGroup, kC == 1 && !kGates && kR != FP64EMU_F32 && S::kT >= 64 ? 4 : 2)
    norm_grad_kernel(NormArgs g, NormGradArgs d) {
  constexpr int kT = S::kT, kN = kPost ? 3 : 1;
  constexpr bool kAhead = kC == 1;
  using Sum = RowSum<kT, kN, S::kGroup, typename GradSums<kPost>::Joint>;
  __shared__ typename Sum::Room room;
  __shared__ float joint[S::kRows > 1 ? 8 * S::kGroup : 1];
  const int t = threadIdx.x % kT, sub = S::sub();
  const Drop drop = drop_of(g.y ? g.threshold : 0, g.rng);
  const int64_t row_chunks = (g.D + 7) / 8;
  struct Column {
    float w[8], post[8], gate[8], dw[8], dpost[8], dgate[8];
    int col, again;                          // first column; leading elements that another thread has, too
    bool in;
  } of[kC];
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    Column& o = of[c];
    const int col = 8 * (c * kT + t), left = (int)g.D - col;
    o.in = left > 0;
    o.again = left > 0 && left < 8 ? 8 - left : 0;
    o.col = col - o.again;
#pragma unroll
    for (int j = 0; j < 8; ++j) o.dw[j] = o.dpost[j] = o.dgate[j] = 0.0f;
  }
  int turn = 0;
  struct Row {
    Eight<kR> v[kC], dr[kC];
    Eight<kY> y[kC], dx[kC], gates[kC];
    float iv, iy;
    __device__ __forceinline__ void from_here(int c, int j) {
      v[c].from_here(j);
      dr[c].from_here(j);
      y[c].from_here(j);
      dx[c].from_here(j);
    }
  };
  auto fetch = [&](int64_t m, Row& o) {
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const int col = of[c].col;
      o.v[c].zero();
      o.dx[c].zero();
      o.dr[c].zero();
      o.y[c].zero();
      if constexpr (kGates) o.gates[c].zero();
      if (m < g.M && of[c].in) {
        o.v[c].whole(S::template row<kR>(g.r, m, g.ld_r), col);
        o.dx[c].whole(S::template row<kY>(d.dx, m, d.ld_dx), col);
        if (d.dr) o.dr[c].whole(S::template row<kR>(d.dr, m, d.ld_dr), col);
        if (g.y) o.y[c].whole(S::template row<kY>(g.y, m, g.ld_y), col);
        if constexpr (kGates) o.gates[c].whole(S::template row<kY>(g.gate, m, g.ld_gate), col);
      }
    }
    o.iv = m < g.M ? g.stats[m] : 0.0f;
    o.iy = kPost && m < g.M ? g.stats[g.M + m] : 0.0f;
  };
  const int64_t step = (int64_t)gridDim.x * S::kRows;
  int64_t m = (int64_t)blockIdx.x * S::kRows + sub;
  Row next;
  if constexpr (kAhead) fetch(m, next);
  {
    EightAny ew[kC], ep[kC], eg[kC];
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const int col = of[c].col, valid = of[c].in ? 8 : 0;
      ew[c].load(g.w_type, g.w, col, valid);
      if constexpr (kPost) ep[c].load(g.post_type, g.post, col, valid);
      if constexpr (!kGates) eg[c].load(g.gate_type, g.gate, col, valid);
    }
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      ew[c].values(g.w_type, g.w, of[c].w);
      if constexpr (kPost) ep[c].values(g.post_type, g.post, of[c].post);
      if constexpr (!kGates) eg[c].values(g.gate_type, g.gate, of[c].gate);
    }
  }
  for (int64_t first = (int64_t)blockIdx.x * S::kRows; first < g.M; first += step, m += step) {
    Row o;
    if constexpr (kAhead) {
      o = next;
      fetch(m + step, next);
    } else {
      fetch(m, o);
    }
    float s[kN] = {};
    uint32_t kept[kC];
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      Column& k = of[c];
      const uint64_t chunk = (uint64_t)(m * row_chunks + c * kT + t);
      kept[c] = kept_of(drop, chunk);
      if (k.again) kept[c] = (kept_of(drop, chunk - 1) | kept[c] << 8) >> (8 - k.again) & 0xff;
      float mine[kN] = {};
      auto element = [&](int j) {
        GradSums<kPost>::add(o.v[c].at(j), o.dx[c].at(j), o.dr[c].at(j), k.w[j], o.iv,
                             kept[c] >> j & 1 ? k.gate[j] * drop.scale : 0.0f, k.post[j], o.y[c].at(j), mine);
      };
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j % 2 == 0) o.from_here(c, j);
        if constexpr (kGates) k.gate[j] = o.gates[c].at(j);
        element(j);
        asm volatile("" : "+v"(mine[0]));
      }
      if (k.again) {                         // (a wave's last thread, at most)
#pragma unroll
        for (int i = 0; i < kN; ++i) mine[i] = 0.0f;
#pragma unroll
        for (int j = 1; j < 8; ++j)
          if (j >= k.again) element(j);
      }
#pragma unroll
      for (int i = 0; i < kN; ++i) s[i] += mine[i];
    }
    const GradRow row = joined_row<Sum, kPost>(s, room, turn, o.iv, o.iy, g.over_d);
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      Column& k = of[c];
      float tv[8], dy[8], dg[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j % 2 == 0) o.from_here(c, j);
        const float v = o.v[c].at(j), dx = o.dx[c].at(j);
        const GradOut e = grad_of<kPost>(row, v, dx, o.dr[c].at(j), k.w[j], kept[c] >> j & 1 ? drop.scale : 0.0f, k.gate[j],
                                         kPost ? k.post[j] : 1.0f, o.y[c].at(j));
        k.dw[j] = fmaf(dx, v * o.iv, k.dw[j]);
        if constexpr (kPost) k.dpost[j] = fmaf(e.dz, e.z, k.dpost[j]);
        if constexpr (!kGates) k.dgate[j] += e.dgate;
        tv[j] = e.t * g.scale;
        dy[j] = e.dy;
        dg[j] = e.dgate;
        asm volatile("" : "+v"(k.dw[j]), "+v"(k.dpost[j]), "+v"(k.dgate[j]));      // (here, and not at the end)
      }
      if (m < g.M && k.in) {
        if (d.dr_out) store8<kR>(S::template row<kR>(d.dr_out, m, d.ld_dr_out), k.col, 8, tv);
        if (d.dy) store8<kY>(S::template row<kY>(d.dy, m, d.ld_dy), k.col, 8, dy);
        if (kGates && d.dgates) put_gates<kY>(d, m, k.col, 8, dg);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    if (d.dw) join_rows<S>(of[c].dw, of[c], d.dw, g.D, joint);
    if (kPost && d.dpost) join_rows<S>(of[c].dpost, of[c], d.dpost, g.D, joint);
    if (!kGates && d.dgate) join_rows<S>(of[c].dgate, of[c], d.dgate, g.D, joint);
  }
}

// Rows of any length: the row's sums, then its gradients, from two readings of it, mostly from memory both times (8192 x 16384
// bfloat16 fetches 1971 MB, four operands once being 1074); 460 us there, and 250 the columns' kernel.  A row's `back` is kept
// for the sums over the rows, which another kernel makes.
template <int kR, int kY, bool kPost>
struct GradAt {
  float v[8], dx[8], dr[8], y[8], w[8], post[8], gate[8];
  uint32_t kept;
  __device__ __forceinline__ GradAt(const NormArgs& g, const NormGradArgs& d, const Drop& drop, int64_t m, int64_t col) {
    const int valid = g.D - col < 8 ? (int)(g.D - col) : 8;
    load8<kR>(g.r, m * g.ld_r + col, valid, v);
    load8<kY>(d.dx, m * d.ld_dx + col, valid, dx);
    load8<kR>(d.dr, m * d.ld_dr + col, d.dr ? valid : 0, dr);
    load8<kY>(g.y, m * g.ld_y + col, g.y ? valid : 0, y);
    load8_any(g.w_type, g.w, col, valid, w);
    load8_any(g.post_type, g.post, col, valid, post);
    load8_any(g.gate_type, g.gate, m * g.ld_gate + col, valid, gate);
    kept = kept_of(drop, (uint64_t)(m * ((g.D + 7) / 8) + col / 8));
  }
  __device__ __forceinline__ GradOut at(const GradRow& r, const Drop& drop, int j) const {
    return grad_of<kPost>(r, v[j], dx[j], dr[j], w[j], kept >> j & 1 ? drop.scale : 0.0f, gate[j], post[j], y[j]);
  }
};

template <int kR, int kY, bool kPost>
__global__ void __launch_bounds__(kLong) norm_grad_long_kernel(NormArgs g, NormGradArgs d) {
  constexpr int kN = kPost ? 3 : 1;
  using Sum = RowSum<kLong, kN, kLong, typename GradSums<kPost>::Joint>;
  using At = GradAt<kR, kY, kPost>;
  __shared__ typename Sum::Room room;
  const Drop drop = drop_of(g.y ? g.threshold : 0, g.rng);
  int turn = 0;
  for (int64_t m = blockIdx.x; m < g.M; m += gridDim.x) {
    const float iv = g.stats[m], iy = kPost ? g.stats[g.M + m] : 1.0f;
    float s[kN] = {};
    for (int64_t col = 8 * threadIdx.x; col < g.D; col += 8 * kLong) {
      const At a(g, d, drop, m, col);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        GradSums<kPost>::add(a.v[j], a.dx[j], a.dr[j], a.w[j], iv, a.kept >> j & 1 ? a.gate[j] * drop.scale : 0.0f,
                             a.post[j], a.y[j], s);
    }
    const GradRow row = joined_row<Sum, kPost>(s, room, turn, iv, iy, g.over_d);
    if (threadIdx.x == 0) d.back[m] = row.back;
    for (int64_t col = 8 * threadIdx.x; col < g.D; col += 8 * kLong) {
      const int valid = g.D - col < 8 ? (int)(g.D - col) : 8;
      const At a(g, d, drop, m, col);
      float t[8], dy[8], dg[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const GradOut e = a.at(row, drop, j);
        t[j] = e.t * g.scale;
        dy[j] = e.dy;
        dg[j] = e.dgate;
      }
      if (d.dr_out) store8<kR>(d.dr_out, m * d.ld_dr_out + col, valid, t);
      if (d.dy) store8<kY>(d.dy, m * d.ld_dy + col, valid, dy);
      if (d.dgates) put_gates<kY>(d, m, col, valid, dg);
    }
  }
}

// The sums over the rows blockIdx.x, + gridDim.x, ..  for the columns of blockIdx.y, from `back`.
template <int kR, int kY, bool kPost>
__global__ void __launch_bounds__(kThreads) norm_grad_columns_kernel(NormArgs g, NormGradArgs d) {
  const Drop drop = drop_of(g.y ? g.threshold : 0, g.rng);
  const int64_t col = 8 * ((int64_t)blockIdx.y * kThreads + threadIdx.x);
  if (col >= g.D) return;
  const int valid = g.D - col < 8 ? (int)(g.D - col) : 8;
  float dw[8] = {}, dpost[8] = {}, dgate[8] = {};
  for (int64_t m = blockIdx.x; m < g.M; m += gridDim.x) {
    const GradRow row{g.stats[m], kPost ? g.stats[g.M + m] : 1.0f, d.back[m], 0.0f};
    const GradAt<kR, kY, kPost> a(g, d, drop, m, col);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const GradOut e = a.at(row, drop, j);
      dw[j] = fmaf(a.dx[j], a.v[j] * row.iv, dw[j]);
      dpost[j] = fmaf(e.dz, e.z, dpost[j]);
      dgate[j] += e.dgate;
    }
  }
  const int64_t to = (int64_t)blockIdx.x * g.D + col;
  if (d.dw) store8<FP64EMU_F32>(d.dw, to, valid, dw);
  if (kPost && d.dpost) store8<FP64EMU_F32>(d.dpost, to, valid, dpost);
  if (d.dgate) store8<FP64EMU_F32>(d.dgate, to, valid, dgate);
}

// ---------------------------------------------------------------------------
// Host side.

constexpr int64_t kMaxHeld = 8192;           // elements of a row that stay in registers
bool grad_held(int64_t D) { return D >= 8 && D <= kMaxHeld; }

// Calls fn with the launch shape of rows of D <= kMaxHeld elements.
template <class Fn>
void for_norm(int64_t D, const Fn& fn) {
  if (D <= 128) fn(RowShape<16>{});
  else if (D <= 512) fn(RowShape<64>{});
  else if (D <= 1024) fn(RowShape<128>{});
  else if (D <= 2048) fn(RowShape<256>{});
  else if (D <= 4096) fn(RowShape<512>{});
  else fn(RowShape<1024>{});
}
// The gradient's, and the chunks a thread has.
template <class Fn>
void for_grad(int64_t D, const Fn& fn) {
  if (D <= 4096) for_norm(D, [&](auto s) {
    if constexpr (s.kT < 1024) fn(s, std::integral_constant<int, 1>{});
  });
  else fn(RowShape<512>{}, std::integral_constant<int, 2>{});
}

// Work groups of a forward pass: 2^19 threads, what the card holds twice over, so that a group loads its weights
// once for many rows (8192 x 8192 both ways 173 us; 205 with eight times as many, 180 with half).
int64_t norm_groups(int64_t M, int64_t D) {
  int64_t groups = std::min<int64_t>(M, 512);
  if (D <= kMaxHeld)
    for_norm(D, [&](auto s) { groups = std::min<int64_t>((M + s.kRows - 1) / s.kRows, (1 << 19) / s.kGroup); });
  return groups;
}
// Of a gradient, as many as run at once, since each leaves D floats for each weight: 16 waves a CU where the
// kernel keeps to 128 registers, else 8 (8192 x 4096: 95 us, float32 117; 119 and 136 with four times as many, 103 and
// 181 with half).
int64_t grad_groups(const fp64emu_norm_t* p) {
  if (!grad_held(p->D)) return std::min<int64_t>(p->M, 512);
  int64_t groups = 0;
  for_grad(p->D, [&](auto s, auto chunks) {
    const bool lean = chunks() == 1 && s.kT >= 64 && p->ld_gate == 0 && p->r_dtype != FP64EMU_F32;
    groups = std::min<int64_t>((p->M + s.kRows - 1) / s.kRows, 256 * (lean ? 1024 : 512) / s.kGroup);
  });
  return groups;
}

template <int kR, int kY>
int launch_norm(const NormArgs& g, bool cols, hipStream_t s) {
  const unsigned groups = (unsigned)norm_groups(g.M, g.D);
  if (g.D > kMaxHeld) {
    norm_long_kernel<kR, kY><<<groups, kLong, 0, s>>>(g);
  } else {
    for_norm(g.D, [&](auto shape) {
      using S = decltype(shape);
      norm_rows_kernel<kR, kY, S><<<groups, S::kGroup, 0, s>>>(g);
    });
  }
  if (int st = check_hip(hipGetLastError(), "norm_f8 launch")) return st;
  if (!cols) return FP64EMU_OK;
  norm_tile_kernel<kR, kY><<<(unsigned)((g.M + kBlk - 1) / kBlk * g.blocks), kThreads, 0, s>>>(g);
  return check_hip(hipGetLastError(), "norm_f8 launch");
}

template <int kR, int kY, bool kPost>
int launch_grad(const NormArgs& g, const NormGradArgs& d, unsigned groups, hipStream_t s) {
  if (!grad_held(g.D)) {
    norm_grad_long_kernel<kR, kY, kPost><<<(unsigned)std::min<int64_t>(g.M, 512), kLong, 0, s>>>(g, d);
    if (int st = check_hip(hipGetLastError(), "norm_f8_backward launch")) return st;
    const unsigned strips = (unsigned)((g.D + 8 * kThreads - 1) / (8 * kThreads));
    norm_grad_columns_kernel<kR, kY, kPost><<<dim3(groups, strips), kThreads, 0, s>>>(g, d);
  } else {
    for_grad(g.D, [&](auto shape, auto chunks) {
      using S = decltype(shape);
      constexpr int kC = decltype(chunks)::value;
      if (g.ld_gate) norm_grad_kernel<kR, kY, S, kC, kPost, true><<<groups, S::kGroup, 0, s>>>(g, d);
      else norm_grad_kernel<kR, kY, S, kC, kPost, false><<<groups, S::kGroup, 0, s>>>(g, d);
    });
  }
  return check_hip(hipGetLastError(), "norm_f8_backward launch");
}

int check_norm(const fp64emu_norm_t* p) {
  if (!p) return invalid("norm must not be NULL");
  if (p->M < 0 || p->D < 0) return invalid("shapes must be non-negative");
  if (p->D == 0) return invalid("rows of nothing have no norm");
  if (p->M >= 1ll << 40 || p->D >= 1ll << 27) return invalid("shapes must be below 2^40 rows of 2^27 elements");
  if (!known_dtype(p->r_dtype) || !known_dtype(p->y_dtype) || !known_dtype(p->w_dtype) ||
      !known_dtype(p->post_dtype) || !known_dtype(p->gate_dtype))
    return invalid("dtype must be FP64EMU_F32, FP64EMU_BF16 or FP64EMU_F16");
  if (p->y_dtype != p->r_dtype && p->r_dtype != FP64EMU_F32)
    return invalid("y's dtype must be r's, or r's FP64EMU_F32");
  if (!(p->eps >= 0x1p-126f)) return invalid("eps must be positive and not denormal");
  if (p->drop < 0 || p->drop > 65535) return invalid("drop must be in 0 .. 65535");
  if (p->M == 0) return FP64EMU_OK;                           // (operands that have no address)
  if (!p->y && (p->post || p->gate || p->drop)) return invalid("post, gate and drop need y");
  if (p->drop && !p->rng) return invalid("drop needs rng");
  return FP64EMU_OK;
}

// Of a call with something to do.
int norm_args(const fp64emu_norm_t* p, NormArgs* g) {
  if (!p->r || !p->w) return invalid("null operand pointer");
  if (p->ld_r < p->D || (p->y && p->ld_y < p->D)) return invalid("rows are shorter than D");
  if (p->gate && p->ld_gate != 0 && p->ld_gate < p->D) return invalid("rows of gate are shorter than D");
  *g = NormArgs{};
  g->r = p->r;
  g->y = p->y;
  g->gate = p->gate;
  g->w = p->w;
  g->post = p->post;
  g->rng = p->rng;
  g->M = p->M;
  g->D = p->D;
  g->ld_r = p->ld_r;
  g->ld_y = p->ld_y;
  g->ld_gate = p->gate ? p->ld_gate : 0;
  g->blocks = (p->D + kBlk - 1) / kBlk;
  g->w_type = p->w_dtype;
  g->post_type = p->post_dtype;
  g->gate_type = p->gate_dtype;
  g->threshold = (uint32_t)p->drop;
  g->scale = p->y ? p->scale : 1.0f;         // (v = r without y)
  g->eps = p->eps;
  g->over_d = 1.0f / (float)p->D;
  if (g->ld_gate && p->gate_dtype != p->y_dtype) return invalid("a gate for each row has y's dtype");
  return FP64EMU_OK;
}

// A matrix of M rows as bytes.
struct Place { const void* p; int64_t width, pitch; };

bool same_place(const Place& a, const Place& b, int64_t M) {
  return a.p == b.p && a.width == b.width && (M == 1 || a.pitch == b.pitch);
}
// Whether two of them have a byte in common; of different pitches, whether their ranges have.
bool overlap(Place a, Place b, int64_t M) {
  if (reinterpret_cast<uintptr_t>(b.p) < reinterpret_cast<uintptr_t>(a.p)) std::swap(a, b);
  const uint64_t d = reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p);
  if (d >= (uint64_t)((M - 1) * a.pitch + a.width)) return false;
  if (M == 1 || a.pitch != b.pitch) return true;
  const uint64_t side = d % (uint64_t)a.pitch;                // rows side by side in one buffer do not
  return side < (uint64_t)a.width || (uint64_t)a.pitch - side < (uint64_t)b.width;
}

// out and x may be an operand itself, whose elements a thread reads before it writes them in their place; any other overlap, and,
// with columns, which read the operands again, any at all, gives rows that were overwritten.
int check_places(const fp64emu_norm_t* p, const void* out, int64_t ld_out, const void* x, int64_t ld_x, bool cols) {
  const auto place = [&](const void* q, int dtype, int64_t ld) { return Place{q, p->D * size_of(dtype), ld * size_of(dtype)}; };
  const Place in[] = {place(p->r, p->r_dtype, p->ld_r), place(p->y, p->y_dtype, p->ld_y),
                      place(p->gate && p->ld_gate ? p->gate : nullptr, p->gate_dtype, p->ld_gate)};
  const Place to[] = {place(out, p->r_dtype, ld_out), place(x, p->y_dtype, ld_x)};
  for (const Place& o : to)
    for (const Place& i : in) {
      if (!o.p || !i.p || !overlap(o, i, p->M)) continue;
      if (cols) return invalid("columns need the operands as they were: out must be elsewhere");
      if (!same_place(o, i, p->M)) return invalid("outputs are an operand itself, rows and all, or apart from it");
    }
  if (out && x && overlap(to[0], to[1], p->M)) return invalid("outputs overlap");
  return FP64EMU_OK;
}

// Calls fn with r's and y's types as constants.
template <class Fn>
int for_types(int r, int y, const Fn& fn) {
#define FP64EMU_TYPES(R, Y) \
  if (r == R && y == Y) return fn(std::integral_constant<int, R>{}, std::integral_constant<int, Y>{});
  FP64EMU_TYPES(FP64EMU_F32, FP64EMU_F32)
  FP64EMU_TYPES(FP64EMU_BF16, FP64EMU_BF16)
  FP64EMU_TYPES(FP64EMU_F16, FP64EMU_F16)
  FP64EMU_TYPES(FP64EMU_F32, FP64EMU_BF16)
  FP64EMU_TYPES(FP64EMU_F32, FP64EMU_F16)
#undef FP64EMU_TYPES
  return invalid("dtype");
}

// wide: dgates is float32.
int norm_backward(const fp64emu_norm_t* p, const float* stats, const fp64emu_norm_grad_t* d, int wide, void* workspace,
                  size_t workspace_bytes, fp64emu_stream_t stream) {
  if (int st = check_norm(p)) return st;
  if (!d) return invalid("gradient must not be NULL");
  if (p->M > 0 && !p->y && (d->dy || d->dpost || d->dgate || d->dgates)) return invalid("gradients of what is absent");
  if ((d->dpost && !p->post) || ((d->dgate || d->dgates) && !p->gate)) return invalid("gradients of what is absent");
  if (d->dgate && d->dgates) return invalid("gate's gradient is a row or a matrix");
  if (d->dgates && p->gate_dtype != p->y_dtype) return invalid("a gate for each row has y's dtype");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  float* const sums[kMaxSums] = {d->dw, d->dpost, d->dgate};
  Sums all{};
  int count = 0;
  if (p->M == 0) {                           // sums of nothing
    for (float* to : sums)
      if (to) all.out[count++] = to;
    all.D = p->D;
    return launch_sums(all, count, s);
  }
  if (!d->dx || !stats) return invalid("null operand pointer");
  if (d->ld_dx < p->D || (d->dr && d->ld_dr < p->D) || (d->dr_out && d->ld_dr_out < p->D) || (d->dy && d->ld_dy < p->D) ||
      (d->dgates && d->ld_dgates < p->D))
    return invalid("rows are shorter than D");
  NormArgs g;
  if (int st = norm_args(p, &g)) return st;
  if ((d->dgate && p->ld_gate != 0) || (d->dgates && p->ld_gate == 0))
    return invalid("dgate is of one gate, dgates of a gate for each row");
  const size_t need = fp64emu_norm_f8_backward_workspace(p);
  if (need && (!workspace || workspace_bytes < need))
    return fp64emu_fail(FP64EMU_EWORKSPACE, "workspace too small: see fp64emu_norm_f8_backward_workspace");
  if (need && !multiple(workspace, 4)) return invalid("workspace must be 4-byte aligned");
  g.stats = const_cast<float*>(stats);
  NormGradArgs a{};
  a.dx = d->dx;
  a.dr = d->dr;
  a.ld_dx = d->ld_dx;
  a.ld_dr = d->ld_dr;
  a.dr_out = d->dr_out;
  a.dy = d->dy;
  a.dgates = d->dgates;
  a.wide = wide;
  a.ld_dr_out = d->ld_dr_out;
  a.ld_dy = d->ld_dy;
  a.ld_dgates = d->ld_dgates;
  const int64_t groups = grad_groups(p);
  float* room = static_cast<float*>(workspace);
  float** const to[kMaxSums] = {&a.dw, &a.dpost, &a.dgate};
  for (int i = 0; i < kMaxSums; ++i) {
    *to[i] = sums[i];
    if (!sums[i] || groups == 1) continue;
    *to[i] = room + (int64_t)count * groups * p->D;
    all.part[count] = *to[i];
    all.out[count++] = sums[i];
  }
  if (!grad_held(p->D)) a.back = room + (groups > 1 ? kMaxSums * groups * p->D : 0);
  all.groups = groups;
  all.D = p->D;
  const int st = for_types(p->r_dtype, p->y_dtype, [&](auto r, auto y) {
    return p->post ? launch_grad<decltype(r)::value, decltype(y)::value, true>(g, a, (unsigned)groups, s)
                   : launch_grad<decltype(r)::value, decltype(y)::value, false>(g, a, (unsigned)groups, s);
  });
  return st ? st : launch_sums(all, count, s);
}

}  // namespace

extern "C" {

int fp64emu_norm_f8(const fp64emu_norm_t* p, void* out, int64_t ld_out, void* x, int64_t ld_x, float* stats,
                    const fp64emu_f8_t* rows, const fp64emu_f8_t* cols, fp64emu_stream_t stream) {
  if (int st = check_norm(p)) return st;
  for (const fp64emu_f8_t* f : {rows, cols})
    if (f && (f->fmt != FP64EMU_E4M3 || f->tiles)) return invalid("outputs are e4m3 with scales by rows");
  if (p->M == 0) return FP64EMU_OK;
  if (!out && !x && !rows && !cols && !stats) return invalid("no output asked for");
  if (out && !p->y) return invalid("a new stream needs y");
  if (cols && !stats) return invalid("columns need stats");
  if (cols && x) return invalid("columns come without x in its plain form");
  if ((out && ld_out < p->D) || (x && ld_x < p->D)) return invalid("rows are shorter than D");
  NormArgs g;
  if (int st = norm_args(p, &g)) return st;
  if (int st = out8(rows, p->D, &g.rows)) return st;
  if (int st = out8(cols, p->M, &g.cols)) return st;
  if (int st = check_places(p, out, ld_out, x, ld_x, cols != nullptr)) return st;
  g.out = out;
  g.ld_out = ld_out;
  g.x = x;
  g.ld_x = ld_x;
  g.stats = stats;
  if (cols && (p->M + kBlk - 1) / kBlk > ((1ll << 31) / kThreads) / g.blocks) return invalid("operand too large for one launch");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return for_types(p->r_dtype, p->y_dtype, [&](auto r, auto y) {
    return launch_norm<decltype(r)::value, decltype(y)::value>(g, cols != nullptr, s);
  });
}

size_t fp64emu_norm_f8_backward_workspace(const fp64emu_norm_t* p) {
  if (check_norm(p) || p->M == 0) return 0;
  const int64_t groups = grad_groups(p);
  const size_t parts = groups > 1 ? 4 * (size_t)kMaxSums * (size_t)(groups * p->D) : 0;
  return parts + (grad_held(p->D) ? 0 : 4 * (size_t)p->M);
}

int fp64emu_norm_f8_backward(const fp64emu_norm_t* p, const float* stats, const fp64emu_norm_grad_t* d, void* workspace,
                             size_t workspace_bytes, fp64emu_stream_t stream) {
  return norm_backward(p, stats, d, 0, workspace, workspace_bytes, stream);
}

int fp64emu_norm_f8_backward_wide(const fp64emu_norm_t* p, const float* stats, const fp64emu_norm_grad_t* d, void* workspace,
                                  size_t workspace_bytes, fp64emu_stream_t stream) {
  return norm_backward(p, stats, d, 1, workspace, workspace_bytes, stream);
}

}  // extern "C"
