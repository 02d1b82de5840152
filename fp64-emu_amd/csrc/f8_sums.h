// Sums over the rows of a matrix that a launch's work groups left in parts: deterministic, since
// what a group takes and the order of the parts follow from the sizes alone.
#pragma once
#include "f8_common.h"

namespace {

constexpr int kMaxSums = 3;
struct Sums {
  const float* part[kMaxSums];               // [groups][D] each
  float* out[kMaxSums];                      // [D]
  int64_t groups, D;
};

// 64 columns a work group of sixteen waves, each at parts wave, wave + 16, ..: few columns have
// many parts, which one wave would wait for one after the other.  512 parts of three times 4096: 5 us.
constexpr int kSumWaves = 16;

__global__ void __launch_bounds__(64 * kSumWaves) sum_groups_kernel(Sums g) {
  __shared__ float joint[kSumWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + lane;
  const float* p = g.part[blockIdx.y];
  float s = 0.0f;
  if (col < g.D) {
#pragma unroll 8
    for (int64_t i = wave; i < g.groups; i += kSumWaves) s += p[i * g.D + col];
  }
  joint[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && col < g.D) {
#pragma unroll
    for (int w = 1; w < kSumWaves; ++w) s += joint[w][lane];
    g.out[blockIdx.y][col] = s;
  }
}

[[maybe_unused]] inline int launch_sums(const Sums& g, int count, hipStream_t s) {
  if (count == 0) return FP64EMU_OK;
  sum_groups_kernel<<<dim3((unsigned)((g.D + 63) / 64), (unsigned)count), 64 * kSumWaves, 0, s>>>(g);
  return check_hip(hipGetLastError(), "column sums launch");
}

}  // namespace
