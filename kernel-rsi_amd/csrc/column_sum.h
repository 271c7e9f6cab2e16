// Column sums of fp32 partial rows: the last step of the norms' weight gradients.
#pragma once

#include "krsi_device.h"

namespace krsi {

constexpr int kColsumWaves = 16;       // waves per column-sum workgroup (64 columns each)

// dw = column sums of the [R, n] fp32 partial rows (R <= 512), in fixed order, in one launch.
// Block = 64 columns (lane = column) and 16 waves: wave w adds rows w, w + 16, ... in order,
// then wave 0 adds the 16 wave sums in wave order and writes dtype DT. Each wave has at most
// 32 rows, all of whose loads it can have in flight.
template <int DT>
__global__ __launch_bounds__(kColsumWaves * kWave) void colsum(const float* __restrict__ in, int64_t R,
                                                               int n, typename Elem<DT>::T* __restrict__ out) {
  __shared__ float s[kColsumWaves][kWave];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x / kWave;
  const int col = blockIdx.x * kWave + lane;
  float acc = 0.f;
  if (col < n) {
#pragma unroll 8
    for (int64_t r = wave; r < R; r += kColsumWaves) acc += in[r * n + col];
  }
  s[wave][lane] = acc;
  __syncthreads();
  if (wave == 0 && col < n) {
    float t = s[0][lane];
#pragma unroll
    for (int w = 1; w < kColsumWaves; ++w) t += s[w][lane];
    out[col] = Elem<DT>::store(t);
  }
}

}  // namespace krsi
