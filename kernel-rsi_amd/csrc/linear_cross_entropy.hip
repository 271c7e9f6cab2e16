// Softmax cross entropy of an output projection's logits, which are never kept, forward and backward, for gfx950.
//   l = x w^T                      x [rows, K], w [V, K] (nn.Linear layout), T = bf16 or fp16; l stays fp32
//   lse_n = log sum_v exp(l_nv),   loss_n = lse_n - l_n,target(n)
//   dl_nv = (exp(l_nv - lse_n) - [v = target(n)]) g_n,   dx = dl w,   dw = dl^T x
// Forward: the products' epilogue reduces each wave's 64 columns of a row to a maximum and a sum of exponentials in
// registers, and keeps the target's logit; a second launch joins a row's pairs, a third adds the losses.
// Backward, in pieces of the vocabulary (512 MB of dl each, or 4096 columns): the products again, whose epilogue
// forms dl, rounded to T; then dw of the piece's rows and the piece's part of dx, which is carried in fp32 from piece to
// piece.
// What dl's rounding takes from the target's entry, the largest of a row, is kept in fp32 per row (its rest) and
// comes back into dx, and into dw's row of the target from the last of the rows that have it (rows of w that many
// targets name average it out). bf16 [2048, 1024], V 32128, 2-norm error of dx: 0.0026 without, 0.0019 with (0.0017
// is the rounding of dx itself).
// dl is held times a power of two that puts the largest |g| at 2^14..2^15: fp16 then keeps its probabilities down to
// 2^-28 in full precision, and the scale comes off exactly where dx and dw are rounded. One power serves all rows, as dw
// adds them: in a row whose weight is 2^-k of the largest fp16 keeps them down to 2^(k - 28) (bf16 everywhere).
//
// What bounds it: the matrix cores (2 rows V K flop forward, 6 backward, 2 of them the logits again). bf16 [8192,
// 4096], V 131072: 6.4 to 6.8 ms of logits by card and run (1370 to 1290 TFLOP/s), backward 20.4 to 20.8 ms (1295 to 1270
// over its three products); the vendor's product of such sizes runs at 1390, 1295 and 1125 TFLOP/s in the three
// orientations. [2048, 1024], V 32128: 131 and 411 us, where 16 stages a tile leave the epilogues a fifth.
#include "chunks.h"
#include "krsi_device.h"
#include "krsi_internal.h"
#include "product_stream.h"

namespace krsi {
namespace {

constexpr int kThreads = 256;
constexpr int kOneBlock = 1024;
// Bytes of dl in the backward, and of the rows' pairs in the forward. Backward at [8192, 1024], V 32128: 1637 us in
// pieces of 128 MB (5), 1500 in pieces of 256 to 1024 (3 to 1); [4099, 2048], V 50257: 2632, 2620 with 256, 2440.
constexpr int64_t kPieceBytes = int64_t(512) << 20;
constexpr int64_t kMinWidth = 4096;  // columns of a piece at least: dx's fp32 sums are read and written once per piece
constexpr int64_t kMaxWidth = 1 << 20;  // columns of a piece: 64 rows of dl stay below 2^31 bytes
constexpr int kMinStages = 8;   // stages of a part of a split sum, at least
constexpr int kMaxSplits = 64;  // parts of a sum

using Large = StreamTile<2, 4, 8, 4>;  // 256 x 256, 8 waves, one workgroup per CU
using Medium = StreamTile<2, 4, 6, 4>;  // 192 x 256, 8 waves: of logits (a TR operand's tile is a power of two wide)
using Small = StreamTile<2, 2, 4, 4>;  // 128 x 128, 4 waves, two per CU

struct Targets {
  const void* p;
  int bytes, V;
  int64_t ignore;
  // In [0, V), or -1: none (ignored, or outside).
  __device__ __forceinline__ int at(int64_t row) const {
    const int64_t t = load_index(p, bytes, row);
    return t >= 0 && t < V && t != ignore ? (int)t : -1;
  }
  __device__ __forceinline__ bool ignored(int64_t row) const { return load_index(p, bytes, row) == ignore; }
};

// ------------------------------------------------------------------ forward
// part [slices][rows]: (maximum, sum of exp(l - maximum)) of a row over the slice's 16 CB columns.
template <int DT, int WM, int WN, int RB, int CB>
__global__ __launch_bounds__(64 * WM * WN, (StreamTile<WM, WN, RB, CB>::kPerCu * WM * WN / 4)) void logits_reduce(
    Operand x, Operand w, int K, Tiles tiles, Targets targets, float2* __restrict__ part,
    float* __restrict__ target_logit) {
  using Tl = StreamTile<WM, WN, RB, CB>;
  __shared__ __attribute__((aligned(512))) uint16_t lds[Tl::kLds];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l16 = lane & 15;
  const int wr = wave / WN, wc = wave % WN;
  const int rows = x.extent, V = w.extent;
  stream_products<DT, false, false, WM, WN, RB, CB>(x, w, K, tiles, lds, [&](const TileAt& t, f32x4(&acc)[RB][CB]) {
    const int col0 = t.n0 + 16 * CB * wc + 4 * g, row0 = t.m0 + 16 * RB * wr + l16;
    const int slice = t.n0 / (16 * CB) + wc;
    // Every step for all rows before the next step: loads, then lane exchanges, overlap (row after row the epilogue
    // took as long as five stages).
    int at[RB];
#pragma unroll
    for (int i = 0; i < RB; ++i) at[i] = targets.at(min(row0 + 16 * i, rows - 1)) - col0;
    auto reduce = [&](auto whole) {  // a tile within the vocabulary, or one that ends past it
      constexpr bool WHOLE = decltype(whole)::value;
      float m[RB], s[RB];
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        m[i] = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < CB; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (!WHOLE && col0 + 16 * j + r >= V) acc[i][j][r] = -__builtin_inff();
            m[i] = fmaxf(m[i], acc[i][j][r]);
          }
      }
#pragma unroll
      for (int i = 0; i < RB; ++i) m[i] = fmaxf(m[i], __shfl_xor(m[i], 16, kWave));
#pragma unroll
      for (int i = 0; i < RB; ++i) m[i] = fmaxf(m[i], __shfl_xor(m[i], 32, kWave));
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const float base = m[i] == -__builtin_inff() ? 0.f : m[i];
        s[i] = 0.f;
#pragma unroll
        for (int j = 0; j < CB; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[i] += __builtin_amdgcn_exp2f((acc[i][j][r] - base) * kLog2e);
      }
#pragma unroll
      for (int i = 0; i < RB; ++i) s[i] += __shfl_xor(s[i], 16, kWave);
#pragma unroll
      for (int i = 0; i < RB; ++i) s[i] += __shfl_xor(s[i], 32, kWave);
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const int row = row0 + 16 * i;
        if (row >= rows) continue;
        if (g == 0) part[(int64_t)slice * rows + row] = float2{m[i], s[i]};
        if ((unsigned)at[i] < 16 * CB && (at[i] & 15) < 4) {
#pragma unroll
          for (int j = 0; j < CB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (at[i] == 16 * j + r) target_logit[row] = acc[i][j][r];
        }
      }
    };
    if (t.n0 + Tl::kCols <= V)
      reduce(std::true_type{});
    else
      reduce(std::false_type{});
  });
}

// lse and loss of each row from its pairs, in a fixed order: 16 rows per workgroup, 64 threads a row, the maximum
// first, then the sums to its base. (With 16 threads a row that joined pair after pair it took 18 us for 2048 rows
// of 502 pairs, a third of the memory's rate at 2048 pairs of 8192 rows.)
constexpr int kJoinRows = 16, kJoinParts = kOneBlock / kJoinRows, kJoinHeld = 8;
__global__ __launch_bounds__(kOneBlock) void join_rows(const float2* __restrict__ part,
                                                       const float* __restrict__ target_logit, Targets targets,
                                                       float* __restrict__ lse, float* __restrict__ loss, int64_t rows,
                                                       int slices) {
  __shared__ float top[kJoinParts][kJoinRows], sum[kJoinParts][kJoinRows];
  const int r = threadIdx.x % kJoinRows, q = threadIdx.x / kJoinRows;
  const int64_t row = (int64_t)blockIdx.x * kJoinRows + r;
  const bool live = row < rows;
  const float2* p = part + (live ? row : 0);
  float m = -__builtin_inff();
  float2 held[kJoinHeld];
#pragma unroll
  for (int k = 0; k < kJoinHeld; ++k) {
    const int at = q + k * kJoinParts;
    held[k] = at < slices ? p[(int64_t)at * rows] : float2{m, 0.f};
  }
#pragma unroll
  for (int k = 0; k < kJoinHeld; ++k) m = fmaxf(m, held[k].x);
#pragma unroll 8
  for (int k = q + kJoinHeld * kJoinParts; k < slices; k += kJoinParts) m = fmaxf(m, p[(int64_t)k * rows].x);
  top[q][r] = m;
  __syncthreads();
  m = top[0][r];
#pragma unroll 8
  for (int k = 1; k < kJoinParts; ++k) m = fmaxf(m, top[k][r]);
  float s = 0.f;
  auto add = [&](float2 a) { s += a.y == 0.f ? 0.f : a.y * __builtin_amdgcn_exp2f((a.x - m) * kLog2e); };
#pragma unroll
  for (int k = 0; k < kJoinHeld; ++k) add(held[k]);
#pragma unroll 8
  for (int k = q + kJoinHeld * kJoinParts; k < slices; k += kJoinParts) add(p[(int64_t)k * rows]);
  sum[q][r] = s;
  __syncthreads();
  if (q != 0 || !live) return;
#pragma unroll 8
  for (int k = 1; k < kJoinParts; ++k) s += sum[k][r];
  const float log_sum = logf(s);
  lse[row] = m + log_sum;
  loss[row] = targets.ignored(row) ? 0.f : targets.at(row) < 0 ? __builtin_nanf("") : (m - target_logit[row]) + log_sum;
}

__device__ __forceinline__ double block_sum(double v, double* s) {
  for (int m = kWave / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  if ((threadIdx.x & (kWave - 1)) == 0) s[threadIdx.x / kWave] = v;
  __syncthreads();
  double t = s[0];
  for (int w = 1; w < kOneBlock / kWave; ++w) t += s[w];
  __syncthreads();
  return t;
}

// total = the losses' sum (over the rows that count, with mean); counted = how many rows are not ignored.
__global__ __launch_bounds__(kOneBlock) void add_losses(const float* __restrict__ loss, Targets targets, int64_t rows,
                                                        bool mean, float* __restrict__ total, float* __restrict__ counted) {
  __shared__ double s[kOneBlock / kWave];
  double sum = 0, n = 0;
  for (int64_t r = threadIdx.x; r < rows; r += kOneBlock) {
    sum += loss[r];
    n += targets.ignored(r) ? 0 : 1;
  }
  sum = block_sum(sum, s);
  n = block_sum(n, s);
  if (threadIdx.x == 0) {
    *counted = (float)n;
    if (total) *total = (float)(mean ? sum / n : sum);
  }
}

// ----------------------------------------------------------------- backward
// What the backward needs of a row, in one load.
struct alignas(16) RowInfo {
  float lse, coef;  // coef 0: no weight
  int target;       // -1: none, or no weight (such a row has no rest and is not the last to name a target)
  int unused;
};

// coef = g_row times 2^k, k such that the largest finite |g| reaches 2^14 .. 2^15; *back = 2^-k. g: the
// loss's gradient for the row (per row, or one for all, over the rows that count with mean); 0 where
// ignored, NaN where the target is outside [0, V). rest and last are cleared. Per row, workgroup 0 finds the
// largest and does all rows; else every workgroup knows it and does its share.
__global__ __launch_bounds__(kOneBlock) void row_weights(const float* __restrict__ dout, bool per_row, bool mean,
                                                         const float* __restrict__ counted, Targets targets,
                                                         int rows, const float* __restrict__ lse,
                                                         RowInfo* __restrict__ info, float* __restrict__ rest,
                                                         int* last, float* __restrict__ back) {
  __shared__ float s[kOneBlock / kWave];
  const int me = blockIdx.x * kOneBlock + threadIdx.x, all = gridDim.x * kOneBlock;
  for (int v = 4 * me; v < targets.V; v += 4 * all)  // the array is padded to whole chunks
    *reinterpret_cast<u32x4*>(last + v) = u32x4{~0u, ~0u, ~0u, ~0u};
  if (per_row && blockIdx.x > 0) return;
  const float one = per_row ? 0.f : *dout * (mean ? 1.f / *counted : 1.f);
  auto weight = [&](int r) {
    if (targets.ignored(r)) return 0.f;
    return targets.at(r) < 0 ? __builtin_nanf("") : per_row ? dout[r] : one;
  };
  auto finite = [](float a) { return a <= 3.4028234663852886e38f ? a : 0.f; };
  float top = finite(fabsf(one));
  if (per_row) {
    for (int r = threadIdx.x; r < rows; r += kOneBlock) top = fmaxf(top, finite(fabsf(weight(r))));
    for (int m = kWave / 2; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, kWave));
    if ((threadIdx.x & (kWave - 1)) == 0) s[threadIdx.x / kWave] = top;
    __syncthreads();
    for (int w = 0; w < kOneBlock / kWave; ++w) top = fmaxf(top, s[w]);
  }
  int k = 0;
  if (top > 0.f) {
    frexpf(top, &k);  // top = f 2^k, f in [1/2, 1)
    k = min(max(15 - k, -126), 126);
  }
  const float scale = ldexpf(1.f, k);
  for (int r = per_row ? threadIdx.x : me; r < rows; r += per_row ? kOneBlock : all) {
    const float c = weight(r) * scale;
    info[r] = RowInfo{lse[r], c, c == 0.f ? -1 : targets.at(r), 0};
    rest[r] = 0.f;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *back = ldexpf(1.f, -k);
}

// dl [rows, ld] of the piece of the vocabulary that starts at v0 (w and its extent are the piece's): zero past it.
// rest[row]: see above; last[v]: the last row whose target is v.
template <int DT, int WM, int WN, int RB, int CB>
__global__ __launch_bounds__(64 * WM * WN, (StreamTile<WM, WN, RB, CB>::kPerCu * WM * WN / 4)) void logits_grad(
    Operand x, Operand w, int K, Tiles tiles, int v0, const RowInfo* __restrict__ info, float* __restrict__ rest,
    int* last, uint16_t* __restrict__ dl, int ld) {
  using Tl = StreamTile<WM, WN, RB, CB>;
  using El = Elem<DT>;
  __shared__ __attribute__((aligned(512))) uint16_t lds[Tl::kLds];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l16 = lane & 15;
  const int wr = wave / WN, wc = wave % WN;
  stream_products<DT, false, false, WM, WN, RB, CB>(x, w, K, tiles, lds, [&](const TileAt& t, f32x4(&acc)[RB][CB]) {
    const int col0 = t.n0 + 16 * CB * wc + 4 * g, row0 = t.m0 + 16 * RB * wr + l16;
    RowInfo of[2];  // of this row and the next
    of[0] = info[min(row0, x.extent - 1)];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const int row = row0 + 16 * i;
      if (i + 1 < RB) of[(i + 1) % 2] = info[min(row + 16, x.extent - 1)];
      if (row >= x.extent) continue;
      const float b = of[i % 2].lse, c = of[i % 2].coef;
      const int at = of[i % 2].target - v0 - col0;
      float d[4 * CB];
#pragma unroll
      for (int j = 0; j < 4 * CB; ++j) d[j] = __builtin_amdgcn_exp2f((acc[i][j / 4][j % 4] - b) * kLog2e) * c;
      if ((unsigned)at < 16 * CB && (at & 15) < 4) {
#pragma unroll
        for (int j = 0; j < 4 * CB; ++j)
          if (at == 16 * (j / 4) + j % 4) {
            d[j] = (__builtin_amdgcn_exp2f((acc[i][j / 4][j % 4] - b) * kLog2e) - 1.f) * c;
            rest[row] = d[j] - El::round(d[j]);
            atomicMax(last + v0 + col0 + at, (int)row);
          }
      }
      if (t.n0 + Tl::kCols > w.extent) {
#pragma unroll
        for (int j = 0; j < 4 * CB; ++j) d[j] = col0 + 16 * (j / 4) + j % 4 < w.extent ? d[j] : 0.f;
      }
      const uint32_t keep = c == 0.f ? 0u : 0xffffffffu;  // a row without weight has no gradient, whatever it holds
#pragma unroll
      for (int j = 0; j < CB; ++j)
        *reinterpret_cast<u32x2*>(dl + (int64_t)row * ld + col0 + 16 * j) =
            u32x2{El::pack2(d[4 * j], d[4 * j + 1]) & keep, El::pack2(d[4 * j + 2], d[4 * j + 3]) & keep};
    }
  });
}

// What comes back into row n of dx: its rest times w[target(n)]; into row v of dw: the rest of row last[v] times
// that row of x. In the units of dl.
struct Rest {
  const float* rest;
  const uint16_t* other;  // w, or x
  const int* last;        // of the piece's vocabulary; NULL: dx
  Targets targets;
  // The row of `other`, -1: nothing, and its factor.
  __device__ __forceinline__ int to(int64_t row) const { return last ? last[row] : targets.at(row); }
  __device__ __forceinline__ float e(int64_t row, int to) const { return rest[last ? max(to, 0) : row]; }
  __device__ __forceinline__ u32x2 chunk(int to, int N, int col) const {
    return *reinterpret_cast<const u32x2*>(other + (int64_t)to * N + col);
  }
  template <int DT>
  static __device__ __forceinline__ f32x4 times(u32x2 raw, float e) {
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = e * Elem<DT>::load((uint16_t)(raw[r / 2] >> (16 * (r % 2))));
    return v;
  }
};

// out [M, N] = a b and the rest, times *back, rounded to T. PART: the sum's parts into part [splits][M][N], added to
// what it holds where `add`.
template <int DT, bool TRA, bool PART, int WM, int WN, int RB, int CB>
__global__ __launch_bounds__(64 * WM * WN, (StreamTile<WM, WN, RB, CB>::kPerCu * WM * WN / 4)) void grad_product(
    Operand a, Operand b, int sum, Tiles tiles, int M, int N, const float* __restrict__ back, Rest rest,
    uint16_t* __restrict__ out, float* __restrict__ part, bool add) {
  using Tl = StreamTile<WM, WN, RB, CB>;
  using El = Elem<DT>;
  __shared__ __attribute__((aligned(512))) uint16_t lds[Tl::kLds];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l16 = lane & 15;
  const int wr = wave / WN, wc = wave % WN;
  stream_products<DT, TRA, true, WM, WN, RB, CB>(a, b, sum, tiles, lds, [&](const TileAt& t, f32x4(&acc)[RB][CB]) {
    const int col0 = t.n0 + 16 * CB * wc + 4 * g, row0 = t.m0 + 16 * RB * wr + l16;
    if constexpr (PART) {
      float* const base = part + ((int64_t)t.split * M + row0) * N + col0;
      // Two rows' chunks requested before the first is added: chunk after chunk waits for memory 32 times.
#pragma unroll
      for (int i = 0; i < RB; i += 2) {
        f32x4 old[2][CB];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < CB; ++j) {
            old[k][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (add && row0 + 16 * (i + k) < M && col0 + 16 * j < N)
              old[k][j] = *reinterpret_cast<const f32x4*>(base + (int64_t)16 * (i + k) * N + 16 * j);
          }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < CB; ++j)
            if (row0 + 16 * (i + k) < M && col0 + 16 * j < N)
              *reinterpret_cast<f32x4*>(base + (int64_t)16 * (i + k) * N + 16 * j) = old[k][j] + acc[i + k][j];
      }
    } else {
      const float scale = *back;
      const bool aligned = ((uintptr_t)out & 7) == 0;
      int to[RB];
      float e[RB];
#pragma unroll
      for (int i = 0; i < RB; ++i) to[i] = rest.to(min(row0 + 16 * i, M - 1));
#pragma unroll
      for (int i = 0; i < RB; ++i) e[i] = rest.e(min(row0 + 16 * i, M - 1), to[i]);
      // Two rows' chunks requested together, by all lanes (a lane without one masks another row's to zeros): with a
      // branch per row, which waits for each row's chunks, the launch takes 12 % longer.
#pragma unroll
      for (int i0 = 0; i0 < RB; i0 += 2) {
        u32x2 raw[2][CB];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t has = lane_mask(to[i0 + k] >= 0);
#pragma unroll
          for (int j = 0; j < CB; ++j) raw[k][j] = rest.chunk(max(to[i0 + k], 0), N, min(col0 + 16 * j, N - 4)) & has;
          e[i0 + k] = __uint_as_float(__float_as_uint(e[i0 + k]) & has);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int i = i0 + k, row = row0 + 16 * i;
#pragma unroll
          for (int j = 0; j < CB; ++j) {
            const int col = col0 + 16 * j;
            const f32x4 v = (acc[i][j] + Rest::times<DT>(raw[k][j], e[i])) * scale;
            if (row >= M || col >= N) continue;
            uint16_t* p = out + (int64_t)row * N + col;
            if (aligned) {
              *reinterpret_cast<u32x2*>(p) = u32x2{El::pack2(v[0], v[1]), El::pack2(v[2], v[3])};
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r) p[r] = El::store(v[r]);
            }
          }
        }
      }
    }
  });
}

// out [M, N] = T(*back times the parts' sum, in order, and the rest); zero where there is none. blockIdx.x: row.
template <int DT>
__global__ __launch_bounds__(kThreads) void add_parts(const float* __restrict__ part, int splits, int64_t M, int N,
                                                      const float* __restrict__ back, Rest rest,
                                                      uint16_t* __restrict__ out) {
  const int col = (blockIdx.y * kThreads + threadIdx.x) * 4;
  if (col >= N) return;
  const int64_t row = blockIdx.x, i = row * N + col;
  f32x4 s{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8  // one part after another waits for memory each time: 18 us for a row of 64 parts, here 5
  for (int k = 0; k < splits; ++k) s += *reinterpret_cast<const f32x4*>(part + k * M * N + i);
  if (splits) {
    const int to = rest.to(row);
    if (to >= 0) s += Rest::times<DT>(rest.chunk(to, N, col), rest.e(row, to));
    s *= *back;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) out[i + r] = Elem<DT>::store(s[r]);
}

// -------------------------------------------------------------------- plans
template <typename Tl>
Tiles tiles_of(int64_t M, int64_t N, int64_t sum, int splits) {
  Tiles t{};
  t.nrb = (int)ceil_div(M, Tl::kRows);
  t.ncb = (int)ceil_div(N, Tl::kCols);
  t.stages = (int)ceil_div(sum, kStage);
  t.per = (int)ceil_div(t.stages, splits);
  t.splits = (int)ceil_div(t.stages, t.per);
  t.total = (int)((int64_t)t.nrb * t.ncb * t.splits);
  return t;
}
struct Plan {
  int tile;  // 0: Large, 1: Medium, 2: Small
  Tiles tiles;
};
// The tile, and (not of logits, which are reduced whole) the parts of the sum, by an estimate in stages of the large
// tile (1.6 us on a CU at full rate): rounds of workgroups times the stages of each and its epilogue (4, or 8 where it
// writes fp32 parts, which all CUs do at once), and the parts' addition (4 M N bytes per part at 5 TB/s). The medium
// tile has three quarters of the work and takes 1.15 times as long for the same (bf16 [300, 1152], V 32128: 29 us, the
// large one 36; [4099, 2048], V 50257: 755, 736); the small one has a quarter, two workgroups per CU share it, and it
// takes 1.2 times as long for the same work (geglu_linear's measurement of the two).
Plan plan_product(int64_t M, int64_t N, int64_t sum, bool logits) {
  Plan best{};
  double least = 0;
  const int64_t stages = ceil_div(sum, kStage), most = logits ? 1 : stages / kMinStages;
  for (int s = 1; s == 1 || (s <= most && s <= kMaxSplits); ++s) {
    for (int tile = 0; tile < 3; ++tile) {
      if (tile == 1 && !logits) continue;
      const Tiles t = tile == 0   ? tiles_of<Large>(M, N, sum, s)
                      : tile == 1 ? tiles_of<Medium>(M, N, sum, s)
                                  : tiles_of<Small>(M, N, sum, s);
      const double each = (t.per + (s > 1 ? 8 : 4)) * (tile == 0 ? 1.0 : tile == 1 ? 0.86 : 0.6);
      const double cost = (double)ceil_div(t.total, 256 * (tile == 2 ? Small::kPerCu : 1)) * each +
                          (s > 1 ? 5e-7 * (double)M * (double)N * s : 0);
      if (best.tiles.total == 0 || cost < least) {
        best = Plan{tile, t};
        least = cost;
      }
    }
  }
  return best;
}

// f(tile) with the plan's tile.
template <int WM_, int WN_, int RB_, int CB_>
struct Shape {
  static constexpr int WM = WM_, WN = WN_, RB = RB_, CB = CB_;
  using Tl = StreamTile<WM, WN, RB, CB>;
};
template <typename F>
void with_grad_tile(const Plan& p, F&& f) {
  if (p.tile == 0)
    f(Shape<2, 4, 8, 4>{});
  else
    f(Shape<2, 2, 4, 4>{});
}
template <typename F>
void with_logits_tile(const Plan& p, F&& f) {
  if (p.tile == 1)
    f(Shape<2, 4, 6, 4>{});
  else
    with_grad_tile(p, f);
}
int rows_of(const Plan& p) { return p.tile == 0 ? Large::kRows : p.tile == 1 ? Medium::kRows : Small::kRows; }
int cols_of(const Plan& p) { return p.tile == 2 ? Small::kCols : Large::kCols; }

struct Forward {
  int chunk;  // rows whose pairs are kept at a time
  size_t part, target_logit, loss, bytes;
};
Forward plan_forward(int64_t rows, int K, int V) {
  Forward f{};
  const int64_t pairs = ceil_div(V, 256) * 4, fit = kPieceBytes / (pairs * (int64_t)sizeof(float2)) / 256 * 256;
  f.chunk = (int)(rows < 2048 || rows < fit ? rows : fit < 2048 ? 2048 : fit);
  size_t at = 0;
  auto take = [&](size_t b) {
    const size_t here = at;
    at += align256(b);
    return here;
  };
  f.part = take((size_t)pairs * f.chunk * sizeof(float2));
  f.target_logit = take((size_t)f.chunk * 4);
  f.loss = take((size_t)rows * 4);
  f.bytes = at;
  return f;
}

struct Backward {
  int width, pieces;  // columns of dl, a multiple of 256
  Plan dx, dw;        // of a whole piece
  size_t info, rest, last, back, dl, dx_part, dw_part, bytes;
};
Backward plan_backward(int64_t rows, int K, int V) {
  Backward b{};
  const int64_t cols = ceil_div(V, 256) * 256, fit = kPieceBytes / (rows * 2) / 256 * 256;
  b.pieces = (int)ceil_div(cols, fit < kMinWidth ? kMinWidth : fit < kMaxWidth ? fit : kMaxWidth);
  b.width = (int)(ceil_div(ceil_div(V, b.pieces), 256) * 256);
  b.pieces = (int)ceil_div(V, b.width);
  const int whole = V < b.width ? V : b.width;
  b.dx = plan_product(rows, K, whole, false);
  b.dw = plan_product(whole, K, rows, false);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t here = at;
    at += align256(n);
    return here;
  };
  b.info = take((size_t)rows * sizeof(RowInfo));
  b.rest = take((size_t)rows * 4);
  b.last = take((size_t)V * 4);
  b.back = take(4);
  b.dl = take((size_t)rows * b.width * 2);
  b.dx_part = take(b.dx.tiles.splits > 1 || b.pieces > 1 ? (size_t)b.dx.tiles.splits * rows * K * 4 : 0);
  b.dw_part = take(b.dw.tiles.splits > 1 ? (size_t)b.dw.tiles.splits * whole * K * 4 : 0);
  b.bytes = at;
  return b;
}

int check(int64_t rows, int32_t k, int32_t v, int32_t target_bytes, int32_t reduction, int32_t dtype) {
  if (dtype != kBf16 && dtype != kF16) return KRSI_ERR_UNSUPPORTED;
  if (target_bytes != 4 && target_bytes != 8) return KRSI_ERR_UNSUPPORTED;
  if (reduction < 0 || reduction > 2) return KRSI_ERR_UNSUPPORTED;
  if (rows < 0 || k <= 0 || v <= 0) return KRSI_ERR_BAD_SHAPE;
  // Whole stages of K; byte offsets of a staged tile below 2^31; grids of less than 2^32 threads.
  if (k % kStage != 0 || k > (1 << 20) || v > (1 << 23) || rows > (1 << 23)) return KRSI_ERR_UNSUPPORTED;
  if (ceil_div(rows, 128) * ceil_div(v, 128) > (1 << 23) || ceil_div(rows, 128) * ceil_div(k, 128) > (1 << 18) ||
      ceil_div(v, 128) * ceil_div(k, 128) > (1 << 23))
    return KRSI_ERR_UNSUPPORTED;
  return KRSI_OK;
}

template <int DT>
int forward(const Operand& x, const Operand& w, int K, const Targets& t, float* loss, float* stats, char* ws,
            int reduction, hipStream_t st) {
  const int rows = x.extent;
  const Forward f = plan_forward(rows, K, w.extent);
  float2* part = (float2*)(ws + f.part);
  float* target_logit = (float*)(ws + f.target_logit);
  float* row_loss = reduction == 0 ? loss : (float*)(ws + f.loss);
  for (int r0 = 0; r0 < rows; r0 += f.chunk) {
    const Operand xr{x.p + (int64_t)r0 * K, K, rows - r0 < f.chunk ? rows - r0 : f.chunk};
    const Targets tr{(const char*)t.p + (int64_t)r0 * t.bytes, t.bytes, t.V, t.ignore};
    const Plan pl = plan_product(xr.extent, w.extent, K, true);
    with_logits_tile(pl, [&](auto s) {
      using S = decltype(s);
      hipLaunchKernelGGL((logits_reduce<DT, S::WM, S::WN, S::RB, S::CB>), dim3(stream_grid<typename S::Tl>(pl.tiles)),
                         dim3(S::Tl::kThreads), 0, st, xr, w, K, pl.tiles, tr, part, target_logit);
    });
    hipLaunchKernelGGL(join_rows, dim3((unsigned)ceil_div(xr.extent, kJoinRows)), dim3(kOneBlock), 0, st,
                       (const float2*)part, (const float*)target_logit, tr, stats + r0, row_loss + r0,
                       (int64_t)xr.extent, pl.tiles.ncb * cols_of(pl) / 64);
  }
  if (reduction != 0)
    hipLaunchKernelGGL(add_losses, dim3(1), dim3(kOneBlock), 0, st, (const float*)row_loss, t, rows, reduction == 1, loss,
                       stats + rows);
  return launch_status();
}

template <int DT, bool TRA>
void launch_product(const Plan& pl, const Operand& a, const Operand& b, int sum, int M, int N, const float* back,
                    const Rest& rest, uint16_t* out, float* part, bool add, hipStream_t st) {
  auto launch = [&](auto s, auto in_parts) {
    using S = decltype(s);
    hipLaunchKernelGGL((grad_product<DT, TRA, decltype(in_parts)::value, S::WM, S::WN, S::RB, S::CB>),
                       dim3(stream_grid<typename S::Tl>(pl.tiles)), dim3(S::Tl::kThreads), 0, st, a, b, sum, pl.tiles, M, N,
                       back, rest, out, part, add);
  };
  with_grad_tile(pl, [&](auto s) {
    if (part)
      launch(s, std::true_type{});
    else
      launch(s, std::false_type{});
  });
}

template <int DT>
int backward(const float* dout, const Operand& x, const Operand& w, int K, const Targets& t, const float* stats,
             uint16_t* dx, uint16_t* dw, char* ws, int reduction, hipStream_t st) {
  const int rows = x.extent, V = w.extent;
  const Backward b = plan_backward(rows, K, V);
  RowInfo* info = (RowInfo*)(ws + b.info);
  float *rest = (float*)(ws + b.rest), *back = (float*)(ws + b.back);
  int* last = (int*)(ws + b.last);
  const Rest to_dx{rest, w.p, nullptr, t};
  uint16_t* dl = (uint16_t*)(ws + b.dl);
  hipLaunchKernelGGL(row_weights, dim3((unsigned)ceil_div(rows + V / 4, 4 * kOneBlock)), dim3(kOneBlock), 0, st, dout,
                     reduction == 0, reduction == 1, stats + rows, t, rows, stats, info, rest, last, back);
  const bool dx_parts = b.dx.tiles.splits > 1 || b.pieces > 1;
  float* dx_part = dx_parts ? (float*)(ws + b.dx_part) : nullptr;
  for (int p = 0; p < b.pieces; ++p) {
    const int v0 = p * b.width, valid = V - v0 < b.width ? V - v0 : b.width;
    const Operand piece{w.p + (int64_t)v0 * K, K, valid};
    const Plan lg = plan_product(rows, b.width, K, true);
    with_logits_tile(lg, [&](auto s) {
      using S = decltype(s);
      hipLaunchKernelGGL((logits_grad<DT, S::WM, S::WN, S::RB, S::CB>), dim3(stream_grid<typename S::Tl>(lg.tiles)),
                         dim3(S::Tl::kThreads), 0, st, x, piece, K, lg.tiles, v0, (const RowInfo*)info, rest, last, dl,
                         b.width);
    });
    if (dx) {
      // The last piece may be shorter: fewer parts, added to those of the pieces before.
      Plan pl = b.dx;
      pl.tiles.stages = (int)ceil_div(valid, kStage);
      pl.tiles.per = pl.tiles.per < pl.tiles.stages ? pl.tiles.per : pl.tiles.stages;
      pl.tiles.splits = (int)ceil_div(pl.tiles.stages, pl.tiles.per);
      pl.tiles.total = pl.tiles.nrb * pl.tiles.ncb * pl.tiles.splits;
      launch_product<DT, false>(pl, Operand{dl, b.width, rows}, Operand{piece.p, K, K}, valid, rows, K, back, to_dx, dx,
                                dx_part, p > 0, st);
    }
    if (dw) {
      Plan pl = b.dw;
      pl.tiles.nrb = (int)ceil_div(valid, rows_of(pl));
      pl.tiles.total = pl.tiles.nrb * pl.tiles.ncb * pl.tiles.splits;
      const bool parts = pl.tiles.splits > 1;
      float* dw_part = parts ? (float*)(ws + b.dw_part) : nullptr;
      uint16_t* out = dw + (int64_t)v0 * K;
      const Rest to_dw{rest, x.p, last + v0, t};
      launch_product<DT, true>(pl, Operand{dl, b.width, b.width}, Operand{x.p, K, K}, rows, valid, K, back, to_dw, out,
                               dw_part, false, st);
      if (parts)
        hipLaunchKernelGGL((add_parts<DT>), dim3((unsigned)valid, (unsigned)ceil_div(K, 4 * kThreads)), dim3(kThreads), 0,
                           st, (const float*)dw_part, pl.tiles.splits, (int64_t)valid, K, (const float*)back, to_dw, out);
    }
  }
  if (dx && dx_parts)
    hipLaunchKernelGGL((add_parts<DT>), dim3((unsigned)rows, (unsigned)ceil_div(K, 4 * kThreads)), dim3(kThreads), 0, st,
                       (const float*)dx_part, b.dx.tiles.splits, rows, K, (const float*)back, to_dx, dx);
  return launch_status();
}

// No rows: the loss of none is 0, its mean NaN; dw is zero.
__global__ void loss_of_none(float* loss, float* counted, bool mean) {
  *loss = mean ? __builtin_nanf("") : 0.f;
  *counted = 0.f;
}

}  // namespace
}  // namespace krsi

extern "C" {

size_t krsi_linear_cross_entropy_fwd_workspace_bytes(int64_t rows, int32_t k, int32_t v) {
  using namespace krsi;
  return rows > 0 && check(rows, k, v, 8, 0, kBf16) == KRSI_OK ? plan_forward(rows, k, v).bytes : 0;
}

size_t krsi_linear_cross_entropy_bwd_workspace_bytes(int64_t rows, int32_t k, int32_t v) {
  using namespace krsi;
  return rows > 0 && check(rows, k, v, 8, 0, kBf16) == KRSI_OK ? plan_backward(rows, k, v).bytes : 0;
}

int krsi_linear_cross_entropy_fwd(const void* x, const void* w, const void* targets, int32_t target_bytes, float* loss,
                                  float* stats, void* workspace, size_t workspace_bytes, int64_t rows, int32_t k,
                                  int32_t v, int64_t ignore_index, int32_t reduction, int32_t dtype, void* stream) {
  using namespace krsi;
  const int rc = check(rows, k, v, target_bytes, reduction, dtype);
  if (rc != KRSI_OK) return rc;
  if (rows == 0) {
    if (reduction == 0) return KRSI_OK;
    if (!loss || !stats) return KRSI_ERR_NULL_POINTER;
    hipLaunchKernelGGL(loss_of_none, dim3(1), dim3(1), 0, as_stream(stream), loss, stats, reduction == 1);
    return launch_status();
  }
  if (!x || !w || !targets || !loss || !stats) return KRSI_ERR_NULL_POINTER;
  if (!aligned16(x) || !aligned16(w)) return KRSI_ERR_MISALIGNED;
  if (!workspace || workspace_bytes < krsi_linear_cross_entropy_fwd_workspace_bytes(rows, k, v))
    return KRSI_ERR_WORKSPACE;
  if (!aligned16(workspace)) return KRSI_ERR_MISALIGNED;
  const Operand xo{(const uint16_t*)x, k, (int)rows}, wo{(const uint16_t*)w, k, v};
  const Targets t{targets, target_bytes, v, ignore_index};
  return dtype == kF16 ? forward<kF16>(xo, wo, k, t, loss, stats, (char*)workspace, reduction, as_stream(stream))
                       : forward<kBf16>(xo, wo, k, t, loss, stats, (char*)workspace, reduction, as_stream(stream));
}

int krsi_linear_cross_entropy_bwd(const float* dout, const void* x, const void* w, const void* targets,
                                  int32_t target_bytes, const float* stats, void* dx, void* dw, void* workspace,
                                  size_t workspace_bytes, int64_t rows, int32_t k, int32_t v, int64_t ignore_index,
                                  int32_t reduction, int32_t dtype, void* stream) {
  using namespace krsi;
  const int rc = check(rows, k, v, target_bytes, reduction, dtype);
  if (rc != KRSI_OK) return rc;
  hipStream_t st = as_stream(stream);
  if (rows == 0) {
    if (!dw) return KRSI_OK;
    hipLaunchKernelGGL((add_parts<kBf16>), dim3((unsigned)v, (unsigned)ceil_div(k, 4 * kThreads)), dim3(kThreads), 0, st,
                       (const float*)nullptr, 0, (int64_t)v, (int)k, (const float*)nullptr, Rest{}, (uint16_t*)dw);
    return launch_status();
  }
  if (!dout || !x || !w || !targets || !stats || (!dx && !dw)) return KRSI_ERR_NULL_POINTER;
  if (!aligned16(x) || !aligned16(w)) return KRSI_ERR_MISALIGNED;
  if (!workspace || workspace_bytes < krsi_linear_cross_entropy_bwd_workspace_bytes(rows, k, v))
    return KRSI_ERR_WORKSPACE;
  if (!aligned16(workspace)) return KRSI_ERR_MISALIGNED;
  const Operand xo{(const uint16_t*)x, k, (int)rows}, wo{(const uint16_t*)w, k, v};
  const Targets t{targets, target_bytes, v, ignore_index};
  return dtype == kF16 ? backward<kF16>(dout, xo, wo, k, t, stats, (uint16_t*)dx, (uint16_t*)dw, (char*)workspace,
                                        reduction, st)
                       : backward<kBf16>(dout, xo, wo, k, t, stats, (uint16_t*)dx, (uint16_t*)dw, (char*)workspace,
                                         reduction, st);
}

}  // extern "C"
