// The addition of a layer's output to the residual stream with the RMS norm of the sum, forward and backward, the
// norm's output in the activations' type or in 8 bits with a scale per row; and rows brought to 8 bits alone.
//   r = T(x + residual)                                   the stream that goes on, rounded once
//   rstd = 1 / sqrt(sum(r^2) / n + eps)                   fp32, kept per row for the backward
//   y = T(w * r * rstd)                                   in fp32, rounded once (krsi_rmsnorm_fwd rounds r * rstd as well, as
//                                                         the formula that it stands in for does: 1.4 times the error)
//   8 bits: z = w * r * rstd in fp32; scale = max(max|z| / 448, 2^-120); q = e4m3(z / scale)
// Backward, of dy and dr (the gradients of y and r): one tensor, the gradient of x and of the residual alike,
//   d = T(dr + rstd * (dn - r * rstd * sum(dn * r * rstd) / n)),  dn = dy * w
//   dw = T(sum over rows of dy * r * rstd)                fp32, per block, then a fixed-order column sum
// 448 is e4m3's largest value. The largest |z| is found as an unsigned integer, in whose order infinity and NaN come
// last: a row that holds one has the scale infinity or NaN, and reads back as NaN throughout.
//
// Bound by HBM: each row is read once, lives in registers in 16-byte chunks and is written once, by WPR waves with VPT
// chunks per lane. The backward is persistent and keeps its share of dw in registers, as RMSNorm's, and w (in LDS for fp32 rows
// of more than 8192 columns). bf16 [32768, 4096]: forward 181 us (5.9 TB/s), backward 171 (6.3), dw's sums 5. fp16
// [8191, 8192] in 8 bits: 72 us (6.5 TB/s). fp32 [2042, 1001]: 7.5, 8.5, 3.8. bf16 [32, 4096] in 8 bits: 3.6 (a launch's
// latency).
#include "chunks.h"
#include "column_sum.h"
#include "krsi_device.h"
#include "krsi_internal.h"

#include <initializer_list>

namespace krsi {
namespace {

constexpr int kBwdMaxBlocks = 512;  // persistent grid of the backward, and the most rows of partial sums
constexpr int kMaxRow = 16384;

// What a row pass does.
constexpr int kAdd = 1, kNorm = 2, k8bit = 4;

constexpr int threads_of(int wpr) { return wpr > 4 ? wpr * kWave : 4 * kWave; }

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m, kWave));
  return v;
}

// The sum (or maximum) of v over the WPR waves of a row; every wave of the workgroup calls it. slots: one per wave.
template <int WPR, typename V, typename Wave, typename Join>
__device__ __forceinline__ V row_reduce(V v, V* slots, Wave&& wave_reduce, Join&& join) {
  v = wave_reduce(v);
  if constexpr (WPR > 1) {
    const int wave = threadIdx.x / kWave, first = wave / WPR * WPR;
    if ((threadIdx.x & (kWave - 1)) == 0) slots[wave] = v;
    __syncthreads();
    v = slots[first];
#pragma unroll
    for (int i = 1; i < WPR; ++i) v = join(v, slots[first + i]);
  }
  return v;
}

// The scale of a row whose largest magnitude has the bits `top`. The maximum is of integers, so NaN stays.
__device__ __forceinline__ float scale_of(uint32_t top) {
  return __uint_as_float(max(__float_as_uint(__uint_as_float(top) * (1.0f / 448.0f)), 0x03800000u));  // 2^-120
}

// E values as e4m3 codes at p, of any alignment.
template <int E>
__device__ __forceinline__ void store_codes(uint8_t* p, const float* f, float inv) {
  uint32_t c[E / 4];
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i] * inv, f[4 * i + 1] * inv, 0, false);
    c[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2] * inv, f[4 * i + 3] * inv, v, true);
  }
  __builtin_memcpy(p, c, sizeof(c));
}
__device__ __forceinline__ uint8_t code_of(float f) {
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(f, 0.f, 0, false);
}

// ------------------------------------------------------------------- rows
template <int DT, int WPR, int VPT, bool RAGGED, int KIND>
__global__ __launch_bounds__(threads_of(WPR)) void row_pass(
    const typename Elem<DT>::T* __restrict__ x, const typename Elem<DT>::T* __restrict__ residual,
    const typename Elem<DT>::T* __restrict__ w, void* __restrict__ y, typename Elem<DT>::T* __restrict__ r,
    float* __restrict__ stat, int64_t rows, int n, float eps) {
  using El = Elem<DT>;
  constexpr int E = El::E, RPB = threads_of(WPR) / kWave / WPR, GT = WPR * kWave;
  __shared__ float sums[threads_of(WPR) / kWave];
  __shared__ uint32_t tops[threads_of(WPR) / kWave];
  const int grp = threadIdx.x / GT, gtid = threadIdx.x - grp * GT;
  const int64_t row = (int64_t)blockIdx.x * RPB + grp;
  const bool live = row < rows;
  const int64_t base = (live ? row : 0) * (int64_t)n;
  const int nch = RAGGED ? (n + E - 1) / E : n / E;

  u32x4 v[VPT], wv[VPT];
  {
    u32x4 a[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = gtid + k * GT;
      const bool ok = live && c < nch;
      v[k] = ok ? stream_chunk<RAGGED>(chunk_at<RAGGED, E>(x + base, c, n)) : u32x4{0u, 0u, 0u, 0u};
      if constexpr (KIND & kAdd)
        a[k] = ok ? stream_chunk<RAGGED>(chunk_at<RAGGED, E>(residual + base, c, n)) : u32x4{0u, 0u, 0u, 0u};
    }
    if constexpr (KIND & kNorm) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = gtid + k * GT;
        wv[k] = c < nch ? load_chunk<RAGGED>(chunk_at<RAGGED, E>(w, c, n)) : u32x4{0u, 0u, 0u, 0u};
      }
    }
    if constexpr (KIND & kAdd) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = gtid + k * GT;
        float f[E], g[E];
        El::unpack(v[k], f);
        El::unpack(a[k], g);
#pragma unroll
        for (int j = 0; j < E; ++j) f[j] += g[j];
        v[k] = El::pack(f);
        if (live && c < nch) store_chunk<RAGGED>(chunk_at<RAGGED, E>(r + base, c, n), v[k]);
      }
    }
  }
  float rstd = 1.f;
  if constexpr (KIND & kNorm) {
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      float f[E];
      El::unpack(v[k], f);
      const int dup = chunk_shared<RAGGED, E>(gtid + k * GT, n);
#pragma unroll
      for (int j = 0; j < E; ++j) ss += RAGGED && j < dup ? 0.f : f[j] * f[j];
    }
    ss = row_reduce<WPR>(ss, sums, wave_sum, [](float a, float b) { return a + b; });
    rstd = 1.0f / __fsqrt_rn(ss / (float)n + eps);
  }
  if constexpr (KIND & k8bit) {
    float z[VPT][E];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      El::unpack(v[k], z[k]);
      if constexpr (KIND & kNorm) {
        float wf[E];
        El::unpack(wv[k], wf);
#pragma unroll
        for (int j = 0; j < E; ++j) z[k][j] = wf[j] * (z[k][j] * rstd);
      }
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (gtid + k * GT < nch) top = max(top, __float_as_uint(z[k][j]) & 0x7fffffffu);
    }
    top = row_reduce<WPR>(top, tops, wave_max, [](uint32_t a, uint32_t b) { return max(a, b); });
    if (!live) return;
    const float scale = scale_of(top), inv = 1.0f / scale;
    if (gtid == 0) stat[row] = scale;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = gtid + k * GT;
      if (c < nch) store_codes<E>((uint8_t*)y + base + chunk_col<RAGGED, E>(c, n), z[k], inv);
    }
  } else {
    if (!live) return;
    if (gtid == 0 && stat) stat[row] = rstd;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = gtid + k * GT;
      if (c < nch) {
        float f[E], wf[E];
        El::unpack(v[k], f);
        El::unpack(wv[k], wf);
#pragma unroll
        for (int j = 0; j < E; ++j) f[j] = wf[j] * (f[j] * rstd);
        const u32x4 ov = El::pack(f);
        store_chunk<RAGGED>(chunk_at<RAGGED, E>((typename El::T*)y + base, c, n), ov);
      }
    }
  }
}

// One wave per row, element by element: rows that no chunk fits, and (8 bits alone) rows longer than the registers hold.
template <int DT, int KIND>
__global__ __launch_bounds__(4 * kWave) void row_scalar(
    const typename Elem<DT>::T* __restrict__ x, const typename Elem<DT>::T* __restrict__ residual,
    const typename Elem<DT>::T* __restrict__ w, void* __restrict__ y, typename Elem<DT>::T* __restrict__ r,
    float* __restrict__ stat, int64_t rows, int n, float eps) {
  using El = Elem<DT>;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  if (row >= rows) return;
  const int64_t base = row * (int64_t)n;
  // The row's value at c, rounded as r is; the same in each pass.
  auto value = [&](int c) {
    const float f = El::load(x[base + c]);
    return KIND & kAdd ? El::round(f + El::load(residual[base + c])) : f;
  };
  float ss = 0.f;
  if constexpr ((KIND & kNorm) != 0) {
    for (int c = lane; c < n; c += kWave) {
      const float f = value(c);
      if constexpr ((KIND & kAdd) != 0) r[base + c] = El::store(f);
      ss += f * f;
    }
    ss = wave_sum(ss);
  }
  const float rstd = KIND & kNorm ? 1.0f / __fsqrt_rn(ss / (float)n + eps) : 1.f;
  if constexpr ((KIND & k8bit) != 0) {
    auto z = [&](int c) { return KIND & kNorm ? El::load(w[c]) * (value(c) * rstd) : value(c); };
    uint32_t top = 0;
    for (int c = lane; c < n; c += kWave) top = max(top, __float_as_uint(z(c)) & 0x7fffffffu);
    const float scale = scale_of(wave_max(top)), inv = 1.0f / scale;
    if (lane == 0) stat[row] = scale;
    for (int c = lane; c < n; c += kWave) ((uint8_t*)y)[base + c] = code_of(z(c) * inv);
  } else {
    if (lane == 0 && stat) stat[row] = rstd;
    for (int c = lane; c < n; c += kWave)
      ((typename El::T*)y)[base + c] = El::store(El::load(w[c]) * (value(c) * rstd));
  }
}

// ---------------------------------------------------------------- backward
// Persistent: block b takes the row groups b, b + grid, ...; all of a block's groups run the same number of steps, so
// that the barriers stay uniform. The next row's loads are out before this one is reduced, but for rows of 16 waves, whose
// registers do not hold both. No register goes to memory: where some did, fp32 [2042, 1001] took 20.3 us, [4096, 16384] 305
// (so 200), bf16 [32768, 4096] 191.
template <int DT, int WPR, int VPT, bool RAGGED, bool DR>
__global__ __launch_bounds__(threads_of(WPR)) void add_rms_bwd(
    const typename Elem<DT>::T* __restrict__ dy, const typename Elem<DT>::T* __restrict__ dr,
    const typename Elem<DT>::T* __restrict__ r, const typename Elem<DT>::T* __restrict__ w,
    const float* __restrict__ rstd, typename Elem<DT>::T* __restrict__ dx, float* __restrict__ part, int64_t rows, int n) {
  using El = Elem<DT>;
  constexpr int E = El::E, WAVES = threads_of(WPR) / kWave, RPB = WAVES / WPR, GT = WPR * kWave;
  __shared__ float red[2][WAVES];
  __shared__ __attribute__((aligned(16))) float comb[4096];
  const int grp = threadIdx.x / GT, gtid = threadIdx.x - grp * GT;
  const int nch = RAGGED ? (n + E - 1) / E : n / E;
  const float inv_n = 1.0f / (float)n;

  // The registers of 16 waves do not hold w beside four chunks a lane of each row: each lane has its part in LDS.
  constexpr bool kStaged = WPR == 16 && VPT == 4;
  __shared__ u32x4 staged[kStaged ? VPT * GT : 1];
  u32x4 wv[kStaged ? 1 : VPT];
  auto weight = [&](int k) { return kStaged ? staged[gtid + k * GT] : wv[kStaged ? 0 : k]; };
  float dw[VPT][E];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int c = gtid + k * GT;
    const u32x4 wc = c < nch ? load_chunk<RAGGED>(chunk_at<RAGGED, E>(w, c, n)) : u32x4{0u, 0u, 0u, 0u};
    if constexpr (kStaged)
      staged[c] = wc;
    else
      wv[k] = wc;
#pragma unroll
    for (int j = 0; j < E; ++j) dw[k][j] = 0.f;
  }

  const int total = (int)rows, groups_total = (int)gridDim.x * RPB;  // fewer than 2^26 rows
  const int iters = (total + groups_total - 1) / groups_total;
  struct Row {
    u32x4 g[VPT], x[VPT], d[DR ? VPT : 1];  // (never unset, which kept all of it in memory)
    float rstd;
  };
  constexpr bool kAhead = WPR < 16;
  auto fetch = [&](int row, Row& q) {
    const bool live = row < total;
    const int64_t base = (live ? row : 0) * (int64_t)n;
    // A lane's addresses are formed here, from its number: kept from row to row they took two registers each, which went to
    // memory.
    int lane = gtid;
    if constexpr (!kAhead) asm volatile("" : "+v"(lane));
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = lane + k * GT;
      const bool ok = live && c < nch;
      q.g[k] = ok ? stream_chunk<RAGGED>(chunk_at<RAGGED, E>(dy + base, c, n)) : u32x4{0u, 0u, 0u, 0u};
      q.x[k] = ok ? stream_chunk<RAGGED>(chunk_at<RAGGED, E>(r + base, c, n)) : u32x4{0u, 0u, 0u, 0u};
      if constexpr (DR) q.d[k] = ok ? stream_chunk<RAGGED>(chunk_at<RAGGED, E>(dr + base, c, n)) : u32x4{0u, 0u, 0u, 0u};
    }
    q.rstd = live ? rstd[row] : 0.f;
  };
  int row = (int)blockIdx.x * RPB + grp;
  Row here;
  fetch(row, here);
  for (int it = 0; it < iters; ++it, row += groups_total) {
    const bool live = row < total;
    const int64_t base = (live ? row : 0) * (int64_t)n;
    Row next;
    if constexpr (kAhead) fetch(row + groups_total, next);
    float sdot = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      float gf[E], xf[E], wf[E];
      El::unpack(here.g[k], gf);
      El::unpack(here.x[k], xf);
      El::unpack(weight(k), wf);
      const int dup = chunk_shared<RAGGED, E>(gtid + k * GT, n);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float nrm = xf[j] * here.rstd;
        dw[k][j] += gf[j] * nrm;
        sdot += RAGGED && j < dup ? 0.f : (gf[j] * wf[j]) * nrm;
      }
    }
    sdot = row_reduce<WPR>(sdot, red[it & 1], wave_sum, [](float a, float b) { return a + b; });
    if (live) {
      const float r1 = here.rstd, sn = sdot * inv_n;
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = gtid + k * GT;
        if (c < nch) {
          float gf[E], xf[E], wf[E], o[E];
          El::unpack(here.g[k], gf);
          El::unpack(here.x[k], xf);
          El::unpack(weight(k), wf);
#pragma unroll
          for (int j = 0; j < E; ++j) o[j] = r1 * (gf[j] * wf[j] - (xf[j] * r1) * sn);
          if constexpr (DR) {
            float df[E];
            El::unpack(here.d[k], df);
#pragma unroll
            for (int j = 0; j < E; ++j) o[j] += df[j];
          }
          const u32x4 ov = El::pack(o);
          store_chunk<RAGGED>(chunk_at<RAGGED, E>(dx + base, c, n), ov);
        }
      }
    }
    if constexpr (kAhead)
      here = next;
    else
      fetch(row + groups_total, here);
  }

  // The RPB row groups' dw into one partial row per block, in group order, through a window of 4096 columns.
  constexpr int WCH = 4096 / E;
  float* prow = part + (int64_t)blockIdx.x * n;
  for (int w0 = 0; w0 < nch; w0 += WCH) {
    for (int gi = 0; gi < RPB; ++gi) {
      if (grp == gi) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
          const int c = gtid + k * GT;
          if (c >= w0 && c < w0 + WCH && c < nch) {
            f32x4* cw = reinterpret_cast<f32x4*>(comb + (c - w0) * E);
            float* pw = prow + chunk_col<RAGGED, E>(c, n);  // shared columns: both chunks have the same sums
#pragma unroll
            for (int q = 0; q < E / 4; ++q) {
              f32x4 v{dw[k][4 * q], dw[k][4 * q + 1], dw[k][4 * q + 2], dw[k][4 * q + 3]};
              if (gi > 0) v = cw[q] + v;
              if (gi < RPB - 1)
                cw[q] = v;
              else
                *reinterpret_cast<f32x4_any*>(pw + 4 * q) = v;
            }
          }
        }
      }
      if constexpr (RPB > 1) __syncthreads();
    }
  }
}

// Rows shorter than a chunk: a thread per column for dw (and the row's sum again in each thread), n < 8 columns.
template <int DT>
__global__ __launch_bounds__(kWave) void add_rms_bwd_short(
    const typename Elem<DT>::T* __restrict__ dy, const typename Elem<DT>::T* __restrict__ dr,
    const typename Elem<DT>::T* __restrict__ r, const typename Elem<DT>::T* __restrict__ w,
    const float* __restrict__ rstd, typename Elem<DT>::T* __restrict__ dx, float* __restrict__ part, int64_t rows, int n) {
  using El = Elem<DT>;
  constexpr int kMost = 8;
  const float inv_n = 1.0f / (float)n;
  float wf[kMost], dw[kMost];
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    wf[j] = j < n ? El::load(w[j]) : 0.f;
    dw[j] = 0.f;
  }
  for (int64_t row = (int64_t)blockIdx.x * kWave + threadIdx.x; row < rows; row += (int64_t)gridDim.x * kWave) {
    const float r1 = rstd[row];
    float dn[kMost], xf[kMost], sdot = 0.f;
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
      const int64_t i = row * n + min(j, n - 1);
      const float g = j < n ? El::load(dy[i]) : 0.f;
      xf[j] = El::load(r[i]) * r1;
      dw[j] += g * xf[j];
      dn[j] = g * wf[j];
      sdot += dn[j] * xf[j];
    }
    const float sn = sdot * inv_n;
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
      const int64_t i = row * n + j;
      if (j < n) dx[i] = El::store(r1 * (dn[j] - xf[j] * sn) + (dr ? El::load(dr[i]) : 0.f));
    }
  }
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    const float sum = wave_sum(dw[j]);
    if (j < n && threadIdx.x == 0) part[(int64_t)blockIdx.x * n + j] = sum;
  }
}

bool vec_ok(int n, int e, std::initializer_list<const void*> ptrs) {
  if (n % e != 0) return false;
  for (const void* p : ptrs)
    if (!aligned16(p)) return false;
  return true;
}

int chunks_per_lane(int nch, int wpr) {
  const int need = (int)ceil_div(nch, (int64_t)wpr * kWave);
  int v = 1;
  while (v < need) v <<= 1;
  return v;
}

struct Rows {
  const void *x, *residual, *w;
  void *y, *r;
  float* stat;
  int64_t rows;
  int n;
  float eps;
  hipStream_t st;
};

template <int DT, int WPR, int VPT, bool RAGGED, int KIND>
void launch_rows(const Rows& a) {
  using T = typename Elem<DT>::T;
  hipLaunchKernelGGL((row_pass<DT, WPR, VPT, RAGGED, KIND>),
                     dim3((unsigned)ceil_div(a.rows, threads_of(WPR) / kWave / WPR)), dim3(threads_of(WPR)), 0, a.st,
                     (const T*)a.x, (const T*)a.residual, (const T*)a.w, a.y, (T*)a.r, a.stat, a.rows, a.n, a.eps);
}

// Waves per row: as few as hold it in four chunks a lane (a row of one wave has no barrier), eight chunks where 16 waves do not.
int row_waves(int nch) { return nch <= 256 ? 1 : nch <= 1024 ? 4 : nch <= 2048 ? 8 : 16; }

template <int DT, bool RAGGED, int KIND>
bool rows_in_chunks(const Rows& a) {
  const int nch = (int)ceil_div(a.n, Elem<DT>::E), wpr = row_waves(nch), vpt = chunks_per_lane(nch, wpr);
#define KRSI_ROW_CASE(W, V)                     \
  if (wpr == W && vpt == V) {                   \
    launch_rows<DT, W, V, RAGGED, KIND>(a);     \
    return true;                                \
  }
  KRSI_ROW_CASE(1, 1) KRSI_ROW_CASE(1, 2) KRSI_ROW_CASE(1, 4) KRSI_ROW_CASE(4, 2) KRSI_ROW_CASE(4, 4)
  KRSI_ROW_CASE(8, 4) KRSI_ROW_CASE(16, 4)
  if constexpr (KIND == k8bit) {
    KRSI_ROW_CASE(16, 8)
  }
#undef KRSI_ROW_CASE
  return false;
}

template <int DT, int KIND>
int row_kernels(const Rows& a) {
  using T = typename Elem<DT>::T;
  constexpr int E = Elem<DT>::E;
  const bool vec = vec_ok(a.n, E, {a.x, a.residual, a.w, a.r}) && (KIND & k8bit ? true : aligned16(a.y));
  // Ragged rows of up to an element per lane: element by element, as RMSNorm's.
  const bool done = vec ? rows_in_chunks<DT, false, KIND>(a) : a.n > kWave && rows_in_chunks<DT, true, KIND>(a);
  if (!done)
    hipLaunchKernelGGL((row_scalar<DT, KIND>), dim3((unsigned)ceil_div(a.rows, 4)), dim3(4 * kWave), 0, a.st,
                       (const T*)a.x, (const T*)a.residual, (const T*)a.w, a.y, (T*)a.r, a.stat, a.rows, a.n, a.eps);
  return launch_status();
}
template <int KIND>
int row_kernels(const Rows& a, int32_t dtype) {
  return dtype == kF16 ? row_kernels<kF16, KIND>(a) : dtype == kF32 ? row_kernels<kF32, KIND>(a) : row_kernels<kBf16, KIND>(a);
}

// Waves per row of the backward, which holds three rows, the next three, w and dw: two chunks a lane, four beyond 2048 chunks.
int bwd_waves(int nch) { return nch <= 128 ? 1 : nch <= 256 ? 2 : nch <= 512 ? 4 : nch <= 1024 ? 8 : 16; }

int64_t bwd_blocks(int64_t rows, int n, int e) {
  const int wpr = bwd_waves((int)ceil_div(n, e));
  const int64_t b = ceil_div(rows, n < e ? kWave : threads_of(wpr) / kWave / wpr);
  return b < kBwdMaxBlocks ? b : kBwdMaxBlocks;
}

struct Bwd {
  const void *dy, *dr, *r, *w;
  const float* rstd;
  void *dx, *dw;
  float* part;
  int64_t rows;
  int n;
  hipStream_t st;
};

template <int DT, int WPR, int VPT, bool RAGGED>
void launch_bwd(const Bwd& a, unsigned blocks) {
  using T = typename Elem<DT>::T;
  const auto kernel = a.dr ? add_rms_bwd<DT, WPR, VPT, RAGGED, true> : add_rms_bwd<DT, WPR, VPT, RAGGED, false>;
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads_of(WPR)), 0, a.st, (const T*)a.dy, (const T*)a.dr, (const T*)a.r,
                     (const T*)a.w, a.rstd, (T*)a.dx, a.part, a.rows, a.n);
}

template <int DT, bool RAGGED>
bool bwd_in_chunks(const Bwd& a, unsigned blocks) {
  const int nch = (int)ceil_div(a.n, Elem<DT>::E), wpr = bwd_waves(nch), vpt = chunks_per_lane(nch, wpr);
#define KRSI_BWD_CASE(W, V)                        \
  if (wpr == W && vpt == V) {                      \
    launch_bwd<DT, W, V, RAGGED>(a, blocks);       \
    return true;                                   \
  }
  KRSI_BWD_CASE(1, 1) KRSI_BWD_CASE(1, 2) KRSI_BWD_CASE(2, 2) KRSI_BWD_CASE(4, 2) KRSI_BWD_CASE(8, 2)
  KRSI_BWD_CASE(16, 2)
  if constexpr (DT == kF32) {
    KRSI_BWD_CASE(16, 4)
  }
#undef KRSI_BWD_CASE
  return false;
}

template <int DT>
int backward(const Bwd& a) {
  using T = typename Elem<DT>::T;
  constexpr int E = Elem<DT>::E;
  const int64_t blocks = bwd_blocks(a.rows, a.n, E);
  if (a.rows) {
    if (a.n < E) {
      hipLaunchKernelGGL((add_rms_bwd_short<DT>), dim3((unsigned)blocks), dim3(kWave), 0, a.st, (const T*)a.dy,
                         (const T*)a.dr, (const T*)a.r, (const T*)a.w, a.rstd, (T*)a.dx, a.part, a.rows, a.n);
    } else {
      const bool vec = vec_ok(a.n, E, {a.dy, a.dr, a.r, a.w, a.dx});
      if (!(vec ? bwd_in_chunks<DT, false>(a, (unsigned)blocks) : bwd_in_chunks<DT, true>(a, (unsigned)blocks)))
        return KRSI_ERR_BAD_SHAPE;
    }
    const int rc = launch_status();
    if (rc != KRSI_OK) return rc;
  }
  hipLaunchKernelGGL((colsum<DT>), dim3((unsigned)ceil_div(a.n, kWave)), dim3(kColsumWaves * kWave), 0, a.st,
                     (const float*)a.part, a.rows ? blocks : (int64_t)0, a.n, (T*)a.dw);
  return launch_status();
}

bool known_dtype(int32_t dt) { return dt == kBf16 || dt == kF16 || dt == kF32; }

// Shapes whose grids stay below 2^32 threads (fp32 rows take the most waves).
int check_rows(int64_t rows, int32_t n, int32_t most, int32_t dtype) {
  if (!known_dtype(dtype)) return KRSI_ERR_UNSUPPORTED;
  if (rows < 0 || n <= 0 || n > most || rows >= (INT64_C(1) << 26) / row_waves((int)ceil_div(n, 4))) return KRSI_ERR_BAD_SHAPE;
  return KRSI_OK;
}
bool finite(float v) { return v == v && v <= 3.0e38f && v >= -3.0e38f; }

}  // namespace
}  // namespace krsi

extern "C" {

int krsi_add_rmsnorm_fwd(const void* x, const void* residual, const void* w, void* y, void* r, float* rstd, int64_t rows,
                         int32_t n, float eps, int32_t dtype, void* stream) {
  using namespace krsi;
  const int rc = check_rows(rows, n, kMaxRow, dtype);
  if (rc != KRSI_OK) return rc;
  if (!finite(eps)) return KRSI_ERR_BAD_SCALE;
  if (rows == 0) return KRSI_OK;
  if (!x || !residual || !w || !y || !r) return KRSI_ERR_NULL_POINTER;
  return row_kernels<kAdd | kNorm>({x, residual, w, y, r, rstd, rows, n, eps, as_stream(stream)}, dtype);
}

int krsi_add_rmsnorm_8bit(const void* x, const void* residual, const void* w, void* q, float* scale, void* r, int64_t rows,
                          int32_t n, float eps, int32_t dtype, void* stream) {
  using namespace krsi;
  const int rc = check_rows(rows, n, kMaxRow, dtype);
  if (rc != KRSI_OK) return rc;
  if (!finite(eps)) return KRSI_ERR_BAD_SCALE;
  if (rows == 0) return KRSI_OK;
  if (!x || !w || !q || !scale || !residual != !r) return KRSI_ERR_NULL_POINTER;
  const Rows a{x, residual, w, q, r, scale, rows, n, eps, as_stream(stream)};
  return residual ? row_kernels<kAdd | kNorm | k8bit>(a, dtype) : row_kernels<kNorm | k8bit>(a, dtype);
}

int krsi_quantize_rows(const void* x, void* q, float* scale, int64_t rows, int32_t n, int32_t dtype, void* stream) {
  using namespace krsi;
  const int rc = check_rows(rows, n, 1 << 20, dtype);
  if (rc != KRSI_OK) return rc;
  if (rows == 0) return KRSI_OK;
  if (!x || !q || !scale) return KRSI_ERR_NULL_POINTER;
  return row_kernels<k8bit>({x, nullptr, nullptr, q, nullptr, scale, rows, n, 0.f, as_stream(stream)}, dtype);
}

size_t krsi_add_rmsnorm_bwd_workspace_bytes(int64_t rows, int32_t n) {
  using namespace krsi;
  if (rows <= 0 || n <= 0 || n > kMaxRow) return 0;
  const int64_t a = bwd_blocks(rows, n, 8), b = bwd_blocks(rows, n, 4);
  return align256((size_t)(a > b ? a : b) * n * sizeof(float));
}

int krsi_add_rmsnorm_bwd(const void* dy, const void* dr, const void* r, const void* w, const float* rstd, void* dx,
                         void* dw, void* workspace, size_t workspace_bytes, int64_t rows, int32_t n, int32_t dtype,
                         void* stream) {
  using namespace krsi;
  const int rc = check_rows(rows, n, kMaxRow, dtype);
  if (rc != KRSI_OK) return rc;
  if (!dw) return KRSI_ERR_NULL_POINTER;
  if (rows > 0) {
    if (!dy || !r || !w || !rstd || !dx) return KRSI_ERR_NULL_POINTER;
    if (!workspace || workspace_bytes < krsi_add_rmsnorm_bwd_workspace_bytes(rows, n)) return KRSI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return KRSI_ERR_MISALIGNED;
  }
  const Bwd a{dy, dr, r, w, rstd, dx, dw, (float*)workspace, rows, n, as_stream(stream)};
  return dtype == kF16 ? backward<kF16>(a) : dtype == kF32 ? backward<kF32>(a) : backward<kBf16>(a);
}

}  // extern "C"
