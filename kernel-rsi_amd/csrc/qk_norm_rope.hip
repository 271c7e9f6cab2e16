// RMS norm of every query and key head, then the rotation by the token's position, for gfx950.
// qkv [tokens, (H + 2 KH) D] holds per token H query heads, KH key heads and KH value heads. For a query or
// key head x [D], with w its kind's weight [D] and (c_i, s_i) row `position` of the rotation table:
//   r = 1 / sqrt(sum x^2 / D + eps),  z = w x r
//   y_a = z_a c_i - z_b s_i,  y_b = z_b c_i + z_a s_i      pair i of the first R columns: (i, i + R/2), or
//                                                          (2 i, 2 i + 1) where interleaved; y = z past R
// Value heads are copied. Everything between the load and the store is fp32: one rounding, at the store.
// Backward, from dy: the pair's inverse rotation gives dz; dw = sum over tokens and heads of dz x r;
//   dn = dz w;  dx = r dn - x r^3 sum(dn x) / D.
//
// What bounds it: HBM (forward 2 bytes moved per byte of qkv; backward dy, q and k in, dqkv out). bf16 [16384, 48
// heads of 128]: forward 69.6 us (5.8 TB/s), backward 112 us (4.8 TB/s); a copy of 2 GB runs at 4.9.
// Outputs are stored past the caches (73 and 114 us without).
// Layout: a lane holds C elements of one half of the pairs and the C elements that they rotate with, so the
// rotation stays in registers; D / (2 C) lanes (rounded up to a power of two, the group) hold a head and reduce its
// square sum by shuffles. C is the widest of 8, 4, 2, 1 (16 bytes at most) that cuts both R / 2 and the rest
// evenly. A wave takes one token's cos and sin into registers and runs that token's heads past them, 64 /
// group at a time, U times with all loads first.
#include "chunks.h"
#include "krsi_device.h"
#include "krsi_internal.h"

#include <type_traits>

namespace krsi {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kBwdBlocks = 1024;  // of a backward, at most: partial rows of dw
// Workgroups of a backward: what the chip holds at once by its registers (8 columns: 182, two waves per SIMD; 4:
// 116, four). bf16 [16384, 48 heads of 128]: 114 us with 512 workgroups, 119 with 1024, 129 with 2048; fp32 [4096,
// 36 heads of 80]: 41, 34, 37.
constexpr int bwd_blocks(int c) { return c == 8 ? kBwdBlocks / 2 : kBwdBlocks; }

// What both directions need of a call, by value.
struct Args {
  const void *x, *wq, *wk, *positions;
  const float* rope;
  int64_t ldx, tokens, table_rows;
  int S, H, KH, D, R, position_bytes;
  int lanes, rotating;  // lanes that hold a head, and how many of them rotate
  int group_shift;      // log2 of the group
  int per;              // waves' worth of heads per token
  float eps;
};

// This lane's columns of a head: C from e0 and C from e1. Interleaved pairs lie within the 2 C columns from e0.
template <int C, bool INTER>
struct Columns {
  int e0, e1;
  __device__ __forceinline__ Columns(const Args& a, int p) {
    e0 = INTER || p >= a.rotating ? 2 * p * C : p * C;
    e1 = INTER || p >= a.rotating ? e0 + C : a.R / 2 + p * C;
  }
};
// Element j of the lane's 2 C as a[i], b[i] of pair i: identity where halves rotate, even and odd where interleaved.
template <int C, bool INTER>
__device__ __forceinline__ constexpr int first_of(int i) { return INTER ? 2 * i : i; }
template <int C, bool INTER>
__device__ __forceinline__ constexpr int second_of(int i) { return INTER ? 2 * i + 1 : C + i; }

__device__ __forceinline__ int64_t position_of(const Args& a, int64_t t) {
  if (!a.positions) return (uint32_t)t % (uint32_t)a.S;
  return load_index(a.positions, a.position_bytes, t);
}

// cos and sin of the lane's pairs at token t: 1 and 0 for lanes past R, NaN for a position outside the table.
template <int C>
__device__ __forceinline__ void load_rotation(const Args& a, int64_t t, int p, float* c, float* s) {
  const int64_t pos = position_of(a, t);
  const bool inside = pos >= 0 && pos < a.table_rows;
  if (p < a.rotating) {
    const float* row = a.rope + (inside ? pos : 0) * a.R + p * C;
    Piece<kF32, C> pc, ps;
    pc.load(row);
    ps.load(row + a.R / 2);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      c[j] = inside ? pc.e[j] : __builtin_nanf("");
      s[j] = inside ? ps.e[j] : __builtin_nanf("");
    }
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      c[j] = 1.f;
      s[j] = 0.f;
    }
  }
}

__device__ __forceinline__ float group_sum(float v, int shift) {
  for (int m = (1 << shift) >> 1; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

template <int DT, int C, int U, bool INTER>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_fwd(Args a, typename Elem<DT>::T* __restrict__ out) {
  using El = Elem<DT>;
  using T = typename El::T;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t wave = (int64_t)blockIdx.x * kWaves + threadIdx.x / kWave;
  const int64_t t = (uint32_t)wave / (uint32_t)a.per;
  if (t >= a.tokens) return;
  const int part = (int)(wave - t * a.per);
  const int p = lane & ((1 << a.group_shift) - 1), sub = lane >> a.group_shift, hp = kWave >> a.group_shift;
  const bool active = p < a.lanes;
  const Columns<C, INTER> col(a, p);
  const int heads = a.H + 2 * a.KH, normed = a.H + a.KH;
  const T* xr = (const T*)a.x + t * a.ldx;
  T* yr = out + t * (int64_t)heads * a.D;

  Piece<DT, C> x0[U], x1[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = (part * U + u) * hp + sub;
    const bool live = active && h < heads;
    const T* src = xr + (int64_t)(live ? h : 0) * a.D;
    x0[u].load(src + (active ? col.e0 : 0));
    x1[u].load(src + (active ? col.e1 : 0));
  }
  float c[C], s[C];
  load_rotation<C>(a, t, p, c, s);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = (part * U + u) * hp + sub;
    const bool live = active && h < heads;
    float v[2 * C], ss = 0.f;
    x0[u].get(v);
    x1[u].get(v + C);
#pragma unroll
    for (int j = 0; j < 2 * C; ++j) ss += v[j] * v[j];
    ss = group_sum(active ? ss : 0.f, a.group_shift);
    if (!live) continue;
    if (h < normed) {
      const float r = 1.0f / __fsqrt_rn(ss / (float)a.D + a.eps);
      const T* w = (const T*)(h < a.H ? a.wq : a.wk);
      Piece<DT, C> w0, w1;
      float wv[2 * C], y[2 * C];
      w0.load(w + col.e0);
      w1.load(w + col.e1);
      w0.get(wv);
      w1.get(wv + C);
#pragma unroll
      for (int j = 0; j < 2 * C; ++j) v[j] = wv[j] * v[j] * r;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const float za = v[first_of<C, INTER>(i)], zb = v[second_of<C, INTER>(i)];
        y[first_of<C, INTER>(i)] = za * c[i] - zb * s[i];
        y[second_of<C, INTER>(i)] = zb * c[i] + za * s[i];
      }
      x0[u].set(y);
      x1[u].set(y + C);
    }
    T* dst = yr + (int64_t)h * a.D;
    x0[u].store_stream(dst + col.e0);
    x1[u].store_stream(dst + col.e1);
  }
}

// A fixed grid of waves walks the (token, part) items and keeps its share of both weights' gradients in
// registers; each workgroup writes one partial row [2, D] of them.
template <int DT, int C, int U, bool INTER>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_bwd(Args a, const typename Elem<DT>::T* __restrict__ dy,
                                                             typename Elem<DT>::T* __restrict__ dx, int64_t lddx,
                                                             float* __restrict__ part_rows) {
  using El = Elem<DT>;
  using T = typename El::T;
  __shared__ float fold[kWaves][2 * 128];
  const int lane = threadIdx.x & (kWave - 1), wv_id = threadIdx.x / kWave;
  const int p = lane & ((1 << a.group_shift) - 1), sub = lane >> a.group_shift, hp = kWave >> a.group_shift;
  const bool active = p < a.lanes;
  const Columns<C, INTER> col(a, p);
  const int heads = a.H + 2 * a.KH, normed = a.H + a.KH;
  float wq[2 * C], wk[2 * C], dwq[2 * C], dwk[2 * C];
  {
    Piece<DT, C> q0, q1, k0, k1;
    q0.load((const T*)a.wq + (active ? col.e0 : 0));
    q1.load((const T*)a.wq + (active ? col.e1 : 0));
    k0.load((const T*)a.wk + (active ? col.e0 : 0));
    k1.load((const T*)a.wk + (active ? col.e1 : 0));
    q0.get(wq);
    q1.get(wq + C);
    k0.get(wk);
    k1.get(wk + C);
  }
#pragma unroll
  for (int j = 0; j < 2 * C; ++j) dwq[j] = dwk[j] = 0.f;

  const int64_t items = a.tokens * a.per;
  for (int64_t it = (int64_t)blockIdx.x * kWaves + wv_id; it < items; it += (int64_t)gridDim.x * kWaves) {
    const int64_t t = (uint32_t)it / (uint32_t)a.per;
    const int part = (int)(it - t * a.per);
    const T* xr = (const T*)a.x + t * a.ldx;
    const T* gr = dy + t * (int64_t)heads * a.D;
    T* dr = dx + t * lddx;
    Piece<DT, C> x0[U], x1[U], g0[U], g1[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = (part * U + u) * hp + sub;
      const int64_t at = (int64_t)(active && h < heads ? h : 0) * a.D;
      const int64_t xat = (int64_t)(active && h < normed ? h : 0) * a.D;
      g0[u].load(gr + at + (active ? col.e0 : 0));
      g1[u].load(gr + at + (active ? col.e1 : 0));
      x0[u].load(xr + xat + (active ? col.e0 : 0));
      x1[u].load(xr + xat + (active ? col.e1 : 0));
    }
    float c[C], s[C];
    load_rotation<C>(a, t, p, c, s);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = (part * U + u) * hp + sub;
      const bool live = active && h < heads;
      float x[2 * C], g[2 * C], dz[2 * C], ss = 0.f, dot = 0.f;
      x0[u].get(x);
      x1[u].get(x + C);
      g0[u].get(g);
      g1[u].get(g + C);
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const float ga = g[first_of<C, INTER>(i)], gb = g[second_of<C, INTER>(i)];
        dz[first_of<C, INTER>(i)] = ga * c[i] + gb * s[i];
        dz[second_of<C, INTER>(i)] = gb * c[i] - ga * s[i];
      }
#pragma unroll
      for (int j = 0; j < 2 * C; ++j) {
        ss += x[j] * x[j];
        dot += dz[j] * (h < a.H ? wq[j] : wk[j]) * x[j];
      }
      ss = group_sum(active ? ss : 0.f, a.group_shift);
      dot = group_sum(active ? dot : 0.f, a.group_shift);
      if (!live) continue;
      if (h < normed) {
        const float r = 1.0f / __fsqrt_rn(ss / (float)a.D + a.eps);
        const float m = r * r * r * (dot / (float)a.D);
#pragma unroll
        for (int j = 0; j < 2 * C; ++j) {
          const float d = dz[j] * x[j] * r;
          dwq[j] += h < a.H ? d : 0.f;
          dwk[j] += h < a.H ? 0.f : d;
          x[j] = r * (dz[j] * (h < a.H ? wq[j] : wk[j])) - x[j] * m;
        }
        g0[u].set(x);
        g1[u].set(x + C);
      }
      T* dst = dr + (int64_t)h * a.D;
      g0[u].store_stream(dst + col.e0);
      g1[u].store_stream(dst + col.e1);
    }
  }

  // The wave's heads, then the workgroup's waves, in a fixed order.
#pragma unroll
  for (int j = 0; j < 2 * C; ++j) {
    for (int m = 1 << a.group_shift; m < kWave; m <<= 1) {
      dwq[j] += __shfl_xor(dwq[j], m, kWave);
      dwk[j] += __shfl_xor(dwk[j], m, kWave);
    }
    if (active && sub == 0) {
      const int e = j < C ? col.e0 + j : col.e1 + j - C;
      fold[wv_id][e] = dwq[j];
      fold[wv_id][a.D + e] = dwk[j];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * a.D; e += kThreads) {
    float v = fold[0][e];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += fold[w][e];
    part_rows[(int64_t)blockIdx.x * 2 * a.D + e] = v;
  }
}

// dwq and dwk: the column sums of the [rows, 2 D] partial rows, in a fixed order: 16 columns per workgroup, thread
// group q of 64 adds rows q, q + 64, ..., then the groups' sums are added in order. (64 columns and 16 groups: 6.6
// us for 1024 rows of 256 columns.) No rows: zero.
constexpr int kSumCols = 16, kSumThreads = 1024, kSumParts = kSumThreads / kSumCols;
template <int DT>
__global__ __launch_bounds__(kSumThreads) void weight_sum(const float* __restrict__ in, int rows, int D,
                                                          typename Elem<DT>::T* __restrict__ dwq,
                                                          typename Elem<DT>::T* __restrict__ dwk) {
  __shared__ float s[kSumParts][kSumCols];
  const int c = threadIdx.x % kSumCols, q = threadIdx.x / kSumCols, col = blockIdx.x * kSumCols + c;
  float acc = 0.f;
#pragma unroll 8
  for (int r = q; r < rows; r += kSumParts) acc += in[(int64_t)r * 2 * D + col];
  s[q][c] = acc;
  __syncthreads();
  if (q != 0) return;
#pragma unroll 8
  for (int k = 1; k < kSumParts; ++k) acc += s[k][c];
  (col < D ? dwq[col] : dwk[col - D]) = Elem<DT>::store(acc);
}

// Elements of a lane's half: the widest power of two, 16 bytes at most, that divides R / 2 and the rest in pairs.
int width_of(int dtype, int D, int R) {
  int c = dtype == kF32 ? 4 : 8;
  while (R % (2 * c) != 0 || D % (2 * c) != 0) c >>= 1;
  return c;
}

constexpr int kU = 2;

void lay_out(Args& a, int c, int u) {
  a.lanes = a.D / (2 * c);
  a.rotating = a.R / (2 * c);
  a.group_shift = 0;
  while ((1 << a.group_shift) < a.lanes) ++a.group_shift;
  a.per = (int)ceil_div(a.H + 2 * (int64_t)a.KH, (int64_t)u * (kWave >> a.group_shift));
}

template <int DT, int C, bool INTER>
int launch_fwd(Args a, void* out, hipStream_t st) {
  lay_out(a, C, kU);
  const int64_t waves = a.tokens * a.per;
  if (waves >= (1 << 26)) return KRSI_ERR_BAD_SHAPE;  // grids of less than 2^32 threads
  hipLaunchKernelGGL((qk_norm_rope_fwd<DT, C, kU, INTER>), dim3((unsigned)ceil_div(waves, kWaves)), dim3(kThreads), 0,
                     st, a, (typename Elem<DT>::T*)out);
  return launch_status();
}

template <int DT, int C, bool INTER>
int launch_bwd(Args a, const void* dy, void* dx, int64_t lddx, void* dwq, void* dwk, float* part, hipStream_t st) {
  using T = typename Elem<DT>::T;
  int blocks = 0;
  if (a.tokens > 0) {
    lay_out(a, C, kU);
    const int64_t waves = a.tokens * a.per;
    if (waves >= (1 << 26)) return KRSI_ERR_BAD_SHAPE;  // grids of less than 2^32 threads
    const int64_t need = ceil_div(waves, kWaves);
    blocks = (int)(need < bwd_blocks(C) ? need : bwd_blocks(C));
    hipLaunchKernelGGL((qk_norm_rope_bwd<DT, C, kU, INTER>), dim3((unsigned)blocks), dim3(kThreads), 0, st, a,
                       (const T*)dy, (T*)dx, lddx, part);
    const int rc = launch_status();
    if (rc != KRSI_OK) return rc;
  }
  hipLaunchKernelGGL((weight_sum<DT>), dim3((unsigned)(2 * a.D / kSumCols)), dim3(kSumThreads), 0, st,
                     (const float*)part, blocks, a.D, (T*)dwq, (T*)dwk);
  return launch_status();
}

// f(dtype, width, interleaved) as constants.
template <int DT, typename F>
int with_width(int c, bool inter, F&& f) {
  auto two = [&](auto w) {
    return inter ? f(std::integral_constant<int, DT>{}, w, std::true_type{})
                 : f(std::integral_constant<int, DT>{}, w, std::false_type{});
  };
  switch (c) {
    case 8:
      if constexpr (DT != kF32) return two(std::integral_constant<int, 8>{});
      return KRSI_ERR_UNSUPPORTED;
    case 4:
      return two(std::integral_constant<int, 4>{});
    case 2:
      return two(std::integral_constant<int, 2>{});
    default:
      return two(std::integral_constant<int, 1>{});
  }
}
template <typename F>
int with_kernel(int dtype, int c, bool inter, F&& f) {
  switch (dtype) {
    case kF16:
      return with_width<kF16>(c, inter, f);
    case kF32:
      return with_width<kF32>(c, inter, f);
    default:
      return with_width<kBf16>(c, inter, f);
  }
}

int check(int64_t tokens, int S, int H, int KH, int D, int R, int64_t table_rows, bool positions, int position_bytes,
          float eps, int interleaved, int dtype, int64_t ld) {
  if (dtype != kBf16 && dtype != kF16 && dtype != kF32) return KRSI_ERR_UNSUPPORTED;
  if (interleaved != 0 && interleaved != 1) return KRSI_ERR_UNSUPPORTED;
  if (tokens < 0 || tokens > 0x7fffffff || S <= 0 || H <= 0 || KH <= 0 || H > 65535 || KH > 65535)
    return KRSI_ERR_BAD_SHAPE;
  if (D % 8 != 0 || D < 8 || D > 128) return KRSI_ERR_UNSUPPORTED;
  if (R <= 0 || R > D || R % 2 != 0 || table_rows <= 0 || ld < (H + 2 * (int64_t)KH) * D) return KRSI_ERR_BAD_SHAPE;
  if (positions ? position_bytes != 4 && position_bytes != 8 : table_rows < S && table_rows < tokens)
    return KRSI_ERR_BAD_SHAPE;
  if (!(eps == eps) || eps > 3.0e38f || eps < -3.0e38f) return KRSI_ERR_BAD_SCALE;
  return KRSI_OK;
}

}  // namespace
}  // namespace krsi

extern "C" {

int krsi_qk_norm_rope_fwd(const void* qkv, int64_t ld_qkv, const void* wq, const void* wk, const float* rope,
                          const void* positions, void* out, int64_t tokens, int32_t S, int32_t H, int32_t KH,
                          int32_t D, int32_t R, int64_t table_rows, int32_t position_bytes, float eps,
                          int32_t interleaved, int32_t dtype, void* stream) {
  using namespace krsi;
  const int rc = check(tokens, S, H, KH, D, R, table_rows, positions != nullptr, position_bytes, eps, interleaved, dtype,
                       ld_qkv);
  if (rc != KRSI_OK) return rc;
  if (tokens == 0) return KRSI_OK;
  if (!qkv || !wq || !wk || !rope || !out) return KRSI_ERR_NULL_POINTER;
  Args a{qkv, wq, wk, positions, rope, ld_qkv, tokens, table_rows, S, H, KH, D, R, position_bytes, 0, 0, 0, 0, eps};
  return with_kernel(dtype, width_of(dtype, D, R), interleaved == 1, [&](auto dt, auto c, auto inter) {
    return launch_fwd<dt(), c(), inter()>(a, out, as_stream(stream));
  });
}

size_t krsi_qk_norm_rope_bwd_workspace_bytes(int32_t D) {
  using namespace krsi;
  return D <= 0 ? 0 : (size_t)kBwdBlocks * 2 * D * sizeof(float);
}

int krsi_qk_norm_rope_bwd(const void* dout, const void* qkv, int64_t ld_qkv, const void* wq, const void* wk,
                          const float* rope, const void* positions, void* dqkv, int64_t ld_dqkv, void* dwq, void* dwk,
                          void* workspace, size_t workspace_bytes, int64_t tokens, int32_t S, int32_t H, int32_t KH,
                          int32_t D, int32_t R, int64_t table_rows, int32_t position_bytes, float eps,
                          int32_t interleaved, int32_t dtype, void* stream) {
  using namespace krsi;
  const int rc = check(tokens, S, H, KH, D, R, table_rows, positions != nullptr, position_bytes, eps, interleaved, dtype,
                       ld_qkv < ld_dqkv ? ld_qkv : ld_dqkv);
  if (rc != KRSI_OK) return rc;
  if (!dwq || !dwk) return KRSI_ERR_NULL_POINTER;
  if (tokens > 0) {
    if (!dout || !qkv || !wq || !wk || !rope || !dqkv) return KRSI_ERR_NULL_POINTER;
    if (!workspace || workspace_bytes < krsi_qk_norm_rope_bwd_workspace_bytes(D)) return KRSI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return KRSI_ERR_MISALIGNED;
  }
  Args a{qkv, wq, wk, positions, rope, ld_qkv, tokens, table_rows, S, H, KH, D, R, position_bytes, 0, 0, 0, 0, eps};
  return with_kernel(dtype, width_of(dtype, D, R), interleaved == 1, [&](auto dt, auto c, auto inter) {
    return launch_bwd<dt(), c(), inter()>(a, dout, dqkv, ld_dqkv, dwq, dwk, (float*)workspace, as_stream(stream));
  });
}

}  // extern "C"
