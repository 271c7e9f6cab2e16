// RMS norm of every query and key head, then the rotation by the token's position, for gfx950.
// qkv [tokens, (H + 2 KH) D] holds per token H query heads, KH key heads and KH value heads. For a query or
// key head x [D], with w its kind's weight [D] and (c_i, s_i) row `position` of the rotation table:
//   r = 1 / sqrt(sum x^2 / D + eps),  z = w x r
//   y_a = z_a c_i - z_b s_i,  y_b = z_b c_i + z_a s_i      pair i of the first R columns: (i, i + R/2), or
//                                                          (2 i, 2 i + 1) where interleaved; y = z past R
// Value heads are copied. Everything between the load and the store is fp32: one rounding, at the store.
// Backward, from dy: the pair's inverse rotation gives dz; dw = sum over tokens and heads of dz x r;
//   dn = dz w;  n = x r;  dx = r (dn - n r sum(dn x) / D).
//
// What bounds it: HBM (forward 2 bytes moved per byte of qkv; backward dy, q and k in, dqkv out). bf16 [16384, 48
// heads of 128]: forward 65 to 70 us by card and run (6.2 to 5.8 TB/s), backward 104 us (5.2 TB/s); a copy of 2 GB
// runs at 4.9. Outputs are stored past the caches (forward 73 us without).
// Layout: a lane holds C elements of one half of the pairs and the C elements that they rotate with, so the
// rotation stays in registers; the lanes of a head (their number rounded up to a power of two, the group) reduce its
// square sum by shuffles. C is the widest of 8, 4, 2, 1 (16 bytes at most) that a half of the rotated columns and
// of the rest holds; where it does not divide them the last lane's columns end at the half's end, and those that
// it shares with the lane before count once in a sum. (With the widest C that divides them, bf16 [16384, 48 heads of
// 72]: 64 / 108 us forward / backward, here 46 / 88; where 36 columns rotate, 98 / 171, here 46 / 88.)
// A wave takes a token's cos and sin into registers and runs that token's heads past them, 64 / group at a time,
// twice with all loads first. Where a token has fewer heads than that, a wave takes as many tokens as fill it
// ([16384, 4 heads of 64]: 9.3 / 29.6 us with one, 4.6 / 14.9).
#include "chunks.h"
#include "krsi_device.h"
#include "krsi_internal.h"

#include <type_traits>

namespace krsi {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kBwdBlocks = 1024;  // of a backward, at most: partial rows of dw
// Workgroups of a backward: what the chip holds at once by its registers (8 columns: 212, two waves per SIMD; 4:
// 112, four). bf16 [16384, 48 heads of 128]: 105 us with 512 workgroups, 109 with 1024; fp32 [4096, 36 heads of
// 80]: 41, 34.
constexpr int bwd_blocks(int c) { return c == 8 ? kBwdBlocks / 2 : kBwdBlocks; }

// What both directions need of a call, by value.
struct Args {
  const void *x, *wq, *wk, *positions;
  const float* rope;
  int64_t ldx, tokens, table_rows;
  int S, H, KH, D, R, position_bytes;
  int lanes, rotating;  // lanes that hold a head, and how many of them rotate
  int group_shift;      // log2 of the group
  int heads_shift;      // log2 of the heads of one token that a wave runs at a time
  int per;              // waves' worth of heads per token; 0: a wave takes more than one token at a time
  float eps;
};

// This lane's columns of a head: C from e0 and C from e1, of which the first dup0 and dup1 are another lane's too.
// Interleaved pairs lie within the 2 C columns from e0.
template <int C, bool INTER>
struct Columns {
  int e0, e1, dup0, dup1;
  bool rotates;
  __device__ __forceinline__ Columns(const Args& a, int p) {
    rotates = p < a.rotating;
    const int i = rotates ? p : p - a.rotating, base = rotates ? 0 : a.R, half = (rotates ? a.R : a.D - a.R) / 2;
    const int at = min(i * C, half - C), dup = i * C - at;  // of a half; of both halves' pairs where interleaved
    e0 = base + (INTER ? 2 * at : at);
    e1 = INTER ? e0 + C : e0 + half;
    dup0 = INTER ? min(2 * dup, C) : dup;
    dup1 = INTER ? max(2 * dup - C, 0) : dup;
  }
  __device__ __forceinline__ bool shared(int j) const { return j < C ? j < dup0 : j - C < dup1; }
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

// cos and sin of the lane's pairs at token t, NaN for a position outside the table. A lane that does not rotate loads
// others and does not use them.
template <int C, bool INTER>
__device__ __forceinline__ void load_rotation(const Args& a, const Columns<C, INTER>& col, int64_t t, float* c,
                                              float* s) {
  const int64_t pos = position_of(a, t);
  const bool inside = pos >= 0 && pos < a.table_rows;
  const float* row = a.rope + (inside ? pos : 0) * a.R + (col.rotates ? INTER ? col.e0 / 2 : col.e0 : 0);
  Piece<kF32, C> pc, ps;
  pc.load(row);
  ps.load(row + a.R / 2);
#pragma unroll
  for (int j = 0; j < C; ++j) {
    c[j] = inside ? pc.e[j] : __builtin_nanf("");
    s[j] = inside ? ps.e[j] : __builtin_nanf("");
  }
}

__device__ __forceinline__ float group_sum(float v, int shift) {
  for (int m = (1 << shift) >> 1; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

// Token and head of a lane group's u-th turn in a wave's item.
constexpr int kU = 2;
struct Turn {
  int64_t t;
  int h;
};
template <bool FEW>
__device__ __forceinline__ Turn turn_of(const Args& a, int64_t item, int sub, int u) {
  if constexpr (FEW) {
    const int tokens_shift = 6 - a.group_shift - a.heads_shift;
    return Turn{((item * kU + u) << tokens_shift) + (sub >> a.heads_shift), sub & ((1 << a.heads_shift) - 1)};
  }
  const int64_t t = (uint32_t)item / (uint32_t)a.per;
  return Turn{t, ((int)(item - t * a.per) * kU + u) * (kWave >> a.group_shift) + sub};
}

// FEW: a wave takes more than one token at a time. (A flag of the call instead costs the others 7 %: their token is a
// scalar.)
template <int DT, int C, bool INTER, bool RAGGED, bool FEW>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_fwd(Args a, int64_t items,
                                                             typename Elem<DT>::T* __restrict__ out) {
  using El = Elem<DT>;
  using T = typename El::T;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t item = (int64_t)blockIdx.x * kWaves + threadIdx.x / kWave;
  if (item >= items) return;
  const int p = lane & ((1 << a.group_shift) - 1), sub = lane >> a.group_shift;
  const bool active = p < a.lanes;
  const Columns<C, INTER> col(a, active ? p : 0);
  const int heads = a.H + 2 * a.KH, normed = a.H + a.KH;

  Turn at[kU];
  bool live[kU];
  Piece<DT, C> x0[kU], x1[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    at[u] = turn_of<FEW>(a, item, sub, u);
    live[u] = active && at[u].h < heads && (!FEW || at[u].t < a.tokens);
    const T* src = (const T*)a.x + (FEW && !live[u] ? 0 : at[u].t) * a.ldx + (live[u] ? at[u].h : 0) * a.D;
    x0[u].load(src + col.e0);
    x1[u].load(src + col.e1);
  }
  float c[C], s[C];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    if (u == 0 || FEW) load_rotation<C, INTER>(a, col, FEW && !live[u] ? 0 : at[u].t, c, s);
    const int h = at[u].h;
    float v[2 * C], ss = 0.f;
    x0[u].get(v);
    x1[u].get(v + C);
#pragma unroll
    for (int j = 0; j < 2 * C; ++j) ss += RAGGED && col.shared(j) ? 0.f : v[j] * v[j];
    ss = group_sum(active ? ss : 0.f, a.group_shift);
    if (!live[u]) continue;
    if (h < normed) {
      const float r = 1.0f / __fsqrt_rn(ss / (float)a.D + a.eps);
      const T* w = (const T*)(h < a.H ? a.wq : a.wk);
      Piece<DT, C> w0, w1;
      float wv[2 * C];
      w0.load(w + col.e0);
      w1.load(w + col.e1);
      w0.get(wv);
      w1.get(wv + C);
#pragma unroll
      for (int j = 0; j < 2 * C; ++j) v[j] = wv[j] * v[j] * r;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const float za = v[first_of<C, INTER>(i)], zb = v[second_of<C, INTER>(i)];
        v[first_of<C, INTER>(i)] = col.rotates ? za * c[i] - zb * s[i] : za;
        v[second_of<C, INTER>(i)] = col.rotates ? zb * c[i] + za * s[i] : zb;
      }
      x0[u].set(v);
      x1[u].set(v + C);
    }
    T* dst = out + at[u].t * (int64_t)(heads * a.D) + h * a.D;
    x0[u].store_stream(dst + col.e0);
    x1[u].store_stream(dst + col.e1);
  }
}

// A fixed grid of waves walks the items and keeps its share of both weights' gradients in registers; each workgroup
// writes one partial row [2, D] of them.
template <int DT, int C, bool INTER, bool RAGGED, bool FEW>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_bwd(Args a, int64_t items,
                                                             const typename Elem<DT>::T* __restrict__ dy,
                                                             typename Elem<DT>::T* __restrict__ dx, int64_t lddx,
                                                             float* __restrict__ part_rows) {
  using El = Elem<DT>;
  using T = typename El::T;
  __shared__ float fold[kWaves][2 * 128];
  const int lane = threadIdx.x & (kWave - 1), wv_id = threadIdx.x / kWave;
  const int p = lane & ((1 << a.group_shift) - 1), sub = lane >> a.group_shift;
  const bool active = p < a.lanes;
  const Columns<C, INTER> col(a, active ? p : 0);
  const int heads = a.H + 2 * a.KH, normed = a.H + a.KH;
  float wq[2 * C], wk[2 * C], dwq[2 * C], dwk[2 * C];
  {
    Piece<DT, C> q0, q1, k0, k1;
    q0.load((const T*)a.wq + col.e0);
    q1.load((const T*)a.wq + col.e1);
    k0.load((const T*)a.wk + col.e0);
    k1.load((const T*)a.wk + col.e1);
    q0.get(wq);
    q1.get(wq + C);
    k0.get(wk);
    k1.get(wk + C);
  }
#pragma unroll
  for (int j = 0; j < 2 * C; ++j) dwq[j] = dwk[j] = 0.f;

  for (int64_t item = (int64_t)blockIdx.x * kWaves + wv_id; item < items; item += (int64_t)gridDim.x * kWaves) {
    Turn at[kU];
    bool live[kU];
    Piece<DT, C> x0[kU], x1[kU], g0[kU], g1[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      at[u] = turn_of<FEW>(a, item, sub, u);
      live[u] = active && at[u].h < heads && (!FEW || at[u].t < a.tokens);
      const int64_t t = FEW && !live[u] ? 0 : at[u].t;
      const int h = live[u] ? at[u].h : 0, hx = h < normed ? h : 0;
      const T *xr = (const T*)a.x + t * a.ldx + hx * a.D, *gr = dy + t * (int64_t)(heads * a.D) + h * a.D;
      g0[u].load(gr + col.e0);
      g1[u].load(gr + col.e1);
      x0[u].load(xr + col.e0);
      x1[u].load(xr + col.e1);
    }
    float c[C], s[C];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (u == 0 || FEW) load_rotation<C, INTER>(a, col, FEW && !live[u] ? 0 : at[u].t, c, s);
      const int h = at[u].h;
      // A head of weight w, whose gradient's share is dw. All lanes of a head take the same branch: they exchange sums.
      auto head = [&](const float(&w)[2 * C], float(&dw)[2 * C]) {
        float x[2 * C], dz[2 * C], ss = 0.f, dot = 0.f;
        x0[u].get(x);
        x1[u].get(x + C);
        g0[u].get(dz);
        g1[u].get(dz + C);
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const float ga = dz[first_of<C, INTER>(i)], gb = dz[second_of<C, INTER>(i)];
          dz[first_of<C, INTER>(i)] = col.rotates ? ga * c[i] + gb * s[i] : ga;
          dz[second_of<C, INTER>(i)] = col.rotates ? gb * c[i] - ga * s[i] : gb;
        }
#pragma unroll
        for (int j = 0; j < 2 * C; ++j) {
          const bool skip = RAGGED && col.shared(j);
          ss += skip ? 0.f : x[j] * x[j];
          dot += skip ? 0.f : dz[j] * w[j] * x[j];
        }
        ss = group_sum(active ? ss : 0.f, a.group_shift);
        dot = group_sum(active ? dot : 0.f, a.group_shift);
        if (!live[u]) return;
        const float r = 1.0f / __fsqrt_rn(ss / (float)a.D + a.eps);
        const float m = dot * r / (float)a.D;
#pragma unroll
        for (int j = 0; j < 2 * C; ++j) {
          const float n = x[j] * r;  // (with r^3 formed, heads below 1e-13 or above 1e12 left its range)
          dw[j] += dz[j] * n;
          x[j] = r * (dz[j] * w[j] - n * m);
        }
        g0[u].set(x);
        g1[u].set(x + C);
      };
      // Heads of both weights in the wave, or few registers to spare: each lane selects its own. (With 8 columns the
      // branches save a twelfth of the time; with 4 they leave three waves per SIMD of four.)
      const int first = __builtin_amdgcn_readfirstlane(h - sub);
      if (FEW || C < 8 || (first < a.H && first + (kWave >> a.group_shift) > a.H)) {
        float w[2 * C], dw[2 * C];
#pragma unroll
        for (int j = 0; j < 2 * C; ++j) w[j] = h < a.H ? wq[j] : wk[j], dw[j] = 0.f;
        if (h < normed) head(w, dw);
#pragma unroll
        for (int j = 0; j < 2 * C; ++j) {
          dwq[j] += h < a.H ? dw[j] : 0.f;
          dwk[j] += h < a.H ? 0.f : dw[j];
        }
      } else if (h < a.H) {
        head(wq, dwq);
      } else if (h < normed) {
        head(wk, dwk);
      }
      if (!live[u]) continue;
      T* dst = dx + at[u].t * lddx + h * a.D;
      g0[u].store_stream(dst + col.e0);
      g1[u].store_stream(dst + col.e1);
    }
  }

  // The wave's heads, then the workgroup's waves, in a fixed order. Lanes that share a column have the same sum of it.
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

// Elements of a lane's half: the widest power of two, 16 bytes at most, that a half of the rotated columns and of
// the others (if there are others) holds. Backward up to 64 columns at most 4: with 8 half as many waves fit the
// registers (bf16 [16384, 48 heads], 40, 48, 56 and 64 columns: 65, 66, 70, 71 us with 8, 56, 58, 60, 63 with 4;
// 96 and 128 columns: 93, 105, and 109, 118).
int width_of(int dtype, int D, int R, bool backward) {
  int c = dtype == kF32 || (backward && D <= 64) ? 4 : 8;
  while (R / 2 < c || (R < D && (D - R) / 2 < c)) c >>= 1;
  return c;
}
bool ragged(int c, int D, int R) { return R / 2 % c != 0 || (D - R) / 2 % c != 0; }

// The lanes' shares of a call, and its items (waves' turns of kU).
int64_t lay_out(Args& a, int c) {
  a.rotating = (int)ceil_div(a.R / 2, c);
  a.lanes = a.rotating + (int)ceil_div((a.D - a.R) / 2, c);
  a.group_shift = 0;
  while ((1 << a.group_shift) < a.lanes) ++a.group_shift;
  const int heads = a.H + 2 * a.KH, at_a_time = kWave >> a.group_shift;
  a.heads_shift = 0;
  while ((1 << a.heads_shift) < heads && (1 << a.heads_shift) < at_a_time) ++a.heads_shift;
  if (2 << a.heads_shift <= at_a_time) {
    a.per = 0;
    return ceil_div(a.tokens, (int64_t)kU * (at_a_time >> a.heads_shift));
  }
  a.per = (int)ceil_div(heads, (int64_t)kU * at_a_time);
  return a.tokens * a.per;
}

template <int DT, int C, bool INTER, bool RAGGED>
int launch_fwd(Args a, void* out, hipStream_t st) {
  const int64_t items = lay_out(a, C);
  if (items >= (1 << 26)) return KRSI_ERR_BAD_SHAPE;  // grids of less than 2^32 threads
  auto launch = [&](auto few) {
    hipLaunchKernelGGL((qk_norm_rope_fwd<DT, C, INTER, RAGGED, decltype(few)::value>),
                       dim3((unsigned)ceil_div(items, kWaves)), dim3(kThreads), 0, st, a, items,
                       (typename Elem<DT>::T*)out);
  };
  a.per ? launch(std::false_type{}) : launch(std::true_type{});
  return launch_status();
}

template <int DT, int C, bool INTER, bool RAGGED>
int launch_bwd(Args a, const void* dy, void* dx, int64_t lddx, void* dwq, void* dwk, float* part, hipStream_t st) {
  using T = typename Elem<DT>::T;
  int blocks = 0;
  if (a.tokens > 0) {
    const int64_t items = lay_out(a, C), need = ceil_div(items, kWaves);
    if (items >= (1 << 26)) return KRSI_ERR_BAD_SHAPE;
    blocks = (int)(need < bwd_blocks(C) ? need : bwd_blocks(C));
    auto launch = [&](auto few) {
      hipLaunchKernelGGL((qk_norm_rope_bwd<DT, C, INTER, RAGGED, decltype(few)::value>), dim3((unsigned)blocks),
                         dim3(kThreads), 0, st, a, items, (const T*)dy, (T*)dx, lddx, part);
    };
    a.per ? launch(std::false_type{}) : launch(std::true_type{});
    const int rc = launch_status();
    if (rc != KRSI_OK) return rc;
  }
  hipLaunchKernelGGL((weight_sum<DT>), dim3((unsigned)(2 * a.D / kSumCols)), dim3(kSumThreads), 0, st,
                     (const float*)part, blocks, a.D, (T*)dwq, (T*)dwk);
  return launch_status();
}

// f(dtype, width, interleaved, ragged) as constants.
template <typename DT, typename C, typename F>
int with_forms(bool inter, bool rag, F&& f) {
  if constexpr (C::value > 1) {
    if (rag)
      return inter ? f(DT{}, C{}, std::true_type{}, std::true_type{}) : f(DT{}, C{}, std::false_type{}, std::true_type{});
  }
  return inter ? f(DT{}, C{}, std::true_type{}, std::false_type{}) : f(DT{}, C{}, std::false_type{}, std::false_type{});
}
template <int DT_, typename F>
int with_width(int c, bool inter, bool rag, F&& f) {
  using DT = std::integral_constant<int, DT_>;
  switch (c) {
    case 8:
      if constexpr (DT_ != kF32) return with_forms<DT, std::integral_constant<int, 8>>(inter, rag, f);
      return KRSI_ERR_UNSUPPORTED;
    case 4:
      return with_forms<DT, std::integral_constant<int, 4>>(inter, rag, f);
    case 2:
      return with_forms<DT, std::integral_constant<int, 2>>(inter, rag, f);
    default:
      return with_forms<DT, std::integral_constant<int, 1>>(inter, rag, f);
  }
}
template <typename F>
int with_kernel(int dtype, int D, int R, bool inter, bool backward, F&& f) {
  const int c = width_of(dtype, D, R, backward);
  const bool rag = ragged(c, D, R);
  switch (dtype) {
    case kF16:
      return with_width<kF16>(c, inter, rag, f);
    case kF32:
      return with_width<kF32>(c, inter, rag, f);
    default:
      return with_width<kBf16>(c, inter, rag, f);
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
  Args a{qkv, wq, wk, positions, rope, ld_qkv, tokens, table_rows, S, H, KH, D, R, position_bytes, 0, 0, 0, 0, 0, eps};
  return with_kernel(dtype, D, R, interleaved == 1, false, [&](auto dt, auto c, auto inter, auto rag) {
    return launch_fwd<dt(), c(), inter(), rag()>(a, out, as_stream(stream));
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
  Args a{qkv, wq, wk, positions, rope, ld_qkv, tokens, table_rows, S, H, KH, D, R, position_bytes, 0, 0, 0, 0, 0, eps};
  return with_kernel(dtype, D, R, interleaved == 1, true, [&](auto dt, auto c, auto inter, auto rag) {
    return launch_bwd<dt(), c(), inter(), rag()>(a, dout, dqkv, ld_dqkv, dwq, dwk, (float*)workspace, as_stream(stream));
  });
}

}  // extern "C"
