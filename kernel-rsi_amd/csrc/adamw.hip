// One AdamW step over any number of tensors in a few launches, and the norm of all gradients.
//   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  w = w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
// g: the gradient times min(1, max_norm / (norm + 1e-6)) where a norm is given; a norm that is not finite leaves everything
// as it is. w: the fp32 master where there is one, and the parameter its rounding; else the parameter itself. All
// arithmetic is fp32, 1 - b^t fp64.
//
// States of 8 bits: e4m3 codes of m and of s = sqrt(v), with an fp32 scale for each 256 elements of a tensor (the largest
// magnitude over 448, at least 2^-120). v changes by 1 - b2 in a step, far less than half a step of any 8-bit type: rounded
// to nearest it would stand still. So codes are rounded up or down at random, m right on average and s right on average in
// its square, v: between the codes k and k + 1 (in units of their spacing) t goes up with probability (t^2 - k^2) / (2 k + 1).
// A root above zero stays above zero, which keeps m / s within bounds. The random numbers are a function of the seed, the
// step, the tensor's number and the element's alone: multiplicative hashing (Knuth) with xor-shifts between.
//
// Bound by HBM: 28 bytes a parameter with 16-bit weights and gradients, masters and 32-bit states; 16 with 8-bit ones. 302 M
// such parameters: 1585 us (5.3 TB/s; plain streams, three read and two written, 5.0) and 905 (5.3); their norm 87 (6.8).
// 145 small tensors: 26 us of kernels, four launches. What a launch needs to know of each tensor comes as an argument by
// value, so nothing is copied to the device beforehand and a captured launch holds its own copy.
#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

#include "chunks.h"
#include "krsi_device.h"
#include "krsi_internal.h"

namespace krsi {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;        // elements that share a scale
// Elements per workgroup of the step: one pass of its lanes with 8-bit states, two with 32-bit ones (302 M parameters, 8-bit
// states: 951 us, workgroups of 8192 1045; both before stores went through the caches).
constexpr int kStepChunk = 4096;
constexpr int kNormChunk = 16384;  // and of the norm, all of whose loads are out at once

// The tensors of a launch, as many as the 4 KB of its arguments hold: P pointers each, its first workgroup of the launch and
// its number in the list.
template <int P>
struct Items {
  static constexpr int kMost = 3840 / (8 * P + 16);
  int32_t first[kMost], number[kMost];
  int64_t n[kMost];
  void* p[kMost][P];
  int32_t count;
};
// Pointers of a step: the four of every tensor, then its master's and its scales', where there are any.
constexpr int kParam = 0, kGrad = 1, kM = 2, kV = 3;
template <bool MASTER, bool SCALES>
constexpr int kPointers = 4 + (MASTER ? 1 : 0) + (SCALES ? 1 : 0);

// What a step needs of a tensor, from the first launch.
struct Factor {
  float rate;   // lr / (1 - b1^t)
  float root;   // 1 / sqrt(1 - b2^t)
  float share;  // of the gradient
  float decay;  // 1 - lr wd
  uint32_t key, go;
  uint32_t pad[2];
};

__device__ __forceinline__ uint32_t mixed(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x6A09E667u;  // the fractions of the roots of 2 and 3
  h = (h ^ (h >> 15)) * 0xBB67AE85u;
  return h ^ (h >> 16);
}
constexpr uint32_t kGolden = 0x9E3779B1u;
__device__ __forceinline__ uint32_t with_word(uint32_t key, uint32_t word) { return mixed(key * 3u + word * kGolden + 1u); }

// The launch's tensor that workgroup b works on. The lanes look at all of them at once: one after the other, each look at the
// arguments waited for the one before it (a small launch took 8 us).
template <int P>
__device__ __forceinline__ int find(const Items<P>& t, int b) {
  const int lane = threadIdx.x & (kWave - 1);
  int before = 0;
#pragma unroll
  for (int i = 0; i < Items<P>::kMost; i += kWave) {
    const int at = min(i + lane, Items<P>::kMost - 1);
    before += __popcll(__ballot(i + lane < t.count && t.first[at] <= b));
  }
  return __builtin_amdgcn_readfirstlane(before - 1);
}

// Pointers that come in a structure are taken for generic ones; these accesses are of global memory.
template <typename T>
using Global = __attribute__((address_space(1))) T;
template <typename T>
__device__ __forceinline__ Global<T>* global(const void* p) {
  return (Global<T>*)(uintptr_t)p;
}

// N consecutive elements of any alignment (N a multiple of a chunk's), or the first `some` of them.
// A lane's 32 or 64 bytes of an fp32 tensor meet their neighbours' in the caches, so loads and stores go through them
// (302 M parameters, 8-bit states: 929 us; stores past them 951, loads too 1350).
template <int DT, int N, bool FULL>
__device__ __forceinline__ void load(const void* p, int64_t i, int some, float* f) {
  using El = Elem<DT>;
  const auto* at = global<const typename El::T>(p) + i;
  if constexpr (FULL) {
#pragma unroll
    for (int q = 0; q < N; q += El::E) {
      const u32x4 c = *(Global<const u32x4_any>*)(at + q);
      El::unpack(c, f + q);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = j < some ? El::load(at[j]) : 0.f;
  }
}
template <int DT, int N, bool FULL>
__device__ __forceinline__ void store(void* p, int64_t i, int some, const float* f) {
  using El = Elem<DT>;
  auto* at = global<typename El::T>(p) + i;
  if constexpr (FULL) {
#pragma unroll
    for (int q = 0; q < N; q += El::E) *(Global<u32x4_any>*)(at + q) = El::pack(f + q);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < some) at[j] = El::store(f[j]);
  }
}

// ------------------------------------------------------------------- norm
template <int DT>
__global__ __launch_bounds__(kThreads) void norm_parts(const Items<1> items, float* __restrict__ part) {
  using El = Elem<DT>;
  __shared__ float red[kThreads / kWave];
  const int which = find(items, blockIdx.x);
  const void* const grad = items.p[which][0];
  const int64_t at = (int64_t)((int)blockIdx.x - items.first[which]) * kNormChunk, end = min(at + kNormChunk, items.n[which]);
  float sum[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) sum[j] = 0.f;
  const int64_t whole = at + (end - at) / 8 * 8;
#pragma unroll 8
  for (int64_t i = at + 8 * threadIdx.x; i < whole; i += 8 * kThreads) {
    float f[8];
#pragma unroll
    for (int q = 0; q < 8; q += El::E) {  // read once, past the caches (604 MB: 118 us through them, 105 so)
      const u32x4 c = __builtin_nontemporal_load((Global<const u32x4_any>*)(global<const typename El::T>(grad) + i + q));
      El::unpack(c, f + q);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] += f[j] * f[j];
  }
  if (threadIdx.x < end - whole) {
    const float f = Elem<DT>::load(global<const typename Elem<DT>::T>(grad)[whole + threadIdx.x]);
    sum[0] += f * f;
  }
  float s = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
  s = wave_sum(s);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// The root of the parts' sum, in every thread of the workgroup: the same bits wherever it is formed.
__device__ __forceinline__ float joined(const float* __restrict__ part, int64_t n, double* red) {
  double s = 0;
#pragma unroll 16
  for (int64_t i = threadIdx.x; i < n; i += kThreads) s += part[i];
  red[threadIdx.x] = s;
  __syncthreads();
#pragma unroll
  for (int w = kThreads / 2; w > 0; w /= 2) {
    if (threadIdx.x < (unsigned)w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  return (float)sqrt(red[0]);
}
__global__ __launch_bounds__(kThreads) void norm_join(const float* __restrict__ part, int64_t n, float* __restrict__ norm) {
  __shared__ double red[kThreads];
  const float v = joined(part, n, red);
  if (threadIdx.x == 0) *norm = v;
}

// ------------------------------------------------------------------- step
constexpr int kMaskWords = 896;
struct Mask {
  uint32_t word[kMaskWords];  // bit i: tensor i of this launch's range has a gradient
};

__global__ __launch_bounds__(kThreads) void step_factors(const Mask mask, int base, int count, int32_t* __restrict__ steps,
                                                         Factor* __restrict__ out, const float* __restrict__ lr_at, float lr,
                                                         double log1, double log2, float wd, float* __restrict__ norm,
                                                         const float* __restrict__ part, int64_t parts, float max_norm,
                                                         uint32_t seed) {
  __shared__ double red[kThreads];
  float total = 0.f;
  if (part) {  // the norm is formed here, by each workgroup
    total = joined(part, parts, red);
    if (base == 0 && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  } else if (norm) {
    total = *norm;
  }
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= count) return;
  Factor f{};
  if ((mask.word[i / 32] >> (i % 32) & 1u) && fabsf(total) <= 3.402823466e38f) {
    const int32_t t = steps[base + i] + 1;
    steps[base + i] = t;
    if (lr_at) lr = *lr_at;
    f.rate = (float)((double)lr / -expm1(t * log1));
    f.root = (float)(1.0 / sqrt(-expm1(t * log2)));
    f.share = norm ? fminf(max_norm / (total + 1e-6f), 1.f) : 1.f;
    f.decay = 1.f - lr * wd;
    f.key = with_word(with_word(mixed(seed), (uint32_t)t), (uint32_t)(base + i));
    f.go = 1;
  }
  out[base + i] = f;
}

// Below kSmall a root is taken of kUp times the number and multiplied by kDown.
constexpr float kSmall = 0x1p-64f, kUp = 0x1p64f, kDown = 0x1p-32f;

struct Rule {
  float b1, c1, b2, c2, eps;  // c: 1 - b, formed in fp64
};

// The stored master's own rounding is the parameter: kept apart from the arithmetic, which the compiler would otherwise
// round to fp16 in one step with it.
template <int N>
__device__ __forceinline__ void settled(float* w) {
#pragma unroll
  for (int j = 0; j < N; ++j) asm volatile("" : "+v"(w[j]));
}

template <int PT, int GT, bool MASTER, bool FULL>
__device__ __forceinline__ void eight32(void* const* p, const Factor& f, const Rule& k, int64_t i, int some) {
  float g[8], m[8], v[8], w[8];
  load<GT, 8, FULL>(p[kGrad], i, some, g);
  load<kF32, 8, FULL>(p[kM], i, some, m);
  load<kF32, 8, FULL>(p[kV], i, some, v);
  if constexpr (MASTER)
    load<kF32, 8, FULL>(p[4], i, some, w);
  else
    load<PT, 8, FULL>(p[kParam], i, some, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = g[j] * f.share;
    m[j] = m[j] * k.b1 + x * k.c1;
    v[j] = v[j] * k.b2 + (x * x) * k.c2;
    // The hardware's root takes a subnormal v for zero: a small one is scaled by 2^64, and its root back.
    const bool small = v[j] < kSmall;
    const float d = __builtin_amdgcn_sqrtf(v[j] * (small ? kUp : 1.f)) * (small ? f.root * kDown : f.root) + k.eps;
    w[j] = w[j] * f.decay - f.rate * m[j] * __builtin_amdgcn_rcpf(d);
  }
  store<kF32, 8, FULL>(p[kM], i, some, m);
  store<kF32, 8, FULL>(p[kV], i, some, v);
  if constexpr (MASTER) {
    settled<8>(w);
    store<kF32, 8, FULL>(p[4], i, some, w);
  }
  store<PT, 8, FULL>(p[kParam], i, some, w);
}

template <int PT, int GT, bool MASTER>
__global__ __launch_bounds__(kThreads) void step32(const Items<kPointers<MASTER, false>> items,
                                                   const Factor* __restrict__ factors, const Rule k) {
  const int which = find(items, blockIdx.x);
  const Factor f = factors[items.number[which]];
  if (!f.go) return;
  void* const* const p = items.p[which];
  const int64_t at = (int64_t)((int)blockIdx.x - items.first[which]) * kStepChunk, n = items.n[which];
#pragma unroll 1
  for (int s = 0; s < kStepChunk / (8 * kThreads); ++s) {
    const int64_t i = at + 8 * (s * kThreads + (int)threadIdx.x), left = n - i;
    if (left <= 0) return;
    if (left >= 8)
      eight32<PT, GT, MASTER, true>(p, f, k, i, 8);
    else
      eight32<PT, GT, MASTER, false>(p, f, k, i, (int)left);
  }
}

// The largest of the 16 lanes of a DPP row, in all of them.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));  // rotations by 1, 2, 4, 8
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));
}
// NaN where the largest magnitude is infinite or NaN (the maximum is of integers, so NaN stays).
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float t = __uint_as_float(top);
  return __uint_as_float(max(__float_as_uint(t * (1.0f / 448.0f) + t * 0.f), 0x03800000u));  // 2^-120
}

// The spacing of e4m3 at a value's size, 2^(max(e, -6) - 3), and its reciprocal.
__device__ __forceinline__ uint32_t spacing_bits(float a) {
  return max(__float_as_uint(a) & 0x7f800000u, 121u << 23) - (3u << 23);
}

__device__ __forceinline__ float rounded_m(float a, uint32_t h) {
  const uint32_t s = spacing_bits(a);
  const float k = floorf(a * __uint_as_float((254u << 23) - s) + (float)(h & 0xffffu) * (1.0f / 65536.0f));
  return fminf(fmaxf(k * __uint_as_float(s), -448.f), 448.f);
}
__device__ __forceinline__ float rounded_root(float b, uint32_t h) {
  const uint32_t s = spacing_bits(b);
  const float t = b * __uint_as_float((254u << 23) - s), low = floorf(t);
  const bool up = (t - low) * (t + low) > (float)(h >> 16) * (1.0f / 65536.0f) * (2.f * low + 1.f) || (low == 0.f && t > 0.f);
  return fminf((low + (up ? 1.f : 0.f)) * __uint_as_float(s), 448.f);
}

// Sixteen codes from p, zeros past `some`.
template <bool FULL>
__device__ __forceinline__ u32x4 load_codes(const void* p, int64_t i, int some) {
  if constexpr (FULL) return *(Global<const u32x4_any>*)(global<const uint8_t>(p) + i);
  u32x4 c{0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < some) c[j / 4] |= (uint32_t)global<const uint8_t>(p)[i + j] << (8 * (j % 4));
  return c;
}
template <bool FULL>
__device__ __forceinline__ void store_codes(void* p, int64_t i, int some, const u32x4& c) {
  if constexpr (FULL) {
    *(Global<u32x4_any>*)(global<uint8_t>(p) + i) = c;
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < some) global<uint8_t>(p)[i + j] = (uint8_t)(c[j / 4] >> (8 * (j % 4)));
  }
}
template <bool HIGH>
__device__ __forceinline__ void two_values(uint32_t codes, float* f) {
  const auto v = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, HIGH);
  f[0] = v[0];
  f[1] = v[1];
}
__device__ __forceinline__ uint32_t four_codes(const float* f) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
}

// The correctly rounded root: the hardware's is a unit off at most, and the residuals of its neighbours say which it is.
// Small numbers are scaled: the hardware takes subnormal ones for zero, and their residuals would be lost (302 M parameters,
// 8-bit states: 895 us so, 927 without, 915 with a branch around it).
__device__ __forceinline__ float exact_root(float x) {
  const bool small = x < kSmall;
  x *= small ? kUp : 1.f;
  const float s = __builtin_amdgcn_sqrtf(x);
  const float below = __uint_as_float(__float_as_uint(s) - 1u), above = __uint_as_float(__float_as_uint(s) + 1u);
  float r = __builtin_fmaf(-below, s, x) <= 0.f ? below : s;
  r = __builtin_fmaf(-above, s, x) > 0.f ? above : r;
  return r * (small ? kDown : 1.f);
}

// 16 elements a lane: a DPP row of 16 lanes has a scale's 256. The states are formed as the formula says it, each operation
// rounded by itself (no fused ones) and the root correctly: a last bit decides now and then which code is stored.
template <int PT, int GT, bool MASTER, bool FULL>
__device__ __forceinline__ void sixteen8(void* const* p, const Factor& f, const Rule& k, int64_t i, int some, int64_t block,
                                         int64_t blocks, uint32_t key) {
#pragma clang fp contract(off)
  Global<float>* const scales = global<float>(p[MASTER ? 5 : 4]) + block;
  const float ms = scales[0], rs = scales[blocks];
  u32x4 mc = load_codes<FULL>(p[kM], i, some), rc = load_codes<FULL>(p[kV], i, some);
  float g[16], w[16], m[16], r[16];
  load<GT, 16, FULL>(p[kGrad], i, some, g);
  if constexpr (MASTER)
    load<kF32, 16, FULL>(p[4], i, some, w);
  else
    load<PT, 16, FULL>(p[kParam], i, some, w);
  uint32_t mtop = 0, rtop = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    two_values<false>(mc[q], m + 4 * q);
    two_values<true>(mc[q], m + 4 * q + 2);
    two_values<false>(rc[q], r + 4 * q);
    two_values<true>(rc[q], r + 4 * q + 2);
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float x = g[j] * f.share, old = r[j] * rs;
    m[j] = (m[j] * ms) * k.b1 + x * k.c1;
    r[j] = exact_root((old * old) * k.b2 + (x * x) * k.c2);
    w[j] = w[j] * f.decay - f.rate * m[j] * __builtin_amdgcn_rcpf(r[j] * f.root + k.eps);
    mtop = max(mtop, __float_as_uint(m[j]) & 0x7fffffffu);
    rtop = max(rtop, __float_as_uint(r[j]) & 0x7fffffffu);
  }
  if constexpr (MASTER) {
    settled<16>(w);
    store<kF32, 16, FULL>(p[4], i, some, w);
  }
  store<PT, 16, FULL>(p[kParam], i, some, w);
  const float mscale = scale_of(row_max(mtop)), rscale = scale_of(row_max(rtop));
  if (threadIdx.x % 16 == 0) {
    scales[0] = mscale;
    scales[blocks] = rscale;
  }
  const float minv = 1.0f / mscale, rinv = 1.0f / rscale;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const uint32_t h = mixed((uint32_t)(i + j) * kGolden + key);
    m[j] = rounded_m(m[j] * minv, h);
    r[j] = rounded_root(r[j] * rinv, h);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    mc[q] = four_codes(m + 4 * q);
    rc[q] = four_codes(r + 4 * q);
  }
  store_codes<FULL>(p[kM], i, some, mc);
  store_codes<FULL>(p[kV], i, some, rc);
}

template <int PT, int GT, bool MASTER>
__global__ __launch_bounds__(kThreads) void step8(const Items<kPointers<MASTER, true>> items,
                                                  const Factor* __restrict__ factors, const Rule k) {
  const int which = find(items, blockIdx.x);
  const Factor f = factors[items.number[which]];
  if (!f.go) return;
  void* const* const p = items.p[which];
  const int64_t n = items.n[which], blocks = (n + kBlock - 1) / kBlock;
  const int64_t at = (int64_t)((int)blockIdx.x - items.first[which]) * kStepChunk;
  const uint32_t key = with_word(f.key, (uint32_t)(at >> 32));
#pragma unroll 1
  for (int s = 0; s < kStepChunk / (16 * kThreads); ++s) {
    const int64_t i = at + 16 * (s * kThreads + (int)threadIdx.x), block = i / kBlock, left = n - i;
    if (block >= blocks) return;  // whole rows of lanes
    // A row of lanes is whole or not as one, for its maximum.
    if ((block + 1) * kBlock <= n)
      sixteen8<PT, GT, MASTER, true>(p, f, k, i, 16, block, blocks, key);
    else
      sixteen8<PT, GT, MASTER, false>(p, f, k, i, (int)max((int64_t)0, left), block, blocks, key);
  }
}

bool known_dtype(int32_t dt) { return dt == kBf16 || dt == kF16 || dt == kF32; }
constexpr int64_t kMostElements = INT64_C(1) << 35;
constexpr int32_t kMostTensors = 1 << 20;

int check_sizes(const int64_t* sizes, int32_t count) {
  if (count < 0 || count > kMostTensors) return KRSI_ERR_BAD_SHAPE;
  if (count && !sizes) return KRSI_ERR_NULL_POINTER;
  int64_t total = 0;
  for (int32_t i = 0; i < count; ++i) {
    if (sizes[i] < 0 || sizes[i] > kMostElements) return KRSI_ERR_BAD_SHAPE;
    total += sizes[i];
    if (total > kMostElements) return KRSI_ERR_BAD_SHAPE;
  }
  return KRSI_OK;
}

// Workgroups of a launch: its threads stay below 2^32.
constexpr int64_t kMostGroups = (INT64_C(1) << 24) - 1;
static_assert(kMostElements / kStepChunk <= kMostGroups, "a tensor fits a launch");

// Calls launch(items, workgroups) for the listed tensors, in as few launches as their number and sizes allow.
// add(i, pointers) fills in tensor i's pointers, or says that it has no part.
template <int P, typename Add, typename Launch>
int in_launches(const int64_t* sizes, int32_t count, int64_t chunk, Add&& add, Launch&& launch) {
  Items<P> t;
  t.count = 0;
  int64_t groups = 0;
  auto flush = [&] {
    if (t.count) launch(t, (unsigned)groups);
    t.count = 0;
    groups = 0;
  };
  for (int32_t i = 0; i < count; ++i) {
    const int64_t need = ceil_div(sizes[i], chunk);
    void* p[P];
    if (!need || !add(i, p)) continue;
    if (t.count == Items<P>::kMost || groups + need > kMostGroups) flush();
    for (int k = 0; k < P; ++k) t.p[t.count][k] = p[k];
    t.n[t.count] = sizes[i];
    t.first[t.count] = (int32_t)groups;
    t.number[t.count++] = i;
    groups += need;
  }
  flush();
  return launch_status();
}

int64_t norm_groups(const int64_t* sizes, int32_t count) {
  int64_t n = 0;
  for (int32_t i = 0; i < count; ++i) n += ceil_div(sizes[i], kNormChunk);
  return n;
}

// The parts of the gradients' norm.
int launch_norm_parts(const void* const* grads, const int64_t* sizes, int32_t count, float* part, int32_t dtype, hipStream_t st,
                      int64_t* parts) {
  *parts = 0;
  return in_launches<1>(
      sizes, count, kNormChunk,
      [&](int32_t i, void** p) {
        p[0] = const_cast<void*>(grads[i]);
        return grads[i] != nullptr;
      },
      [&](const Items<1>& t, unsigned groups) {
        const auto kernel = dtype == kF16 ? norm_parts<kF16> : dtype == kF32 ? norm_parts<kF32> : norm_parts<kBf16>;
        hipLaunchKernelGGL(kernel, dim3(groups), dim3(kThreads), 0, st, t, part + *parts);
        *parts += groups;
      });
}

struct Lists {
  void* const* params;
  const void* const* grads;
  void *const *m, *const *v;
  float *const *masters, *const *scales;
  const int64_t* sizes;
  int32_t count;
  const Factor* factors;
  Rule rule;
  hipStream_t st;
};

template <int BITS, int PT, int GT, bool MASTER>
int launch_step(const Lists& a) {
  constexpr int P = kPointers<MASTER, BITS == 8>;
  return in_launches<P>(
      a.sizes, a.count, kStepChunk,
      [&](int32_t i, void** p) {
        p[kParam] = a.params[i], p[kGrad] = const_cast<void*>(a.grads[i]), p[kM] = a.m[i], p[kV] = a.v[i];
        if (MASTER) p[4] = a.masters[i];
        if (BITS == 8) p[P - 1] = a.scales[i];
        return a.grads[i] != nullptr;
      },
      [&](const Items<P>& t, unsigned groups) {
        if constexpr (BITS == 8)
          hipLaunchKernelGGL((step8<PT, GT, MASTER>), dim3(groups), dim3(kThreads), 0, a.st, t, a.factors, a.rule);
        else
          hipLaunchKernelGGL((step32<PT, GT, MASTER>), dim3(groups), dim3(kThreads), 0, a.st, t, a.factors, a.rule);
      });
}
template <int BITS, int PT, int GT>
int launch_step(const Lists& a) {
  return a.masters ? launch_step<BITS, PT, GT, true>(a) : launch_step<BITS, PT, GT, false>(a);
}
template <int BITS>
int launch_step(const Lists& a, int32_t pt, int32_t gt) {
  if (pt == kF32) return launch_step<BITS, kF32, kF32, false>(a);
  if (pt == kBf16) return gt == kBf16 ? launch_step<BITS, kBf16, kBf16>(a) : launch_step<BITS, kBf16, kF32>(a);
  return gt == kF16 ? launch_step<BITS, kF16, kF16>(a) : launch_step<BITS, kF16, kF32>(a);
}

bool in_range(double v) { return std::isfinite(v) && std::fabs(v) <= 3.0e38; }

}  // namespace
}  // namespace krsi

extern "C" {

size_t krsi_grad_norm_workspace_bytes(const int64_t* sizes, int32_t count) {
  using namespace krsi;
  if (check_sizes(sizes, count) != KRSI_OK) return 0;
  return align256((size_t)(norm_groups(sizes, count) + 1) * sizeof(float));
}

int krsi_grad_norm(const void* const* grads, const int64_t* sizes, int32_t count, float* norm, void* workspace,
                   size_t workspace_bytes, int32_t dtype, void* stream) {
  using namespace krsi;
  if (!known_dtype(dtype)) return KRSI_ERR_UNSUPPORTED;
  int rc = check_sizes(sizes, count);
  if (rc != KRSI_OK) return rc;
  if (!norm || (count && !grads)) return KRSI_ERR_NULL_POINTER;
  if (!workspace || workspace_bytes < krsi_grad_norm_workspace_bytes(sizes, count)) return KRSI_ERR_WORKSPACE;
  if (!aligned16(workspace)) return KRSI_ERR_MISALIGNED;
  float* part = (float*)workspace;
  const hipStream_t st = as_stream(stream);
  int64_t parts;
  rc = launch_norm_parts(grads, sizes, count, part, dtype, st, &parts);
  if (rc != KRSI_OK) return rc;
  hipLaunchKernelGGL(norm_join, dim3(1), dim3(kThreads), 0, st, (const float*)part, parts, norm);
  return launch_status();
}

size_t krsi_adamw_workspace_bytes(const int64_t* sizes, int32_t count) {
  using namespace krsi;
  if (check_sizes(sizes, count) != KRSI_OK) return 0;
  return align256((size_t)count * sizeof(Factor)) + align256((size_t)(norm_groups(sizes, count) + 1) * sizeof(float));
}

int krsi_adamw_step(void* const* params, const void* const* grads, void* const* exp_avgs, void* const* exp_avg_sqs,
                    float* const* masters, float* const* scales, const int64_t* sizes, int32_t count, int32_t* steps,
                    const float* lr_at, float lr, double beta1, double beta2, float eps, float weight_decay,
                    float* norm, int32_t norm_given, float max_norm, uint32_t seed, int32_t state_bits, int32_t dtype,
                    int32_t grad_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace krsi;
  if (!known_dtype(dtype) || (grad_dtype != dtype && grad_dtype != kF32) || (masters && dtype == kF32))
    return KRSI_ERR_UNSUPPORTED;
  if ((state_bits != 8 && state_bits != 32) || (state_bits == 8) != (scales != nullptr)) return KRSI_ERR_UNSUPPORTED;
  int rc = check_sizes(sizes, count);
  if (rc != KRSI_OK) return rc;
  // A subnormal eps has no reciprocal in fp32: an element that never had a gradient would step by 0 times infinity.
  if ((!lr_at && !in_range(lr)) || !in_range(eps) || eps < 0 || (eps > 0 && eps < 0x1p-126f) || !in_range(weight_decay) ||
      !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || (norm && !(max_norm >= 0)) || norm_given < 0 || norm_given > 1)
    return KRSI_ERR_BAD_SCALE;
  if (count == 0) return KRSI_OK;
  if (!params || !grads || !exp_avgs || !exp_avg_sqs || !steps) return KRSI_ERR_NULL_POINTER;
  if (!workspace || workspace_bytes < krsi_adamw_workspace_bytes(sizes, count)) return KRSI_ERR_WORKSPACE;
  if (!aligned16(workspace)) return KRSI_ERR_MISALIGNED;
  // Nothing that is written twice, or meets what else is written: two workgroups would race on it.
  struct Span {
    uintptr_t begin, end;
    bool operator<(const Span& o) const { return begin < o.begin; }
  };
  const std::unique_ptr<Span[]> spans(new (std::nothrow) Span[5 * (size_t)count]);
  if (!spans) return KRSI_ERR_TOO_LARGE;
  const int64_t width = dtype == kF32 ? 4 : 2, state = state_bits / 8;
  int64_t used = 0;
  auto written = [&](const void* p, int64_t bytes) { spans[used++] = Span{(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes}; };
  for (int32_t i = 0; i < count; ++i) {
    if (!grads[i] || !sizes[i]) continue;
    if (!params[i] || !exp_avgs[i] || !exp_avg_sqs[i] || (masters && !masters[i]) || (scales && !scales[i]))
      return KRSI_ERR_NULL_POINTER;
    written(params[i], sizes[i] * width);
    written(exp_avgs[i], sizes[i] * state);
    written(exp_avg_sqs[i], sizes[i] * state);
    if (masters) written(masters[i], sizes[i] * 4);
    if (scales) written(scales[i], 8 * ceil_div(sizes[i], kBlock));
  }
  std::sort(spans.get(), spans.get() + used);
  for (int64_t i = 1; i < used; ++i)
    if (spans[i].begin < spans[i - 1].end) return KRSI_ERR_BAD_SHAPE;

  Factor* factors = (Factor*)workspace;
  float* part = (float*)((char*)workspace + align256((size_t)count * sizeof(Factor)));
  const hipStream_t st = as_stream(stream);
  const bool norm_here = norm && !norm_given;
  int64_t parts = 0;
  // An error that an earlier call has left is not this one's: reported after the first launches, it would have the caller make
  // the step again.
  (void)hipGetLastError();
  if (norm_here) {
    rc = launch_norm_parts(grads, sizes, count, part, grad_dtype, st, &parts);
    if (rc != KRSI_OK) return rc;
  }
  for (int32_t base = 0; base < count; base += 32 * kMaskWords) {
    const int32_t here = std::min(count - base, 32 * kMaskWords);
    Mask mask{};
    for (int32_t i = 0; i < here; ++i)
      if (grads[base + i]) mask.word[i / 32] |= 1u << (i % 32);
    hipLaunchKernelGGL(step_factors, dim3((unsigned)ceil_div(here, kThreads)), dim3(kThreads), 0, st, mask, base, here, steps,
                       factors, lr_at, lr, std::log(beta1), std::log(beta2), weight_decay, norm,
                       norm_here ? (const float*)part : nullptr, parts, max_norm, seed);
  }
  rc = launch_status();
  if (rc != KRSI_OK) return rc;
  const Rule rule{(float)beta1, (float)(1 - beta1), (float)beta2, (float)(1 - beta2), eps};
  const Lists a{params, grads, exp_avgs, exp_avg_sqs, masters, scales, sizes, count, factors, rule, st};
  return state_bits == 8 ? launch_step<8>(a, dtype, grad_dtype) : launch_step<32>(a, dtype, grad_dtype);
}

}  // extern "C"
