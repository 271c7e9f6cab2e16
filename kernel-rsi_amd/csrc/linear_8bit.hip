// Product of 8-bit rows: out[m, n] = T( xs[m] * ws[n] * sum_k x[m, k] w[n, k] ), x [rows, K] and w [F, K] e4m3 with an fp32
// scale per row of each, sums in fp32 on v_mfma_f32_16x16x128_f8f6f4 (scaled products: the unscaled form, the scales
// are the epilogue's).
//
// The instruction adds the products of eight consecutive bytes of a lane first, aligned to the largest of them and cut below
// 2^-13 of its power of two; everything else is added as fp32 (measured with single products). That is 1e-4 of an output of
// random rows, where the codes' rounding is 2.6e-2 of it and a bf16 output's 2^-9; the instruction has twice the rate of the
// 16x16x32 form.
// A lane of 16 g + l16 gives an operand 32 bytes of row l16. Which summed index a byte stands for only has to be the same in
// both operands, so a lane takes the 16-byte chunks g and 4 + g of 128 summed indices, whose reads do not conflict.
//
// Many rows: one stream of stages per workgroup, 128 summed indices each, memory -> LDS directly, double-buffered,
// persistent over tiles. Few rows: bound by the weight, which goes from memory to registers, once.
#include "krsi_device.h"
#include "krsi_internal.h"
#include "lds_dma.h"
#include "product_stream.h"

namespace krsi {
namespace {

constexpr int kStage8 = 128;  // summed indices (bytes) per stage
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Frag {
  u32x4 lo, hi;
};
__device__ __forceinline__ f32x4 product(const Frag& a, const Frag& b, const f32x4& c) {
  const i32x8 av{(int)a.lo[0], (int)a.lo[1], (int)a.lo[2], (int)a.lo[3], (int)a.hi[0], (int)a.hi[1], (int)a.hi[2], (int)a.hi[3]};
  const i32x8 bv{(int)b.lo[0], (int)b.lo[1], (int)b.lo[2], (int)b.lo[3], (int)b.hi[0], (int)b.hi[1], (int)b.hi[2], (int)b.hi[3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 0, 0, 0, 0, 0, 0);
}

// Four outputs of a row from column col on.
template <int OT>
__device__ __forceinline__ void store_out(typename Elem<OT>::T* out, int64_t row, int col, int F, const f32x4& acc, float xs,
                                          const float* ws) {
  using T = typename Elem<OT>::T;
  T* p = out + row * F + col;
  if (col + 4 <= F) {
    T v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = Elem<OT>::store(acc[r] * xs * ws[r]);
    __builtin_memcpy(p, v, sizeof(v));
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col + r < F) p[r] = Elem<OT>::store(acc[r] * xs * ws[r]);
  }
}
// The scales of columns col .. col + 3 (past the end: of the last).
__device__ __forceinline__ void load_scales(const float* ws, int col, int F, float* s) {
#pragma unroll
  for (int r = 0; r < 4; ++r) s[r] = ws[min(col + r, F - 1)];
}

// ---------------------------------------------------------------- many rows
template <int WM, int WN, int RB, int CB>
struct Tile8 {
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int kRows = 16 * RB * WM, kCols = 16 * CB * WN;
  static constexpr int kA = kRows * kStage8, kB = kCols * kStage8;  // bytes of a staged tile
  static constexpr int kADma = kA / 16 / kThreads, kBDma = kB / 16 / kThreads, kDma = kADma + kBDma;
  static constexpr int kPerCu = 160 * 1024 / (2 * (kA + kB));
  static constexpr int kStep = kThreads / 8;  // staged rows from request to request
  static_assert(kA / 16 % kThreads == 0 && kB / 16 % kThreads == 0 && kStep % 16 == 0 && RB % 4 == 0, "whole requests");
};

template <int OT, int WM, int WN, int RB, int CB>
__global__ __launch_bounds__(64 * WM * WN, (Tile8<WM, WN, RB, CB>::kPerCu * WM * WN / 4)) void
linear_8bit_stream(const uint8_t* __restrict__ x, const uint8_t* __restrict__ w, const float* __restrict__ xs,
                   const float* __restrict__ ws, typename Elem<OT>::T* __restrict__ out, int rows, int K, int F, const Tiles tiles) {
  using Tl = Tile8<WM, WN, RB, CB>;
  __shared__ __attribute__((aligned(512))) uint8_t lds[2 * (Tl::kA + Tl::kB)];
  uint8_t *const As = lds, *const Bs = lds + 2 * Tl::kA;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, l16 = lane & 15;
  const int wr = wave / WN, wc = wave % WN, wv = __builtin_amdgcn_readfirstlane(wave);

  // Chunk q = i * threads + tid of a staged tile is position q % 8 of row q / 8, which holds chunk (q % 8) ^ swizzle(row):
  // the same one in every request, whose rows lie whole swizzle periods apart. A tile's resource ends with its last row, and the
  // range check is of the lane's offset alone; the stage's place in the rows is the scalar offset, which is not checked, so
  // what lies past K in the last stage, and all of a stage past that one, is not asked for by an offset past any resource.
  constexpr int kOffs = Tl::kADma > Tl::kBDma ? Tl::kADma : Tl::kBDma;
  const int srow = tid >> 3, chunk = (tid & 7) ^ stage_swizzle<false>(srow);
  uint32_t off[kOffs];
#pragma unroll
  for (int i = 0; i < kOffs; ++i) off[i] = opaque((uint32_t)((srow + i * Tl::kStep) * K + 16 * chunk));
  const uint32_t past = opaque(16 * chunk >= K - (tiles.stages - 1) * kStage8 ? kPastEnd : 0u);

  struct Source {
    rsrc_t a, b;
  };
  auto source = [&](const TileAt& t) {
    return Source{make_rsrc(x + (int64_t)t.m0 * K, (uint32_t)(min(Tl::kRows, rows - t.m0) * K)),
                  make_rsrc(w + (int64_t)t.n0 * K, (uint32_t)(min(Tl::kCols, F - t.n0) * K))};
  };
  // Which stage of which tile, and what is past its end.
  struct Stage {
    Source s;
    int k0;
    uint32_t past;
  };
  auto stage_of = [&](const Source& s, int st) {
    return Stage{s, st * kStage8, st + 1 < tiles.stages ? 0u : st < tiles.stages ? past : kPastEnd};
  };
  auto request = [&](const Stage& s, int buf, int i) {
    const bool of_a = i < Tl::kADma;
    const int k = of_a ? i : i - Tl::kADma;
    uint8_t* const to = of_a ? As + buf * Tl::kA : Bs + buf * Tl::kB;
    dma16_at(of_a ? s.s.a : s.s.b, off[k] | s.past, s.k0,
             (uint32_t)(uintptr_t)(lds_void*)(to + (k * Tl::kThreads + 64 * wv) * 16));
  };

  // Row block o of a staged tile: rows 16 o + l16, chunks g and 4 + g. The swizzle depends on l16 alone.
  const int lo = l16 * kStage8 + 16 * (g ^ stage_swizzle<false>(l16)), hi = l16 * kStage8 + 16 * ((4 + g) ^ stage_swizzle<false>(l16));
  auto frag = [&](const uint8_t* t, int o) {
    return Frag{*reinterpret_cast<const u32x4*>(t + 16 * o * kStage8 + lo), *reinterpret_cast<const u32x4*>(t + 16 * o * kStage8 + hi)};
  };
  Frag a[4], b[CB];  // row block i of the stage is in a[i % 4]
  auto read_a = [&](int i, int buf) { a[i % 4] = frag(As + buf * Tl::kA, RB * wr + i); };
  auto read_b = [&](int j, int buf) { b[j] = frag(Bs + buf * Tl::kB, CB * wc + j); };
  f32x4 acc[RB][CB];

  // The products of row blocks 2 p and 2 p + 1, b by b. The reads of the pair after, and with the last pair, which only
  // needs registers, the next stage's first pair and each b after its last use, and the requests of the stage after that.
  constexpr int kProducts = 2 * CB;
  auto pair = [&](int p, int buf, const Stage& d) {
    const bool last = p == RB / 2 - 1;
#pragma unroll
    for (int m = 0; m < kProducts; ++m) {
      const int j = m / 2, i = 2 * p + m % 2;
      acc[i][j] = product(b[j], a[i % 4], acc[i][j]);
      if (m < 2) read_a(last ? m : 2 * p + 2 + m, last ? buf ^ 1 : buf);
      if (last && m % 2 == 1) read_b(j, buf ^ 1);
#pragma unroll
      for (int q = 0; q < Tl::kDma; ++q)
        if (last && q * kProducts / Tl::kDma == m) request(d, buf, q);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  int v = blockIdx.x, buf = 0;
  if (v >= tiles.total) return;
  TileAt here = tile_at<Tl::kRows, Tl::kCols>(tiles, v);
  Source cur = source(here);
  Stage st = stage_of(cur, 0);
#pragma unroll
  for (int i = 0; i < Tl::kDma; ++i) request(st, 0, i);
  wait_and_sync();
  TileAt next = tile_at<Tl::kRows, Tl::kCols>(tiles, min(v + (int)gridDim.x, tiles.total - 1));
  Source nxt = source(next);
  st = stage_of(cur, 1);
#pragma unroll
  for (int i = 0; i < Tl::kDma; ++i) request(st, 1, i);
  read_a(0, 0);
  read_a(1, 0);
#pragma unroll
  for (int j = 0; j < CB; ++j) read_b(j, 0);
  for (;;) {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < CB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < tiles.stages; ++k) {
#pragma unroll
      for (int p = 0; p < RB / 2 - 1; ++p) pair(p, buf, st);
      wait_and_sync();
      // Stage k + 2 of this tile, or the first or second of the next one (after the last tile some tile's, not used).
      const bool in = k + 2 < tiles.stages;
      st = stage_of(Source{in ? cur.a : nxt.a, in ? cur.b : nxt.b}, in ? k + 2 : k + 2 - tiles.stages);
      pair(RB / 2 - 1, buf, st);
      buf ^= 1;
    }
#pragma unroll
    for (int j = 0; j < CB; ++j) {
      const int col = here.n0 + 16 * (CB * wc + j) + 4 * g;
      float s[4];
      load_scales(ws, min(col, F - 1), F, s);
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const int row = here.m0 + 16 * (RB * wr + i) + l16;
        if (row < rows && col < F) store_out<OT>(out, row, col, F, acc[i][j], xs[row], s);
      }
    }
    v += gridDim.x;
    if (v >= tiles.total) break;
    here = next;
    cur = nxt;
    next = tile_at<Tl::kRows, Tl::kCols>(tiles, min(v + (int)gridDim.x, tiles.total - 1));
    nxt = source(next);
  }
  wait_and_sync();  // the unused requests land before the workgroup's LDS is released
}

// ----------------------------------------------------------------- few rows
// A workgroup has 16 CB columns and all rows (16 RB at most); its waves take stages in turn, and their sums are added in the
// order of the waves. Stages past the end read as zero.
constexpr int kFewWaves = 8;

template <int OT, int RB, int CB>
__global__ __launch_bounds__(64 * kFewWaves) void linear_8bit_few(const uint8_t* __restrict__ x, const uint8_t* __restrict__ w,
                                                                  const float* __restrict__ xs, const float* __restrict__ ws,
                                                                  typename Elem<OT>::T* __restrict__ out, int rows, int K,
                                                                  int F) {
  __shared__ f32x4 part[kFewWaves][RB * CB][64];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), n0 = blockIdx.x * 16 * CB;
  const rsrc_t xr = make_rsrc(x, (uint32_t)(rows * K)), wr = make_rsrc(w + (int64_t)n0 * K, (uint32_t)(min(16 * CB, F - n0) * K));
  auto frag = [&](rsrc_t r, int o, int k0) {
    const int at = (16 * o + l16) * K, lo = k0 + 16 * g, hi = lo + 64;
    return Frag{__builtin_amdgcn_raw_buffer_load_b128(r, lo < K ? at + lo : (int)kPastEnd, 0, 0),
                __builtin_amdgcn_raw_buffer_load_b128(r, hi < K ? at + hi : (int)kPastEnd, 0, 0)};
  };
  f32x4 acc[RB][CB];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < CB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k0 = wave * kStage8; k0 < K; k0 += kFewWaves * kStage8) {
    Frag a[RB], b[CB];
#pragma unroll
    for (int j = 0; j < CB; ++j) b[j] = frag(wr, j, k0);
#pragma unroll
    for (int i = 0; i < RB; ++i) a[i] = frag(xr, i, k0);
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < CB; ++j) acc[i][j] = product(b[j], a[i], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < CB; ++j) part[wave][i * CB + j][lane] = acc[i][j];
  __syncthreads();
  for (int o = wave; o < RB * CB; o += kFewWaves) {
    f32x4 sum = part[0][o][lane];
#pragma unroll
    for (int q = 1; q < kFewWaves; ++q) sum += part[q][o][lane];
    const int row = 16 * (o / CB) + l16, col = n0 + 16 * (o % CB) + 4 * g;
    if (row >= rows || col >= F) continue;
    float s[4];
    load_scales(ws, col, F, s);
    store_out<OT>(out, row, col, F, sum, xs[row], s);
  }
}

struct Call {
  const uint8_t *x, *w;
  const float *xs, *ws;
  void* out;
  int64_t rows;
  int K, F;
  hipStream_t st;
};

constexpr int kCus = 256;
constexpr int kFewRows = 64;

template <int OT, int RB, int CB>
int launch_few(const Call& c) {
  hipLaunchKernelGGL((linear_8bit_few<OT, RB, CB>), dim3((unsigned)ceil_div(c.F, 16 * CB)), dim3(64 * kFewWaves), 0, c.st, c.x,
                     c.w, c.xs, c.ws, (typename Elem<OT>::T*)c.out, (int)c.rows, c.K, c.F);
  return launch_status();
}

template <int OT, int WM, int WN, int RB, int CB>
int launch_stream(const Call& c) {
  using Tl = Tile8<WM, WN, RB, CB>;
  Tiles t;
  t.nrb = (int)ceil_div(c.rows, Tl::kRows);
  t.ncb = (int)ceil_div(c.F, Tl::kCols);
  t.splits = 1;
  t.per = t.stages = (int)ceil_div(c.K, kStage8);
  if ((int64_t)t.nrb * t.ncb > (1 << 23)) return KRSI_ERR_UNSUPPORTED;
  t.total = t.nrb * t.ncb;
  // The stream reaches one tile ahead, two stages: with one stage per tile every workgroup takes one tile.
  const int resident = t.stages >= 2 ? kCus * Tl::kPerCu : t.total;
  hipLaunchKernelGGL((linear_8bit_stream<OT, WM, WN, RB, CB>), dim3((unsigned)(t.total < resident ? t.total : resident)),
                     dim3(Tl::kThreads), 0, c.st, c.x, c.w, c.xs, c.ws, (typename Elem<OT>::T*)c.out, (int)c.rows, c.K, c.F, t);
  return launch_status();
}

template <int OT>
int launch(const Call& c) {
  if (c.rows <= 16) return launch_few<OT, 1, 1>(c);
  if (c.rows <= 32) return launch_few<OT, 2, 1>(c);
  if (c.rows <= kFewRows) return launch_few<OT, 4, 2>(c);
  // Rounds of the chip, by a tile's work: 256 x 256, 128 x 128 (two to a CU), 64 x 128 (three).
  const int64_t large = ceil_div(ceil_div(c.rows, 256) * ceil_div(c.F, 256), kCus) * 8;
  const int64_t mid = ceil_div(ceil_div(c.rows, 128) * ceil_div(c.F, 128), 2 * kCus) * 5;
  const int64_t small = ceil_div(ceil_div(c.rows, 64) * ceil_div(c.F, 128), 3 * kCus) * 4;
  if (large <= mid && large <= small) return launch_stream<OT, 2, 4, 8, 4>(c);
  if (mid <= small) return launch_stream<OT, 2, 2, 4, 4>(c);
  return launch_stream<OT, 1, 4, 4, 2>(c);
}

}  // namespace
}  // namespace krsi

extern "C" {

int krsi_linear_8bit(const void* x, const void* w, const float* x_scale, const float* w_scale, void* out, int64_t rows,
                     int32_t k, int32_t f, int32_t out_dtype, void* stream) {
  using namespace krsi;
  if (out_dtype != kBf16 && out_dtype != kF16 && out_dtype != kF32) return KRSI_ERR_UNSUPPORTED;
  if (rows < 0 || k <= 0 || f <= 0) return KRSI_ERR_BAD_SHAPE;
  // Byte offsets into a tile stay below 2^31, element offsets of rows and columns below 2^31.
  if (k % 16 || k > (1 << 20) || rows > (1 << 23) || f > (1 << 23)) return KRSI_ERR_UNSUPPORTED;
  if (ceil_div(rows, 64) * ceil_div(f, 128) > (1 << 23)) return KRSI_ERR_UNSUPPORTED;
  if (rows == 0) return KRSI_OK;
  if (!x || !w || !x_scale || !w_scale || !out) return KRSI_ERR_NULL_POINTER;
  if (!aligned16(x) || !aligned16(w)) return KRSI_ERR_MISALIGNED;
  const Call c{(const uint8_t*)x, (const uint8_t*)w, x_scale, w_scale, out, rows, k, f, as_stream(stream)};
  return out_dtype == kF16 ? launch<kF16>(c) : out_dtype == kF32 ? launch<kF32>(c) : launch<kBf16>(c);
}

}  // extern "C"
