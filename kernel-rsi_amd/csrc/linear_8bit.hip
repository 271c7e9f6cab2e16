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
// Many rows: one stream of stages per workgroup, 128 summed indices each, memory -> LDS directly, persistent over tiles. A
// stage's products go in pairs of row blocks; its barrier stands before the last pair, whose operands are in registers by
// then. LDS holds the stages that DA and DB say, so that a request has that many stages' time (256 x 256 tiles: three of x and
// two of w, all of a CU's 160 KB). 8192 x 8192 x 8192, random rows: 365 to 391 us (3010 to 2810 TFLOP/s), the matrix cores busy 77 % of
// the cycles at 1.86 GHz. In turn with it on one card at 391: the vendor's library 342 with one scale for all, 384 with a scale per
// row; zeros 285, 256 and 317. A step that cost: registers that went to memory in the loop, and a load waited for in it, each
// waited for every request in flight.
// Few rows (64 at most): bound by the weight, which goes from memory to registers, once. One row, [8192, 4096]: 7.5 us (4.5
// TB/s; a read of as much takes 5.4), [28672, 8192]: 39.5 (5.9 TB/s). 33 to 64 rows: bound by the reads of x by every
// workgroup through L2 (x [48, 4112], w [5633, 4112]: 10.3 us).
// Few outputs of a long sum: the sum in parts, whose fp32 sums a second launch adds in their order (x [64, 8192], w [8192, 8192]:
// 27.2 us by the kernel for few rows, 33.2 by whole tiles, 19.9 in four parts; [512, 8192] x [1024, 8192]: 20.5 -> 15.0).
#include "chunks.h"
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

// Four outputs of a row at p, or as many as are `left` before its end.
template <int OT>
__device__ __forceinline__ void store_out(typename Elem<OT>::T* p, int left, const f32x4& acc, float xs, const float* ws) {
  using T = typename Elem<OT>::T;
  if (left >= 4) {
    T v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = Elem<OT>::store(acc[r] * xs * ws[r]);
    __builtin_memcpy(p, v, sizeof(v));
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < left) p[r] = Elem<OT>::store(acc[r] * xs * ws[r]);
  }
}
// Two column blocks' outputs of a row, eight columns to a lane: lane groups 0 and 2 get columns 0 - 7 and 8 - 15 of the first
// block, 1 and 3 of the second, so that a store writes 64 bytes of each row. Stored past the caches, they leave the tiles in flight in L2
// (8192 x 4096 x 16384: 483 us with eight bytes a lane, 464 so, 423 past the caches).
template <int OT>
__device__ __forceinline__ void store_two(bool live, typename Elem<OT>::T* p, const f32x4& a, const f32x4& b, float xs, const float* sa,
                                          const float* sb) {
  static_assert(sizeof(*p) == 2, "16-bit outputs");
  uint32_t v[2][2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const uint32_t lo = Elem<OT>::pack2(a[2 * q] * xs * sa[2 * q], a[2 * q + 1] * xs * sa[2 * q + 1]);
    const uint32_t hi = Elem<OT>::pack2(b[2 * q] * xs * sb[2 * q], b[2 * q + 1] * xs * sb[2 * q + 1]);
    const auto r = __builtin_amdgcn_permlane16_swap(lo, hi, false, false);  // lo's odd groups with hi's even ones
    v[0][q] = r[0];
    v[1][q] = r[1];
  }
  if (live) __builtin_nontemporal_store(u32x4{v[0][0], v[0][1], v[1][0], v[1][1]}, reinterpret_cast<u32x4_any*>(p));
}
// The scales of columns col .. col + 3 (past the end: of the last).
__device__ __forceinline__ void load_scales(const float* ws, int col, int F, float* s) {
#pragma unroll
  for (int r = 0; r < 4; ++r) s[r] = ws[min(col + r, F - 1)];
}

// ---------------------------------------------------------------- many rows
// Every LDS access of the wave done and all of its vector memory requests but the newest N, then the workgroup's barrier.
template <int N>
__device__ __forceinline__ void wait_for() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// DA and DB: the stages of x and of w that LDS holds.
template <int WM, int WN, int RB, int CB, int DA, int DB>
struct Tile8 {
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int kRows = 16 * RB * WM, kCols = 16 * CB * WN;
  static constexpr int kA = kRows * kStage8, kB = kCols * kStage8;  // bytes of a staged tile
  static constexpr int kADma = kA / 16 / kThreads, kBDma = kB / 16 / kThreads, kDma = kADma + kBDma;
  static constexpr int kLds = DA * kA + DB * kB;
  static constexpr int kPerCu = 160 * 1024 / kLds;
  static constexpr int kStep = kThreads / 8;  // staged rows from request to request
  // At the barrier that lets the next stage be read: requests that may still be on their way, those for later ones.
  static constexpr int kLater = (DB - 2) * kDma + (DA > DB ? kADma : 0);
  static_assert(DB >= 2 && (DA == DB || (DA == 3 && DB == 2)) && RB >= 4 && DA * kDma < 64, "requests that the wait can count");
  static_assert(kA / 16 % kThreads == 0 && kB / 16 % kThreads == 0 && kStep % 16 == 0 && RB % 4 == 0, "whole requests");
};

// SPLIT: a tile of a part of the sum, whose fp32 sums go to `part` [splits, rows, F]; a workgroup takes one.
template <int OT, int WM, int WN, int RB, int CB, int DA, int DB, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN, (Tile8<WM, WN, RB, CB, DA, DB>::kPerCu * WM * WN / 4)) void
linear_8bit_stream(const uint8_t* __restrict__ x, const uint8_t* __restrict__ w, const float* __restrict__ xs,
                   const float* __restrict__ ws, typename Elem<OT>::T* __restrict__ out, float* __restrict__ part, int rows, int K, int F,
                   const Tiles tiles) {
  using Tl = Tile8<WM, WN, RB, CB, DA, DB>;
  __shared__ __attribute__((aligned(512))) uint8_t lds[Tl::kLds];
  uint8_t *const As = lds, *const Bs = lds + DA * Tl::kA;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, l16 = lane & 15;
  const int wr = wave / WN, wc = wave % WN, wv = __builtin_amdgcn_readfirstlane(wave), wru = wv / WN, wcu = wv % WN;
  const rsrc_t xsr = make_rsrc(xs, (uint32_t)rows * 4u), wsr = make_rsrc(ws, (uint32_t)F * 4u);

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
  // Request i of this thread for x's part of a stage, into the buffer at byte `to`, and for w's.
  auto request = [&](bool of_a, const Stage& s, int to, int i) {
    dma16_at(of_a ? s.s.a : s.s.b, off[i] | s.past, s.k0,
             (uint32_t)(uintptr_t)(lds_void*)((of_a ? As : Bs) + to + (i * Tl::kThreads + 64 * wv) * 16));
  };

  // Row block o of a staged tile: rows 16 o + l16, chunks g and 4 + g. The swizzle depends on l16 alone.
  const int lo = l16 * kStage8 + 16 * (g ^ stage_swizzle<false>(l16)), hi = l16 * kStage8 + 16 * ((4 + g) ^ stage_swizzle<false>(l16));
  auto frag = [&](const uint8_t* t, int o) {
    return Frag{*reinterpret_cast<const u32x4*>(t + 16 * o * kStage8 + lo), *reinterpret_cast<const u32x4*>(t + 16 * o * kStage8 + hi)};
  };
  Frag a[4], b[CB];  // row block i of the stage is in a[i % 4]
  auto read_a = [&](int i, int at) { a[i % 4] = frag(As + at, RB * wr + i); };
  auto read_b = [&](int j, int at) { b[j] = frag(Bs + at, CB * wc + j); };
  f32x4 acc[RB][CB];

  // Stage k's buffers are at a0 and b0, the next one's at a1 and b1, the one's before at ap.
  int ap = (DA - 1) * Tl::kA, a0 = 0, a1 = Tl::kA, b0 = 0, b1 = Tl::kB;
  // The products of row blocks 2 p and 2 p + 1, b by b. The reads of the pair after, and with the last pair, which only
  // needs registers, the next stage's first pair and each b after its last use, and the requests of w's stage k + DB. Where x's
  // ring is the longer one, its stage k - 1 + DA is asked for over the pairs before, into the buffer of stage k - 1, else
  // stage k + DA after w's: requests all in the last pair got in each other's way (8192 x 8192 x 8192: 407 us, so 379;
  // in that pair's first half 416). Equal rings would lose a stage's time by it (200 x 4096 x 4096: 12.1 us, 12.9).
  constexpr int kProducts = 2 * CB;
  constexpr bool kSpread = DA > DB;
  constexpr int kAhead = kSpread ? DA - 1 : DA;
  auto pair = [&](int p, const Stage& da, const Stage& db) {
    const bool last = p == RB / 2 - 1;
#pragma unroll
    for (int m = 0; m < kProducts; ++m) {
      const int j = m / 2, i = 2 * p + m % 2;
      acc[i][j] = product(b[j], a[i % 4], acc[i][j]);
      if (m < 2) read_a(last ? m : 2 * p + 2 + m, last ? a1 : a0);
      if (last && m % 2 == 1) read_b(j, b1);
#pragma unroll
      for (int q = 0; q < Tl::kBDma; ++q)
        if (last && q * kProducts / (kSpread ? Tl::kBDma : Tl::kDma) == m) request(false, db, b0, q);
#pragma unroll
      for (int q = 0; q < Tl::kADma; ++q)
        if (kSpread ? !last && q * (RB / 2 - 1) * kProducts / Tl::kADma == p * kProducts + m
                    : last && (Tl::kBDma + q) * kProducts / Tl::kDma == m)
          request(true, da, kSpread ? ap : a0, q);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  int v = blockIdx.x;
  if (v >= tiles.total) return;
  TileAt here = tile_at<Tl::kRows, Tl::kCols>(tiles, v);
  Source cur = source(here);
  TileAt next = tile_at<Tl::kRows, Tl::kCols>(tiles, min(v + (int)gridDim.x, tiles.total - 1));
  Source nxt = source(next);
  // Stage s of this tile, or where it is past its end, of the next one (after the last tile some tile's, not used).
  auto ahead = [&](int s) {
    if constexpr (SPLIT) return stage_of(cur, here.s0 + s < here.s1 ? here.s0 + s : tiles.stages);
    const bool in = s < tiles.stages;
    return stage_of(Source{in ? cur.a : nxt.a, in ? cur.b : nxt.b}, in ? s : s - tiles.stages);
  };
  // Stage by stage, so that the first may be read before the last are here.
#pragma unroll
  for (int s = 0; s < DA; ++s) {
    const Stage st = ahead(s);
#pragma unroll
    for (int i = 0; i < Tl::kBDma; ++i)
      if (s < DB) request(false, st, s * Tl::kB, i);
#pragma unroll
    for (int i = 0; i < Tl::kADma; ++i)
      if (s < kAhead) request(true, st, s * Tl::kA, i);
  }
  wait_for<(DB - 1) * Tl::kDma + (kAhead - DB) * Tl::kADma>();
  read_a(0, 0);
  read_a(1, 0);
#pragma unroll
  for (int j = 0; j < CB; ++j) read_b(j, 0);
  for (;;) {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < CB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int stages = SPLIT ? here.s1 - here.s0 : tiles.stages;
    for (int k = 0; k < stages; ++k) {
      const Stage db = ahead(k + DB), da = ahead(k + kAhead);
#pragma unroll
      for (int p = 0; p < RB / 2 - 1; ++p) pair(p, da, db);
      // After an epilogue, whose loads and stores are counted too, everything is waited for.
      if (k == 0 && v != (int)blockIdx.x)
        wait_for<0>();
      else
        wait_for<Tl::kLater>();
      pair(RB / 2 - 1, da, db);
      ap = a0, a0 = a1, b0 = b1;
      a1 = a1 + Tl::kA == DA * Tl::kA ? 0 : a1 + Tl::kA;
      b1 = b1 + Tl::kB == DB * Tl::kB ? 0 : b1 + Tl::kB;
    }
    if constexpr (SPLIT) {
      float* at = part + ((int64_t)here.split * rows + here.m0 + 16 * RB * wru) * F + here.n0 + 16 * CB * wcu;
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const bool live = l16 < rows - here.m0 - 16 * RB * wru - 16 * i;
#pragma unroll
        for (int j = 0; j < CB; ++j) {
          const int left = F - here.n0 - 16 * CB * wcu - 4 * g - 16 * j;
          float* p = at + (l16 * F + 4 * g) + 16 * j;
          if (live && left >= 4) {
            *reinterpret_cast<f32x4_any*>(p) = acc[i][j];
          } else if (live) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (r < left) p[r] = acc[i][j][r];
          }
        }
        at += 16 * (int64_t)F;
      }
      break;
    }
    // All scales first: loaded one by one between the stores, each waited for the requests in flight before it as well. One to a
    // lane, and given round by the lanes' exchange: in each lane that needs them they took seven registers more. What lies
    // past an end reads as zero. Places are a wave's own plus a lane's 32-bit offset: with a pointer for each row, the loop's
    // registers went to memory and back.
    const int m = here.m0 + 16 * RB * wru, n = here.n0 + 16 * CB * wcu;
    constexpr int kX = (16 * RB + 63) / 64, kW = (16 * CB + 63) / 64;
    uint32_t lx[kX], lw[kW];
#pragma unroll
    for (int i = 0; i < kX; ++i) lx[i] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(xsr, opaque(4 * (m + lane) + 256 * i), 0, 0);
#pragma unroll
    for (int j = 0; j < kW; ++j) lw[j] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(wsr, opaque(4 * (n + lane) + 256 * j), 0, 0);
    // Used here, on every path: a load that some path leaves unused is waited for where its register is next written, which
    // was in the loop over the stages, in each of them and for all requests in flight.
#pragma unroll
    for (int i = 0; i < kX; ++i) asm volatile("" : "+v"(lx[i]));
#pragma unroll
    for (int j = 0; j < kW; ++j) asm volatile("" : "+v"(lw[j]));
    const int lx4 = opaque(4 * l16), lw4 = opaque(16 * g);  // the lanes' addresses, four bytes each
    auto from = [&](uint32_t v, int l) { return __uint_as_float((uint32_t)__builtin_amdgcn_ds_bpermute(l, (int)v)); };
    typename Elem<OT>::T* at = out + (int64_t)m * F + n;
    const bool wide = OT != kF32 && n + 16 * CB <= F;  // all of the wave's columns are there
#pragma unroll
    for (int j = 0; j < CB; j += 2) {
      __builtin_amdgcn_sched_barrier(0);  // not all exchanges before the first store
      float sw[2][4];
#pragma unroll
      for (int r = 0; r < 8; ++r) sw[r / 4][r % 4] = from(lw[j / 4], lw4 + 64 * (j % 4 + r / 4) + 4 * (r % 4));
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const float sx = from(lx[i / 4], lx4 + 64 * (i % 4));
        const bool live = l16 < rows - m - 16 * i;
        typename Elem<OT>::T* to = at + (int64_t)(16 * i) * F + 16 * j;
        if constexpr (OT != kF32) {
          if (wide)  // every lane has its part in the exchange, also of a row that is not there
            store_two<OT>(live, to + (l16 * F + 16 * (g & 1) + 8 * (g >> 1)), acc[i][j], acc[i][j + 1], sx, sw[0], sw[1]);
        }
        if (!wide) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
            if (live) store_out<OT>(to + (l16 * F + 4 * g) + 16 * q, F - n - 4 * g - 16 * (j + q), acc[i][j + q], sx, sw[q]);
        }
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

// The parts' sum, in their order, times the scales: four columns a thread.
template <int OT>
__global__ __launch_bounds__(256) void linear_8bit_join(const float* __restrict__ part, const float* __restrict__ xs,
                                                        const float* __restrict__ ws, typename Elem<OT>::T* __restrict__ out,
                                                        int rows, int F, int splits) {
  const int col = 4 * (blockIdx.x * 256 + (int)threadIdx.x), row = blockIdx.y;
  if (col >= F) return;
  const int64_t at = (int64_t)row * F + col, step = (int64_t)rows * F;
  const float x = xs[row];
  if (col + 4 <= F) {
    f32x4 sum = *reinterpret_cast<const f32x4_any*>(part + at);
    for (int p = 1; p < splits; ++p) sum += *reinterpret_cast<const f32x4_any*>(part + p * step + at);
    const f32x4 w = *reinterpret_cast<const f32x4_any*>(ws + col);
    const float s[4] = {w[0], w[1], w[2], w[3]};
    store_out<OT>(out + at, 4, sum, x, s);
  } else {
    for (int r = 0; r < F - col; ++r) {
      float sum = part[at + r];
      for (int p = 1; p < splits; ++p) sum += part[p * step + at + r];
      out[at + r] = Elem<OT>::store(sum * x * ws[col + r]);
    }
  }
}

// ----------------------------------------------------------------- few rows
// A workgroup has 16 CB columns and all rows (16 RB at most); its waves take stages in turn, and their sums are added in the
// order of the waves. Stages past the end read as zero.
constexpr int kFewWaves = 8;

template <int OT, int RB, int CB, int U>
__global__ __launch_bounds__(64 * kFewWaves) void linear_8bit_few(const uint8_t* __restrict__ x, const uint8_t* __restrict__ w,
                                                                  const float* __restrict__ xs, const float* __restrict__ ws,
                                                                  typename Elem<OT>::T* __restrict__ out, int rows, int K,
                                                                  int F) {
  __shared__ f32x4 part[kFewWaves][RB * CB][64];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), n0 = blockIdx.x * 16 * CB;
  const rsrc_t xr = make_rsrc(x, (uint32_t)(rows * K)), wr = make_rsrc(w + (int64_t)n0 * K, (uint32_t)(min(16 * CB, F - n0) * K));
  // Both chunks of a row's stage at k0; one past K is not asked for (nor, by the resource, one past the rows).
  auto frag = [&](rsrc_t r, int o, int k0) {
    const int at = (16 * o + l16) * K, lo = k0 + 16 * g, hi = lo + 64;
    return Frag{__builtin_amdgcn_raw_buffer_load_b128(r, opaque(lo < K ? at + lo : (int)kPastEnd), 0, 0),
                __builtin_amdgcn_raw_buffer_load_b128(r, opaque(hi < K ? at + hi : (int)kPastEnd), 0, 0)};
  };
  f32x4 acc[RB][CB];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < CB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // U stages of a wave at a time, all loads before the products. Workgroups begin at different places of the rows, which they
  // would otherwise ask of the same part of L2 at once ([16, 4096] x [4096, 4096] 6.8 -> 5.8 us).
  const int iters = (K + U * kFewWaves * kStage8 - 1) / (U * kFewWaves * kStage8);
  int turn = (int)(blockIdx.x % (unsigned)iters);
  for (int it = 0; it < iters; ++it, turn = turn + 1 == iters ? 0 : turn + 1) {
    const int k0 = (turn * U * kFewWaves + wave) * kStage8;
    Frag a[U][RB], b[U][CB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < CB; ++j) b[u][j] = frag(wr, j, k0 + u * kFewWaves * kStage8);
#pragma unroll
      for (int i = 0; i < RB; ++i) a[u][i] = frag(xr, i, k0 + u * kFewWaves * kStage8);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < CB; ++j) acc[i][j] = product(b[u][j], a[u][i], acc[i][j]);
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
    store_out<OT>(out + (int64_t)row * F + col, F - col, sum, xs[row], s);
  }
}

struct Call {
  const uint8_t *x, *w;
  const float *xs, *ws;
  void* out;
  float* part;
  int64_t rows;
  int K, F;
  hipStream_t st;
};

constexpr int kCus = 256;
constexpr int kFewRows = 64;

template <int OT, int RB, int CB, int U>
int launch_few(const Call& c) {
  hipLaunchKernelGGL((linear_8bit_few<OT, RB, CB, U>), dim3((unsigned)ceil_div(c.F, 16 * CB)), dim3(64 * kFewWaves), 0, c.st, c.x,
                     c.w, c.xs, c.ws, (typename Elem<OT>::T*)c.out, (int)c.rows, c.K, c.F);
  return launch_status();
}

template <int OT, int WM, int WN, int RB, int CB, int DA, int DB, bool SPLIT = false>
int launch_stream(const Call& c, int splits = 1) {
  using Tl = Tile8<WM, WN, RB, CB, DA, DB>;
  Tiles t;
  t.nrb = (int)ceil_div(c.rows, Tl::kRows);
  t.ncb = (int)ceil_div(c.F, Tl::kCols);
  t.splits = splits;
  t.stages = (int)ceil_div(c.K, kStage8);
  t.per = (int)ceil_div(t.stages, splits);
  if ((int64_t)t.nrb * t.ncb > (1 << 23)) return KRSI_ERR_UNSUPPORTED;
  t.total = t.nrb * t.ncb * splits;
  // The stream reaches one tile ahead, DA stages: with fewer every workgroup takes one tile.
  const int resident = !SPLIT && t.stages >= DA ? kCus * Tl::kPerCu : t.total;
  hipLaunchKernelGGL((linear_8bit_stream<OT, WM, WN, RB, CB, DA, DB, SPLIT>),
                     dim3((unsigned)(t.total < resident ? t.total : resident)), dim3(Tl::kThreads), 0, c.st, c.x, c.w, c.xs,
                     c.ws, (typename Elem<OT>::T*)c.out, c.part, (int)c.rows, c.K, c.F, t);
  const int rc = launch_status();
  if (!SPLIT || rc != KRSI_OK) return rc;
  hipLaunchKernelGGL((linear_8bit_join<OT>), dim3((unsigned)ceil_div(c.F, 1024), (unsigned)c.rows), dim3(256), 0, c.st,
                     (const float*)c.part, c.xs, c.ws, (typename Elem<OT>::T*)c.out, (int)c.rows, c.F, splits);
  return launch_status();
}

// Which kernel a size takes, by its cost in hundredths of a us as measured.
enum Kind { kFew, kLarge, kMid, kSmall };
struct Plan {
  Kind kind;
  int splits;
};
Plan plan_of(int64_t rows, int K, int F) {
  const int64_t stages = ceil_div(K, kStage8);
  // Rounds of the chip, each its stages and an end. Two workgroups of the smaller tiles share a CU, and a round that gives each
  // CU one at most takes about half of a full one.
  auto cost = [&](int64_t tiles, int64_t depth, int full, int full_end, int part, int part_end) {
    const int64_t per = full == part ? kCus : 2 * kCus, last = tiles % per;
    return tiles / per * (full * depth + full_end) +
           (last == 0 ? 0 : last > kCus ? full * depth + full_end : part * depth + part_end);
  };
  auto tiles = [&](int m, int n) { return ceil_div(rows, m) * ceil_div(F, n); };
  Plan best{kLarge, 1};
  int64_t least = cost(tiles(256, 256), stages, 133, 800, 133, 800);
  auto consider = [&](int64_t c, Plan p) {
    if (c < least) least = c, best = p;
  };
  consider(cost(tiles(128, 128), stages, 102, 400, 55, 340), Plan{kMid, 1});
  consider(cost(tiles(64, 128), stages, 72, 350, 38, 290), Plan{kSmall, 1});
  // The sum in parts, each four stages at least, where that fills the chip: the parts' bytes both ways and a launch come on top.
  for (int s = 2; s <= 16; s *= 2) {
    const int64_t per = ceil_div(stages, s), parts = ceil_div(stages, per);
    if (per < 4 || tiles(64, 128) * parts > 2 * kCus) break;
    consider(cost(tiles(64, 128) * parts, per, 72, 350, 38, 290) + 300 + rows * F * parts * 8 / 40000, Plan{kSmall, (int)parts});
  }
  if (rows <= kFewRows) {
    const bool two = rows > 32 || (rows > 16 && F >= 32 * kCus);  // column blocks to a workgroup
    const int64_t wide = two ? 32 : 16, each = rows <= 16 ? 8 : rows > 32 ? 9 * rows / 16 : two ? 26 : 17;
    consider(250 + ceil_div(F, wide * kCus) * stages * each, Plan{kFew, 1});
  }
  return best;
}

template <int OT>
int launch(const Call& c) {
  const Plan p = plan_of(c.rows, c.K, c.F);
  switch (p.kind) {
    case kFew:
      // Two column blocks share their reads of x where that leaves a workgroup for each CU ([32, 4096] x [4096, 4096]: 8.0 us
      // with one, 9.5 with two; x [8192, 4096]: 13.4, 10.3).
      if (c.rows <= 16) return launch_few<OT, 1, 1, 2>(c);
      if (c.rows <= 32) return c.F >= 32 * kCus ? launch_few<OT, 2, 2, 2>(c) : launch_few<OT, 2, 1, 2>(c);
      return launch_few<OT, 4, 2, 1>(c);
    case kLarge: return launch_stream<OT, 2, 4, 8, 4, 3, 2>(c);
    case kMid: return launch_stream<OT, 2, 2, 4, 4, 3, 2>(c);
    default:
      return p.splits > 1 ? launch_stream<OT, 1, 4, 4, 2, 3, 3, true>(c, p.splits) : launch_stream<OT, 1, 4, 4, 2, 3, 3>(c);
  }
}

int check_sizes(int64_t rows, int32_t k, int32_t f) {
  if (rows < 0 || k <= 0 || f <= 0) return KRSI_ERR_BAD_SHAPE;
  // Byte offsets into a tile stay below 2^31, a launch's threads below 2^32.
  if (k % 16 || k > (1 << 20) || rows > (1 << 23) || f > (1 << 23)) return KRSI_ERR_UNSUPPORTED;
  if (ceil_div(rows, 64) * ceil_div(f, 128) > (1 << 23)) return KRSI_ERR_UNSUPPORTED;
  return KRSI_OK;
}

}  // namespace
}  // namespace krsi

extern "C" {

size_t krsi_linear_8bit_workspace_bytes(int64_t rows, int32_t k, int32_t f) {
  using namespace krsi;
  if (check_sizes(rows, k, f) != KRSI_OK || rows == 0) return 0;
  const Plan p = plan_of(rows, k, f);
  return p.splits > 1 ? align256((size_t)p.splits * rows * f * sizeof(float)) : 0;
}

int krsi_linear_8bit(const void* x, const void* w, const float* x_scale, const float* w_scale, void* out, void* workspace,
                     size_t workspace_bytes, int64_t rows, int32_t k, int32_t f, int32_t out_dtype, void* stream) {
  using namespace krsi;
  if (out_dtype != kBf16 && out_dtype != kF16 && out_dtype != kF32) return KRSI_ERR_UNSUPPORTED;
  const int rc = check_sizes(rows, k, f);
  if (rc != KRSI_OK) return rc;
  if (rows == 0) return KRSI_OK;
  if (!x || !w || !x_scale || !w_scale || !out) return KRSI_ERR_NULL_POINTER;
  if (!aligned16(x) || !aligned16(w)) return KRSI_ERR_MISALIGNED;
  const size_t need = krsi_linear_8bit_workspace_bytes(rows, k, f);
  if (need && (!workspace || workspace_bytes < need)) return KRSI_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return KRSI_ERR_MISALIGNED;
  const Call c{(const uint8_t*)x, (const uint8_t*)w, x_scale, w_scale, out, (float*)workspace, rows, k, f, as_stream(stream)};
  return out_dtype == kF16 ? launch<kF16>(c) : out_dtype == kF32 ? launch<kF32>(c) : launch<kBf16>(c);
}

}  // extern "C"
