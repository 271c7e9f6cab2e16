// Products of 16-bit matrices on MFMA v_mfma_f32_16x16x32, fp32 accumulate, as one stream of stages per workgroup.
//   out[m, n] = sum_k a[m, k] b[n, k]
// Each operand lies in memory with the summed index contiguous (rows) or the output index contiguous (TR: row k
// holds all m or n).
//   * A workgroup of WM x WN waves computes (16 RB WM) x (16 CB WN) outputs, a wave 16 RB x 16 CB of them.
//   * The sum goes in stages of 64 through double-buffered LDS, memory -> LDS directly, 16-byte chunks swizzled
//     so that operand reads (128-bit rows; transposed 64-bit where TR) do not conflict.
//   * One barrier per stage, before its last products, whose operands are in registers by then: they cover the
//     barrier, the requests of the stage after the next and the first reads of the next stage.
//   * Persistent: workgroup b takes tiles b, b + grid, ... as one stream, so that a tile's epilogue covers the
//     first loads of the next tile.
//   * What lies past an end reads as zero (buffer range check).
#pragma once

#include <type_traits>

#include "krsi_device.h"
#include "lds_dma.h"
#include "relpos_common.h"

namespace krsi {

constexpr int kStage = 64;           // summed index per stage
constexpr uint32_t kPastEnd = 0x7ffffff0u;  // past every resource

// Every vector memory request and LDS access of the wave done, then the workgroup's barrier.
__device__ __forceinline__ void wait_and_sync() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Position of 16-byte chunk j of staged row r is j ^ swizzle: rows of 8 chunks (the summed index contiguous) for
// 128-bit reads of 16 rows; rows of 16 chunks or more (TR) for transposed 64-bit reads of rows 0-3 and 8-11 (or
// 4-7 and 12-15) of 16 x 2 chunks.
template <bool TR>
__device__ __forceinline__ int stage_swizzle(int r) {
  return TR ? ((r & 3) | ((r >> 3) & 1) << 2) << 1 : (r >> 1) & 7;
}

// All sizes fit 31 bits (in 64 the loop's scalars did not fit their registers); element offsets take 64.
struct Operand {
  const uint16_t* p;
  int ld;      // elements between rows
  int extent;  // of the output index
};

template <int WM, int WN, int RB, int CB>
struct StreamTile {
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int kRows = 16 * RB * WM, kCols = 16 * CB * WN;
  static constexpr int kA = kRows * kStage, kB = kCols * kStage;  // 16-bit elements of a staged tile
  static constexpr int kADma = kA / 8 / kThreads, kBDma = kB / 8 / kThreads, kDma = kADma + kBDma;
  static constexpr int kPerCu = 160 * 1024 / (4 * (kA + kB));     // workgroups whose two buffers a CU holds
  static constexpr int kLds = 2 * (kA + kB);
  static_assert(kA / 8 % kThreads == 0 && kB / 8 % kThreads == 0, "whole chunks per thread");
};

// The tiles of a product, in an order that keeps what an XCD has in flight on few row and column blocks: each XCD
// takes a contiguous range of tiles, which walk a group's row blocks, then the columns. Parts of a split sum are
// whole ranges of their own.
struct Tiles {
  int nrb, ncb, splits, per, stages;  // row and column blocks, parts of the sum, stages of a part and in all
  int total;
};
constexpr int kTileGroup = 4;

struct TileAt {
  int m0, n0, split, s0, s1;  // stages [s0, s1)
};
template <int ROWS, int COLS>
__device__ __forceinline__ TileAt tile_at(const Tiles& t, int v) {
  const int vv = xcd_tile(v, t.total), tiles = t.nrb * t.ncb, split = vv / tiles, tile = vv - split * tiles;
  const int per_group = kTileGroup * t.ncb, grp = tile / per_group, in_grp = tile - grp * per_group;
  const int gsz = min(kTileGroup, t.nrb - grp * kTileGroup);
  return TileAt{(grp * kTileGroup + in_grp % gsz) * ROWS, in_grp / gsz * COLS, split, split * t.per,
                min(t.stages, (split + 1) * t.per)};
}

// Calls epilogue(tile, acc) for every tile of this workgroup: acc[i][j][r] is row 16 (RB wr + i) + l16, column
// 16 (CB wc + j) + 4 g + r of the tile, for lane 16 g + l16 of wave (wr, wc). The grid is the tiles, or fewer
// where every part of the sum has two stages at least. lds: Tl::kLds elements on a 512-byte boundary.
template <int DT, bool TRA, bool TRB, int WM, int WN, int RB, int CB, typename Epilogue>
__device__ __forceinline__ void stream_products(const Operand a, const Operand b, int sum, const Tiles tiles,
                                                uint16_t* lds, Epilogue&& epilogue) {
  using Tl = StreamTile<WM, WN, RB, CB>;
  uint16_t *const As = lds, *const Bs = lds + 2 * Tl::kA;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, l16 = lane & 15;
  const int wr = wave / WN, wc = wave % WN;
  const int wv = __builtin_amdgcn_readfirstlane(wave);

  using TagA = std::bool_constant<TRA>;
  using TagB = std::bool_constant<TRB>;
  // Chunk q = i * threads + tid of a staged tile: row q / chunks of it. Request i's rows lie a whole number of
  // swizzle periods (16 rows) below request 0's, so one byte offset per lane serves all requests of an operand, whose
  // resource starts i steps further on (a register per request cost spills in the products of two TR operands).
  constexpr int kAStep = TRA ? Tl::kThreads * 8 / Tl::kRows : Tl::kThreads * 8 / kStage;  // rows from request to request
  constexpr int kBStep = TRB ? Tl::kThreads * 8 / Tl::kCols : Tl::kThreads * 8 / kStage;
  static_assert(kAStep % 16 == 0 && kBStep % 16 == 0, "whole swizzle periods");
  auto offset = [&](auto tr, const Operand& o, int o0, int width) {
    constexpr bool TR = decltype(tr)::value;
    const int chunks = TR ? width / 8 : kStage / 8, r = tid / chunks;
    const int col = 8 * ((tid & (chunks - 1)) ^ stage_swizzle<TR>(r));
    return opaque(TR && o0 + col >= o.extent ? kPastEnd : (uint32_t)(r * o.ld + col) * 2u);
  };
  uint32_t aoff, boff;  // they depend on the tile only where TR meets the extent's end
  auto offsets_a = [&](const TileAt& t) { aoff = offset(TagA{}, a, t.m0, Tl::kRows); };
  auto offsets_b = [&](const TileAt& t) { boff = offset(TagB{}, b, t.n0, Tl::kCols); };
  // A stage's memory: base and bytes up to the operand's end (less than 2^31), none where the stage lies past it.
  struct Stage {
    const uint16_t *a, *b;
    int abytes, bbytes;
  };
  auto stage_of = [&](const TileAt& t, int st) {
    const int k0 = st * kStage, left = max(min(sum - k0, kStage), 0);
    Stage s;
    if constexpr (TRA) {
      s.a = a.p + (int64_t)k0 * a.ld + t.m0;
      s.abytes = 2 * (left * a.ld - t.m0);
    } else {
      s.a = a.p + (int64_t)t.m0 * a.ld + k0;
      s.abytes = 2 * (min(a.extent - t.m0, Tl::kRows) * a.ld - k0);
    }
    if constexpr (TRB) {
      s.b = b.p + (int64_t)k0 * b.ld + t.n0;
      s.bbytes = 2 * (left * b.ld - t.n0);
    } else {
      s.b = b.p + (int64_t)t.n0 * b.ld + k0;
      s.bbytes = 2 * (min(b.extent - t.n0, Tl::kCols) * b.ld - k0);
    }
    return s;
  };
  auto request = [&](const Stage& s, int buf, int i) {
    const bool of_a = i < Tl::kADma;
    const int k = of_a ? i : i - Tl::kADma;
    const int ahead = of_a ? k * kAStep * a.ld : k * kBStep * b.ld;
    const int left = (of_a ? s.abytes : s.bbytes) - 2 * ahead;
    uint16_t* const to = of_a ? As + buf * Tl::kA : Bs + buf * Tl::kB;
    dma16(make_rsrc((of_a ? s.a : s.b) + ahead, (uint32_t)max(left, 0)), of_a ? aoff : boff,
          (uint32_t)(uintptr_t)(lds_void*)(to + (k * Tl::kThreads + 64 * wv) * 8));
  };

  // Operand reads of k-step s (32 of the stage's 64): outputs 16 o + l16, summed indices 32 s + 8 g .. + 7. A TR
  // read's chunk differs from that of o = 0 in bits of the address alone (rows are 256 bytes at least): one address
  // register per operand and an exclusive or per read, redone in each stage rather than kept.
  const int trow = 8 * g + (l16 >> 2), tsw = stage_swizzle<true>(trow), tb = (l16 & 3) >> 1, te = 4 * (l16 & 1);
  auto tr_base = [&](const uint16_t* t, int width) {
    return (uint32_t)(uintptr_t)(lds_void*)t + 2u * (uint32_t)(trow * width + 8 * (tb ^ tsw) + te);
  };
  uint32_t abase = 0, bbase = 0;
  if (TRA) abase = tr_base(As, Tl::kRows);
  if (TRB) bbase = tr_base(Bs, Tl::kCols);
  auto read_operand = [&](auto tr, const uint16_t* t, uint32_t base, int tile, int width, int buf, int s, int o) {
    if constexpr (decltype(tr)::value) {
      const uint32_t at = (base ^ (uint32_t)(o << 5)) + 2u * (uint32_t)(buf * tile + 32 * s * width);
      const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)at));
      const u32x2 y =
          __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(at + 8u * width)));
      return u32x4{x[0], x[1], y[0], y[1]};
    } else {
      return *reinterpret_cast<const u32x4*>(t + buf * tile + (16 * o + l16) * kStage +
                                             8 * ((4 * s + g) ^ stage_swizzle<false>(l16)));
    }
  };
  u32x4 ra[2][RB], rb[2][CB];
  constexpr int kReads = RB + CB, kProducts = RB * CB, kEvery = kProducts / Tl::kDma;
  static_assert(kReads * 2 <= kProducts && kEvery >= 2, "one k-step's products hold its reads and requests");
  auto read = [&](int s, int buf, int o) {
    if (o < CB)
      rb[s][o] = read_operand(TagB{}, Bs, bbase, Tl::kB, Tl::kCols, buf, s, CB * wc + o);
    else
      ra[s][o - CB] = read_operand(TagA{}, As, abase, Tl::kA, Tl::kRows, buf, s, RB * wr + o - CB);
  };
  f32x4 acc[RB][CB];
  // The products of k-step s, the reads of the next k-step after the even ones, in k-step 1 the requests of the
  // stage after the next spread over them. b first: a lane holds four columns of one row.
  auto products = [&](int s, int rbuf, const Stage& d) {
    if (TRA) abase = opaque(abase);
    if (TRB) bbase = opaque(bbase);
#pragma unroll
    for (int m = 0; m < kProducts; ++m) {
      const int i = m / CB, j = m % CB;
      acc[i][j] = mfma16x16x32<DT>(rb[s][j], ra[s][i], acc[i][j]);
      if (m % 2 == 0 && m / 2 < kReads) read(s ^ 1, rbuf, m / 2);
      if (s == 1 && m % kEvery == 1 && m / kEvery < Tl::kDma) request(d, rbuf ^ 1, m / kEvery);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  int v = blockIdx.x, buf = 0;
  if (v >= tiles.total) return;
  TileAt here = tile_at<Tl::kRows, Tl::kCols>(tiles, v);
  offsets_a(here);
  offsets_b(here);
  Stage st = stage_of(here, here.s0);
#pragma unroll
  for (int i = 0; i < Tl::kDma; ++i) request(st, 0, i);
  wait_and_sync();
#pragma unroll
  for (int o = 0; o < kReads; ++o) read(0, 0, o);
  TileAt next = tile_at<Tl::kRows, Tl::kCols>(tiles, min(v + (int)gridDim.x, tiles.total - 1));
  st = stage_of(here, here.s0 + 1);
#pragma unroll
  for (int i = 0; i < Tl::kDma; ++i) request(st, 1, i);
  for (;;) {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < CB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = here.s0; k < here.s1; ++k) {
      products(0, buf, st);
      wait_and_sync();
      // Stage k + 2 of this tile, or the first or second of the next one (after the last tile some tile's, not used).
      const bool in = k + 2 < here.s1;
      if (k + 2 == here.s1 || (k + 1 == here.s1 && here.s1 - here.s0 == 1)) {
        if (TRA) offsets_a(next);
        if (TRB) offsets_b(next);
      }
      st = in ? stage_of(here, k + 2) : stage_of(next, next.s0 + k + 2 - here.s1);
      products(1, buf ^ 1, st);
      buf ^= 1;
    }
    epilogue(here, acc);
    v += gridDim.x;
    if (v >= tiles.total) break;
    here = next;
    next = tile_at<Tl::kRows, Tl::kCols>(tiles, min(v + (int)gridDim.x, tiles.total - 1));
  }
  wait_and_sync();  // the unused requests land before the workgroup's LDS is released
}

// Workgroups of a launch over the tiles: what the chip holds at once, or all where a part of the sum has one stage.
template <typename Tl>
inline unsigned stream_grid(const Tiles& t) {
  const int last = t.stages - (t.splits - 1) * t.per;
  const int64_t resident = t.per >= 2 && last >= 2 ? 256 * Tl::kPerCu : t.total;
  return (unsigned)(t.total < resident ? t.total : resident);
}

}  // namespace krsi
