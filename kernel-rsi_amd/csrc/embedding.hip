// Token embedding with scaling, and its gradient, for gfx950.
//   out[t, :]    = T(scale table[tok_t, :])                            a token outside [0, V): NaN
//   dtable[v, :] = T(scale sum of g[t, :] over the t with tok_t = v)   every row written, zero where there is none
// The sums are fp32, in an order that the tokens alone decide; no float atomics, so dtable is bitwise
// reproducible. Tokens outside [0, V) and the padding token have no part in them.
//
// What bounds both: HBM (forward: the named rows in, out; backward: g in, dtable out, most of whose rows are zeros).
// bf16 [32768, 4096], V 131072: forward 72 us, backward 302 (of 1.34 GB: 4.4 TB/s); [8191, 1024], V 32128: 5 and 33
// (of 83 MB), where group_tokens' latency and the last rows' sums are a half each; 500 tokens there: 2.4 and 23. From
// about 100000 tokens on, group_tokens' two passes over all tokens in each workgroup are the larger part.
//
// Backward in three launches:
//   group_tokens  one launch that sorts the positions by token, stably. Workgroup j owns the rows v = j (mod
//                 groups), so that neighbouring ids, of which the low ones are often the frequent ones, go to
//                 different workgroups. Each reads all tokens (from L2): it counts its own per row and
//                 wave in LDS and the tokens of lower groups (its offset), then places its positions in order.
//                 That is latency; the launch's other workgroups meanwhile write dtable's zeros, most of its bytes,
//                 as one stream whatever the rows' alignment.
//   sum_rows      rows of at most a piece of tokens, found from their first sorted place: a wave (or a part of one,
//                 where rows are short) adds them in order and writes the row; and, per piece of 16 or 32
//                 sorted places, fp32 partial sums of longer rows.
//   sum_pieces    longer rows: their pieces' partial sums, in order.
#include "chunks.h"
#include "krsi_device.h"
#include "krsi_internal.h"

namespace krsi {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kGroupThreads = 1024;
constexpr int kGroupWaves = kGroupThreads / kWave;
constexpr int kGroupRows = 1024;   // most rows of a group: one per thread in its scan, 64 KB of counters
constexpr int kGroups = 256;       // groups at least (fewer for fewer rows): a workgroup per CU
constexpr int kFillChunks = 8;     // 16-byte chunks of zeros that a thread of group_tokens writes: 128 KB per workgroup
// Sorted positions per piece, log2. Short pieces spread the frequent tokens' rows wider, and cost a partial row each.
// Where they cross depends on the ids, which the host does not know, more than on the columns. The backward with 16
// and with 32, us, bf16, V 32128, rows of 256 / 1024 / 4096: ids as frequent as 1 / id,
//   4096 tokens 21 / 25 / 75 and 24 / 29 / 85;  8192: 22 / 31 / 81 and 24 / 36 / 89;  12288: 27 / 38 / 87 and 28 / 43 / 92;
//   16384: 30 / 41 / 98 and 30 / 45 / 96;  24576: 39 / 53 / 125 and 36 / 49 / 114;
// half of the tokens one id, 4096: 27 / 31 / 78 and 23 / 29 / 86;  8192: 40 / 48 / 97 and 31 / 43 / 96;
//   12288: 55 / 64 / 113 and 42 / 55 / 102;  ids of one frequency: the same. Of the first kind 64 is slower than 32 from
// 2048 to 32768 tokens (1024 columns or more), and 8 slower than 16 from 8192 on.
int piece_shift_of(int64_t n) { return n <= 8192 ? 4 : 5; }
constexpr int kHeld = 8;           // tokens that a thread of group_tokens keeps from its count to its placing
constexpr int kSumWaves = 16;
constexpr int kSumPieces = 8;      // pieces whose rows a workgroup of sum_pieces looks after
constexpr int kSumCols = 256;      // columns per workgroup of sum_pieces

// A wave holds 64 >> shift rows at a time; chunk k of a lane is chunk lane_in_row + k (1 << shift) of the row.
// The last chunk of a row that no chunk divides ends at the row's end: both chunks' lanes have the same
// values in the columns that they share.
template <int C>
__device__ __forceinline__ int chunk_start(int c, int D) { return min(c * C, D - C); }

template <int DT, int C, int K>
__global__ __launch_bounds__(kThreads) void embedding_fwd(const void* __restrict__ tokens, int token_bytes,
                                                          const typename Elem<DT>::T* __restrict__ table,
                                                          typename Elem<DT>::T* __restrict__ out, int64_t n, int V,
                                                          int D, int nch, int shift, float scale) {
  const int lane = threadIdx.x & (kWave - 1), in_row = lane & ((1 << shift) - 1);
  const int64_t wave = (int64_t)blockIdx.x * kWaves + threadIdx.x / kWave;
  const int64_t t = (wave << (6 - shift)) + (lane >> shift);
  if (t >= n) return;
  const int64_t tok = load_index(tokens, token_bytes, t);
  const bool inside = tok >= 0 && tok < V;
  const auto* src = table + (inside ? tok : 0) * D;
  auto* dst = out + t * D;
  const int c0 = blockIdx.y * (K << shift) + in_row;
  Piece<DT, C> v[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = c0 + (k << shift);
    if (c < nch) v[k].load(src + chunk_start<C>(c, D));
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = c0 + (k << shift);
    if (c >= nch) continue;
    float f[C];
    v[k].get(f);
#pragma unroll
    for (int j = 0; j < C; ++j) f[j] = inside ? f[j] * scale : __builtin_nanf("");
    v[k].set(f);
    v[k].store_stream(dst + chunk_start<C>(c, D));  // bf16 [32768, 4096]: 82.5 -> 72 us
  }
}

// Positions grouped by token. order[i]: the position at sorted place i; row_of[i]: its token; of row v, start[v] and
// count[v]; *total: places in all.
struct Groups {
  int32_t *order, *row_of, *start, *count, *total;
  int piece_shift;
};

// Workgroups from `groups` on: zeros into [zeros, zeros + bytes), kFillChunks 16-byte chunks per thread between its
// unaligned ends.
__device__ __forceinline__ void write_zeros(char* zeros, int64_t bytes, int block) {
  const int64_t head = min((int64_t)(-(intptr_t)zeros & 15), bytes), chunks = (bytes - head) / 16;
  u32x4* p = reinterpret_cast<u32x4*>(zeros + head);
  const int64_t first = (int64_t)block * (kGroupThreads * kFillChunks) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < kFillChunks; ++k)
    if (first + k * kGroupThreads < chunks) __builtin_nontemporal_store(u32x4{0u, 0u, 0u, 0u}, p + first + k * kGroupThreads);
  if (block == 0 && threadIdx.x < 16) {
    const int64_t tail = head + chunks * 16 + threadIdx.x;
    if (threadIdx.x < head) zeros[threadIdx.x] = 0;
    if (tail < bytes) zeros[tail] = 0;
  }
}

__global__ __launch_bounds__(kGroupThreads) void group_tokens(const void* __restrict__ tokens, int token_bytes, int n,
                                                              int V, int group_shift, int64_t padding, Groups out,
                                                              char* __restrict__ zeros, int64_t bytes) {
  __shared__ int count[kGroupWaves][kGroupRows];
  __shared__ int sums[2][kGroupWaves];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int groups = 1 << group_shift, j = blockIdx.x, mask = groups - 1;
  if (j >= groups) {
    write_zeros(zeros, bytes, j - groups);
    return;
  }
  for (int w = 0; w < kGroupWaves; ++w) count[w][tid] = 0;
  // Each wave goes over a contiguous part of the tokens, so that order by wave, then by place in it, is theirs.
  const int per = (n + kGroupThreads - 1) / kGroupThreads * kWave;
  const int64_t first = (int64_t)wave * per;
  const int begin = (int)(first < n ? first : n), end = (int)(first + per < n ? first + per : n);
  int held[kHeld];
  auto load = [&](int i0) {  // the lane's tokens of kHeld rounds; -1: none, or one that is not counted
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int i = i0 + k * kWave + lane;
      const int64_t t = i < end ? load_index(tokens, token_bytes, i) : -1;
      held[k] = t >= 0 && t < V && t != padding ? (int)t : -1;
    }
  };
  load(begin);
  __syncthreads();
  int lower = 0;
  for (int i0 = begin; i0 < end; i0 += kHeld * kWave) {
    if (i0 != begin) load(i0);
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int t = held[k];
      lower += t >= 0 && (t & mask) < j;
      if (t >= 0 && (t & mask) == j) atomicAdd(&count[wave][t >> group_shift], 1);
    }
  }
  for (int m = kWave / 2; m >= 1; m >>= 1) lower += __shfl_xor(lower, m, kWave);
  if (lane == 0) sums[0][wave] = lower;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < kGroupWaves; ++w) base += sums[0][w];
  // Thread r: row r of the group. Exclusive sums over the waves, then over the rows.
  int all = 0;
  for (int w = 0; w < kGroupWaves; ++w) {
    const int c = count[w][tid];
    count[w][tid] = all;
    all += c;
  }
  int scan = all;  // inclusive over the wave's rows
  for (int m = 1; m < kWave; m <<= 1) {
    const int up = __shfl_up(scan, m, kWave);
    if (lane >= m) scan += up;
  }
  if (lane == kWave - 1) sums[1][wave] = scan;
  __syncthreads();
  int at = base + scan - all;
  for (int w = 0; w < wave; ++w) at += sums[1][w];
  for (int w = 0; w < kGroupWaves; ++w) count[w][tid] += at;
  const int64_t v = j + ((int64_t)tid << group_shift);
  if (v < V && all) {
    out.start[v] = at;
    out.count[v] = all;
  }
  if (j == groups - 1 && tid == kGroupThreads - 1) *out.total = at + all;
  __syncthreads();
  // The lanes of one row take consecutive places, in lane order.
  for (int i0 = begin; i0 < end; i0 += kHeld * kWave) {
    if (per > kHeld * kWave) load(i0);
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int t = held[k], row = t >> group_shift;
      const bool mine = t >= 0 && (t & mask) == j;
      uint64_t left = __ballot(mine);
      while (left) {
        const int leader = __builtin_ctzll(left);
        const int its_row = __builtin_amdgcn_readlane(row, leader);
        const uint64_t same = __ballot(mine && row == its_row);
        int place = 0;
        if (lane == leader) place = atomicAdd(&count[wave][row], __popcll(same));
        place = __builtin_amdgcn_readlane(place, leader);
        if (same >> lane & 1) {
          const int p = place + __popcll(same & ((uint64_t(1) << lane) - 1));
          out.order[p] = i0 + k * kWave + lane;
          out.row_of[p] = t;
        }
        left &= ~same;
      }
    }
  }
}

// acc[k][:] = sum over the sorted places [from, to) of the lane's chunks of g, in order. Batches of B places, whose
// positions and then rows are all requested before the first is added: one place after another is two memory
// latencies each (a piece of 32 rows: 30 us).
template <int DT, int C, int K, int B>
__device__ __forceinline__ void add_batch(float (&acc)[K][C], const typename Elem<DT>::T* g, const int32_t* order, int at,
                                          int D, int nch, int c0, int step) {
  Piece<DT, C> v[B][K];
  int pos[B];
#pragma unroll
  for (int i = 0; i < B; ++i) pos[i] = order[at + i];
#pragma unroll
  for (int i = 0; i < B; ++i)
#pragma unroll
    for (int k = 0; k < K; ++k) v[i][k].load(g + (int64_t)pos[i] * D + chunk_start<C>(min(c0 + k * step, nch - 1), D));
#pragma unroll
  for (int i = 0; i < B; ++i)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float f[C];
      v[i][k].get(f);
#pragma unroll
      for (int j = 0; j < C; ++j) acc[k][j] += f[j];
    }
}
template <int DT, int C, int K>
__device__ __forceinline__ void add_places(float (&acc)[K][C], const typename Elem<DT>::T* g, const int32_t* order,
                                           int from, int to, int D, int nch, int c0, int step) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < C; ++j) acc[k][j] = 0.f;
  constexpr int B = K >= 4 ? 4 : 8;
  for (; from + B <= to; from += B) add_batch<DT, C, K, B>(acc, g, order, from, D, nch, c0, step);
  for (; from + 2 <= to; from += 2) add_batch<DT, C, K, 2>(acc, g, order, from, D, nch, c0, step);
  if (from < to) add_batch<DT, C, K, 1>(acc, g, order, from, D, nch, c0, step);
}

// Workgroups below piece_blocks: a wave per piece, its parts of longer rows into part [pieces][2][D] (slot 0: of
// a row that starts at or before the piece's first place, slot 1: after it). The others: rows, by the sorted
// place that is a row's first.
template <int DT, int C, int K>
__global__ __launch_bounds__(kThreads) void sum_rows(const typename Elem<DT>::T* __restrict__ g, Groups in,
                                                     typename Elem<DT>::T* __restrict__ dtable,
                                                     float* __restrict__ part, int piece_blocks, int D, int nch,
                                                     int shift, float scale) {
  const int lane = threadIdx.x & (kWave - 1);
  const int wave_in_block = threadIdx.x / kWave;
  const int piece = 1 << in.piece_shift;
  float acc[K][C];
  if ((int)blockIdx.x < piece_blocks) {
    const int64_t p = (int64_t)blockIdx.x * kWaves + wave_in_block, a = p << in.piece_shift;
    const int total = *in.total;
    if (a >= total) return;
    const int from = (int)a, to = a + piece < total ? from + piece : total;
    const int head = in.row_of[from], tail = in.row_of[to - 1];
    const int c0 = blockIdx.y * (K * kWave) + lane;
    auto write = [&](int slot) {
      float* dst = part + (2 * p + slot) * D;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = c0 + k * kWave;
        if (c < nch) __builtin_memcpy(dst + chunk_start<C>(c, D), acc[k], sizeof(acc[k]));
      }
    };
    if (in.count[head] > piece) {
      add_places<DT, C, K>(acc, g, in.order, from, min(to, in.start[head] + in.count[head]), D, nch, c0, kWave);
      write(0);
    }
    if (in.count[tail] > piece && in.start[tail] > from) {
      add_places<DT, C, K>(acc, g, in.order, in.start[tail], to, D, nch, c0, kWave);
      write(1);
    }
    return;
  }
  const int64_t wave = (int64_t)(blockIdx.x - piece_blocks) * kWaves + wave_in_block;
  const int64_t place = (wave << (6 - shift)) + (lane >> shift);
  if (place >= *in.total) return;
  const int64_t v = in.row_of[place];
  const int start = in.start[v], count = in.count[v];
  if (place != start || count > piece) return;
  const int c0 = blockIdx.y * (K << shift) + (lane & ((1 << shift) - 1));
  add_places<DT, C, K>(acc, g, in.order, start, start + count, D, nch, c0, 1 << shift);
  auto* dst = dtable + v * D;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = c0 + (k << shift);
    if (c >= nch) continue;
    Piece<DT, C> o;
#pragma unroll
    for (int j = 0; j < C; ++j) acc[k][j] *= scale;
    o.set(acc[k]);
    o.store(dst + chunk_start<C>(c, D));
  }
}

// Workgroup (x, y): the longer rows whose first piece is one of 8 x .. 8 x + 7, columns 256 y .. + 255. Wave w adds
// pieces w, w + 16, ... of the row, then the waves' sums are added in order.
template <int DT>
__global__ __launch_bounds__(kSumWaves * kWave) void sum_pieces(const float* __restrict__ part, Groups in,
                                                                typename Elem<DT>::T* __restrict__ dtable, int D,
                                                                float scale) {
  __shared__ float s[kSumWaves][kSumCols];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int total = *in.total;
  const int piece = 1 << in.piece_shift;
  const int64_t p_lane = (int64_t)blockIdx.x * kSumPieces + lane, a = p_lane * piece;
  int row = 0;
  bool begins = false;
  if (lane < kSumPieces && a < total) {
    row = in.row_of[(a + piece < total ? a + piece : total) - 1];
    begins = in.count[row] > piece && in.start[row] >= a;
  }
  uint64_t left = __ballot(begins);
  while (left) {
    const int l = __builtin_ctzll(left);
    left &= left - 1;
    const int v = __builtin_amdgcn_readlane(row, l), start = in.start[v];
    const int64_t p = (int64_t)blockIdx.x * kSumPieces + l, last = ((int64_t)start + in.count[v] - 1) >> in.piece_shift;
    const int slot = start == p << in.piece_shift ? 0 : 1;
    float acc[kSumCols / kWave] = {};
#pragma unroll 4
    for (int64_t q = p + wave; q <= last; q += kSumWaves) {
      const float* src = part + (2 * q + (q == p ? slot : 0)) * D;
#pragma unroll
      for (int k = 0; k < kSumCols / kWave; ++k) {
        const int col = blockIdx.y * kSumCols + k * kWave + lane;
        if (col < D) acc[k] += src[col];
      }
    }
#pragma unroll
    for (int k = 0; k < kSumCols / kWave; ++k) s[wave][k * kWave + lane] = acc[k];
    __syncthreads();
    const int col = blockIdx.y * kSumCols + threadIdx.x;
    if (threadIdx.x < kSumCols && col < D) {
      float t = s[0][threadIdx.x];
      for (int w = 1; w < kSumWaves; ++w) t += s[w][threadIdx.x];
      dtable[(int64_t)v * D + col] = Elem<DT>::store(t * scale);
    }
    __syncthreads();
  }
}

// Rows as chunks: elements per chunk, chunks, log2 of the lanes of a row, chunks per lane, blocks of columns.
struct Cut {
  int c, nch, shift, k, blocks;
};
Cut cut_rows(int dtype, int D) {
  const int wide = dtype == kF32 ? 4 : 8;
  Cut r{D >= wide ? wide : 1, 0, 0, 1, 1};
  r.nch = (int)ceil_div(D, r.c);
  while (r.shift < 6 && (1 << r.shift) < r.nch) ++r.shift;
  if (r.nch > kWave) r.k = r.nch > 2 * kWave ? 4 : 2;
  r.blocks = (int)ceil_div(r.nch, (int64_t)r.k << r.shift);
  return r;
}

// f(dtype, chunk, chunks per lane) as constants.
template <int N>
struct Int {
  static constexpr int value = N;
};
template <int DT, typename F>
int with_cut(const Cut& r, F&& f) {
  constexpr int E = Elem<DT>::E;
  if (r.c == 1) return f(Int<DT>{}, Int<1>{}, Int<1>{});
  switch (r.k) {
    case 1:
      return f(Int<DT>{}, Int<E>{}, Int<1>{});
    case 2:
      return f(Int<DT>{}, Int<E>{}, Int<2>{});
    default:
      return f(Int<DT>{}, Int<E>{}, Int<4>{});
  }
}
template <typename F>
int with_kernel(int dtype, const Cut& r, F&& f) {
  switch (dtype) {
    case kF16:
      return with_cut<kF16>(r, f);
    case kF32:
      return with_cut<kF32>(r, f);
    default:
      return with_cut<kBf16>(r, f);
  }
}

int group_shift_of(int V) {
  int s = 0;
  while ((1 << s) < kGroups && (1 << s) < V) ++s;
  while (ceil_div(V, (int64_t)1 << s) > kGroupRows) ++s;
  return s;
}

struct Workspace {
  size_t order, row_of, start, count, total, part, bytes;
  int64_t pieces;  // 0: no row can be a long one
};
Workspace lay_out(int64_t n, int V, int D) {
  Workspace w{};
  const int64_t piece = (int64_t)1 << piece_shift_of(n);
  w.pieces = n > piece ? ceil_div(n, piece) : 0;
  size_t at = 0;
  auto take = [&](size_t b) {
    const size_t here = at;
    at += align256(b);
    return here;
  };
  w.order = take((size_t)n * 4);
  w.row_of = take((size_t)n * 4);
  w.start = take((size_t)V * 4);
  w.count = take((size_t)V * 4);
  w.total = take(4);
  w.part = take((size_t)w.pieces * 2 * D * 4);
  w.bytes = at;
  return w;
}

int check(int64_t n, int V, int D, int token_bytes, float scale, int dtype) {
  if (dtype != kBf16 && dtype != kF16 && dtype != kF32) return KRSI_ERR_UNSUPPORTED;
  if (n < 0 || n > (1 << 25) || V <= 0 || V > (1 << 24) || D <= 0 || D > (1 << 20))
    return KRSI_ERR_BAD_SHAPE;
  if (token_bytes != 4 && token_bytes != 8) return KRSI_ERR_UNSUPPORTED;
  if (!(scale == scale) || scale > 3.0e38f || scale < -3.0e38f) return KRSI_ERR_BAD_SCALE;
  return KRSI_OK;
}

}  // namespace
}  // namespace krsi

extern "C" {

int krsi_embedding_fwd(const void* tokens, int32_t token_bytes, const void* table, void* out, int64_t n, int32_t V,
                       int32_t D, float scale, int32_t dtype, void* stream) {
  using namespace krsi;
  const int rc = check(n, V, D, token_bytes, scale, dtype);
  if (rc != KRSI_OK) return rc;
  if (n == 0) return KRSI_OK;
  if (!tokens || !table || !out) return KRSI_ERR_NULL_POINTER;
  const Cut r = cut_rows(dtype, D);
  const int64_t waves = ceil_div(n, kWave >> r.shift);
  return with_kernel(dtype, r, [&](auto dt, auto c, auto k) {
    constexpr int DT = decltype(dt)::value;
    using T = typename Elem<DT>::T;
    hipLaunchKernelGGL((embedding_fwd<DT, decltype(c)::value, decltype(k)::value>),
                       dim3((unsigned)ceil_div(waves, kWaves), (unsigned)r.blocks), dim3(kThreads), 0, as_stream(stream),
                       tokens, (int)token_bytes, (const T*)table, (T*)out, n, (int)V, (int)D, r.nch, r.shift, scale);
    return launch_status();
  });
}

size_t krsi_embedding_bwd_workspace_bytes(int64_t n, int32_t V, int32_t D) {
  using namespace krsi;
  return check(n, V, D, 8, 1.f, kBf16) == KRSI_OK ? lay_out(n, V, D).bytes : 0;
}

int krsi_embedding_bwd(const void* dout, const void* tokens, int32_t token_bytes, void* dtable, void* workspace,
                       size_t workspace_bytes, int64_t n, int32_t V, int32_t D, int64_t padding, float scale,
                       int32_t dtype, void* stream) {
  using namespace krsi;
  const int rc = check(n, V, D, token_bytes, scale, dtype);
  if (rc != KRSI_OK) return rc;
  if (!dtable || (n > 0 && (!dout || !tokens))) return KRSI_ERR_NULL_POINTER;
  const Workspace w = lay_out(n, V, D);
  if (!workspace || workspace_bytes < w.bytes) return KRSI_ERR_WORKSPACE;
  if (!aligned16(workspace)) return KRSI_ERR_MISALIGNED;
  char* base = static_cast<char*>(workspace);
  const Groups g{(int32_t*)(base + w.order), (int32_t*)(base + w.row_of), (int32_t*)(base + w.start),
                 (int32_t*)(base + w.count), (int32_t*)(base + w.total), piece_shift_of(n)};
  float* part = (float*)(base + w.part);
  hipStream_t st = as_stream(stream);
  const int gs = group_shift_of(V);
  const int64_t bytes = (int64_t)V * D * (dtype == kF32 ? 4 : 2);
  const int64_t fill = ceil_div(bytes, 16 * kGroupThreads * kFillChunks);
  hipLaunchKernelGGL(group_tokens, dim3((1u << gs) + (unsigned)fill),
                     dim3(kGroupThreads), 0, st, tokens, (int)token_bytes, (int)n, (int)V, gs, padding, g, (char*)dtable,
                     bytes);
  if (n == 0) return launch_status();
  const Cut r = cut_rows(dtype, D);
  const int piece_blocks = (int)ceil_div(w.pieces, kWaves);
  const int64_t row_blocks = ceil_div(ceil_div(n, kWave >> r.shift), kWaves);
  return with_kernel(dtype, r, [&](auto dt, auto c, auto k) {
    constexpr int DT = decltype(dt)::value;
    using T = typename Elem<DT>::T;
    hipLaunchKernelGGL((sum_rows<DT, decltype(c)::value, decltype(k)::value>),
                       dim3((unsigned)(piece_blocks + row_blocks), (unsigned)r.blocks), dim3(kThreads), 0, st,
                       (const T*)dout, g, (T*)dtable, part, piece_blocks, (int)D, r.nch, r.shift, scale);
    if (w.pieces)
      hipLaunchKernelGGL((sum_pieces<DT>),
                         dim3((unsigned)ceil_div(w.pieces, kSumPieces), (unsigned)ceil_div(D, kSumCols)),
                         dim3(kSumWaves * kWave), 0, st, (const float*)part, g, (T*)dtable, (int)D, scale);
    return launch_status();
  });
}

}  // extern "C"
