// Products of rows grouped by leaf: every leaf g owns the rows [begin[g], begin[g + 1]) and a linear map W_g [P x F].
//   leaf products:  y_i = W_g x_i                       for the rows i of leaf g
//   leaf Gram:      P_g = sum over the rows i of leaf g of a_i b_i^T
// The first is the linear part of leaves with several outputs; its gradient in x is the same product with the transposed maps,
// its gradient in W the second, which also gives the normal equations X^T H X of linear leaves (a = h x).
// Sums are held in fp32 and rounded once to the output's type.
//
// A leaf's rows are cut into tiles (of a Gram matrix: slices of rows); which tile is whose is known only on the device. Every block
// counts the leaves' tiles when it starts and walks the tiles with the grid's stride.
//   16-bit types  tcgen05.mma, accumulators in tensor memory            (LeafTensorKernel)
//   fp32          fused multiply-adds, so that fp32 products stay exact   (LeafProductsFloatKernel, LeafGramFloatKernel)
#include "kernels.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

namespace fb {

namespace {

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr int kSms = 148;

// Boundary i inside [0, rows).
__device__ __forceinline__ int Boundary(const LeafWindows& w, int i) {
  const long long b = w.begin_bits == 32 ? static_cast<const int*>(w.begin)[i] : static_cast<const long long*>(w.begin)[i];
  return static_cast<int>(min(max(b, 0LL), w.rows));
}
// Tiles of `rows` rows in [b, e); `least`: tiles of a leaf without rows.
__device__ __forceinline__ int TilesIn(int b, int e, int rows, int least) { return max(least, static_cast<int>((static_cast<unsigned int>(e - b) + static_cast<unsigned int>(rows) - 1u) / static_cast<unsigned int>(rows))); }

// The tiles of all leaves one behind the other: `rows` rows each, a leaf's last one shorter. Up to kSpans leaves are looked up by
// bisection; more are counted in spans of several leaves.
// A leaf starts where the one before it ended. That is its own boundary unless boundaries fall again: then a row belongs to the first
// leaf that has it, so no boundaries make more tiles than rows / tile rows + leaves, or rows that two leaves work on.
constexpr int kSpans = 1024;
struct TileMap {
  int before[kSpans + 1];        // tiles before span i
  int row[kSpans + 1];           // its first row
  int per, spans, first_row, last_row;      // rows of all leaves: [first_row, last_row)
  // tiles of span i (its leaves: [i * p, end)), whose first row is *b; *b: the row behind it. falls: whether a boundary fell again
  __device__ __forceinline__ static int CountSpan(const LeafWindows& w, int i, int p, int rows, int least, int* b, int* falls) {
    int c = 0;
    for (int g = i * p; g < min(w.leaves, (i + 1) * p); ++g) {
      const int next = Boundary(w, g + 1), e = max(*b, next);
      *falls |= next < *b ? 1 : 0;
      c += TilesIn(*b, e, rows, least);
      *b = e;
    }
    return c;
  }
  // All threads of the block; `least`: tiles of a leaf without rows.
  __device__ void Build(const LeafWindows& w, int rows, int least) {
    const int p = (w.leaves + kSpans - 1) / kSpans, n = (w.leaves + p - 1) / p;
    if (threadIdx.x == 0) { per = p; spans = n; }
    int falls = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      int b = Boundary(w, i * p);
      row[i] = b;
      if (i == 0) first_row = b;
      before[i + 1] = CountSpan(w, i, p, rows, least, &b, &falls);
      if (i == n - 1) row[n] = last_row = b;
    }
    if (__syncthreads_or(falls) != 0) {
      // where spans start when rows before them have been taken: the highest boundary so far
#pragma unroll 1
      for (int i = threadIdx.x; i < n; i += blockDim.x) { int b = Boundary(w, i * p); CountSpan(w, i, p, rows, least, &b, &falls); before[i + 1] = b; }
      __syncthreads();
      if (threadIdx.x == 0) {
#pragma unroll 1
        for (int i = 0; i < n; ++i) row[i + 1] = max(row[i], before[i + 1]);
        last_row = row[n];
      }
      __syncthreads();
#pragma unroll 1
      for (int i = threadIdx.x; i < n; i += blockDim.x) { int b = row[i]; before[i + 1] = CountSpan(w, i, p, rows, least, &b, &falls); }
      __syncthreads();
    }
    if (threadIdx.x < 32) {
      const int each = (n + 31) / 32, lo = min(n, static_cast<int>(threadIdx.x) * each), hi = min(n, lo + each);
      int sum = 0;
      for (int i = lo; i < hi; ++i) sum += before[i + 1];
      int scan = sum;
      for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, scan, o); if (static_cast<int>(threadIdx.x) >= o) scan += v; }
      scan -= sum;
      __syncwarp();
      for (int i = lo; i < hi; ++i) { scan += before[i + 1]; before[i + 1] = scan; }
      if (threadIdx.x == 0) before[0] = 0;
    }
    __syncthreads();
  }
  __device__ __forceinline__ int Total() const { return before[spans]; }
  // the row behind leaf g, which starts at row b
  __device__ __forceinline__ int End(const LeafWindows& w, int g, int b) const { return per == 1 ? row[g + 1] : max(b, Boundary(w, g + 1)); }
  // tile -> leaf, its first row and the end of the rows that it covers, and the rows [begin, last) of the whole leaf. `span`: where the last
  // search of an earlier tile ended (0 at first); the next tile is mostly a few leaves on.
  __device__ __forceinline__ void Find(const LeafWindows& w, int tile, int rows, int least, int* span, int* leaf, int* first, int* end, int* begin, int* last) const {
    int lo = *span;
    if (before[lo + 1] <= tile && lo + 1 < spans) ++lo;
    if (before[lo + 1] <= tile) { int hi = spans; while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (before[mid] <= tile) lo = mid; else hi = mid; } }
    *span = lo;
    int g = lo * per, left = tile - before[lo], b = row[lo], e = End(w, g, b);
    if (per > 1) {
      for (int c = TilesIn(b, e, rows, least); left >= c && g + 1 < w.leaves; c = TilesIn(b, e, rows, least)) { left -= c; ++g; b = e; e = End(w, g, b); }
    }
    *leaf = g; *begin = b; *last = e;
    *first = static_cast<int>(min(static_cast<long long>(e), b + static_cast<long long>(left) * rows)); *end = static_cast<int>(min(static_cast<long long>(e), static_cast<long long>(*first) + rows));
  }
};

// Rows that belong to no leaf: zero. All threads of the grid, when the map is built.
template <typename T>
__device__ __forceinline__ void ZeroLeaflessRows(const TileMap& map, const LeafWindows& w, T* y, int outputs) {
  if (map.first_row == 0 && map.last_row == w.rows) return;
  const long long head = static_cast<long long>(map.first_row) * outputs, tail = static_cast<long long>(map.last_row) * outputs, total = w.rows * outputs;
  const long long t = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x, stride = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i = t; i < head; i += stride) y[i] = FromFloat<T>(0.f);
  for (long long i = tail + t; i < total; i += stride) y[i] = FromFloat<T>(0.f);
}

// ------------------------------------------------------------------------------------------------------- fp32 ----
struct F2 { unsigned long long v; };
__device__ __forceinline__ F2 MakeF2(float x, float y) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ void Split(F2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 Fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
__device__ __forceinline__ unsigned int Smem32(const void* p) { return static_cast<unsigned int>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void CopyCommit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING> __device__ __forceinline__ void CopyWait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// 4 bytes global -> shared, zero when !in
__device__ __forceinline__ void CopyFloat(float* dst, const float* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(Smem32(dst)), "l"(src), "r"(in ? 4 : 0) : "memory");
}
// Copies blocks of `all` lines of `width` floats (a multiple of 4), `pitch` apart in shared memory, in pieces of `vec` floats;
// neighbouring threads take neighbouring pieces. What a thread copies where is worked out once and walked by adding.
template <int THREADS>
struct CopyPlan {
  int all, vec, per, line0, piece0, lines_on, pieces_on, pitch;
  __device__ __forceinline__ CopyPlan(int all_, int width, int pitch_, int vec_) {
    all = all_; vec = vec_; pitch = pitch_; per = width / vec;
    lines_on = THREADS / per; pieces_on = THREADS - lines_on * per;
    line0 = static_cast<int>(threadIdx.x) / per; piece0 = static_cast<int>(threadIdx.x) - line0 * per;
  }
  template <int BYTES, bool WHOLE>
  __device__ __forceinline__ void Walk(float* dst, const float* src, int lines, long long stride, int along) const {
    constexpr int V = BYTES / 4;
    const float* from = src + line0 * stride + piece0 * V;
    unsigned int to = Smem32(dst + line0 * pitch + piece0 * V);
    const long long from_on = lines_on * stride + pieces_on * V, from_wrap = stride - per * V;
    const unsigned int to_on = 4u * (lines_on * pitch + pieces_on * V), to_wrap = 4u * (pitch - per * V);
    int piece = piece0;
    const int end = min(all, lines);
#pragma unroll 2
    for (int line = line0; line < end;) {
      const int valid = WHOLE ? BYTES : 4 * max(0, min(V, along - piece * V));
      const float* at = WHOLE || valid > 0 ? from : src;
      if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(at), "r"(valid) : "memory");
      else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(to), "l"(at), "r"(valid), "n"(BYTES) : "memory");
      line += lines_on; piece += pieces_on; from += from_on; to += to_on;
      if (piece >= per) { piece -= per; ++line; from += from_wrap; to += to_wrap; }
    }
  }
  // the source has `lines` lines, `stride` apart, of `along` floats (zero beyond); lines that it does not have are left as they are
  __device__ __forceinline__ void Copy(float* dst, const float* src, int lines, long long stride, int along) const {
    const bool whole = along >= per * vec;
    if (vec == 4) { if (whole) Walk<16, true>(dst, src, lines, stride, along); else Walk<16, false>(dst, src, lines, stride, along); }
    else if (vec == 2) Walk<8, false>(dst, src, lines, stride, along);
    else Walk<4, false>(dst, src, lines, stride, along);
  }
};

// Products. Tile: ROWS = 32 * TM * WR rows x OUTS = TN * WO outputs, up to kDepth features a step. x and the maps lie in shared
// memory as they do in memory, line by line, the pitch an odd number of 16-byte pieces: 32 lanes then read 4 features of 32 rows
// without bank conflicts, the outputs' features are read by whole warps at once. A lane has TM rows, 32 apart, and TN outputs; a
// 64-bit register holds the sums over even and over odd features, added at the end. Steps (of all the block's tiles, one behind the
// other) go through a ring of kRing buffers.
// `width` and `pitch` of the launch: features a step, in multiples of 4, and their pitch.
constexpr int kDepth = 32, kRing = 3;
struct FloatShape { int width, pitch, x_vec, w_vec; bool w_by_output; };
template <int TM, int TN, int WR, int WO>
struct FloatTile {
  static constexpr int ROWS = 32 * TM * WR, OUTS = TN * WO, THREADS = 32 * WR * WO;
  static int Bytes(int pitch) { return (kRing * (ROWS + OUTS) * pitch + (WO == 1 ? ROWS * OUTS : 0)) * 4; }
};
template <int TM, int TN, int WR, int WO>
__global__ void __launch_bounds__(32 * WR * WO, 512 / (32 * WR * WO)) LeafProductsFloatKernel(LeafProductsArgs a, FloatShape shape) {
  using Tile = FloatTile<TM, TN, WR, WO>;
  extern __shared__ __align__(16) float s_float[];
  __shared__ TileMap map;
  const int pitch = shape.pitch, buffer = (Tile::ROWS + Tile::OUTS) * pitch;
  map.Build(a.leaves, Tile::ROWS, 0);
  ZeroLeaflessRows(map, a.leaves, static_cast<float*>(a.y), a.outputs);
  const int across = (a.outputs + Tile::OUTS - 1) / Tile::OUTS;
  const int tiles = map.Total() * across, grid = gridDim.x;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, wr = warp % WR, wo = warp / WR;
  const CopyPlan<Tile::THREADS> x_plan(Tile::ROWS, shape.width, pitch, shape.x_vec), w_plan(Tile::OUTS, shape.width, pitch, shape.w_vec);
  struct At { int t, span, row0, leaf, rows, out0, f0; };
  auto find = [&](At& at) {
    int end, begin, last;
    const int which = at.t / across;
    map.Find(a.leaves, which, Tile::ROWS, 0, &at.span, &at.leaf, &at.row0, &end, &begin, &last);
    at.rows = end - at.row0; at.out0 = (at.t - which * across) * Tile::OUTS; at.f0 = 0;
  };
  auto advance = [&](At& at) { at.f0 += shape.width; if (at.f0 >= a.features) { at.t += grid; if (at.t < tiles) find(at); } };
  auto copy = [&](const At& at, int slot) {
    if (at.t < tiles) {
      float* to = s_float + slot * buffer;
      x_plan.Copy(to, static_cast<const float*>(a.x) + at.row0 * a.x_stride + at.f0, at.rows, a.x_stride, a.features - at.f0);
      to += Tile::ROWS * pitch;
      const float* w = static_cast<const float*>(a.weight) + at.leaf * a.weight_leaf_stride + at.out0 * a.weight_out_stride + at.f0 * a.weight_in_stride;
      const int outs = a.outputs - at.out0;
      if (!shape.w_by_output) {
        w_plan.Copy(to, w, outs, a.weight_out_stride, a.features - at.f0);
      } else {      // the outputs are contiguous (or nothing is): value by value, neighbouring threads along the outputs
        for (int e = threadIdx.x; e < Tile::OUTS * shape.width; e += Tile::THREADS) {
          const int o = e % Tile::OUTS, f = e / Tile::OUTS;
          const bool in = o < outs && at.f0 + f < a.features;
          CopyFloat(to + o * pitch + f, in ? w + o * a.weight_out_stride + f * a.weight_in_stride : w, in);
        }
      }
    }
    CopyCommit();
  };
  At now, ahead;
  now.t = blockIdx.x; now.span = 0;
  if (now.t < tiles) find(now);
  ahead = now;
  int slot = 0;
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) { copy(ahead, i); if (ahead.t < tiles) advance(ahead); }
  F2 acc[TM][TN];
  while (now.t < tiles) {
    if (now.f0 == 0) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = MakeF2(0.f, 0.f);
    }
    CopyWait<kRing - 2>();
    __syncthreads();
    copy(ahead, (slot + kRing - 1) % kRing);      // the buffer that everyone has left
    if (ahead.t < tiles) advance(ahead);
    const float* xs = s_float + slot * buffer + (wr * 32 * TM + lane) * pitch;
    const float* ws = s_float + slot * buffer + (Tile::ROWS + wo * TN) * pitch;
    // beyond the last feature both sides are zero; rows and outputs that do not exist hold anything, and are not stored
    const int depth = wr * 32 * TM < now.rows ? min(shape.width, a.features - now.f0) : 0;
    for (int f = 0; f < depth; f += 4) {
      ulonglong2 xv[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) xv[i] = *reinterpret_cast<const ulonglong2*>(xs + 32 * i * pitch + f);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(ws + j * pitch + f);
#pragma unroll
        for (int i = 0; i < TM; ++i) { acc[i][j] = Fma2(F2{xv[i].x}, F2{w.x}, acc[i][j]); acc[i][j] = Fma2(F2{xv[i].y}, F2{w.y}, acc[i][j]); }
      }
    }
    if (now.f0 + shape.width >= a.features) {
      const int outs = min(Tile::OUTS, a.outputs - now.out0);
      float* y = static_cast<float*>(a.y) + static_cast<long long>(now.row0) * a.outputs + now.out0;
      if constexpr (WO == 1) {
        // narrow outputs: a tile's rows are one piece of memory when the tile holds all outputs; a warp's rows go through shared memory
        float* s_y = s_float + kRing * buffer + wr * 32 * TM * Tile::OUTS;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) if (j < outs) { float lo, hi; Split(acc[i][j], lo, hi); s_y[(lane + 32 * i) * outs + j] = lo + hi; }
        __syncwarp();
        const int first = wr * 32 * TM, rows = max(0, min(32 * TM, now.rows - first));
        if (outs == a.outputs) for (int e = lane; e < rows * outs; e += 32) y[static_cast<long long>(first) * outs + e] = s_y[e];
        else for (int e = lane; e < rows * outs; e += 32) y[static_cast<long long>(first + e / outs) * a.outputs + e % outs] = s_y[e];
        __syncwarp();
      } else {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int r = wr * 32 * TM + lane + 32 * i;
          if (r >= now.rows) continue;
          float* to = y + static_cast<long long>(r) * a.outputs + wo * TN;
          float v[TN];
#pragma unroll
          for (int j = 0; j < TN; ++j) { float lo, hi; Split(acc[i][j], lo, hi); v[j] = lo + hi; }
          if (wo * TN + TN <= outs && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < TN; j += 4) *reinterpret_cast<float4*>(to + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < TN; ++j) if (wo * TN + j < outs) to[j] = v[j];
          }
        }
      }
    }
    advance(now);
    slot = (slot + 1) % kRing;
  }
  CopyWait<0>();
}

// Where the sums of a slice go: -1 straight to the output (its leaf has no other), else a place of the workspace. Of the leaves with
// several slices, first slices start more than a slice apart, and so do the others: 2 places per `rows` rows are enough.
__device__ __forceinline__ int SliceSlot(int leaf_begin, int leaf_end, int row0, int rows) { return leaf_end - leaf_begin <= rows ? -1 : 2 * (row0 / rows) + (row0 == leaf_begin ? 0 : 1); }

// Gram matrices. Tile: AC = TA * GA columns of a x BC = TB * GB columns of b, RD rows a step through a ring of kRing buffers; SLICES
// groups of GA * GB threads take every SLICES-th row each and are added up at the end, in order.
template <int TA, int TB, int GA, int GB, int SLICES, int RD>
struct FloatGramTile {
  static constexpr int AC = TA * GA, BC = TB * GB, GROUP = GA * GB, THREADS = GROUP * SLICES;
  static constexpr int kLoad = kRing * RD * (AC + BC) * 4, kSum = SLICES * AC * BC * 4, kBytes = kLoad > kSum ? kLoad : kSum;
};
// A leaf of one slice is written to out; the sums of the slices of longer leaves go to partial [slot][a_cols][b_cols].
template <int TA, int TB, int GA, int GB, int SLICES, int RD>
__global__ void __launch_bounds__(GA * GB * SLICES, 2) LeafGramFloatKernel(LeafGramArgs a, int rows_per_slice, int a_vec, int b_vec, float* partial) {
  using Tile = FloatGramTile<TA, TB, GA, GB, SLICES, RD>;
  extern __shared__ __align__(16) float s_float[];
  __shared__ TileMap map;
  map.Build(a.leaves, rows_per_slice, 1);
  const int across_a = (a.a_cols + Tile::AC - 1) / Tile::AC, across_b = (a.b_cols + Tile::BC - 1) / Tile::BC;
  const int across = across_a * across_b, tiles = map.Total() * across;
  const int slice = threadIdx.x / Tile::GROUP, member = threadIdx.x % Tile::GROUP, ga = member / GB, gb = member % GB;
  int span = 0;
  for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int which = t / across, rest = t - which * across;
    int leaf, row0, end, leaf_begin, leaf_end;
    map.Find(a.leaves, which, rows_per_slice, 1, &span, &leaf, &row0, &end, &leaf_begin, &leaf_end);
    const int a0 = rest / across_b * Tile::AC, b0 = rest % across_b * Tile::BC, a_in = min(Tile::AC, a.a_cols - a0), b_in = min(Tile::BC, a.b_cols - b0);
    const CopyPlan<Tile::THREADS> a_plan(RD, (a_in + 3) & ~3, Tile::AC, a_vec), b_plan(RD, (b_in + 3) & ~3, Tile::BC, b_vec);
    const float* pa = static_cast<const float*>(a.a) + row0 * a.a_stride + a0; const float* pb = static_cast<const float*>(a.b) + row0 * a.b_stride + b0;
    const int rows = end - row0, steps = (rows + RD - 1) / RD;
    auto copy = [&](int step) {
      if (step < steps) {
        float* to = s_float + step % kRing * RD * (Tile::AC + Tile::BC);
        const int r0 = step * RD;
        a_plan.Copy(to, pa + r0 * a.a_stride, rows - r0, a.a_stride, a_in);
        b_plan.Copy(to + RD * Tile::AC, pb + r0 * a.b_stride, rows - r0, a.b_stride, b_in);
      }
      CopyCommit();
    };
    F2 acc[TA][TB / 2];
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
      for (int j = 0; j < TB / 2; ++j) acc[i][j] = MakeF2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) copy(i);
    for (int step = 0; step < steps; ++step) {
      CopyWait<kRing - 2>();
      __syncthreads();
      copy(step + kRing - 1);                     // the buffer that everyone has left
      // columns beyond the operands hold anything; they reach only sums that are not stored
      const float* as = s_float + step % kRing * RD * (Tile::AC + Tile::BC) + ga * TA; const float* bs = s_float + (step % kRing * (Tile::AC + Tile::BC) + Tile::AC) * RD + gb * TB;
      const int here = min(RD, rows - step * RD);
#pragma unroll 4
      for (int r = slice; r < here; r += SLICES) {
        F2 bv[TB / 2]; float av[TA];
#pragma unroll
        for (int j = 0; j < TB / 4; ++j) { const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(bs + r * Tile::BC + 4 * j); bv[2 * j].v = q.x; bv[2 * j + 1].v = q.y; }
#pragma unroll
        for (int i = 0; i < TA / 4; ++i) { const float4 q = *reinterpret_cast<const float4*>(as + r * Tile::AC + 4 * i); av[4 * i] = q.x; av[4 * i + 1] = q.y; av[4 * i + 2] = q.z; av[4 * i + 3] = q.w; }
#pragma unroll
        for (int i = 0; i < TA; ++i) {
          const F2 v = MakeF2(av[i], av[i]);
#pragma unroll
          for (int j = 0; j < TB / 2; ++j) acc[i][j] = Fma2(v, bv[j], acc[i][j]);
        }
      }
    }
    CopyWait<0>();
    __syncthreads();
    const int slot = SliceSlot(leaf_begin, leaf_end, row0, rows_per_slice);
    float* to = slot >= 0 ? partial + static_cast<long long>(slot) * a.a_cols * a.b_cols : static_cast<float*>(a.out) + static_cast<long long>(leaf) * a.a_cols * a.b_cols;
    float* s_sum = s_float;                  // the row buffers are free now
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
      for (int j = 0; j < TB / 2; ++j) {
        float v0, v1; Split(acc[i][j], v0, v1);
        float* p = s_sum + (slice * Tile::AC + ga * TA + i) * Tile::BC + gb * TB + 2 * j;
        p[0] = v0; p[1] = v1;
      }
    __syncthreads();
    for (int e = threadIdx.x; e < Tile::AC * Tile::BC; e += Tile::THREADS) {
      const int ca = e / Tile::BC, cb = e % Tile::BC;
      if (ca >= a_in || cb >= b_in) continue;
      float v = 0.f;
#pragma unroll
      for (int s = 0; s < SLICES; ++s) v += s_sum[s * Tile::AC * Tile::BC + e];
      to[static_cast<long long>(a0 + ca) * a.b_cols + b0 + cb] = v;
    }
    __syncthreads();
  }
}

// --------------------------------------------------------------------------------------- few columns, any type ----
// With at most 32 outputs and short rows the products are a matter of bandwidth: 12 warps per SM, each by itself, walk through tiles of
// rows that come by asynchronous copies into the warp's own ring, so that about 90 KB per SM are on their way and no warp waits
// for another. A warp's tiles are neighbours, so a leaf's map is loaded (as fp32) when the leaf changes. fp32 sums over even and
// over odd features in one 64-bit register.
constexpr int kNarrowWarps = 12, kNarrowThreads = 32 * kNarrowWarps, kNarrowRing = 2, kNarrowRowBytes = 256;
// Copies rows to lines `pitch` bytes apart, in pieces of `piece` bytes; by one warp. What is worked out once: where a lane starts.
struct WarpCopy {
  int piece, per, pitch, row_bytes, line0, piece0, lines_on, pieces_on;
  __device__ __forceinline__ WarpCopy(int row_bytes_, int pitch_, int piece_, int lane) {
    piece = piece_; pitch = pitch_; row_bytes = row_bytes_; per = (row_bytes + piece - 1) / piece;
    lines_on = 32 / per; pieces_on = 32 - lines_on * per; line0 = lane / per; piece0 = lane - line0 * per;
  }
  template <int BYTES>
  __device__ __forceinline__ void Walk(unsigned int to, const char* from, long long stride, int rows) const {
    from += line0 * stride + piece0 * BYTES; to += line0 * pitch + piece0 * BYTES;
    const long long from_on = lines_on * stride + pieces_on * BYTES, from_wrap = stride - per * BYTES;
    const int to_on = lines_on * pitch + pieces_on * BYTES, to_wrap = pitch - per * BYTES;
    int p = piece0;
#pragma unroll 2
    for (int line = line0; line < rows;) {
      const int valid = min(BYTES, row_bytes - p * BYTES);
      if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid) : "memory");
      else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(to), "l"(from), "r"(valid), "n"(BYTES) : "memory");
      line += lines_on; p += pieces_on; from += from_on; to += to_on;
      if (p >= per) { p -= per; ++line; from += from_wrap; to += to_wrap; }
    }
  }
  __device__ __forceinline__ void Copy(void* to, const void* from, long long stride_bytes, int rows) const {
    const unsigned int dst = Smem32(to); const char* src = static_cast<const char*>(from);
    if (piece == 16) Walk<16>(dst, src, stride_bytes, rows); else if (piece == 8) Walk<8>(dst, src, stride_bytes, rows); else Walk<4>(dst, src, stride_bytes, rows);
  }
};
// 16 bytes of a row as pairs of fp32
__device__ __forceinline__ void Pairs(const uint4& q, F2 (&p)[2], const float*) { p[0] = MakeF2(__uint_as_float(q.x), __uint_as_float(q.y)); p[1] = MakeF2(__uint_as_float(q.z), __uint_as_float(q.w)); }
__device__ __forceinline__ F2 Pair(unsigned int w, const __nv_bfloat16*) { return MakeF2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ F2 Pair(unsigned int w, const __half*) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w)); return MakeF2(f.x, f.y); }
template <typename T> __device__ __forceinline__ void Pairs(const uint4& q, F2 (&p)[4], const T* t) { p[0] = Pair(q.x, t); p[1] = Pair(q.y, t); p[2] = Pair(q.z, t); p[3] = Pair(q.w, t); }

// A warp's share of the tiles of `rows` rows, one behind the other: [first, last) of them.
struct WarpTiles {
  int left, leaf, row, leaf_begin, leaf_end, least;
  __device__ __forceinline__ WarpTiles(const TileMap& map, const LeafWindows& w, int rows, int least_) {
    least = least_;
    const int total = map.Total(), warps = gridDim.x * kNarrowWarps, me = blockIdx.x * kNarrowWarps + threadIdx.x / 32;
    const int each = total / warps, more = total - each * warps, first = me * each + min(me, more);
    left = each + (me < more ? 1 : 0); leaf = row = leaf_begin = leaf_end = 0;
    if (left > 0) { int span = 0, end; map.Find(w, first, rows, least, &span, &leaf, &row, &end, &leaf_begin, &leaf_end); }
  }
  __device__ __forceinline__ void Next(const TileMap& map, const LeafWindows& w, int rows) {
    if (--left <= 0) return;
    if (leaf_end - row > rows) row += rows;
    else {
      do { ++leaf; row = leaf_begin = leaf_end; leaf_end = map.End(w, leaf, row); } while (least == 0 && row >= leaf_end && leaf + 1 < w.leaves);
    }
  }
};

// Shared memory for a tile's outputs, 0 where the place of its rows (`stage` bytes) is enough.
__host__ __device__ constexpr int NarrowOutputBytes(int tm, int outputs, int size, int stage) { const int bytes = (32 * tm * outputs * size + 15) / 16 * 16; return bytes <= stage ? 0 : bytes; }
template <typename T, int TM, int TN>
__global__ void __launch_bounds__(kNarrowThreads, 1) LeafProductsNarrowKernel(LeafProductsArgs a, int pitch, int piece) {
  constexpr int ROWS = 32 * TM, V = 16 / sizeof(T);
  extern __shared__ __align__(16) unsigned char s_bytes[];
  __shared__ TileMap map;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, w_pitch = (a.features + V - 1) / V * V;      // features of a map's line in shared memory
  const int stage = ROWS * pitch, y_bytes = NarrowOutputBytes(TM, a.outputs, static_cast<int>(sizeof(T)), stage), of_warp = kNarrowRing * stage + TN * w_pitch * 4 + y_bytes;
  unsigned char* s_x = s_bytes + warp * of_warp;
  float* s_w = reinterpret_cast<float*>(s_x + kNarrowRing * stage);
  for (int i = lane; i < of_warp / 16; i += 32) reinterpret_cast<uint4*>(s_x)[i] = make_uint4(0u, 0u, 0u, 0u);      // what no copy writes stays zero
  map.Build(a.leaves, ROWS, 0);
  ZeroLeaflessRows(map, a.leaves, static_cast<T*>(a.y), a.outputs);
  WarpTiles now(map, a.leaves, ROWS, 0);
  WarpTiles ahead = now;
  const WarpCopy plan(a.features * static_cast<int>(sizeof(T)), pitch, piece, lane);
  auto copy = [&](int slot) {
    if (ahead.left > 0) {
      plan.Copy(s_x + slot * stage, static_cast<const T*>(a.x) + static_cast<long long>(ahead.row) * a.x_stride, a.x_stride * static_cast<long long>(sizeof(T)), min(ROWS, ahead.leaf_end - ahead.row));
      ahead.Next(map, a.leaves, ROWS);
    }
    CopyCommit();
  };
  copy(0);
  int slot = 0, loaded = -1;
  for (; now.left > 0; now.Next(map, a.leaves, ROWS), slot ^= 1) {
    const int rows = min(ROWS, now.leaf_end - now.row);
    copy(slot ^ 1);
    if (now.leaf != loaded) {
      loaded = now.leaf;
      const T* w = static_cast<const T*>(a.weight) + loaded * a.weight_leaf_stride;
      const bool by_feature = a.weight_in_stride == 1;
      const int along = by_feature ? a.features : a.outputs, lines = by_feature ? a.outputs : a.features;
      const long long along_on = by_feature ? a.weight_in_stride : a.weight_out_stride, line_on = by_feature ? a.weight_out_stride : a.weight_in_stride;
      const int s_along = by_feature ? 1 : w_pitch, s_line = by_feature ? w_pitch : 1;
#pragma unroll 8
      for (int line = 0; line < lines; ++line)
        for (int c = lane; c < along; c += 32) s_w[line * s_line + c * s_along] = ToFloat(w[line * line_on + c * along_on]);
    }
    CopyWait<1>();
    __syncwarp();
    F2 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = MakeF2(0.f, 0.f);
    const unsigned char* xs = s_x + slot * stage + lane * pitch;
    for (int f = 0; f < a.features; f += V) {
      F2 xv[TM][V / 2];
#pragma unroll
      for (int i = 0; i < TM; ++i) Pairs(*reinterpret_cast<const uint4*>(xs + 32 * i * pitch + f * static_cast<int>(sizeof(T))), xv[i], static_cast<const T*>(nullptr));
#pragma unroll
      for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int h = 0; h < V / 4; ++h) {
          const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(s_w + j * w_pitch + f + 4 * h);
#pragma unroll
          for (int i = 0; i < TM; ++i) { acc[i][j] = Fma2(xv[i][2 * h], F2{w.x}, acc[i][j]); acc[i][j] = Fma2(xv[i][2 * h + 1], F2{w.y}, acc[i][j]); }
        }
      }
    }
    // the tile's outputs are one piece of memory; they go there through the place of its rows, which only this warp has read, or, where
    // that is too small, through a place of their own
    __syncwarp();
    T* s_y = reinterpret_cast<T*>(y_bytes > 0 ? reinterpret_cast<unsigned char*>(s_w + TN * w_pitch) : s_x + slot * stage);
    const int count = rows * a.outputs;
    T* y = static_cast<T*>(a.y) + static_cast<long long>(now.row) * a.outputs;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
        if (j < a.outputs) {
          float lo, hi; Split(acc[i][j], lo, hi);
          s_y[(lane + 32 * i) * a.outputs + j] = FromFloat<T>(lo + hi);
        }
    __syncwarp();
    {
      if (sizeof(T) == 4 || (reinterpret_cast<uintptr_t>(y) & 3) != 0) { for (int e = lane; e < count; e += 32) y[e] = s_y[e]; }
      else {
        for (int e = lane; e < count / 2; e += 32) reinterpret_cast<unsigned int*>(y)[e] = reinterpret_cast<const unsigned int*>(s_y)[e];
        if ((count & 1) != 0 && lane == 0) y[count - 1] = s_y[count - 1];
      }
      __syncwarp();
      // the features' padding has to be zero again
      const int row_bytes = a.features * static_cast<int>(sizeof(T)), pad = (row_bytes + 15) / 16 * 16 - row_bytes;
      if (pad > 0 && y_bytes == 0) for (int l = lane; l < ROWS; l += 32) for (int b = 0; b < pad; b += static_cast<int>(sizeof(T))) *reinterpret_cast<T*>(s_x + slot * stage + l * pitch + row_bytes + b) = FromFloat<T>(0.f);
      __syncwarp();
    }
  }
  CopyWait<0>();
}

// Gram matrices of at most 4 GA columns of a and 4 GB of b (GA GB = 32): a lane has 4 x 4 of the sums, a warp a slice of a leaf's rows.
constexpr int kGramRows = 32;
constexpr int GramRing(int size) { return size == 4 ? 2 : 4; }      // of all warps: 147 KB
template <typename T> __device__ __forceinline__ void Four(const void* p, float (&v)[4]);
template <> __device__ __forceinline__ void Four<float>(const void* p, float (&v)[4]) { const float4 q = *static_cast<const float4*>(p); v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w; }
template <> __device__ __forceinline__ void Four<__nv_bfloat16>(const void* p, float (&v)[4]) { const uint2 q = *static_cast<const uint2*>(p); Split(Pair(q.x, static_cast<const __nv_bfloat16*>(nullptr)), v[0], v[1]); Split(Pair(q.y, static_cast<const __nv_bfloat16*>(nullptr)), v[2], v[3]); }
template <> __device__ __forceinline__ void Four<__half>(const void* p, float (&v)[4]) { const uint2 q = *static_cast<const uint2*>(p); Split(Pair(q.x, static_cast<const __half*>(nullptr)), v[0], v[1]); Split(Pair(q.y, static_cast<const __half*>(nullptr)), v[2], v[3]); }
template <typename T, typename O, int GA, int GB>
__global__ void __launch_bounds__(kNarrowThreads, 1) LeafGramNarrowKernel(LeafGramArgs a, int rows_per_slice, int a_piece, int b_piece, float* partial) {
  constexpr int A_PITCH = 4 * GA * static_cast<int>(sizeof(T)), B_PITCH = 4 * GB * static_cast<int>(sizeof(T)), STAGE = kGramRows * (A_PITCH + B_PITCH), RING = GramRing(static_cast<int>(sizeof(T)));
  extern __shared__ __align__(16) unsigned char s_bytes[];
  __shared__ TileMap map;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, ga = lane / GB, gb = lane % GB;
  unsigned char* mine = s_bytes + warp * RING * STAGE;
  map.Build(a.leaves, rows_per_slice, 1);
  const WarpCopy a_plan(a.a_cols * static_cast<int>(sizeof(T)), A_PITCH, a_piece, lane), b_plan(a.b_cols * static_cast<int>(sizeof(T)), B_PITCH, b_piece, lane);
  for (WarpTiles slice(map, a.leaves, rows_per_slice, 1); slice.left > 0; slice.Next(map, a.leaves, rows_per_slice)) {
    const int rows = max(0, min(rows_per_slice, slice.leaf_end - slice.row));
    const T* pa = static_cast<const T*>(a.a) + static_cast<long long>(slice.row) * a.a_stride; const T* pb = static_cast<const T*>(a.b) + static_cast<long long>(slice.row) * a.b_stride;
    auto copy = [&](int r0) {
      if (r0 < rows) {
        unsigned char* to = mine + r0 / kGramRows % RING * STAGE;
        const int n = min(kGramRows, rows - r0);
        a_plan.Copy(to, pa + r0 * a.a_stride, a.a_stride * static_cast<long long>(sizeof(T)), n);
        b_plan.Copy(to + kGramRows * A_PITCH, pb + r0 * a.b_stride, a.b_stride * static_cast<long long>(sizeof(T)), n);
      }
      CopyCommit();
    };
    F2 acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i][0] = acc[i][1] = MakeF2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) copy(i * kGramRows);
    for (int r0 = 0; r0 < rows; r0 += kGramRows) {
      __syncwarp();                                 // every lane has left the buffer that is filled now
      copy(r0 + (RING - 1) * kGramRows);
      CopyWait<RING - 1>();
      __syncwarp();
      const unsigned char* as = mine + r0 / kGramRows % RING * STAGE + ga * 4 * sizeof(T); const unsigned char* bs = mine + r0 / kGramRows % RING * STAGE + kGramRows * A_PITCH + gb * 4 * sizeof(T);
      const int here = min(kGramRows, rows - r0);
#pragma unroll 8
      for (int r = 0; r < here; ++r) {              // columns beyond the operands hold anything; they reach only sums that are not stored
        float av[4], bv[4];
        Four<T>(as + r * A_PITCH, av); Four<T>(bs + r * B_PITCH, bv);
        const F2 b0 = MakeF2(bv[0], bv[1]), b1 = MakeF2(bv[2], bv[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const F2 v = MakeF2(av[i], av[i]); acc[i][0] = Fma2(v, b0, acc[i][0]); acc[i][1] = Fma2(v, b1, acc[i][1]); }
      }
    }
    CopyWait<0>();
    __syncwarp();
    const int slot = SliceSlot(slice.leaf_begin, slice.leaf_end, slice.row, rows_per_slice);
    const long long size = static_cast<long long>(a.a_cols) * a.b_cols;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float v[2]; Split(acc[i][j], v[0], v[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int ca = ga * 4 + i, cb = gb * 4 + 2 * j + h;
          if (ca >= a.a_cols || cb >= a.b_cols) continue;
          if (slot >= 0) partial[slot * size + ca * a.b_cols + cb] = v[h]; else static_cast<O*>(a.out)[slice.leaf * size + ca * a.b_cols + cb] = FromFloat<O>(v[h]);
        }
      }
  }
}

// Adds the sums of the slices of each leaf that has several, always in the same order. Few slices: a thread adds all of its four sums'
// slices. More: a warp has 32 neighbouring sums and an eighth of the slices, the eighths are added up at the end (the only form before:
// 31 slices of 15 leaves' 513 x 1000 sums, half of them joined, took 151 us, a block's two barriers for every 32 sums).
constexpr int kFewSlices = 16;
template <typename O>
__global__ void __launch_bounds__(256) LeafGramJoinKernel(LeafGramArgs a, int rows_per_slice, const float* __restrict__ partial) {
  __shared__ float s_part[8][32];
  const long long size = static_cast<long long>(a.a_cols) * a.b_cols;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int g = blockIdx.y; g < a.leaves.leaves; g += gridDim.y) {
    const int b = Boundary(a.leaves, g), e = max(b, Boundary(a.leaves, g + 1));      // where boundaries fall again: any slices of the workspace
    if (e - b <= rows_per_slice) continue;
    const int slices = TilesIn(b, e, rows_per_slice, 1), each = (slices + 7) / 8, first = warp * each, last = min(slices, first + each);
    const float* of_leaf = partial + 2LL * (b / rows_per_slice) * size;      // first slice here, the others one place and two places apart
    if (slices <= kFewSlices) {
      const long long on = 2 * size;
      for (long long i0 = static_cast<long long>(blockIdx.x) * 1024 + threadIdx.x; i0 < size; i0 += static_cast<long long>(gridDim.x) * 1024) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = i0 + 256 * j < size ? __ldg(of_leaf + i0 + 256 * j) : 0.f;
        const float* from = of_leaf + size + i0;
#pragma unroll 2
        for (int s = 1; s < slices; ++s) {
          from += on;
#pragma unroll
          for (int j = 0; j < 4; ++j) if (i0 + 256 * j < size) v[j] += __ldg(from + 256 * j);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) if (i0 + 256 * j < size) static_cast<O*>(a.out)[g * size + i0 + 256 * j] = FromFloat<O>(v[j]);
      }
      continue;
    }
    for (long long i0 = static_cast<long long>(blockIdx.x) * 32; i0 < size; i0 += static_cast<long long>(gridDim.x) * 32) {
      const long long i = i0 + lane;
      float v = 0.f;
      if (i < size) {
#pragma unroll 8
        for (int s = first; s < last; ++s) v += __ldg(of_leaf + (2 * s + (s == 0 ? 0 : 1)) * size + i);
      }
      s_part[warp][lane] = v;
      __syncthreads();
      if (warp == 0 && i < size) {
        v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += s_part[w][lane];
        static_cast<O*>(a.out)[g * size + i] = FromFloat<O>(v);
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------------------------- 16-bit types ----
// Lines that do not start on 16-byte boundaries, copied to lines that do: tensor-map copies need it, and the tensor cores read an
// operand many times. A thread writes 8 values; it reads whole words and shifts where the line starts between two.
__global__ void __launch_bounds__(256) PackLinesKernel(const unsigned short* __restrict__ from, long long stride, long long lines, int along, unsigned short* __restrict__ to, int to_stride) {
  const int pieces = to_stride / 8;
  const long long total = lines * pieces;
  for (long long e = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; e < total; e += static_cast<long long>(gridDim.x) * 256) {
    const long long line = e / pieces;
    const int c = static_cast<int>(e - line * pieces) * 8;
    const unsigned short* src = from + line * stride + c;
    unsigned int w[4];
    const bool odd = (reinterpret_cast<uintptr_t>(src) & 2) != 0;
    if (c + 8 <= along && (!odd || (c > 0 && c + 9 <= along))) {       // the words read lie within the line
      const unsigned int* words = reinterpret_cast<const unsigned int*>(odd ? src - 1 : src);
      unsigned int v[5];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __ldg(words + i);
      v[4] = odd ? __ldg(words + 4) : 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = odd ? __funnelshift_r(v[i], v[i + 1], 16) : v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned int lo = c + 2 * i < along ? __ldg(src + 2 * i) : 0u, hi = c + 2 * i + 1 < along ? __ldg(src + 2 * i + 1) : 0u;
        w[i] = lo | (hi << 16);
      }
    }
    reinterpret_cast<uint4*>(to + line * to_stride)[c / 8] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// D [128 x N] += A [128 x 64] B [64 x N] steps on the tensor cores, N <= 256, accumulators in tensor memory (two sets, so that
// one tile is stored while the next is summed). Products: A = 128 rows of x, B = N outputs of the leaf's map, the steps walk the
// features. Gram: A = 128 columns of one side, B = N of the other, the steps walk the slice's rows.
// Operands lie in shared memory in the 128-byte-swizzled layout: lines of 64 values, the 16-byte piece c of line l at piece
// c ^ (l % 8). A line is a row / output with 64 features (K-major), or a feature / row with 64 outputs / columns (MN-major), whatever
// is contiguous in memory. An operand whose lines start on 16-byte boundaries comes by tensor-map copies (TMA) issued by one thread;
// others go through the copying warps in pieces of 8 or 4 bytes or single values. Rows of a neighbouring leaf in an x tile
// reach only outputs that are not stored; in a Gram's last step, where they would be summed, the copying warps bring the rows
// that belong to the slice and zeros (unless the slice ends at a multiple of 16 rows, the depth of an instruction).
// Warps: 0-3 store the accumulators, 4-11 copy, 12 issues the matrix instructions. Every wait is bounded (a try lasts 4 us: 4 s); one
// that gives up makes all roles leave, and no role waits again: a phase that never completes would look complete to the wait for the
// next one but one, whose parity is the other. The outputs of every tile that is not finished are NaN then. What is in flight is waited
// for before the block ends.
constexpr int kDepthTc = 64, kTileM = 128, kMostN = 256;
constexpr int kCopyWarps = 8, kCopyThreads = 32 * kCopyWarps, kTcThreads = 128 + kCopyThreads + 32;
constexpr int kMostStages = 8;
constexpr int kLag = 5, kLagFew = 2;               // a stage is handed over when so many younger ones are on their way (of 8; of fewer stages)
constexpr int kABytes = kTileM * 128;
// Outputs go through shared memory, 64 columns of a warp's 32 rows at a time, so that a row is stored by neighbouring lanes: eight with 16
// bytes each, or value by value where rows do not start on 16-byte boundaries (stored by its own lane, value by value, 200000 x 100 -> 100
// took 130 us, of it 100 for the stores; by its own lane in 16-byte pieces, 50000 x 512 -> 1000 took 88 us, so 77).
constexpr int kStorePitch = 33, kStoreBytes = 4 * 32 * kStorePitch * 4;      // words: a row's 64 values and one to spare


__device__ __forceinline__ void BarInit(unsigned long long* bar, unsigned int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(Smem32(bar)), "r"(count) : "memory"); }
__device__ __forceinline__ void BarArrive(unsigned long long* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(Smem32(bar)) : "memory"); }
__device__ __forceinline__ bool BarTry(unsigned long long* bar, unsigned int parity) {
  unsigned int ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(Smem32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
constexpr int kWaitTries = 1 << 20, kDrainTries = 1 << 12;
// false: the tries ran out, here or in another role
__device__ __forceinline__ bool BarWait(unsigned long long* bar, unsigned int parity, int tries, volatile int* stop) {
  do { if (BarTry(bar, parity)) return true; if (*stop != 0) return false; } while (--tries > 0);
  *stop = 1;
  return false;
}
__device__ __forceinline__ void MmaCommit(unsigned long long* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(Smem32(bar)) : "memory");
}
// 128-byte swizzle. K-major: 8-line groups `stride` = 1024 bytes apart. MN-major: 8-line groups 1024 bytes apart, blocks of 64 values
// `lead` = 8192 bytes apart.
__device__ __forceinline__ unsigned long long OperandDesc(unsigned int addr, unsigned int lead) {
  return static_cast<unsigned long long>((addr & 0x3FFFFu) >> 4) | (static_cast<unsigned long long>(lead >> 4) << 16) | (static_cast<unsigned long long>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void Mma16(unsigned int d, unsigned long long da, unsigned long long db, unsigned int idesc, bool accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
               ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(0u) : "memory");
}
__device__ __forceinline__ void TmemLoad16(unsigned int addr, unsigned int* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(addr) : "memory");
}

__device__ __forceinline__ void BarExpect(unsigned long long* bar, unsigned int bytes) { asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(Smem32(bar)), "r"(bytes) : "memory"); }
__device__ __forceinline__ void BarArriveExpect(unsigned long long* bar, unsigned int bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(Smem32(bar)), "r"(bytes) : "memory"); }
__device__ __forceinline__ void TmaLoad2D(unsigned int dst, const CUtensorMap* map, int x, int y, unsigned long long* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(reinterpret_cast<unsigned long long>(map)), "r"(x), "r"(y), "r"(Smem32(bar)) : "memory");
}
__device__ __forceinline__ void TmaLoad3D(unsigned int dst, const CUtensorMap* map, int x, int y, int z, unsigned long long* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(reinterpret_cast<unsigned long long>(map)), "r"(x), "r"(y), "r"(z), "r"(Smem32(bar)) : "memory");
}

// One operand's part of a tile in memory: `lines` lines `stride` values apart, `along` values each.
struct OperandView { const unsigned short* base; long long stride; int lines, along; };

// `valid` of 8 values to a 16-byte piece of shared memory, the rest zero.
__device__ __forceinline__ void CopyPiece(unsigned int dst, const unsigned short* src, int valid, int vec) {
  if (vec == 8) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(2 * valid) : "memory");
  } else if (vec == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = max(0, min(4, valid - 4 * h));
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + 8 * h), "l"(n > 0 ? src + 4 * h : src), "r"(2 * n) : "memory");
    }
  } else if (vec == 2) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int n = max(0, min(2, valid - 2 * h));
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * h), "l"(n > 0 ? src + 2 * h : src), "r"(2 * n) : "memory");
    }
  } else {
    unsigned int w[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const unsigned int lo = 2 * h < valid ? __ldg(src + 2 * h) : 0u, hi = 2 * h + 1 < valid ? __ldg(src + 2 * h + 1) : 0u;
      w[h] = lo | (hi << 16);
    }
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
  }
}
// Lines of `depth` (a multiple of 16) features from k0 on.
__device__ __forceinline__ void CopyKMajor(unsigned int dst, const OperandView& o, int tile_lines, int k0, int depth, int vec, int tid) {
  const int c = tid & 7;
  if (c * 8 >= depth) return;
  const int along = max(0, min(8, o.along - (k0 + 8 * c)));
#pragma unroll 4
  for (int l = tid >> 3; l < tile_lines; l += kCopyThreads / 8) {
    const int valid = l < o.lines ? along : 0;
    CopyPiece(dst + l * 128 + ((c ^ (l & 7)) << 4), valid > 0 ? o.base + l * o.stride + k0 + 8 * c : o.base, valid, vec);
  }
}
// `depth` lines from k0 on, of `pieces` 16-byte pieces.
__device__ __forceinline__ void CopyMnMajor(unsigned int dst, const OperandView& o, int pieces, int k0, int depth, int vec, int tid) {
  const int bits = 32 - __clz(pieces - 1), c = tid & ((1 << bits) - 1);      // pieces 2..32
  if (c >= pieces) return;
  const int along = max(0, min(8, o.along - 8 * c));
#pragma unroll 4
  for (int l = tid >> bits; l < depth; l += kCopyThreads >> bits) {
    const int valid = k0 + l < o.lines ? along : 0;
    CopyPiece(dst + (c >> 3) * 8192 + l * 128 + (((c & 7) ^ (l & 7)) << 4), valid > 0 ? o.base + (k0 + l) * o.stride + 8 * c : o.base, valid, vec);
  }
}

// What a launch walks, for both products.
struct TensorArgs {
  LeafWindows leaves; int tile_rows, least;                     // rows per tile or slice; tiles of a leaf without rows
  const unsigned short *a, *b; long long a_stride, b_stride, b_leaf_stride;
  int a_tma, b_tma, b_leaf_on;                                  // operand by tensor map; 1: its third coordinate is the leaf
  int a_vec, b_vec, a_size, b_size, depth;                      // columns of a Gram's sides; outputs (b_size) and features (depth) of products
  int n, across_a, across_b, stages, stage_bytes, tmem_cols, wait_tries;
  unsigned int idesc;
  void* out; float* partial; long long out_row_stride, out_col_stride;
};
enum { kProductsK, kProductsMn, kGram };

template <typename T, typename O, int MODE>
__global__ void __launch_bounds__(kTcThreads, 1) LeafTensorKernel(const __grid_constant__ TensorArgs a, const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map) {
  extern __shared__ unsigned char s_raw[];
  __shared__ TileMap map;
  __shared__ unsigned long long s_full[kMostStages], s_empty[kMostStages], s_done[2], s_free[2], s_cut, s_go;
  __shared__ unsigned int s_tmem; __shared__ int s_stop, s_go_stage;
  unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(Smem32(&s_tmem)), "r"(a.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) { BarInit(s_full + i, a.a_tma != 0 && a.b_tma != 0 ? 1 : kCopyWarps); BarInit(s_empty + i, 1); }
    for (int i = 0; i < 2; ++i) { BarInit(s_done + i, 1); BarInit(s_free + i, 4); }
    BarInit(&s_cut, kCopyWarps); BarInit(&s_go, 1);
    s_stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  map.Build(a.leaves, a.tile_rows, a.least);
  if constexpr (MODE != kGram) ZeroLeaflessRows(map, a.leaves, static_cast<O*>(a.out), a.b_size);
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned int tmem = *reinterpret_cast<volatile unsigned int*>(&s_tmem);
  volatile int* stop = &s_stop;
  const int across = a.across_a * a.across_b;
  const int tiles = map.Total() * across;
  int issued = 0, last_stage = 0; unsigned int last_parity = 0;      // steps copied (first copying thread) or multiplied (issuing thread); the latter's last stage
  // Products: the row tiles of the leaves, `across_b` output tiles each. Gram: slices, across_a x across_b tiles each.
  struct Tile { int leaf, which, m0, n0, depth, row0, end, leaf_begin, leaf_end; };
  int span = 0;
  auto tile_of = [&](int t) {
    Tile r;
    r.which = t / across;
    const int rest = t - r.which * across;
    map.Find(a.leaves, r.which, a.tile_rows, a.least, &span, &r.leaf, &r.row0, &r.end, &r.leaf_begin, &r.leaf_end);
    r.m0 = MODE == kGram ? rest / a.across_b * kTileM : 0; r.n0 = rest % a.across_b * a.n;
    r.depth = MODE == kGram ? r.end - r.row0 : a.depth;
    return r;
  };

  if (warp >= 4 && warp < 12) {
    const int tid = threadIdx.x - 128;
    const bool both = a.a_tma != 0 && a.b_tma != 0;
    const int lag = a.stages > kLag + 1 ? kLag : kLagFew;
    int it = 0, cuts = 0, fill = 0;
    unsigned int fill_parity = 1;            // of the stage's use before: flips when the ring starts over (the first use waits for nothing)
    bool ok = true;
    auto hand_over = [&](int step) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // this thread's copies -> visible to the tensor core's reads
      __syncwarp();
      if (lane == 0) BarArrive(s_full + step % a.stages);
    };
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const Tile tile = tile_of(t);
      OperandView va, vb;
      const int rows = tile.end - tile.row0;
      va.stride = a.a_stride; vb.stride = a.b_stride;
      if constexpr (MODE == kGram) {
        va.base = a.a + static_cast<long long>(tile.row0) * a.a_stride + tile.m0; va.lines = rows; va.along = a.a_size - tile.m0;
        vb.base = a.b + static_cast<long long>(tile.row0) * a.b_stride + tile.n0; vb.lines = rows; vb.along = a.b_size - tile.n0;
      } else {
        va.base = a.a + static_cast<long long>(tile.row0) * a.a_stride; va.lines = rows; va.along = a.depth;
        if constexpr (MODE == kProductsK) { vb.base = a.b + tile.leaf * a.b_leaf_stride + tile.n0 * a.b_stride; vb.lines = a.b_size - tile.n0; vb.along = a.depth; }
        else { vb.base = a.b + tile.leaf * a.b_leaf_stride + tile.n0; vb.lines = a.depth; vb.along = a.b_size - tile.n0; }
      }
      auto load = [&](bool ta, bool tb, int st, int k0) {      // one thread
        const unsigned int sa = Smem32(stages + static_cast<size_t>(st) * a.stage_bytes), sb = sa + kABytes;
        const int b_boxes = (a.n + 63) / 64;
        if (ta) {
          if constexpr (MODE == kGram) { for (int i = 0; i < 2; ++i) TmaLoad2D(sa + i * 8192, &a_map, tile.m0 + 64 * i, tile.row0 + k0, s_full + st); }
          else TmaLoad2D(sa, &a_map, k0, tile.row0, s_full + st);
        }
        if (tb) {
          if constexpr (MODE == kProductsK) { TmaLoad3D(sb, &b_map, k0, tile.n0, tile.leaf * a.b_leaf_on, s_full + st); }
          else if constexpr (MODE == kGram) { for (int i = 0; i < b_boxes; ++i) TmaLoad2D(sb + i * 8192, &b_map, tile.n0 + 64 * i, tile.row0 + k0, s_full + st); }
          else { for (int i = 0; i < b_boxes; ++i) TmaLoad3D(sb + i * 8192, &b_map, tile.n0 + 64 * i, k0, tile.leaf * a.b_leaf_on, s_full + st); }
        }
      };
      auto copy = [&](bool ca, bool cb, int st, int k0) {      // all copying warps
        const unsigned int sa = Smem32(stages + static_cast<size_t>(st) * a.stage_bytes), sb = sa + kABytes;
        const int depth = min(kDepthTc, (tile.depth - k0 + 15) & ~15);
        if (ca) { if constexpr (MODE == kGram) CopyMnMajor(sa, va, kTileM / 8, k0, depth, a.a_vec, tid); else CopyKMajor(sa, va, kTileM, k0, depth, a.a_vec, tid); }
        if (cb) { if constexpr (MODE == kProductsK) CopyKMajor(sb, vb, a.n, k0, depth, a.b_vec, tid); else CopyMnMajor(sb, vb, a.n / 8, k0, depth, a.b_vec, tid); }
        CopyCommit();
      };
      const unsigned int a_bytes = kABytes, b_bytes = MODE == kProductsK ? a.n * 128 : (a.n + 63) / 64 * 8192;
      if (both) {
        // One thread fills the stages; all warps come together only for a Gram's ragged last step.
        const int steps = (tile.depth + kDepthTc - 1) / kDepthTc, cut = MODE == kGram && (tile.depth & 15) != 0 ? 1 : 0;
        if (tid == 0) {
          for (int i = 0; i < steps - cut; ++i) {
            if (it >= a.stages && !BarWait(s_empty + fill, fill_parity, a.wait_tries, stop)) { ok = false; break; }
            BarArriveExpect(s_full + fill, a_bytes + b_bytes);
            load(true, true, fill, i * kDepthTc);
            ++it;
            if (++fill == a.stages) { fill = 0; fill_parity ^= 1u; }
          }
        }
        ok = __all_sync(0xffffffffu, ok) != 0;      // the filling thread's warp leaves as a whole: it meets at barriers below
        if (cut != 0 && ok) {
          // the filling thread alone knows when the stage is free: the others skip steps, and a parity tells neighbouring uses apart only
          if (tid == 0) { if (it >= a.stages) ok = BarWait(s_empty + fill, fill_parity, a.wait_tries, stop); if (ok) { s_go_stage = fill; BarArrive(&s_go); } }
          __syncwarp();
          ok = ok && BarWait(&s_go, cuts & 1, a.wait_tries, stop);
          ok = __all_sync(0xffffffffu, ok) != 0;
          if (ok) {
            const int st = *const_cast<volatile int*>(&s_go_stage);
            copy(true, true, st, (steps - 1) * kDepthTc);
            CopyWait<0>();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) BarArrive(&s_cut);
            if (tid == 0) {
              ok = BarWait(&s_cut, cuts & 1, a.wait_tries, stop);
              if (ok) { BarArrive(s_full + st); ++it; if (++fill == a.stages) { fill = 0; fill_parity ^= 1u; } }
            }
            ok = __all_sync(0xffffffffu, ok) != 0;
          }
          ++cuts;
        }
      } else {
        for (int k0 = 0; k0 < tile.depth; k0 += kDepthTc, ++it) {
          const int st = it % a.stages;
          if (it >= a.stages) ok = __all_sync(0xffffffffu, BarWait(s_empty + st, ((it / a.stages) - 1) & 1, a.wait_tries, stop)) != 0;      // one decision per warp
          if (!ok) break;
          const bool cut = MODE == kGram && ((tile.depth - k0) & 15) != 0 && tile.depth - k0 < kDepthTc;
          const bool ta = a.a_tma != 0 && !cut, tb = a.b_tma != 0 && !cut;
          if (tid == 0 && (ta || tb)) { BarExpect(s_full + st, (ta ? a_bytes : 0) + (tb ? b_bytes : 0)); load(ta, tb, st, k0); }
          copy(!ta, !tb, st, k0);
          if (it >= lag) { if (lag == kLag) CopyWait<kLag>(); else CopyWait<kLagFew>(); hand_over(it - lag); }
        }
      }
    }
    CopyWait<0>();
    if (!both) for (int step = max(0, it - lag); step < it; ++step) hand_over(step);
    issued = it;
  } else if (warp == 12) {
    if (lane == 0) {
      // One thread feeds the tensor cores: its own instructions must take less time than the matrix instructions that they issue (512
      // cycles a step), so stages, parities and descriptors are carried along by adding (worked out anew: 1000 cycles a step).
      int set = 0, st = 0;
      unsigned int parity = 0;
      bool ok = true;
      const unsigned long long a_desc0 = OperandDesc(Smem32(stages), MODE == kGram ? 8192 : 16), b_desc0 = OperandDesc(Smem32(stages) + kABytes, MODE == kProductsK ? 16 : 8192);
      const unsigned int stage_on = static_cast<unsigned int>(a.stage_bytes) >> 4;
      // 16 deep at a time: 32 bytes on inside a K-major line, 16 lines on in MN-major order
      constexpr unsigned int kAOn = MODE == kGram ? 2048 >> 4 : 32 >> 4, kBOn = MODE == kProductsK ? 32 >> 4 : 2048 >> 4;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const Tile tile = tile_of(t);
        if (tile.depth == 0) continue;
        const int acc = set & 1;
        if (set >= 2 && !BarWait(s_free + acc, ((set >> 1) - 1) & 1, a.wait_tries, stop)) { ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned int d = tmem + acc * (a.tmem_cols / 2);
        bool fresh = true;
        for (int left = tile.depth; left > 0; left -= kDepthTc) {
          if (!BarWait(s_full + st, parity, a.wait_tries, stop)) { ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const unsigned long long da = a_desc0 + static_cast<unsigned long long>(st * stage_on), db = b_desc0 + static_cast<unsigned long long>(st * stage_on);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (16 * k < left) { Mma16(d, da + k * kAOn, db + k * kBOn, a.idesc, !fresh); fresh = false; }
          MmaCommit(s_empty + st);
          ++issued;
          if (++st == a.stages) { st = 0; parity ^= 1u; }
        }
        if (ok) { MmaCommit(s_done + acc); ++set; }
      }
      last_stage = st == 0 ? a.stages - 1 : st - 1; last_parity = st == 0 ? parity ^ 1u : parity;
    }
    __syncwarp();
  } else {
    int set = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
      const Tile tile = tile_of(t);
      const int acc = set & 1;
      if (tile.depth > 0) {
        ok = ok && BarWait(s_done + acc, (set >> 1) & 1, a.wait_tries, stop);
        ok = __all_sync(0xffffffffu, ok);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        ++set;
      }
      const unsigned int sums = tmem + acc * (a.tmem_cols / 2) + (static_cast<unsigned int>(warp * 32) << 16);
      const int n_end = min(a.n, a.b_size - tile.n0);
      if constexpr (MODE != kGram) {
        const bool pieces = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_row_stride % 8 == 0;
        unsigned int* s_words = reinterpret_cast<unsigned int*>(stages + static_cast<size_t>(a.stages) * a.stage_bytes) + warp * 32 * kStorePitch;
        O* rows_out = static_cast<O*>(a.out) + (tile.row0 + warp * 32) * a.out_row_stride + tile.n0;
        const int rows = max(0, min(32, tile.end - tile.row0 - warp * 32));
        for (int c0 = 0; c0 < n_end; c0 += 64) {
#pragma unroll 1
          for (int h = 0; h < 2 && c0 + 32 * h < a.n; ++h) {
            unsigned int v[32];
            if (ok) {
              TmemLoad16(sums + c0 + 32 * h, v);
              if (c0 + 32 * h + 16 < a.n) TmemLoad16(sums + c0 + 32 * h + 16, v + 16);
              asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = 0x7fc00000u;
            }
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              union { O o[8]; unsigned int w[4]; uint4 q; } u;
#pragma unroll
              for (int j = 0; j < 8; ++j) u.o[j] = FromFloat<O>(__uint_as_float(v[8 * p + j]));
              if (pieces) reinterpret_cast<uint4*>(s_words)[8 * lane + ((4 * h + p) ^ (lane & 7))] = u.q;      // eight lanes then write to all banks
              else {
#pragma unroll
                for (int j = 0; j < 4; ++j) s_words[lane * kStorePitch + 16 * h + 4 * p + j] = u.w[j];
              }
            }
          }
          __syncwarp();
          const int cols = min(64, n_end - c0);
          const O* s_row = reinterpret_cast<const O*>(s_words);
          if (pieces) {
            const int p = lane & 7;
            if (8 * p < cols) {
#pragma unroll
              for (int r = lane >> 3; r < 32; r += 4)
                if (r < rows) *reinterpret_cast<uint4*>(rows_out + r * a.out_row_stride + c0 + 8 * p) = reinterpret_cast<const uint4*>(s_words)[8 * r + (p ^ (r & 7))];
            }
          } else if (cols > 32) {
            for (int r = 0; r < rows; ++r) {
              O* to = rows_out + static_cast<long long>(r) * a.out_row_stride + c0; const O* from = s_row + r * 2 * kStorePitch;
              to[lane] = from[lane];
              if (32 + lane < cols) to[32 + lane] = from[32 + lane];
            }
          } else {      // several rows at a time
            const int at_once = 32 / cols, r_on = lane / cols, c = lane - r_on * cols;
            if (r_on < at_once)
              for (int r = r_on; r < rows; r += at_once) rows_out[static_cast<long long>(r) * a.out_row_stride + c0 + c] = s_row[r * 2 * kStorePitch + c];
          }
          __syncwarp();
        }
      } else {
        const int m = warp * 32 + lane, m_end = min(kTileM, a.a_size - tile.m0);
        const long long at = (tile.m0 + m) * a.out_row_stride + tile.n0 * a.out_col_stride;
        const int slot = SliceSlot(tile.leaf_begin, tile.leaf_end, tile.row0, a.tile_rows);
        O* out = static_cast<O*>(a.out) + static_cast<long long>(tile.leaf) * a.a_size * a.b_size + at;
        float* part = slot >= 0 ? a.partial + static_cast<long long>(slot) * a.a_size * a.b_size + at : nullptr;
        for (int c0 = 0; c0 < n_end; c0 += 16) {
          unsigned int v[16];
          if (tile.depth > 0 && ok) {
            TmemLoad16(sums + c0, v);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = tile.depth == 0 ? 0u : 0x7fc00000u;
          }
          if (m < m_end) {
            if (part != nullptr) {
#pragma unroll
              for (int j = 0; j < 16; ++j) if (c0 + j < n_end) part[(c0 + j) * a.out_col_stride] = __uint_as_float(v[j]);
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j) if (c0 + j < n_end) out[(c0 + j) * a.out_col_stride] = FromFloat<O>(__uint_as_float(v[j]));
            }
          }
          __syncwarp();      // the next read of tensor memory is one of the whole warp
        }
      }
      if (tile.depth > 0 && ok) {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) BarArrive(s_free + acc);
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*stop != 0) {      // a role left early: copies in flight still write shared memory, matrix instructions still read it and write their sums
    if (threadIdx.x == 128 && (a.a_tma != 0 || a.b_tma != 0))
      for (int step = max(0, issued - a.stages); step < issued; ++step)
        for (int i = 0; i < kDrainTries && !BarTry(s_full + step % a.stages, (step / a.stages) & 1); ++i) {}
    if (warp == 12 && lane == 0 && issued > 0) for (int i = 0; i < kDrainTries && !BarTry(s_empty + last_stage, last_parity); ++i) {}
    __syncthreads();
  }
  if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
}

std::atomic<int> g_wait_tries{kWaitTries};

template <typename F> void DispatchHalf(int dtype, F&& f) {
  switch (dtype) {
    case kOpFloat16: f(static_cast<__half*>(nullptr)); return;
    case kOpBFloat16: f(static_cast<__nv_bfloat16*>(nullptr)); return;
    default: Log::Fatal("leaf products: unknown type code %d", dtype);
  }
}

inline void CheckTiles(long long tiles) { if (tiles > 0x7ff00000LL) Log::Fatal("leaf products: %lld tiles are not covered", tiles); }
inline int PackedStride(int along) { return (along + 7) / 8 * 8; }
void LaunchPack(const unsigned short* from, long long stride, long long lines, int along, unsigned short* to, cudaStream_t s) {
  const long long pieces = lines * (PackedStride(along) / 8);
  PackLinesKernel<<<static_cast<unsigned int>(std::max(1LL, std::min<long long>(kSms * 16, (pieces + 255) / 256))), 256, 0, s>>>(from, stride, lines, along, to, PackedStride(along));
  FB_LAUNCHED(); FB_KERNEL_CHECK();
}
// Widest pieces (in values) that an operand's start and strides allow.
inline int PieceWidth(const void* p, long long stride0, long long stride1) {
  for (int v = 8; v > 1; v /= 2) if (reinterpret_cast<uintptr_t>(p) % (2 * v) == 0 && stride0 % v == 0 && stride1 % v == 0) return v;
  return 1;
}
// N of the tiles of `size` columns: as few tiles as 256 allows, evenly filled.
inline int TileN(int size) { const int tiles = (size + kMostN - 1) / kMostN; return ((size + tiles - 1) / tiles + 15) / 16 * 16; }

PFN_cuTensorMapEncodeTiled_v12000 TensorMapEncoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr; cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}
// Map of `along` x `lines` (x `leaves`) values, boxes of 64 x box_lines, 128-byte swizzle. false: such an operand is copied by the warps.
template <typename T>
bool EncodeMap(CUtensorMap* map, const void* p, int dims, long long along, long long lines, long long leaves, long long line_stride, long long leaf_stride, int box_lines) {
  const PFN_cuTensorMapEncodeTiled_v12000 encode = TensorMapEncoder();
  if (encode == nullptr || PieceWidth(p, line_stride, leaf_stride) != 8 || line_stride < along || (dims == 3 && leaves > 1 && leaf_stride <= 0)) return false;
  const cuuint64_t size[3] = {static_cast<cuuint64_t>(along), static_cast<cuuint64_t>(lines), static_cast<cuuint64_t>(leaves)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(line_stride) * 2, static_cast<cuuint64_t>(leaves > 1 ? leaf_stride : line_stride * lines) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_lines), 1}, step[3] = {1, 1, 1};
  const CUtensorMapDataType type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode(map, type, dims, const_cast<void*>(p), size, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, typename O, int MODE>
void LaunchTensor(TensorArgs a, long long most_tiles, cudaStream_t s) {
  CUtensorMap a_map = CUtensorMap(), b_map = CUtensorMap();
  const long long rows = a.leaves.rows;
  // a map shared by all leaves (stride 0) is one leaf to the tensor map
  const bool shared = a.b_leaf_stride == 0 || a.leaves.leaves == 1;
  a.b_leaf_on = shared ? 0 : 1;
  const long long leaves = shared ? 1 : a.leaves.leaves;
  if (MODE == kGram) {
    a.a_tma = EncodeMap<T>(&a_map, a.a, 2, a.a_size, rows, 1, a.a_stride, 0, kDepthTc); a.b_tma = EncodeMap<T>(&b_map, a.b, 2, a.b_size, rows, 1, a.b_stride, 0, kDepthTc);
  } else {
    a.a_tma = EncodeMap<T>(&a_map, a.a, 2, a.depth, rows, 1, a.a_stride, 0, kTileM);
    if (MODE == kProductsK) a.b_tma = EncodeMap<T>(&b_map, a.b, 3, a.depth, a.b_size, leaves, a.b_stride, a.b_leaf_stride, a.n);
    else a.b_tma = EncodeMap<T>(&b_map, a.b, 3, a.b_size, a.depth, leaves, a.b_stride, a.b_leaf_stride, kDepthTc);
  }
  const int store_bytes = MODE == kGram ? 0 : kStoreBytes, most_bytes = 216 * 1024;
  a.stage_bytes = kABytes + (a.n + 63) / 64 * 64 * 128;
  a.stages = std::min(kMostStages, (most_bytes - 1024 - store_bytes) / a.stage_bytes);
  a.tmem_cols = 32; while (a.tmem_cols < a.n) a.tmem_cols *= 2;
  a.tmem_cols *= 2;
  // D fp32; A, B fp16 (0) or bf16 (1), their majors; N, M
  const unsigned int type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  a.idesc = (1u << 4) | (type << 7) | (type << 10) | (MODE == kGram ? 1u << 15 : 0u) | (MODE != kProductsK ? 1u << 16 : 0u) | (static_cast<unsigned int>(a.n >> 3) << 17) | (static_cast<unsigned int>(kTileM >> 4) << 24);
  a.wait_tries = g_wait_tries.load(std::memory_order_relaxed);
  CheckTiles(most_tiles);
  const int bytes = a.stages * a.stage_bytes + 1024 + store_bytes;
  static PerDevice allowed;
  AllowSharedMemory(LeafTensorKernel<T, O, MODE>, most_bytes, &allowed);
  LeafTensorKernel<T, O, MODE><<<static_cast<unsigned int>(std::min<long long>(most_tiles, kSms)), kTcThreads, bytes, s>>>(a, a_map, b_map);
}

// Widest pieces (in floats) of a side whose lines start at p, `stride` apart.
inline int FloatPieces(const void* p, long long stride) {
  for (int v = 4; v > 1; v /= 2) if (reinterpret_cast<uintptr_t>(p) % (4 * v) == 0 && stride % v == 0) return v;
  return 1;
}
// At most so many slices: whole ones, and every leaf's last.
inline long long LeafGramTiles(const LeafGramArgs& a) { return a.leaves.rows / std::max(1, LeafGramSliceRows(a)) + a.leaves.leaves; }
template <int TM, int TN, int WR, int WO>
void LaunchFloatProducts(const LeafProductsArgs& a, cudaStream_t s) {
  using Tile = FloatTile<TM, TN, WR, WO>;
  FloatShape shape;
  shape.width = std::min(kDepth, (a.features + 3) / 4 * 4); shape.pitch = shape.width / 4 % 2 == 0 ? shape.width + 4 : shape.width;
  shape.x_vec = FloatPieces(a.x, a.x_stride); shape.w_by_output = a.weight_in_stride != 1 && a.features > 1;
  shape.w_vec = std::min(FloatPieces(a.weight, a.weight_out_stride), FloatPieces(a.weight, a.weight_leaf_stride));
  const int bytes = Tile::Bytes(shape.pitch);
  static PerDevice allowed;
  AllowSharedMemory(LeafProductsFloatKernel<TM, TN, WR, WO>, Tile::Bytes(kDepth + 4), &allowed);
  // as many blocks as are resident, by shared memory (224 KB) and by threads (8 warps of 255 registers, 16 of 128)
  const int per_sm = std::max(1, std::min(224 * 1024 / (bytes + 6 * 1024), 512 / Tile::THREADS));
  const long long tiles = ((a.leaves.rows + Tile::ROWS - 1) / Tile::ROWS + a.leaves.leaves) * ((a.outputs + Tile::OUTS - 1) / Tile::OUTS);
  CheckTiles(tiles);
  LeafProductsFloatKernel<TM, TN, WR, WO><<<static_cast<unsigned int>(std::min<long long>(tiles, kSms * per_sm)), Tile::THREADS, bytes, s>>>(a, shape);
}
// Pieces (in bytes) of rows that start at p, `stride` bytes apart; 2: not for asynchronous copies
inline int BytePieces(const void* p, long long stride) {
  for (int v = 16; v > 2; v /= 2) if (reinterpret_cast<uintptr_t>(p) % v == 0 && stride % v == 0) return v;
  return 2;
}
// Shared memory of a warp: its ring of rows (an odd number of 16-byte pieces apart) and its leaf's map.
inline int NarrowPitch(int row_bytes) { const int pieces = (row_bytes + 15) / 16; return 16 * (pieces | 1); }
inline int NarrowBytes(int tm, int tn, int size, int features, int outputs) {
  const int v = 16 / size, stage = 32 * tm * NarrowPitch(features * size);
  return kNarrowRing * stage + tn * ((features + v - 1) / v * v) * 4 + NarrowOutputBytes(tm, outputs, size, stage);
}
constexpr int kNarrowMostBytes = 216 * 1024;
inline int NarrowOutputs(int outputs) { return outputs <= 16 ? (outputs + 1) / 2 * 2 : (outputs + 3) / 4 * 4; }      // sums that a lane holds per row
// Rows short enough for the warps' rings, on 4-byte boundaries; outputs that fit a lane's registers.
inline bool NarrowProducts(const LeafProductsArgs& a) {
  const int size = a.dtype == kOpFloat32 ? 4 : 2, tn = NarrowOutputs(a.outputs);
  return a.outputs <= 32 && a.features * size <= kNarrowRowBytes && BytePieces(a.x, a.x_stride * size) >= 4 && kNarrowWarps * NarrowBytes(tn <= 16 ? 2 : 1, tn, size, a.features, a.outputs) <= kNarrowMostBytes;
}
template <typename T, int TM, int TN>
void LaunchNarrowProducts(const LeafProductsArgs& a, cudaStream_t s) {
  constexpr int kSize = static_cast<int>(sizeof(T));
  const int bytes = kNarrowWarps * NarrowBytes(TM, TN, kSize, a.features, a.outputs);
  static PerDevice allowed;
  AllowSharedMemory(LeafProductsNarrowKernel<T, TM, TN>, kNarrowMostBytes, &allowed);
  const long long tiles = (a.leaves.rows + 32 * TM - 1) / (32 * TM) + a.leaves.leaves;
  LeafProductsNarrowKernel<T, TM, TN><<<static_cast<unsigned int>(std::max(1LL, std::min<long long>((tiles + kNarrowWarps - 1) / kNarrowWarps, kSms))), kNarrowThreads, bytes, s>>>(
      a, NarrowPitch(a.features * kSize), BytePieces(a.x, a.x_stride * kSize));
}
template <typename T>
void LaunchNarrowProducts(const LeafProductsArgs& a, cudaStream_t s) {
  switch (NarrowOutputs(a.outputs)) {
    case 2: LaunchNarrowProducts<T, 2, 2>(a, s); return;
    case 4: LaunchNarrowProducts<T, 2, 4>(a, s); return;
    case 6: LaunchNarrowProducts<T, 2, 6>(a, s); return;
    case 8: LaunchNarrowProducts<T, 2, 8>(a, s); return;
    case 10: LaunchNarrowProducts<T, 2, 10>(a, s); return;
    case 12: LaunchNarrowProducts<T, 2, 12>(a, s); return;
    case 14: LaunchNarrowProducts<T, 2, 14>(a, s); return;
    case 16: LaunchNarrowProducts<T, 2, 16>(a, s); return;
    case 20: LaunchNarrowProducts<T, 1, 20>(a, s); return;
    case 24: LaunchNarrowProducts<T, 1, 24>(a, s); return;
    case 28: LaunchNarrowProducts<T, 1, 28>(a, s); return;
    default: LaunchNarrowProducts<T, 1, 32>(a, s);
  }
}
inline bool NarrowGram(const LeafGramArgs& a) {
  const int size = a.dtype == kOpFloat32 ? 4 : 2;
  return ((a.a_cols <= 16 && a.b_cols <= 32) || (a.a_cols <= 32 && a.b_cols <= 16)) && BytePieces(a.a, a.a_stride * size) >= 4 && BytePieces(a.b, a.b_stride * size) >= 4;
}
template <typename T, typename O, int GA, int GB>
void LaunchNarrowGram(const LeafGramArgs& a, float* workspace, cudaStream_t s) {
  constexpr int kSize = static_cast<int>(sizeof(T)), kBytes = kNarrowWarps * GramRing(kSize) * kGramRows * 4 * (GA + GB) * kSize;
  static PerDevice allowed;
  AllowSharedMemory(LeafGramNarrowKernel<T, O, GA, GB>, kBytes, &allowed);
  const int rows = LeafGramSliceRows(a);
  LeafGramNarrowKernel<T, O, GA, GB><<<static_cast<unsigned int>(std::max(1LL, std::min<long long>((LeafGramTiles(a) + kNarrowWarps - 1) / kNarrowWarps, kSms))), kNarrowThreads, kBytes, s>>>(
      a, rows, BytePieces(a.a, a.a_stride * kSize), BytePieces(a.b, a.b_stride * kSize), rows < a.leaves.rows ? workspace : nullptr);
}
template <typename T, typename O>
void LaunchNarrowGram(const LeafGramArgs& a, float* workspace, cudaStream_t s) {
  if (a.a_cols <= 16 && a.b_cols <= 32) LaunchNarrowGram<T, O, 4, 8>(a, workspace, s); else LaunchNarrowGram<T, O, 8, 4>(a, workspace, s);
}
template <int TA, int TB, int GA, int GB, int SLICES, int RD>
void LaunchFloatGram(const LeafGramArgs& a, float* workspace, cudaStream_t s) {
  using Tile = FloatGramTile<TA, TB, GA, GB, SLICES, RD>;
  static PerDevice allowed;
  AllowSharedMemory(LeafGramFloatKernel<TA, TB, GA, GB, SLICES, RD>, Tile::kBytes, &allowed);
  const long long across = static_cast<long long>((a.a_cols + Tile::AC - 1) / Tile::AC) * ((a.b_cols + Tile::BC - 1) / Tile::BC);
  const int rows = LeafGramSliceRows(a);
  const bool split = rows < a.leaves.rows;
  const long long tiles = LeafGramTiles(a) * across;
  const int per_sm = std::max(1, std::min(224 * 1024 / (Tile::kBytes + 6 * 1024), 1024 / Tile::THREADS));
  CheckTiles(tiles);
  LeafGramFloatKernel<TA, TB, GA, GB, SLICES, RD><<<static_cast<unsigned int>(std::min<long long>(tiles, kSms * per_sm)), Tile::THREADS, Tile::kBytes, s>>>(
      a, rows, FloatPieces(a.a, a.a_stride), FloatPieces(a.b, a.b_stride), split ? workspace : nullptr);
}
// Gram tiles: 128 columns of b x N columns of a, so that the lanes of a store have neighbouring columns of an output row.
inline long long GramTiles(const LeafGramArgs& a) { const int n = TileN(a.a_cols); return (a.b_cols + 127LL) / 128 * ((a.a_cols + n - 1) / n); }
// Operands that are packed first (see PackLinesKernel). An operand that is read once only, because the other side fits one tile, is
// not worth two more passes over it.
inline bool Unaligned(const void* p, long long stride, long long along) { return PieceWidth(p, stride, 0) != 8 && stride >= along; }
struct GramPacking {
  bool a, b;
  explicit GramPacking(const LeafGramArgs& g) {
    const bool half = g.dtype != kOpFloat32 && !NarrowGram(g);
    a = half && g.b_cols > kTileM && Unaligned(g.a, g.a_stride, g.a_cols);
    b = half && g.a_cols > kTileM && Unaligned(g.b, g.b_stride, g.b_cols);
  }
};
// Products: x is read once per tile of outputs, a map once per tile of its leaf's rows.
struct ProductsPacking {
  bool x, w; long long w_lines; int w_along;
  explicit ProductsPacking(const LeafProductsArgs& p) {
    const bool half = p.dtype != kOpFloat32 && !NarrowProducts(p), by_feature = p.weight_in_stride == 1 || p.features == 1;
    w_lines = by_feature ? p.outputs : p.features; w_along = by_feature ? p.features : p.outputs;
    const long long line_stride = by_feature ? p.weight_out_stride : p.weight_in_stride;
    x = half && p.outputs > kTileM && Unaligned(p.x, p.x_stride, p.features);
    // whole dense maps only: one run of lines for all leaves
    w = half && p.leaves.rows > 2LL * kTileM * p.leaves.leaves && p.leaves.leaves > 1 && line_stride == w_along && p.weight_leaf_stride == w_lines * line_stride &&
        PieceWidth(p.weight, line_stride, p.weight_leaf_stride) != 8;
  }
};

}  // namespace

int SetLeafWaitTries(int tries) { return g_wait_tries.exchange(tries < 1 ? kWaitTries : tries); }

// Rows of a leaf that one block (narrow: one warp) sums up. Slices short enough that uneven leaves even out (4 per SM, 2 per warp), long
// enough that a slice's work outweighs its sums' way through the workspace, and that the workspace stays within 128 MB.
int LeafGramSliceRows(const LeafGramArgs& a) {
  long long outputs = GramTiles(a), least = 1024, per_sm = 4;
  const long long size = static_cast<long long>(a.a_cols) * a.b_cols;
  if (NarrowGram(a)) { outputs = 1; least = 128; per_sm = 2 * kNarrowWarps; }
  else if (a.dtype == kOpFloat32) { outputs = (a.a_cols + 63LL) / 64 * ((a.b_cols + 63) / 64); least = 256; }
  const long long wanted = std::max(1LL, std::min(per_sm * kSms / outputs, (16LL << 20) / size));
  const long long rows = std::max(least, ((a.leaves.rows + wanted - 1) / wanted + 63) / 64 * 64);
  return static_cast<int>(std::min<long long>(rows, std::max(1LL, a.leaves.rows)));
}
// floats of the slices' sums, in whole 16-byte pieces
static long long GramSumFloats(const LeafGramArgs& a) {
  const long long rows = LeafGramSliceRows(a);
  return rows < a.leaves.rows ? (2 * ((a.leaves.rows - 1) / rows + 1) * a.a_cols * a.b_cols + 3) / 4 * 4 : 0;
}
long long LeafGramWorkspace(const LeafGramArgs& a) {
  const GramPacking packing(a);
  return GramSumFloats(a) + a.leaves.rows * ((packing.a ? PackedStride(a.a_cols) : 0) + (packing.b ? PackedStride(a.b_cols) : 0)) / 2;
}
long long LeafProductsWorkspace(const LeafProductsArgs& a) {
  const ProductsPacking packing(a);
  return (packing.x ? a.leaves.rows * PackedStride(a.features) / 2 : 0) + (packing.w ? a.leaves.leaves * packing.w_lines * PackedStride(packing.w_along) / 2 : 0);
}
template <typename T, typename O>
static void LaunchTensorGram(const LeafGramArgs& a, float* workspace, cudaStream_t s) {
  const int rows = LeafGramSliceRows(a);
  const bool split = rows < a.leaves.rows;
  TensorArgs t = TensorArgs();
  t.leaves = a.leaves; t.tile_rows = rows; t.least = 1;
  t.a = static_cast<const unsigned short*>(a.b); t.a_stride = a.b_stride; t.a_size = a.b_cols;
  t.b = static_cast<const unsigned short*>(a.a); t.b_stride = a.a_stride; t.b_size = a.a_cols;
  unsigned short* packed = reinterpret_cast<unsigned short*>(workspace + (split ? GramSumFloats(a) : 0));
  const GramPacking packing(a);
  if (packing.b) { t.a_stride = PackedStride(a.b_cols); LaunchPack(t.a, a.b_stride, a.leaves.rows, a.b_cols, packed, s); t.a = packed; packed += a.leaves.rows * t.a_stride; }
  if (packing.a) { t.b_stride = PackedStride(a.a_cols); LaunchPack(t.b, a.a_stride, a.leaves.rows, a.a_cols, packed, s); t.b = packed; }
  t.a_vec = PieceWidth(t.a, t.a_stride, 0); t.b_vec = PieceWidth(t.b, t.b_stride, 0);
  t.n = TileN(t.b_size); t.across_a = (t.a_size + kTileM - 1) / kTileM; t.across_b = (t.b_size + t.n - 1) / t.n;
  t.out = a.out; t.partial = split ? workspace : nullptr; t.out_row_stride = 1; t.out_col_stride = a.b_cols;
  LaunchTensor<T, O, kGram>(t, LeafGramTiles(a) * t.across_a * t.across_b, s);
}

void LaunchLeafProducts(const LeafProductsArgs& a, float* workspace, cudaStream_t s) {
  if (a.leaves.rows <= 0) return;
  if (NarrowProducts(a)) {
    if (a.dtype == kOpFloat32) LaunchNarrowProducts<float>(a, s);
    else DispatchHalf(a.dtype, [&](auto* p) { LaunchNarrowProducts<std::remove_pointer_t<decltype(p)>>(a, s); });
  } else if (a.dtype == kOpFloat32) {
    if (a.outputs <= 16) LaunchFloatProducts<2, 16, 4, 1>(a, s);
    else if (a.outputs <= 32) LaunchFloatProducts<2, 16, 2, 2>(a, s);
    else LaunchFloatProducts<4, 8, 1, 8>(a, s);
  } else DispatchHalf(a.dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    TensorArgs t = TensorArgs();
    const bool by_feature = a.weight_in_stride == 1 || a.features == 1;
    if (!by_feature && a.weight_out_stride != 1 && a.outputs != 1) Log::Fatal("leaf products: the maps' features or outputs have to be contiguous");
    t.leaves = a.leaves; t.tile_rows = kTileM; t.least = 0;
    t.a = static_cast<const unsigned short*>(a.x); t.a_stride = a.x_stride;
    t.b = static_cast<const unsigned short*>(a.weight); t.b_stride = by_feature ? a.weight_out_stride : a.weight_in_stride; t.b_leaf_stride = a.weight_leaf_stride;
    unsigned short* packed = reinterpret_cast<unsigned short*>(workspace);
    const ProductsPacking packing(a);
    if (packing.x) { t.a_stride = PackedStride(a.features); LaunchPack(t.a, a.x_stride, a.leaves.rows, a.features, packed, s); t.a = packed; packed += a.leaves.rows * t.a_stride; }
    if (packing.w) {
      t.b_stride = PackedStride(packing.w_along); t.b_leaf_stride = packing.w_lines * t.b_stride;
      LaunchPack(t.b, packing.w_along, a.leaves.leaves * packing.w_lines, packing.w_along, packed, s); t.b = packed;
    }
    t.a_vec = PieceWidth(t.a, t.a_stride, 0); t.b_vec = PieceWidth(t.b, t.b_stride, t.b_leaf_stride);
    t.b_size = a.outputs; t.depth = a.features; t.n = TileN(a.outputs); t.across_a = 1; t.across_b = (a.outputs + t.n - 1) / t.n;
    t.out = a.y; t.out_row_stride = a.outputs; t.out_col_stride = 1;
    const long long tiles = ((a.leaves.rows + kTileM - 1) / kTileM + a.leaves.leaves) * t.across_b;
    if (by_feature) LaunchTensor<T, T, kProductsK>(t, tiles, s); else LaunchTensor<T, T, kProductsMn>(t, tiles, s);
  });
  FB_LAUNCHED(); FB_KERNEL_CHECK();
}

void LaunchLeafGram(const LeafGramArgs& a, float* workspace, cudaStream_t s) {
  const int rows = LeafGramSliceRows(a);
  const bool split = rows < a.leaves.rows, same = a.out_dtype == a.dtype;
  if (!same && a.out_dtype != kOpFloat32) Log::Fatal("leaf Gram: sums of type code %d as type code %d", a.dtype, a.out_dtype);
  if (NarrowGram(a)) {
    if (a.dtype == kOpFloat32) LaunchNarrowGram<float, float>(a, workspace, s);
    else DispatchHalf(a.dtype, [&](auto* p) { using T = std::remove_pointer_t<decltype(p)>; if (same) LaunchNarrowGram<T, T>(a, workspace, s); else LaunchNarrowGram<T, float>(a, workspace, s); });
  } else if (a.dtype == kOpFloat32) {
    LaunchFloatGram<8, 8, 8, 8, 4, 32>(a, workspace, s);
  } else {
    DispatchHalf(a.dtype, [&](auto* p) { using T = std::remove_pointer_t<decltype(p)>; if (same) LaunchTensorGram<T, T>(a, workspace, s); else LaunchTensorGram<T, float>(a, workspace, s); });
  }
  FB_LAUNCHED(); FB_KERNEL_CHECK();
  if (!split) return;
  const long long size = static_cast<long long>(a.a_cols) * a.b_cols;
  const dim3 grid(static_cast<unsigned int>(std::min(256LL, (size + 31) / 32)), std::min(a.leaves.leaves, 1024));
  if (a.out_dtype == kOpFloat32) LeafGramJoinKernel<float><<<grid, 256, 0, s>>>(a, rows, workspace);
  else DispatchHalf(a.out_dtype, [&](auto* p) { LeafGramJoinKernel<std::remove_pointer_t<decltype(p)>><<<grid, 256, 0, s>>>(a, rows, workspace); });
  FB_LAUNCHED(); FB_KERNEL_CHECK();
}

}  // namespace fb
