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

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

// Window of leaf g inside [0, rows): whatever the caller's boundaries hold, no access leaves the arrays.
__device__ __forceinline__ void LeafWindow(const LeafWindows& w, int g, long long* begin, long long* end) {
  const long long b = w.begin_bits == 32 ? static_cast<const int*>(w.begin)[g] : static_cast<const long long*>(w.begin)[g];
  const long long e = w.begin_bits == 32 ? static_cast<const int*>(w.begin)[g + 1] : static_cast<const long long*>(w.begin)[g + 1];
  *begin = min(max(b, 0LL), w.rows); *end = min(max(e, *begin), w.rows);
}

// The tiles of all leaves one behind the other: `rows` rows each, a leaf's last one shorter. Up to kSpans leaves are looked up by
// bisection; more are counted in spans of several leaves.
constexpr int kSpans = 1024;
struct TileMap {
  int before[kSpans + 1];        // tiles before span i
  int per, spans;
  __device__ __forceinline__ static int Count(const LeafWindows& w, int g, int rows, int least) {
    long long b, e; LeafWindow(w, g, &b, &e);
    return max(least, static_cast<int>((e - b + rows - 1) / rows));
  }
  // All threads of the block; `least`: tiles of a leaf without rows.
  __device__ void Build(const LeafWindows& w, int rows, int least) {
    const int p = (w.leaves + kSpans - 1) / kSpans, n = (w.leaves + p - 1) / p;
    if (threadIdx.x == 0) { per = p; spans = n; }
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      int c = 0;
      for (int g = i * p; g < min(w.leaves, (i + 1) * p); ++g) c += Count(w, g, rows, least);
      before[i + 1] = c;
    }
    __syncthreads();
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
  // tile -> leaf, its first row and the end of the rows that it covers
  __device__ __forceinline__ void Find(const LeafWindows& w, int tile, int rows, int least, int* leaf, long long* first, long long* end) const {
    int lo = 0, hi = spans;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (before[mid] <= tile) lo = mid; else hi = mid; }
    int g = lo * per, left = tile - before[lo];
    if (per > 1) for (int c = Count(w, g, rows, least); left >= c; c = Count(w, g, rows, least)) { left -= c; ++g; }
    long long b, e; LeafWindow(w, g, &b, &e);
    *leaf = g; *first = min(e, b + static_cast<long long>(left) * rows); *end = min(e, *first + rows);
  }
};

// ------------------------------------------------------------------------------------------------------- fp32 ----
struct F2 { unsigned long long v; };
__device__ __forceinline__ F2 MakeF2(float x, float y) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ void Split(F2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 Fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
__device__ __forceinline__ unsigned int Smem32(const void* p) { return static_cast<unsigned int>(__cvta_generic_to_shared(p)); }
// 4 bytes global -> shared, zero when !in; asynchronous
__device__ __forceinline__ void Copy4(float* dst, const float* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(Smem32(dst)), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ void CopyCommit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING> __device__ __forceinline__ void CopyWait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// Tile: ROWS = 32 * TM * WR rows x OUTS = TN * WO outputs, kDepth features at a time, double-buffered. A lane has TM rows, 32 apart,
// and TN neighbouring outputs, two to a 64-bit register; x lies [feature][row] (odd pitch: the transposing copies and the reads of
// 32 neighbouring rows are both free of bank conflicts), w [feature][output], read by whole warps at once.
constexpr int kDepth = 32;
template <int TM, int TN, int WR, int WO>
struct FloatTile {
  static constexpr int ROWS = 32 * TM * WR, OUTS = TN * WO, THREADS = 32 * WR * WO, XP = ROWS + 1, WP = OUTS + 4;
  static constexpr int kBytes = 2 * kDepth * (XP + WP) * 4;
};
template <int TM, int TN, int WR, int WO>
__global__ void __launch_bounds__(32 * WR * WO) LeafProductsFloatKernel(LeafProductsArgs a) {
  using Tile = FloatTile<TM, TN, WR, WO>;
  extern __shared__ __align__(16) float s_float[];
  __shared__ TileMap map;
  float* s_x = s_float + 2 * kDepth * Tile::WP;      // w first: its rows are read 16 bytes at a time
  float* s_w = s_float;
  map.Build(a.leaves, Tile::ROWS, 0);
  const int across = (a.outputs + Tile::OUTS - 1) / Tile::OUTS;
  const long long tiles = static_cast<long long>(map.Total()) * across;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, wr = warp % WR, wo = warp / WR;
  for (long long t = blockIdx.x; t < tiles; t += gridDim.x) {
    int leaf; long long row0, end;
    map.Find(a.leaves, static_cast<int>(t / across), Tile::ROWS, 0, &leaf, &row0, &end);
    const int out0 = static_cast<int>(t % across) * Tile::OUTS, rows = static_cast<int>(end - row0), outs = min(Tile::OUTS, a.outputs - out0);
    const float* x = static_cast<const float*>(a.x) + row0 * a.x_stride;
    const float* w = static_cast<const float*>(a.weight) + leaf * a.weight_leaf_stride + out0 * a.weight_out_stride;
    auto load = [&](int f0, int buf) {
      float* to = s_x + buf * kDepth * Tile::XP;
#pragma unroll 4
      for (int e = threadIdx.x; e < Tile::ROWS * kDepth; e += Tile::THREADS) {      // lanes: neighbouring features of a row
        const int r = e / kDepth, f = e % kDepth;
        const bool in = r < rows && f0 + f < a.features;
        Copy4(to + f * Tile::XP + r, in ? x + r * a.x_stride + f0 + f : x, in);
      }
      to = s_w + buf * kDepth * Tile::WP;
      for (int e = threadIdx.x; e < Tile::OUTS * kDepth; e += Tile::THREADS) {
        // lanes along whichever of the two is contiguous
        const int o = a.weight_out_stride == 1 ? e % Tile::OUTS : e / kDepth, f = a.weight_out_stride == 1 ? e / Tile::OUTS : e % kDepth;
        const bool in = o < outs && f0 + f < a.features;
        Copy4(to + f * Tile::WP + o, in ? w + o * a.weight_out_stride + (f0 + f) * a.weight_in_stride : w, in);
      }
      CopyCommit();
    };
    F2 acc[TM][TN / 2];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN / 2; ++j) acc[i][j] = MakeF2(0.f, 0.f);
    load(0, 0);
    int buf = 0;
    for (int f0 = 0; f0 < a.features; f0 += kDepth, buf ^= 1) {
      if (f0 + kDepth < a.features) { load(f0 + kDepth, buf ^ 1); CopyWait<1>(); } else CopyWait<0>();
      __syncthreads();
      const float* xs = s_x + buf * kDepth * Tile::XP + wr * 32 * TM + lane;
      const float* ws = s_w + buf * kDepth * Tile::WP + wo * TN;
      const int depth = min(kDepth, a.features - f0);
#pragma unroll 4
      for (int f = 0; f < depth; ++f) {
        F2 wv[TN / 2];
#pragma unroll
        for (int j = 0; j < TN / 4; ++j) { const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(ws + f * Tile::WP + 4 * j); wv[2 * j].v = q.x; wv[2 * j + 1].v = q.y; }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const float v = xs[f * Tile::XP + 32 * i];
          const F2 xv = MakeF2(v, v);
#pragma unroll
          for (int j = 0; j < TN / 2; ++j) acc[i][j] = Fma2(xv, wv[j], acc[i][j]);
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int r = wr * 32 * TM + lane + 32 * i;
      if (r >= rows) continue;
      float* y = static_cast<float*>(a.y) + (row0 + r) * a.outputs + out0 + wo * TN;
#pragma unroll
      for (int j = 0; j < TN / 2; ++j) {
        float v0, v1; Split(acc[i][j], v0, v1);
        if (wo * TN + 2 * j < outs) y[2 * j] = v0;
        if (wo * TN + 2 * j + 1 < outs) y[2 * j + 1] = v1;
      }
    }
  }
}

// Tile: AC = TA * GA columns of a x BC = TB * GB columns of b, kRowsDeep rows at a time; SLICES groups of GA * GB threads take every
// SLICES-th row each and are added up at the end, in order.
constexpr int kRowsDeep = 32;
template <int TA, int TB, int GA, int GB, int SLICES>
struct FloatGramTile {
  static constexpr int AC = TA * GA, BC = TB * GB, GROUP = GA * GB, THREADS = GROUP * SLICES, AP = AC + 4, BP = BC + 4;
  static constexpr int kLoad = 2 * kRowsDeep * (AP + BP) * 4, kSum = SLICES > 1 ? SLICES * AC * BC * 4 : 0, kBytes = kLoad > kSum ? kLoad : kSum;
};
// `partial` null: one slice of rows per leaf, written to out; else slice t's sums go to partial [slice][a_cols][b_cols].
template <int TA, int TB, int GA, int GB, int SLICES>
__global__ void __launch_bounds__(GA * GB * SLICES) LeafGramFloatKernel(LeafGramArgs a, int rows_per_slice, float* partial) {
  using Tile = FloatGramTile<TA, TB, GA, GB, SLICES>;
  extern __shared__ __align__(16) float s_float[];
  __shared__ TileMap map;
  float* s_a = s_float; float* s_b = s_float + 2 * kRowsDeep * Tile::AP;
  map.Build(a.leaves, rows_per_slice, 1);
  const int across_a = (a.a_cols + Tile::AC - 1) / Tile::AC, across_b = (a.b_cols + Tile::BC - 1) / Tile::BC;
  const long long tiles = static_cast<long long>(map.Total()) * across_a * across_b;
  const int slice = threadIdx.x / Tile::GROUP, member = threadIdx.x % Tile::GROUP, ga = member / GB, gb = member % GB;
  for (long long t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int which = static_cast<int>(t / (across_a * across_b)), rest = static_cast<int>(t % (across_a * across_b));
    int leaf; long long row0, end;
    map.Find(a.leaves, which, rows_per_slice, 1, &leaf, &row0, &end);
    const int a0 = rest / across_b * Tile::AC, b0 = rest % across_b * Tile::BC, a_in = min(Tile::AC, a.a_cols - a0), b_in = min(Tile::BC, a.b_cols - b0);
    const float* pa = static_cast<const float*>(a.a) + a0; const float* pb = static_cast<const float*>(a.b) + b0;
    auto load = [&](long long r0, int buf) {
#pragma unroll 2
      for (int e = threadIdx.x; e < kRowsDeep * Tile::AC; e += Tile::THREADS) {
        const int r = e / Tile::AC, c = e % Tile::AC;
        const bool in = r0 + r < end && c < a_in;
        Copy4(s_a + (buf * kRowsDeep + r) * Tile::AP + c, in ? pa + (r0 + r) * a.a_stride + c : static_cast<const float*>(a.a), in);
      }
#pragma unroll 2
      for (int e = threadIdx.x; e < kRowsDeep * Tile::BC; e += Tile::THREADS) {
        const int r = e / Tile::BC, c = e % Tile::BC;
        const bool in = r0 + r < end && c < b_in;
        Copy4(s_b + (buf * kRowsDeep + r) * Tile::BP + c, in ? pb + (r0 + r) * a.b_stride + c : static_cast<const float*>(a.b), in);
      }
      CopyCommit();
    };
    F2 acc[TA][TB / 2];
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
      for (int j = 0; j < TB / 2; ++j) acc[i][j] = MakeF2(0.f, 0.f);
    if (row0 < end) load(row0, 0);
    int buf = 0;
    for (long long r0 = row0; r0 < end; r0 += kRowsDeep, buf ^= 1) {
      if (r0 + kRowsDeep < end) { load(r0 + kRowsDeep, buf ^ 1); CopyWait<1>(); } else CopyWait<0>();
      __syncthreads();
#pragma unroll 2
      for (int r = slice; r < kRowsDeep; r += SLICES) {
        const float* as = s_a + (buf * kRowsDeep + r) * Tile::AP + ga * TA; const float* bs = s_b + (buf * kRowsDeep + r) * Tile::BP + gb * TB;
        F2 bv[TB / 2]; float av[TA];
#pragma unroll
        for (int j = 0; j < TB / 4; ++j) { const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(bs + 4 * j); bv[2 * j].v = q.x; bv[2 * j + 1].v = q.y; }
#pragma unroll
        for (int i = 0; i < TA / 4; ++i) { const float4 q = *reinterpret_cast<const float4*>(as + 4 * i); av[4 * i] = q.x; av[4 * i + 1] = q.y; av[4 * i + 2] = q.z; av[4 * i + 3] = q.w; }
#pragma unroll
        for (int i = 0; i < TA; ++i) {
          const F2 v = MakeF2(av[i], av[i]);
#pragma unroll
          for (int j = 0; j < TB / 2; ++j) acc[i][j] = Fma2(v, bv[j], acc[i][j]);
        }
      }
      __syncthreads();
    }
    float* to = partial != nullptr ? partial + static_cast<long long>(which) * a.a_cols * a.b_cols : static_cast<float*>(a.out) + static_cast<long long>(leaf) * a.a_cols * a.b_cols;
    if constexpr (SLICES == 1) {
#pragma unroll
      for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < TB / 2; ++j) {
          float v[2]; Split(acc[i][j], v[0], v[1]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int ca = ga * TA + i, cb = gb * TB + 2 * j + h;
            if (ca < a_in && cb < b_in) to[static_cast<long long>(a0 + ca) * a.b_cols + b0 + cb] = v[h];
          }
        }
    } else {
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
}

// Adds the partial sums of each leaf's slices, in order.
template <typename O>
__global__ void __launch_bounds__(256) LeafGramJoinKernel(LeafGramArgs a, int rows_per_slice, const float* __restrict__ partial) {
  __shared__ TileMap map;
  map.Build(a.leaves, rows_per_slice, 1);
  const long long size = static_cast<long long>(a.a_cols) * a.b_cols;
  for (int g = blockIdx.y; g < a.leaves.leaves; g += gridDim.y) {
    int first = map.before[g / map.per];
    for (int o = g / map.per * map.per; o < g; ++o) first += TileMap::Count(a.leaves, o, rows_per_slice, 1);
    const int slices = TileMap::Count(a.leaves, g, rows_per_slice, 1);
    for (long long e = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; e < size; e += static_cast<long long>(gridDim.x) * 256) {
      float v = 0.f;
      for (int s = 0; s < slices; ++s) v += partial[(first + s) * size + e];
      static_cast<O*>(a.out)[g * size + e] = FromFloat<O>(v);
    }
  }
}

// ------------------------------------------------------------------------------------- 16-bit types, any shape ----
constexpr int kTile = 16;

// Block (x: 16 outputs, y: slice of a leaf's rows, z: leaf): 16 x 16 outputs at a time through shared memory.
template <typename T>
__global__ void __launch_bounds__(kTile * kTile) LeafProductsKernel(LeafProductsArgs a) {
  __shared__ float s_x[kTile][kTile + 1], s_w[kTile][kTile + 1];
  const int tx = threadIdx.x % kTile, ty = threadIdx.x / kTile;
  for (int g = blockIdx.z; g < a.leaves.leaves; g += gridDim.z) {
    long long begin, end; LeafWindow(a.leaves, g, &begin, &end);
    const T* w = static_cast<const T*>(a.weight) + g * a.weight_leaf_stride;
    for (long long r0 = begin + static_cast<long long>(blockIdx.y) * kTile; r0 < end; r0 += static_cast<long long>(gridDim.y) * kTile) {
      for (int p0 = blockIdx.x * kTile; p0 < a.outputs; p0 += gridDim.x * kTile) {
        float acc = 0.f;
        for (int f0 = 0; f0 < a.features; f0 += kTile) {
          s_x[ty][tx] = (r0 + ty < end && f0 + tx < a.features) ? ToFloat(static_cast<const T*>(a.x)[(r0 + ty) * a.x_stride + f0 + tx]) : 0.f;
          s_w[ty][tx] = (p0 + ty < a.outputs && f0 + tx < a.features) ? ToFloat(w[(p0 + ty) * a.weight_out_stride + (f0 + tx) * a.weight_in_stride]) : 0.f;
          __syncthreads();
          for (int f = 0; f < kTile; ++f) acc = fmaf(s_x[ty][f], s_w[tx][f], acc);
          __syncthreads();
        }
        if (r0 + ty < end && p0 + tx < a.outputs) static_cast<T*>(a.y)[(r0 + ty) * a.outputs + p0 + tx] = FromFloat<T>(acc);
      }
    }
  }
}

template <typename T, typename O>
__global__ void __launch_bounds__(kTile * kTile) LeafGramKernel(LeafGramArgs a) {
  __shared__ float s_a[kTile][kTile + 1], s_b[kTile][kTile + 1];
  const int tx = threadIdx.x % kTile, ty = threadIdx.x / kTile;
  for (int g = blockIdx.z; g < a.leaves.leaves; g += gridDim.z) {
    long long begin, end; LeafWindow(a.leaves, g, &begin, &end);
    for (int p0 = blockIdx.y * kTile; p0 < a.a_cols; p0 += gridDim.y * kTile)
      for (int q0 = blockIdx.x * kTile; q0 < a.b_cols; q0 += gridDim.x * kTile) {
        float acc = 0.f;
        for (long long r0 = begin; r0 < end; r0 += kTile) {
          s_a[ty][tx] = (r0 + ty < end && p0 + tx < a.a_cols) ? ToFloat(static_cast<const T*>(a.a)[(r0 + ty) * a.a_stride + p0 + tx]) : 0.f;
          s_b[ty][tx] = (r0 + ty < end && q0 + tx < a.b_cols) ? ToFloat(static_cast<const T*>(a.b)[(r0 + ty) * a.b_stride + q0 + tx]) : 0.f;
          __syncthreads();
          for (int r = 0; r < kTile; ++r) acc = fmaf(s_a[r][ty], s_b[r][tx], acc);
          __syncthreads();
        }
        if (p0 + ty < a.a_cols && q0 + tx < a.b_cols) static_cast<O*>(a.out)[(static_cast<long long>(g) * a.a_cols + p0 + ty) * a.b_cols + q0 + tx] = FromFloat<O>(acc);
      }
  }
}

// Rows that belong to no leaf: zero.
template <typename T>
__global__ void __launch_bounds__(256) LeaflessRowsKernel(LeafProductsArgs a) {
  long long first, last, unused;
  LeafWindow(a.leaves, 0, &first, &unused); LeafWindow(a.leaves, a.leaves.leaves - 1, &unused, &last);
  const long long head = first * a.outputs, tail = last * a.outputs, total = a.leaves.rows * a.outputs, stride = static_cast<long long>(gridDim.x) * blockDim.x;
  const long long t = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (long long i = t; i < head; i += stride) static_cast<T*>(a.y)[i] = FromFloat<T>(0.f);
  for (long long i = tail + t; i < total; i += stride) static_cast<T*>(a.y)[i] = FromFloat<T>(0.f);
}

template <typename F> void DispatchHalf(int dtype, F&& f) {
  switch (dtype) {
    case kOpFloat16: f(static_cast<__half*>(nullptr)); return;
    case kOpBFloat16: f(static_cast<__nv_bfloat16*>(nullptr)); return;
    default: Log::Fatal("leaf products: unknown type code %d", dtype);
  }
}

inline unsigned int Tiles(long long n, long long most) { return static_cast<unsigned int>(std::max(1LL, std::min(most, (n + kTile - 1) / kTile))); }

template <int TM, int TN, int WR, int WO>
void LaunchFloatProducts(const LeafProductsArgs& a, int per_sm, cudaStream_t s) {
  using Tile = FloatTile<TM, TN, WR, WO>;
  static PerDevice allowed;
  AllowSharedMemory(LeafProductsFloatKernel<TM, TN, WR, WO>, Tile::kBytes, &allowed);
  const long long tiles = ((a.leaves.rows + Tile::ROWS - 1) / Tile::ROWS + a.leaves.leaves) * ((a.outputs + Tile::OUTS - 1) / Tile::OUTS);
  LeafProductsFloatKernel<TM, TN, WR, WO><<<static_cast<unsigned int>(std::min<long long>(tiles, kSms * per_sm)), Tile::THREADS, Tile::kBytes, s>>>(a);
}
template <int TA, int TB, int GA, int GB, int SLICES>
void LaunchFloatGram(const LeafGramArgs& a, int per_sm, float* workspace, cudaStream_t s) {
  using Tile = FloatGramTile<TA, TB, GA, GB, SLICES>;
  static PerDevice allowed;
  AllowSharedMemory(LeafGramFloatKernel<TA, TB, GA, GB, SLICES>, Tile::kBytes, &allowed);
  const long long across = static_cast<long long>((a.a_cols + Tile::AC - 1) / Tile::AC) * ((a.b_cols + Tile::BC - 1) / Tile::BC);
  const int rows = LeafGramSliceRows(a);
  const bool split = rows < a.leaves.rows;
  const long long tiles = (split ? LeafGramSlices(a) : a.leaves.leaves) * across;
  LeafGramFloatKernel<TA, TB, GA, GB, SLICES><<<static_cast<unsigned int>(std::min<long long>(tiles, kSms * per_sm)), Tile::THREADS, Tile::kBytes, s>>>(a, rows, split ? workspace : nullptr);
}
// narrow sides: few outputs / both sides of a Gram matrix within one small tile
constexpr int kNarrow = 16;

}  // namespace

// Rows of a leaf that one block sums up: all of them where the output tiles and the leaves alone fill the machine, else shorter
// slices, whose sums are added in a second step.
int LeafGramSliceRows(const LeafGramArgs& a) {
  const long long tile = a.dtype == kOpFloat32 ? (a.a_cols <= kNarrow && a.b_cols <= 2 * kNarrow ? kNarrow * 2 * kNarrow : 64 * 64) : 128 * 256;
  const long long outputs = std::max(1LL, (static_cast<long long>(a.a_cols) * a.b_cols + tile - 1) / tile);
  const long long wanted = std::max(1LL, 4LL * kSms / outputs);        // slices, over all leaves
  const long long rows = std::max(256LL, ((a.leaves.rows + wanted - 1) / wanted + 63) / 64 * 64);
  return static_cast<int>(std::min<long long>(rows, std::max(1LL, a.leaves.rows)));
}
long long LeafGramSlices(const LeafGramArgs& a) { const int rows = LeafGramSliceRows(a); return (a.leaves.rows + rows - 1) / rows + a.leaves.leaves; }
long long LeafGramWorkspace(const LeafGramArgs& a) {
  if (a.dtype != kOpFloat32) return 0;
  return LeafGramSliceRows(a) < a.leaves.rows ? LeafGramSlices(a) * a.a_cols * a.b_cols : 0;
}

void LaunchLeafProducts(const LeafProductsArgs& a, cudaStream_t s) {
  if (a.leaves.rows <= 0) return;
  if (a.dtype == kOpFloat32) {
    LeaflessRowsKernel<float><<<64, 256, 0, s>>>(a);
    FB_LAUNCHED(); FB_KERNEL_CHECK();
    if (a.outputs <= kNarrow) LaunchFloatProducts<2, 16, 4, 1>(a, 3, s);
    else if (a.outputs <= 64) LaunchFloatProducts<4, 8, 1, 8>(a, 3, s);
    else LaunchFloatProducts<4, 16, 1, 8>(a, 2, s);
  } else DispatchHalf(a.dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    LeaflessRowsKernel<T><<<64, 256, 0, s>>>(a);
    FB_LAUNCHED(); FB_KERNEL_CHECK();
    LeafProductsKernel<T><<<dim3(Tiles(a.outputs, 64), Tiles(a.leaves.rows, 64), std::min(a.leaves.leaves, 1024)), kTile * kTile, 0, s>>>(a);
  });
  FB_LAUNCHED(); FB_KERNEL_CHECK();
}

void LaunchLeafGram(const LeafGramArgs& a, float* workspace, cudaStream_t s) {
  if (a.dtype == kOpFloat32) {
    if (a.out_dtype != kOpFloat32) Log::Fatal("leaf Gram: sums of type code %d as type code %d", a.dtype, a.out_dtype);
    if (a.a_cols <= kNarrow && a.b_cols <= 2 * kNarrow) LaunchFloatGram<4, 4, 4, 8, 8>(a, 3, workspace, s);
    else LaunchFloatGram<8, 8, 8, 8, 4>(a, 2, workspace, s);
    FB_LAUNCHED(); FB_KERNEL_CHECK();
    if (LeafGramSliceRows(a) < a.leaves.rows) {
      const long long size = static_cast<long long>(a.a_cols) * a.b_cols;
      LeafGramJoinKernel<float><<<dim3(static_cast<unsigned int>(std::min(64LL, (size + 255) / 256)), std::min(a.leaves.leaves, 1024)), 256, 0, s>>>(a, LeafGramSliceRows(a), workspace);
      FB_LAUNCHED(); FB_KERNEL_CHECK();
    }
    return;
  }
  const dim3 grid(Tiles(a.b_cols, 64), Tiles(a.a_cols, 64), std::min(a.leaves.leaves, 1024));
  DispatchHalf(a.dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    if (a.out_dtype == a.dtype) LeafGramKernel<T, T><<<grid, kTile * kTile, 0, s>>>(a);
    else if (a.out_dtype == kOpFloat32) LeafGramKernel<T, float><<<grid, kTile * kTile, 0, s>>>(a);
    else Log::Fatal("leaf Gram: sums of type code %d as type code %d", a.dtype, a.out_dtype);
  });
  FB_LAUNCHED(); FB_KERNEL_CHECK();
}

}  // namespace fb
