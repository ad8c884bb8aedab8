// Class scores -> log probability of a given class, log of the normaliser, entropy and top alternatives of every row, and the
// gradient in the scores of a loss made of these.
//
// Row i, classes j, scores s_j, m = max_j s_j:
//   S = sum_j e^(s_j - m),  T = sum_j e^(s_j - m) (s_j - m)
//   log_norm = m + log S,  log p_j = s_j - m - log S,  entropy = log S - T / S          (p log p = 0 where p = 0)
//   top: the classes of the largest scores, equal scores by rising class
//   d loss / d s_j = p_j (a + b log p_j) + (upstream gradients of log p_j itself),  b = -g_entropy,
//   a = g_log_norm - g_log_prob - sum g_top - g_entropy * entropy
// Everything is summed in fp32 whatever the type of the scores; only the gradient is rounded to that type, once, at the end.
// A row whose scores are all -inf has no distribution: log_norm and log probabilities -inf, entropy 0, no alternatives, gradient 0.
// A row with a NaN or +inf has NaN everywhere and no alternatives.
//
// The forward kernels read every score once from memory, and so do the gradient kernels as long as log_norm is small enough to hold
// the probabilities (kTrustedLogNorm), and write every value once: bound by bandwidth, in 16-bit types shared with the exponentials.
// (S, T) are kept relative to a running maximum and rescaled when it grows, so partial results of any split of a row can be
// joined. Which threads share a row goes by the number of classes and by what is contiguous:
//   few classes                 a thread per row, the row in registers           (ClassLogProbsFewKernel)
//   some, contiguous rows       8 lanes per row, the row in their registers      (ClassLogProbsSomeKernel)
//   contiguous rows             a warp, or a block or cluster of blocks, per row  (ClassLogProbsWarpKernel, ClassLogProbsBlockKernel)
//   contiguous columns, others  rows gathered in shared memory, a warp per row    (ClassLogProbsTileKernel); very many classes: 32
//                               rows per block, the classes over its warps          (ClassLogProbsColumnKernel)
#include "kernels.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace cg = cooperative_groups;

namespace fb {

namespace {

// log_norm in fp32 gives p to a relative 2^-24 |log_norm|: beyond this size the gradient takes the row's maximum and sum again, once per
// block of a row's chunks, or, where a thread has a row, once per slice of its classes. That costs much more than the gradient itself:
// scores shifted by 100 take 1354 us instead of 206 at 8191 x 32001 bf16, 883 instead of 29 at 4099 x 2000 fp32 class-major.
constexpr float kTrustedLogNorm = 64.f;
constexpr float kLowestExponent = -200.f;     // 2^x is 0 in fp32 from here on; keeps 0 * (-inf) out of T
constexpr float kLn2 = 0.69314718055994530942f;

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float NanF() { return __int_as_float(0x7fc00000); }
__device__ __forceinline__ float InfF() { return __int_as_float(0x7f800000); }
__device__ __forceinline__ float MaxNan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

__device__ __forceinline__ long long LabelOf(const ClassScoresArgs& a, long long row) {
  if (a.label_bits == 0) return -1;
  return a.label_bits == 32 ? static_cast<const int*>(a.labels)[row] : static_cast<const long long*>(a.labels)[row];
}

// 16 bytes of scores
template <typename T> struct Pack { static constexpr int N = 16 / sizeof(T); };
__device__ __forceinline__ void Unpack(const uint4& q, float (&v)[4], const float*) {
  v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
}
__device__ __forceinline__ void Unpack2(unsigned int u, float& lo, float& hi, const __nv_bfloat16*) { lo = __uint_as_float(u << 16); hi = __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ void Unpack2(unsigned int u, float& lo, float& hi, const __half*) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u)); lo = f.x; hi = f.y;
}
template <typename T>
__device__ __forceinline__ void Unpack(const uint4& q, float (&v)[8], const T* t) { Unpack2(q.x, v[0], v[1], t); Unpack2(q.y, v[2], v[3], t); Unpack2(q.z, v[4], v[5], t); Unpack2(q.w, v[6], v[7], t); }
__device__ __forceinline__ float Max(const uint4& q, const float*) { return MaxNan(MaxNan(__uint_as_float(q.x), __uint_as_float(q.y)), MaxNan(__uint_as_float(q.z), __uint_as_float(q.w))); }
__device__ __forceinline__ unsigned int Max2(unsigned int a, unsigned int b, const __half*) { unsigned int r; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ unsigned int Max2(unsigned int a, unsigned int b, const __nv_bfloat16*) { unsigned int r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
template <typename T>
__device__ __forceinline__ float Max(const uint4& q, const T* t) { float lo, hi; Unpack2(Max2(Max2(q.x, q.y, t), Max2(q.z, q.w, t), t), lo, hi, t); return MaxNan(lo, hi); }
__device__ __forceinline__ uint4 AllRuledOut(const float*) { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
__device__ __forceinline__ uint4 AllRuledOut(const __nv_bfloat16*) { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
__device__ __forceinline__ uint4 AllRuledOut(const __half*) { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }

// Pairs of fp32 values in one 64-bit register: one instruction for two elements.
struct F2 { unsigned long long v; };
__device__ __forceinline__ F2 MakeF2(float x, float y) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ void Split(F2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 Add2(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ F2 Mul2(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ F2 Fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
__device__ __forceinline__ float Exp2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }   // 2 ulp; e^x below is 2^(x log2 e)
constexpr float kLog2E = 1.44269504088896340736f;

// Exponents are taken to base 2 against the rounded product B = m log2 e: x_j = s_j log2 e - B is one fused multiply-add. The rounding
// of B shifts all x alike, by half a step of B at most, and the results are put together from the same x and B, so it drops out as
// long as 2^shift is far from fp32's ends. Up to |m| = 2^24 the shift is at most 1 (at 2^31 it would pass 64, at 2^33 every term
// overflow or vanish). Beyond kHugeScore x = (s_j - m) log2 e, without a shift: neighbouring scores differ by 2 or more there, and
// the subtraction loses nothing that e^x could show.
constexpr float kHugeScore = 16777216.f;
__device__ __forceinline__ bool Huge(float m) { return !(fabsf(m) <= kHugeScore); }
__device__ __forceinline__ float Exponent(float v, float m) { return Huge(m) ? (v - m) * kLog2E : fmaf(v, kLog2E, -__fmul_rn(m, kLog2E)); }
// what the exponents of a part with maximum m are too high by: m log2 e - B
__device__ __forceinline__ float Shift(float m) { return Huge(m) ? 0.f : fmaf(m, kLog2E, -__fmul_rn(m, kLog2E)); }
// how much lower the exponents are when the maximum goes from m to `to` (> m); with one side beyond kHugeScore the other's shift counts
__device__ __forceinline__ float Lower(float m, float to) {
  return fmaxf(Huge(m) || Huge(to) ? (m - to) * kLog2E - Shift(m) + Shift(to) : __fsub_rn(__fmul_rn(m, kLog2E), __fmul_rn(to, kLog2E)), kLowestExponent);
}

// The running sums of a part of a row, relative to its maximum m (-inf: nothing yet; a NaN or +inf among the scores makes s NaN):
// s = sum 2^x, t = sum 2^x x.
struct Sums {
  float m = -INFINITY, s = 0.f, t = 0.f;
  __device__ __forceinline__ void Raise(float to) {     // to > m
    const float d = Lower(m, to), f = Exp2(d);
    t = (t + s * d) * f; s *= f; m = to;
  }
  __device__ __forceinline__ float Base() const { return m == -INFINITY ? 0.f : m; }
  __device__ __forceinline__ void Add(float v, float base) { const float x = MaxNan(Exponent(v, base), kLowestExponent), e = Exp2(x); s += e; t = fmaf(e, x, t); }
  __device__ __forceinline__ void AddOne(float v) { if (v > m) Raise(v); Add(v, Base()); }
  __device__ __forceinline__ void Join(float m2, float s2, float t2) {
    if (m2 > m) { const float m1 = m, s1 = s, t1 = t; m = m2; s = s2; t = t2; m2 = m1; s2 = s1; t2 = t1; }
    const float d = m2 == -INFINITY ? kLowestExponent : m2 == m ? 0.f : Lower(m2, m), f = Exp2(d);
    t += (t2 + s2 * d) * f; s += s2 * f;
  }
  // Over LANES neighbouring lanes: one maximum, one rescaling, then plain sums.
  template <int LANES = 32>
  __device__ __forceinline__ void JoinLanes() {
    float most = m;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (most > m) Raise(most);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, o); t += __shfl_xor_sync(0xffffffffu, t, o); }
    m = most;
  }
};
// The same for 16 bytes of scores at a time, two sums side by side.
// In a pair's product 2^x * x a ruled-out score must not give 0 * (-inf): 16-bit scores are lifted to a finite low value first, two
// per instruction. That is exact as long as the maximum is far above that value, and needs exponents by one multiply-add: maxima up
// to kMost in size; elsewhere every exponent is clamped by itself.
template <typename T> struct FarBelow;
template <> struct FarBelow<__half> { static constexpr unsigned int kLow = 0xfbfffbffu; static constexpr float kMost = 60000.f; };               // -65504
template <> struct FarBelow<__nv_bfloat16> { static constexpr unsigned int kLow = 0xf14af14au; static constexpr float kMost = kHugeScore; };     // -1.0e30
template <typename T>
struct PairSums {
  float m = -INFINITY; F2 s = MakeF2(0.f, 0.f), t = MakeF2(0.f, 0.f);
  __device__ __forceinline__ void Raise(float to) {
    const float d = Lower(m, to), f = Exp2(d);
    const F2 d2 = MakeF2(d, d), f2 = MakeF2(f, f);
    t = Mul2(Fma2(s, d2, t), f2); s = Mul2(s, f2); m = to;
  }
  __device__ __forceinline__ void AddExponents(F2 x) {
    float x0, x1; Split(x, x0, x1);
    const F2 e = MakeF2(Exp2(x0), Exp2(x1));
    s = Add2(s, e); t = Fma2(e, x, t);
  }
  // COUNT pieces of 16 bytes
  template <int COUNT>
  __device__ __forceinline__ void Add16(const uint4 (&all)[COUNT]) {
    constexpr int N = Pack<T>::N;
    const float base = m == -INFINITY ? 0.f : m;
    const T* type = nullptr;
    if constexpr (sizeof(T) == 2) {
      if (fabsf(base) <= FarBelow<T>::kMost) {
        const unsigned int low = FarBelow<T>::kLow;
        const float minus_b = -__fmul_rn(base, kLog2E);
        const F2 minus_base = MakeF2(minus_b, minus_b), scale = MakeF2(kLog2E, kLog2E);
#pragma unroll
        for (int u = 0; u < COUNT; ++u) {
          uint4 q = all[u];
          q.x = Max2(q.x, low, type); q.y = Max2(q.y, low, type); q.z = Max2(q.z, low, type); q.w = Max2(q.w, low, type);
          float v[N]; Unpack(q, v, type);
#pragma unroll
          for (int i = 0; i < N; i += 2) AddExponents(Fma2(MakeF2(v[i], v[i + 1]), scale, minus_base));
        }
        return;
      }
    }
#pragma unroll
    for (int u = 0; u < COUNT; ++u) {
      float v[N]; Unpack(all[u], v, type);
#pragma unroll
      for (int i = 0; i < N; i += 2) AddExponents(MakeF2(MaxNan(Exponent(v[i], base), kLowestExponent), MaxNan(Exponent(v[i + 1], base), kLowestExponent)));
    }
  }
  __device__ __forceinline__ Sums Total() const { Sums r; float a, b; Split(s, a, b); r.s = a + b; Split(t, a, b); r.t = a + b; r.m = m; return r; }
};
// The largest of COUNT pieces.
template <int COUNT, typename T>
__device__ __forceinline__ float MaxOf(const uint4 (&q)[COUNT], const T* t) {
  if constexpr (sizeof(T) == 2) {
    unsigned int w = Max2(Max2(q[0].x, q[0].y, t), Max2(q[0].z, q[0].w, t), t);
#pragma unroll
    for (int u = 1; u < COUNT; ++u) w = Max2(w, Max2(Max2(q[u].x, q[u].y, t), Max2(q[u].z, q[u].w, t), t), t);
    float lo, hi; Unpack2(w, lo, hi, t);
    return MaxNan(lo, hi);
  } else {
    float r = Max(q[0], t);
#pragma unroll
    for (int u = 1; u < COUNT; ++u) r = MaxNan(r, Max(q[u], t));
    return r;
  }
}

// The results of a row from its sums.
struct RowResult {
  float m, log_sum, shift, entropy; bool none, bad;      // log_sum: to base 2, with the exponents' shift
  __device__ explicit RowResult(const Sums& r) {
    none = r.m == -INFINITY && !(r.s != r.s); bad = !none && !(fabsf(r.m) < InfF() && r.s < InfF());   // a NaN sum fails the comparison
    m = r.m; log_sum = log2f(r.s); shift = Shift(m); entropy = none ? 0.f : bad ? NanF() : fmaxf((log_sum - r.t / r.s) * kLn2, 0.f);
  }
  __device__ __forceinline__ float LogProb(float v) const { return none || v == -INFINITY ? (bad ? NanF() : -INFINITY) : bad ? NanF() : Huge(m) || Huge(v) ? (v - m) - (log_sum - shift) * kLn2 : fminf((Exponent(v, m) - log_sum) * kLn2, 0.f); }
  __device__ __forceinline__ float LogNorm() const { return none ? -INFINITY : bad ? NanF() : m + (log_sum - shift) * kLn2; }
  __device__ __forceinline__ void Store(const ClassScoresArgs& a, long long row, long long y, float label_score) const {
    a.log_norm[row] = LogNorm(); a.entropy[row] = entropy;
    if (a.log_prob != nullptr) a.log_prob[row] = y < 0 ? 0.f : y >= a.classes ? NanF() : LogProb(label_score);
  }
  __device__ __forceinline__ void StoreTop(const ClassScoresArgs& a, long long at, float v, int cls) const {   // v -inf: no such alternative
    const bool is = !bad && !none && v > -INFINITY;
    a.top_log_prob[at] = is ? LogProb(v) : bad ? NanF() : -INFINITY; a.top_class[at] = is ? cls : -1;
  }
};

// ------------------------------------------------------------------------------------------------ few classes ----
// The results of a row whose scores are in registers.
template <int MOST>
__device__ __forceinline__ void FinishRow(const ClassScoresArgs& a, long long row, long long y, float (&v)[MOST]) {
  if (row >= a.rows) return;
  Sums sums;
  float m = v[0];
#pragma unroll
  for (int j = 1; j < MOST; ++j) m = MaxNan(m, v[j]);
  sums.m = m;
  const float b = sums.Base();
#pragma unroll
  for (int j = 0; j < MOST; ++j) sums.Add(v[j], b);
  const RowResult res(sums);
  float given = 0.f;
#pragma unroll
  for (int j = 0; j < MOST; ++j) if (j == y) given = v[j];
  res.Store(a, row, y, given);
  for (int t = 0; t < a.top_k; ++t) {
    float best = -INFINITY; int cls = -1;
#pragma unroll
    for (int j = 0; j < MOST; ++j) if (v[j] > best) { best = v[j]; cls = j; }
#pragma unroll
    for (int j = 0; j < MOST; ++j) if (j == cls) v[j] = -INFINITY;
    res.StoreTop(a, row * a.top_k + t, best, cls);
  }
}
// A thread has ROWS rows, each row's scores in MOST registers. Class-major scores are read straight into them, 32 rows per instruction,
// all rows' loads before the first use; rows go through shared memory (an odd row pitch there, so that neither side meets bank
// conflicts).
constexpr int kFewThreads = 128, kFewClasses = 64;
template <typename T, int MOST, bool BY_CLASS, int ROWS>
__global__ void __launch_bounds__(kFewThreads) ClassLogProbsFewKernel(ClassScoresArgs a) {
  __shared__ float s_rows[BY_CLASS ? 1 : kFewThreads * (MOST + 1)];
  const int K = static_cast<int>(a.classes);
  const long long row0 = static_cast<long long>(blockIdx.x) * (kFewThreads * ROWS);
  const T* base = static_cast<const T*>(a.scores);
  float v[ROWS][MOST]; long long y[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) { const long long row = row0 + i * kFewThreads + threadIdx.x; y[i] = row < a.rows ? LabelOf(a, row) : -1; }
  if constexpr (BY_CLASS) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const long long row = row0 + i * kFewThreads + threadIdx.x;
#pragma unroll
      for (int j = 0; j < MOST; ++j) v[i][j] = j < K && row < a.rows ? ToFloat(base[row * a.row_stride + j * a.class_stride]) : -INFINITY;
    }
  } else {
    static_assert(ROWS == 1, "rows in shared memory: one per thread");
    const int rows = static_cast<int>(min(static_cast<long long>(kFewThreads), a.rows - row0)), pitch = K | 1;
    for (int e = threadIdx.x, r = e / K, j = e - r * K; e < rows * K; e += kFewThreads) {
      s_rows[r * pitch + j] = ToFloat(base[(row0 + r) * a.row_stride + j * a.class_stride]);
      j += kFewThreads % K; r += kFewThreads / K;
      if (j >= K) { j -= K; ++r; }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < MOST; ++j) v[0][j] = j < K ? s_rows[threadIdx.x * pitch + j] : -INFINITY;
  }
  FinishRow<MOST>(a, row0 + threadIdx.x, y[0], v[0]);
  if constexpr (ROWS == 2) FinishRow<MOST>(a, row0 + kFewThreads + threadIdx.x, y[1], v[1]);
}

// Rows of up to kSomeClasses contiguous classes: 8 lanes per row, PER scores each in registers. An alternative at a time: the best of a
// lane's scores, of the 8 lanes', and out of the registers.
constexpr int kSomeClasses = 256;
// s: the row (any row where !is_row; a warp's lanes stay together)
template <typename T, int PER>
__device__ __forceinline__ void SomeRow(const ClassScoresArgs& a, long long row, bool is_row, const T* s, int lane8) {
  const int K = static_cast<int>(a.classes);
  const long long y = is_row ? LabelOf(a, row) : -1;
  float v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = is_row && lane8 + 8 * i < K ? ToFloat(s[lane8 + 8 * i]) : -INFINITY;
  const float given = lane8 == 0 && y >= 0 && y < K ? ToFloat(s[y]) : 0.f;
  Sums sums;
  sums.m = v[0];
#pragma unroll
  for (int i = 1; i < PER; ++i) sums.m = MaxNan(sums.m, v[i]);
  const float b = sums.Base();
#pragma unroll
  for (int i = 0; i < PER; ++i) sums.Add(v[i], b);
  sums.JoinLanes<8>();
  const RowResult res(sums);
  if (is_row && lane8 == 0) res.Store(a, row, y, given);
  for (int t = 0; t < a.top_k; ++t) {
    float best = -INFINITY; int cls = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PER; ++i) if (v[i] > best) { best = v[i]; cls = lane8 + 8 * i; }
    const int mine = cls;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      const float bo = __shfl_xor_sync(0xffffffffu, best, o); const int co = __shfl_xor_sync(0xffffffffu, cls, o);
      if (bo > best || (bo == best && co < cls)) { best = bo; cls = co; }
    }
    if (mine == cls) {
#pragma unroll
      for (int i = 0; i < PER; ++i) if (lane8 + 8 * i == cls) v[i] = -INFINITY;
    }
    if (is_row && lane8 == 0) res.StoreTop(a, row * a.top_k + t, best, cls);
  }
}
template <typename T, int PER>
__global__ void __launch_bounds__(128) ClassLogProbsSomeKernel(ClassScoresArgs a) {
  const long long row = static_cast<long long>(blockIdx.x) * 16 + threadIdx.x / 8;
  const bool is_row = row < a.rows;
  SomeRow<T, PER>(a, row, is_row, static_cast<const T*>(a.scores) + (is_row ? row : 0) * a.row_stride, threadIdx.x & 7);
}

// -------------------------------------------------------------------------------------------- contiguous rows ----
// A warp, or 8 warps of a block, walk a row (or a block cluster's share of one), kUnroll 16-byte pieces per thread at a time. The
// pieces come by asynchronous copies through a ring of chunks, every thread its own pieces, so that a thread waits only for itself;
// the copies run ahead into the next row, which covers the end of a row. Scores before the first 16-byte boundary and behind
// the last come one by one.
// Alternatives: every thread notes the maximum of its pieces, the chunk that held it, and the best that any other of its chunks held.
// With V the top_k-th largest of these maxima, only the threads whose maximum reaches V can hold one of the top_k best
// scores: about top_k of them, each mostly with that one score, so little more than one chunk of each is read again (from
// L2; the whole share where another chunk reaches V too). The scores that reach V are listed and the short list is ranked by counting.
constexpr int kUnroll = 4;
struct Entry { float v; int cls; };
__device__ __forceinline__ bool Before(const Entry& a, const Entry& b) { return a.v > b.v || (a.v == b.v && a.cls < b.cls); }
// Order of scores as unsigned numbers, -inf 0, zeros of both signs alike; types of 16 bits need fewer.
template <typename T> struct KeyBits { static constexpr int kBits = 16, kShift = 16; };
template <> struct KeyBits<__half> { static constexpr int kBits = 19, kShift = 13; };
template <> struct KeyBits<float> { static constexpr int kBits = 32, kShift = 0; };
template <typename T>
__device__ __forceinline__ unsigned int OrderKey(float v) {
  const unsigned int u = __float_as_uint(v + 0.f);
  return v == -INFINITY ? 0u : ((u & 0x80000000u) != 0 ? ~u : u | 0x80000000u) >> KeyBits<T>::kShift;
}

// The score of a key; below the finite scores (key 1: anything but -inf) the lowest finite one.
template <typename T>
__device__ __forceinline__ float KeyScore(unsigned int k) {
  constexpr int kShift = KeyBits<T>::kShift;
  const bool positive = (k & (1u << (31 - kShift))) != 0;
  const unsigned int low = kShift > 0 ? (1u << kShift) - 1u : 0u;
  return fmaxf(__uint_as_float(positive ? (k << kShift) & 0x7fffffffu : ~((k << kShift) | low)), -3.402823466e38f);      // a NaN pattern gives way
}

// The `rank`-th largest (1-based) of PER numbers per lane, of `bits` bits: bit by bit, the largest value that at least `rank` numbers
// reach (0: there are fewer). Run by one warp.
template <int PER>
__device__ __forceinline__ unsigned int KthLargest(const unsigned int (&mine)[PER], int rank, int bits) {
  if (rank == 1) {
    unsigned int best = mine[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) best = max(best, mine[i]);
    return __reduce_max_sync(0xffffffffu, best);
  }
  unsigned int found = 0u;
  for (int bit = bits - 1; bit >= 0; --bit) {
    const unsigned int probe = found | (1u << bit);
    int c = 0;
    if constexpr (PER == 1) c = __popc(__ballot_sync(0xffffffffu, mine[0] >= probe));
    else {
#pragma unroll
      for (int i = 0; i < PER; ++i) c += mine[i] >= probe ? 1 : 0;
      c = __reduce_add_sync(0xffffffffu, c);
    }
    if (c >= rank) found = probe;
  }
  return found;
}

// A share of a row: part `part` of `parts`, of whole rounds of `group` threads.
template <typename T>
struct RowShare {
  const T* s; const uint4* body; int K, head, tail, v_begin, v_end; bool first, last_part;
  __device__ __forceinline__ RowShare(const ClassScoresArgs& a, long long row, int part, int parts, int group) {
    constexpr int N = Pack<T>::N;
    s = static_cast<const T*>(a.scores) + row * a.row_stride; K = static_cast<int>(a.classes);
    head = min(K, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(s) & 15)) & 15) / static_cast<int>(sizeof(T)));
    const int vectors = (K - head) / N;
    tail = head + vectors * N; body = reinterpret_cast<const uint4*>(s + head);
    const int each = ((vectors + parts - 1) / parts + group - 1) / group * group;
    v_begin = min(vectors, part * each); v_end = min(vectors, v_begin + each);
    first = part == 0; last_part = part == parts - 1;
  }
  // a whole row in shared memory, padded with -inf to 16-byte pieces
  __device__ __forceinline__ RowShare(const T* row, int classes) {
    s = row; K = classes; head = 0; v_begin = 0; v_end = (classes + Pack<T>::N - 1) / Pack<T>::N; tail = v_end * Pack<T>::N; body = reinterpret_cast<const uint4*>(row); first = last_part = true;
  }
  // the scores outside the 16-byte pieces, one per thread (-inf: none)
  __device__ __forceinline__ float Head(int tid) const { return first && tid < head ? ToFloat(s[tid]) : -INFINITY; }
  __device__ __forceinline__ float Tail(int tid) const { return last_part && tid < K - tail ? ToFloat(s[tail + tid]) : -INFINITY; }
};

// The walk of GROUP threads through the rows row, row + stride, ... with RING chunks of shared memory per thread.
template <typename T, int GROUP, int RING>
struct Walk {
  const ClassScoresArgs& a; uint4* mine; unsigned int stride; int tid, part, parts, slot, ahead_slot, ahead_at, ahead_end; unsigned int ahead_row; const uint4* ahead_body;
  __device__ __forceinline__ Walk(const ClassScoresArgs& args, uint4* ring, unsigned int row, unsigned int stride_, int tid_, int part_, int parts_) : a(args) {
    mine = ring + threadIdx.x; stride = stride_; tid = tid_; part = part_; parts = parts_; slot = ahead_slot = 0; ahead_row = row;
    const RowShare<T> r(a, row, part, parts, GROUP);
    ahead_body = r.body; ahead_at = r.v_begin; ahead_end = r.v_end;
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) CopyAhead();
  }
  __device__ __forceinline__ void CopyAhead() {
    if (ahead_row < a.rows) {
      const unsigned int to = static_cast<unsigned int>(__cvta_generic_to_shared(mine + ahead_slot * (kUnroll * 256)));
      const uint4* from = ahead_body + ahead_at + tid;
      if (ahead_at + GROUP * kUnroll <= ahead_end) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + u * (256 * 16)), "l"(from + u * GROUP) : "memory");
      } else {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (ahead_at + u * GROUP + tid < ahead_end) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + u * (256 * 16)), "l"(from + u * GROUP) : "memory");
      }
      ahead_at += GROUP * kUnroll;
      if (ahead_at >= ahead_end) {
        ahead_row += stride;
        if (ahead_row < a.rows) { const RowShare<T> n(a, ahead_row, part, parts, GROUP); ahead_body = n.body; ahead_at = n.v_begin; ahead_end = n.v_end; }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ahead_slot = ahead_slot == RING - 1 ? 0 : ahead_slot + 1;
  }
  // of this thread (a lone warp: of each of a lane's 4 pieces by itself): the maximum, the chunk (its first piece) that held it, and
  // the best of the other chunks
  static constexpr int kOf = GROUP == 32 ? kUnroll : 1;
  float best[kOf], second[kOf]; int best_at[kOf];
  __device__ __forceinline__ void Note(int u, float most, int at) { if (most > best[u]) { second[u] = best[u]; best[u] = most; best_at[u] = at; } else second[u] = fmaxf(second[u], most); }
  __device__ __forceinline__ float NotePieces(const uint4 (&q)[kUnroll], int at) {
    float most = -INFINITY;
#pragma unroll
    for (int u = 0; u < kOf; ++u) { const uint4 one[1] = {q[u]}; const float m = MaxOf(one, static_cast<const T*>(nullptr)); Note(u, m, at); most = MaxNan(most, m); }
    return most;
  }
  // This thread's sums of the pieces of the next row's share; m is its maximum.
  __device__ __forceinline__ Sums Row(const RowShare<T>& r) {
    const T* type = nullptr;
    PairSums<T> pairs;
    int at = r.v_begin;
#pragma unroll
    for (int u = 0; u < kOf; ++u) { best[u] = second[u] = -INFINITY; best_at[u] = at; }
    do {                                         // a share without pieces takes one empty step
      CopyAhead();
      asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
      const uint4* from = mine + slot * (kUnroll * 256);
      if (GROUP == 32 || at + GROUP * kUnroll <= r.v_end) {
        uint4 q[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) q[u] = GROUP > 32 || at + u * GROUP + tid < r.v_end ? from[u * 256] : AllRuledOut(type);
        float most;
        if constexpr (kOf == 1) { most = MaxOf(q, type); Note(0, most, at); } else most = NotePieces(q, at);
        if (most > pairs.m) pairs.Raise(most);
        pairs.Add16(q);
      } else {                                   // the last chunk, piece by piece
        float most = -INFINITY;
#pragma unroll 1
        for (int u = 0; u < kUnroll && (u == 0 || at + u * GROUP + (tid & ~31) < r.v_end); ++u) {
          const uint4 one[1] = {at + u * GROUP + tid < r.v_end ? from[u * 256] : AllRuledOut(type)};
          const float here = MaxOf(one, type);
          most = fmaxf(most, here);
          if (here > pairs.m) pairs.Raise(here);
          pairs.Add16(one);
        }
        Note(0, most, at);
      }
      at += GROUP * kUnroll;
      slot = slot == RING - 1 ? 0 : slot + 1;
    } while (at < r.v_end);
    return pairs.Total();
  }
};

// One warp finds the alternatives of a share that GROUP walkers have walked, in chunks of CHUNK pieces of each. The walkers are a block's
// threads (256, chunks of 4), or, where a warp walks alone, the 4 pieces of a lane's chunk taken by themselves (128, of 1), so
// that there are enough walkers for 32 alternatives.
template <int GROUP>
struct TopShared {
  static constexpr int kFlagged = 64, kCandidates = GROUP == 128 ? 128 : 256;
  Entry list[kMaxTopClasses], cand[kCandidates];
  int flagged[kFlagged], flagged_at[kFlagged], num_flagged, num_cand;      // threads; the chunk to look at (-1: all of the thread's share)
};
template <int GROUP, typename T>
struct Alternatives {
  static constexpr int N = Pack<T>::N, PER = GROUP / 32, CHUNK = GROUP == 128 ? 1 : kUnroll;
  TopShared<GROUP>& sh; const RowShare<T>& r; int top_k, lane;
  // f(score, class) for the scores that reach `limit` among piece `at` of the share (each lane its own; at >= v_end: none)
  template <int COUNT, typename F>
  __device__ __forceinline__ void Pieces(const int (&at)[COUNT], float limit, F&& f) const {
    uint4 q[COUNT];
#pragma unroll
    for (int u = 0; u < COUNT; ++u) q[u] = at[u] < r.v_end ? r.body[at[u]] : AllRuledOut(static_cast<const T*>(nullptr));
#pragma unroll
    for (int u = 0; u < COUNT; ++u) {
      const uint4 one[1] = {q[u]};
      if (!(MaxOf(one, static_cast<const T*>(nullptr)) >= limit)) continue;
      float v[N];
      Unpack(q[u], v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int k = 0; k < N; ++k) if (v[k] >= limit) f(v[k], r.head + at[u] * N + k);
    }
  }
  // the same for what the flagged threads have to look at, and for the ends of the row
  template <typename F>
  __device__ __forceinline__ void Scores(int num_flagged, float limit, F&& f) const {
    const float head_v = r.Head(lane), tail_v = r.Tail(lane);
    if (head_v >= limit) f(head_v, lane);
    if (tail_v >= limit) f(tail_v, r.tail + lane);
    constexpr int kAtOnce = CHUNK == 1 ? 2 : 4;
    for (int e0 = lane; e0 < CHUNK * num_flagged; e0 += 32 * kAtOnce) {
      int at[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int e = e0 + 32 * u, which = e / CHUNK;
        const int chunk = which < num_flagged ? sh.flagged_at[which] : -1;
        at[u] = chunk >= 0 ? chunk + (e % CHUNK) * GROUP + sh.flagged[which] : 0x7fffffff;
      }
      Pieces(at, limit, f);
    }
    for (int which = 0; which < num_flagged; ++which) {
      if (sh.flagged_at[which] >= 0) continue;
      for (int p = r.v_begin + sh.flagged[which] + lane * GROUP; p < r.v_end; p += 32 * GROUP * 2) {
        const int at[2] = {p, p + 32 * GROUP};
        Pieces(at, limit, f);
      }
    }
  }
  // Ranks the first `count` candidates into the list; returns how many that leaves.
  __device__ __forceinline__ int Rank(int count) {
    for (int i = lane; i < count; i += 32) {
      const Entry e = sh.cand[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += Before(sh.cand[j], e) ? 1 : 0;
      if (rank < top_k) sh.list[rank] = e;
    }
    __syncwarp();
    return min(count, top_k);
  }
  // Of the threads lane, lane + 32, ...: OrderKeys of their maxima and of the best of their other chunks, and the chunk of the maximum.
  // Returns the number of alternatives found, in the list.
  __device__ __forceinline__ int Find(const unsigned int (&keys)[PER], const unsigned int (&second)[PER], const int (&chunk)[PER]) {
    const unsigned int limit = max(1u, KthLargest<PER>(keys, top_k, KeyBits<T>::kBits));      // key 0: a thread without a score
    int flagged = 0, last = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned int in = __ballot_sync(0xffffffffu, keys[i] >= limit);
      const int at = flagged + __popc(in & ((1u << lane) - 1u));
      if (keys[i] >= limit && at < TopShared<GROUP>::kFlagged) { sh.flagged[at] = lane + 32 * i; sh.flagged_at[at] = second[i] >= limit ? -1 : chunk[i]; }
      flagged += __popc(in);
    }
    if (lane == 0) sh.num_cand = 0;
    __syncwarp();
    if (flagged > TopShared<GROUP>::kFlagged) flagged = Ties(keys, limit, &last);
    const float limit_score = KeyScore<T>(limit);
    Scores(flagged, limit_score, [&](float v, int cls) {
      if (v > limit_score || cls <= last) { const int at = atomicAdd(&sh.num_cand, 1); if (at < TopShared<GROUP>::kCandidates) { sh.cand[at].v = v; sh.cand[at].cls = cls; } }
    });
    __syncwarp();
    const int count = sh.num_cand;
    return count <= TopShared<GROUP>::kCandidates ? Rank(count) : OneByOne(flagged, limit_score);
  }
  // Very many equal maxima: of the threads with maximum `limit` only those count that reach it at the lowest classes. *last: the
  // highest of these classes.
  __device__ __noinline__ int Ties(const unsigned int (&keys)[PER], unsigned int limit, int* last) {
    unsigned int order[PER];
    int higher = 0;
    for (int i = 0; i < PER; ++i) {
      order[i] = 0u;
      higher += keys[i] > limit ? 1 : 0;
      if (keys[i] != limit) continue;
      const int thread = lane + 32 * i;
      int at = 0x7fffffff;
      for (int p = r.v_begin + thread; p < r.v_end && at == 0x7fffffff; p += GROUP) {
        float v[N];
        Unpack(r.body[p], v, static_cast<const T*>(nullptr));
#pragma unroll
        for (int k = N - 1; k >= 0; --k) if (OrderKey<T>(v[k]) == limit) at = r.head + p * N + k;
      }
      order[i] = 0x80000000u - static_cast<unsigned int>(at);
    }
    higher = __reduce_add_sync(0xffffffffu, higher);
    const unsigned int kth = KthLargest<PER>(order, top_k - higher, 32);
    *last = static_cast<int>(0x80000000u - kth);
    if (lane == 0) sh.num_flagged = 0;
    __syncwarp();
    for (int i = 0; i < PER; ++i) if (keys[i] > limit || order[i] >= kth) { const int at = atomicAdd(&sh.num_flagged, 1); sh.flagged[at] = lane + 32 * i; sh.flagged_at[at] = -1; }
    __syncwarp();
    return sh.num_flagged;
  }
  // More candidates than the list holds (few threads own very many of the best scores): one alternative per pass.
  __device__ __noinline__ int OneByOne(int num_flagged, float limit) {
    Entry before; before.v = INFINITY; before.cls = -1;
    int t = 0;
    for (; t < top_k; ++t) {
      Entry best; best.v = -INFINITY; best.cls = 0x7fffffff;
      Scores(num_flagged, limit, [&](float v, int cls) { Entry e; e.v = v; e.cls = cls; if (v > -INFINITY && Before(before, e) && Before(e, best)) best = e; });
      for (int o = 16; o > 0; o >>= 1) {
        Entry e; e.v = __shfl_xor_sync(0xffffffffu, best.v, o); e.cls = __shfl_xor_sync(0xffffffffu, best.cls, o);
        if (Before(e, best)) best = e;
      }
      if (best.cls == 0x7fffffff) break;
      if (lane == 0) sh.list[t] = best;
      before = best;
    }
    __syncwarp();
    return t;
  }
};

// A warp per row, 8 warps per block, each walking rows with the grid's stride. TOP: alternatives are wanted.
constexpr int kWarpRing = 3;
template <typename T, bool TOP>
__global__ void __launch_bounds__(256, 4) ClassLogProbsWarpKernel(ClassScoresArgs a) {
  extern __shared__ __align__(16) uint4 s_ring[];      // [kWarpRing][kUnroll][256]
  __shared__ TopShared<128> s_top[TOP ? 8 : 1];
  const int lane = threadIdx.x % 32;
  const unsigned int stride = gridDim.x * 8;      // unsigned: row + stride may pass 2^31
  unsigned int row = blockIdx.x * 8 + threadIdx.x / 32;
  if (row >= a.rows) return;                     // whole warps
  Walk<T, 32, kWarpRing> walk(a, s_ring, row, stride, lane, 0, 1);
  long long y = LabelOf(a, row);
  for (; row < a.rows; row += stride) {
    const RowShare<T> r(a, row, 0, 1, 32);
    const float head_v = r.Head(lane), tail_v = r.Tail(lane), given = lane == 0 && y >= 0 && y < r.K ? ToFloat(r.s[y]) : 0.f;
    const long long y_next = row + stride < a.rows ? LabelOf(a, row + stride) : -1;
    Sums sums = walk.Row(r);
    if (head_v != -INFINITY) sums.AddOne(head_v);
    if (tail_v != -INFINITY) sums.AddOne(tail_v);
    sums.JoinLanes();
    const RowResult res(sums);
    if (lane == 0) res.Store(a, row, y, given);
    if constexpr (TOP) {
      Alternatives<128, T> alt{s_top[threadIdx.x / 32], r, a.top_k, lane};
      unsigned int keys[kUnroll], second[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) { keys[u] = OrderKey<T>(walk.best[u]); second[u] = OrderKey<T>(walk.second[u]); }
      const int have = alt.Find(keys, second, walk.best_at);
      if (lane < a.top_k) { const Entry e = alt.sh.list[lane]; res.StoreTop(a, static_cast<long long>(row) * a.top_k + lane, lane < have ? e.v : -INFINITY, e.cls); }
      __syncwarp();
    }
    y = y_next;
  }
}

// 8 warps walk a row (with a cluster of blocks: a share of it), a ninth joins their sums, finds the alternatives and writes the results
// while they are in the next row. Named barriers: kFull (walkers arrive, the ninth waits), kFree (the other way round, as soon as it has
// the maxima in registers). 56 registers a thread: 4 blocks, 32 walking warps on an SM; with 24 of them the walk takes a fifth longer.
constexpr int kBlockRing = 3, kBlockThreads = 288;
enum { kFull = 1, kFree = 2, kWalkers = 3, kJoined = 4 };
template <int ID, int THREADS = kBlockThreads> __device__ __forceinline__ void BarrierSync() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(THREADS) : "memory"); }
template <int ID> __device__ __forceinline__ void BarrierArrive() { asm volatile("bar.arrive %0, %1;" ::"n"(ID), "n"(kBlockThreads) : "memory"); }
template <typename T, bool TOP>
__global__ void __launch_bounds__(kBlockThreads, 4) ClassLogProbsBlockKernel(ClassScoresArgs a) {
  extern __shared__ __align__(16) uint4 s_ring[];      // [kBlockRing][kUnroll][256]
  __shared__ TopShared<256> s_top[1];
  __shared__ unsigned int s_key[256], s_second[256]; __shared__ int s_chunk[256];
  __shared__ float s_m[8], s_s[8], s_t[8];
  __shared__ float s_share[3]; __shared__ int s_have;                  // of a cluster's block: its share's sums and number of alternatives
  __shared__ Entry s_joined[kMaxTopClasses]; __shared__ int s_count[8];
  Entry (*s_join)[kMaxTopClasses] = reinterpret_cast<Entry (*)[kMaxTopClasses]>(s_top[0].cand);      // 8 lists, when the candidates are done with
  static_assert(TopShared<256>::kCandidates >= 8 * kMaxTopClasses, "the lists of a cluster's blocks");
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int parts = static_cast<int>(cg::this_cluster().num_blocks()), part = static_cast<int>(cg::this_cluster().block_rank());
  const unsigned int stride = gridDim.x / parts, row0 = blockIdx.x / parts;      // the grid has no more clusters than rows
  if (warp < 8) {
    Walk<T, 256, kBlockRing> walk(a, s_ring, row0, stride, threadIdx.x, part, parts);
    for (unsigned int row = row0; row < a.rows; row += stride) {
      const RowShare<T> r(a, row, part, parts, 256);
      const float head_v = r.Head(threadIdx.x), tail_v = r.Tail(threadIdx.x);
      Sums sums = walk.Row(r);
      if (head_v != -INFINITY) sums.AddOne(head_v);
      if (tail_v != -INFINITY) sums.AddOne(tail_v);
      sums.JoinLanes();
      if (row != row0) BarrierSync<kFree>();
      if constexpr (TOP) { s_key[threadIdx.x] = OrderKey<T>(walk.best[0]); s_second[threadIdx.x] = OrderKey<T>(walk.second[0]); s_chunk[threadIdx.x] = walk.best_at[0]; }
      if (lane == 0) { s_m[warp] = sums.m; s_s[warp] = sums.s; s_t[warp] = sums.t; }
      BarrierArrive<kFull>();
      if (parts > 1) {
        // the first block joins the lists of all, read from their shared memory: warp w has block w's list, lane i its entry i. The lists
        // are sorted, so an entry's rank is, list by list and by bisection, how many come before it.
        cg::this_cluster().sync();
        if (TOP && part == 0) {
          int n = 0;
          Entry e; e.v = -INFINITY; e.cls = 0x7fffffff;
          if (warp < parts) {
            n = *cg::this_cluster().map_shared_rank(&s_have, warp);
            e = cg::this_cluster().map_shared_rank(&s_top[0], warp)->list[lane];      // beyond n: not an entry
            s_join[warp][lane] = e;
          }
          if (lane == 0) s_count[warp] = n;
          BarrierSync<kWalkers, 256>();
          if (lane < n) {
            int rank = 0;
#pragma unroll
            for (int p = 0; p < 8; ++p) {
              const int m = s_count[p];
              int before = 0;
#pragma unroll
              for (int step = 32; step > 0; step >>= 1) if (before + step <= m && Before(s_join[p][before + step - 1], e)) before += step;
              rank += before;
            }
            if (rank < a.top_k) s_joined[rank] = e;
          }
          BarrierSync<kJoined>();
        }
        cg::this_cluster().sync();
      }
    }
    return;
  }
  long long y = LabelOf(a, row0);
  for (unsigned int row = row0; row < a.rows; row += stride) {
    const RowShare<T> r(a, row, part, parts, 256);
    const float given = lane == 0 && y >= 0 && y < r.K ? ToFloat(r.s[y]) : 0.f;
    const long long y_next = row + stride < a.rows ? LabelOf(a, row + stride) : -1;
    Alternatives<256, T> alt{s_top[0], r, a.top_k, lane};
    BarrierSync<kFull>();
    Sums sums;
    if (lane < 8) { sums.m = s_m[lane]; sums.s = s_s[lane]; sums.t = s_t[lane]; }
    int have = 0;
    if constexpr (TOP) {
      unsigned int keys[8], second[8]; int chunk[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) { keys[i] = s_key[lane + 32 * i]; second[i] = s_second[lane + 32 * i]; chunk[i] = s_chunk[lane + 32 * i]; }
      if (row + stride < a.rows) BarrierArrive<kFree>();
      sums.JoinLanes();
      have = alt.Find(keys, second, chunk);
    } else {
      if (row + stride < a.rows) BarrierArrive<kFree>();
      sums.JoinLanes();
    }
    if (parts > 1) {
      if (lane == 0) { s_share[0] = sums.m; s_share[1] = sums.s; s_share[2] = sums.t; s_have = have; }
      cg::this_cluster().sync();
      if (part == 0) {
        Sums other;
        if (lane < parts) { const float* o = cg::this_cluster().map_shared_rank(&s_share[0], lane); other.m = o[0]; other.s = o[1]; other.t = o[2]; }
        other.JoinLanes();
        sums = other;
        if constexpr (TOP) {
          BarrierSync<kJoined>();      // the walkers have joined the lists
          have = 0;
          for (int p = 0; p < 8; ++p) have += s_count[p];
          have = min(have, a.top_k);
        }
      }
      cg::this_cluster().sync();           // no block goes on while its shared memory is read
    }
    if (part == 0) {
      const RowResult res(sums);
      if (lane == 0) res.Store(a, row, y, given);
      if constexpr (TOP) if (lane < a.top_k) { const Entry e = parts > 1 ? s_joined[lane] : alt.sh.list[lane]; res.StoreTop(a, static_cast<long long>(row) * a.top_k + lane, lane < have ? e.v : -INFINITY, e.cls); }
    }
    __syncwarp();
    y = y_next;
  }
}

// ----------------------------------------------------------------------------------------- contiguous columns ----
// A block turns tile_rows rows of class-major scores (or of any strides) into rows in shared memory, read as they lie: neighbouring
// lanes have neighbouring rows. Then a warp per row, as above. Rows of up to kTileMostBytes / 8 bytes.
// (Against the kernel below, which keeps a list per thread: 2479 x 2000 fp32 with 32 alternatives 230 -> 36 us.)
constexpr int kTileBytes = 72 * 1024, kTileMostBytes = 200 * 1024;
// PER > 0: at most 8 PER classes, 8 lanes per row.
template <typename T, bool TOP, int PER>
__global__ void __launch_bounds__(256) ClassLogProbsTileKernel(ClassScoresArgs a, int tile_rows, int pitch) {
  constexpr int N = Pack<T>::N;
  extern __shared__ __align__(16) unsigned char s_tile[];
  __shared__ TopShared<128> s_top[TOP ? 8 : 1];
  const int K = static_cast<int>(a.classes), warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long row0 = static_cast<long long>(blockIdx.x) * tile_rows;
  const int rows = static_cast<int>(min(static_cast<long long>(tile_rows), a.rows - row0));
  {
    const int r = threadIdx.x % tile_rows, step = 256 / tile_rows;
    if (r < rows) {
      const T* from = static_cast<const T*>(a.scores) + (row0 + r) * a.row_stride;
      T* to = reinterpret_cast<T*>(s_tile + r * pitch);
      int c = threadIdx.x / tile_rows;
      for (; c + 7 * step < K; c += 8 * step) {
        T v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = from[(c + u * step) * a.class_stride];
#pragma unroll
        for (int u = 0; u < 8; ++u) to[c + u * step] = v[u];
      }
      for (; c < (K + N - 1) / N * N; c += step) to[c] = c < K ? from[c * a.class_stride] : FromFloat<T>(-INFINITY);
    }
  }
  __syncthreads();
  if constexpr (PER > 0) {
    for (int i0 = 0; i0 < rows; i0 += 32) {
      const int i = i0 + threadIdx.x / 8;
      SomeRow<T, PER>(a, row0 + i, i < rows, reinterpret_cast<const T*>(s_tile + min(i, rows - 1) * pitch), threadIdx.x & 7);
    }
    return;
  }
  for (int i = warp; i < rows; i += 8) {
    const long long row = row0 + i;
    const RowShare<T> r(reinterpret_cast<const T*>(s_tile + i * pitch), K);
    const long long y = LabelOf(a, row);
    PairSums<T> pairs;
    float best[kUnroll], second[kUnroll]; int best_at[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) { best[u] = second[u] = -INFINITY; best_at[u] = 0; }
    for (int at = 0; at < r.v_end; at += 32 * kUnroll) {
      uint4 q[kUnroll];
      float most = -INFINITY;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        q[u] = at + 32 * u + lane < r.v_end ? r.body[at + 32 * u + lane] : AllRuledOut(static_cast<const T*>(nullptr));
        const uint4 one[1] = {q[u]};
        const float m = MaxOf(one, static_cast<const T*>(nullptr));
        if (m > best[u]) { second[u] = best[u]; best[u] = m; best_at[u] = at; } else second[u] = fmaxf(second[u], m);
        most = MaxNan(most, m);
      }
      if (most > pairs.m) pairs.Raise(most);
      pairs.Add16(q);
    }
    Sums sums = pairs.Total();
    sums.JoinLanes();
    const RowResult res(sums);
    if (lane == 0) res.Store(a, row, y, y >= 0 && y < K ? ToFloat(r.s[y]) : 0.f);
    if constexpr (TOP) {
      Alternatives<128, T> alt{s_top[warp], r, a.top_k, lane};
      unsigned int keys[kUnroll], seconds[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) { keys[u] = OrderKey<T>(best[u]); seconds[u] = OrderKey<T>(second[u]); }
      const int have = alt.Find(keys, seconds, best_at);
      if (lane < a.top_k) { const Entry e = alt.sh.list[lane]; res.StoreTop(a, row * a.top_k + lane, lane < have ? e.v : -INFINITY, e.cls); }
      __syncwarp();
    }
  }
}

// 32 rows per block (lane = row, so class-major scores are read 32 rows at a time), the classes dealt out over the warps; every
// thread keeps its own sums and its own sorted list, joined per row at the end.
constexpr int kColumnUnroll = 8;
template <typename T>
__global__ void __launch_bounds__(1024) ClassLogProbsColumnKernel(ClassScoresArgs a) {
  extern __shared__ Entry s_lists[];                 // [warps][top_k][32]
  __shared__ float s_m[32][32], s_s[32][32], s_t[32][32]; __shared__ int s_have[32][32];
  const int warps = blockDim.x / 32, w = threadIdx.x / 32, lane = threadIdx.x % 32, K = static_cast<int>(a.classes), k = a.top_k;
  const long long row = static_cast<long long>(blockIdx.x) * 32 + lane;
  const bool is_row = row < a.rows;
  const T* s = static_cast<const T*>(a.scores) + (is_row ? row : 0) * a.row_stride;
  Entry* list = s_lists + static_cast<size_t>(w) * k * 32 + lane;
  Sums sums; int have = 0; float threshold = -INFINITY;
  auto consider = [&](float v, int cls) {
    if (!(v > threshold)) return;                    // classes rise within a thread: equal scores lose
    int at = have < k ? have : k - 1;
    for (; at > 0 && list[(at - 1) * 32].v < v; --at) list[at * 32] = list[(at - 1) * 32];
    list[at * 32].v = v; list[at * 32].cls = cls;
    if (have < k) ++have;
    if (have == k) threshold = list[(k - 1) * 32].v;
  };
  for (int c0 = w; c0 < K; c0 += warps * kColumnUnroll) {
    float v[kColumnUnroll];
#pragma unroll
    for (int u = 0; u < kColumnUnroll; ++u) { const int c = c0 + u * warps; v[u] = c < K && is_row ? ToFloat(s[c * a.class_stride]) : -INFINITY; }
    float most = v[0];
#pragma unroll
    for (int u = 1; u < kColumnUnroll; ++u) most = MaxNan(most, v[u]);
    if (most > sums.m) sums.Raise(most);
    const float base = sums.Base();
#pragma unroll
    for (int u = 0; u < kColumnUnroll; ++u) { sums.Add(v[u], base); if (k > 0) consider(v[u], c0 + u * warps); }
  }
  s_m[w][lane] = sums.m; s_s[w][lane] = sums.s; s_t[w][lane] = sums.t; s_have[w][lane] = have;
  __syncthreads();
  if (w != 0 || !is_row) return;
  for (int o = 1; o < warps; ++o) sums.Join(s_m[o][lane], s_s[o][lane], s_t[o][lane]);
  const RowResult res(sums);
  const long long y = LabelOf(a, row);
  res.Store(a, row, y, y >= 0 && y < K ? ToFloat(s[y * a.class_stride]) : 0.f);
  // the warps' sorted lists are merged; s_have turns into "taken so far" in s_m (as an int)
  for (int o = 0; o < warps; ++o) s_m[o][lane] = __int_as_float(0);
  for (int t = 0; t < k; ++t) {
    Entry best; best.v = -INFINITY; best.cls = 0x7fffffff; int from = -1;
    for (int o = 0; o < warps; ++o) {
      const int taken = __float_as_int(s_m[o][lane]);
      if (taken < s_have[o][lane]) { const Entry e = s_lists[(static_cast<size_t>(o) * k + taken) * 32 + lane]; if (Before(e, best)) { best = e; from = o; } }
    }
    if (from >= 0) s_m[from][lane] = __int_as_float(__float_as_int(s_m[from][lane]) + 1);
    res.StoreTop(a, row * k + t, from >= 0 ? best.v : -INFINITY, best.cls);
  }
}

// --------------------------------------------------------------------------------------------------- gradient ----
// What the gradient needs of a row: p_j = e^(s_j - m - log_sum), d_j = p_j (a - h log p_j), + g_label at the label.
struct RowGrad {
  float m, log_sum, a, h, g_label; int label; bool none, bad, again;
  __device__ __forceinline__ RowGrad() {}
  __device__ __forceinline__ RowGrad(const ClassScoresArgs& s, const ClassGradArgs& g, long long row) {
    float top = 0.f;
    for (int t = 0; t < s.top_k; ++t) top += Top(s, g, row, t);
    Set(s, g, row, top);
  }
  __device__ __forceinline__ static float Top(const ClassScoresArgs& s, const ClassGradArgs& g, long long row, int t) {
    const int c = s.top_class[row * s.top_k + t]; const float v = g.g_top[row * s.top_k + t];
    return c >= 0 && c < s.classes ? v : 0.f;
  }
  // top: the sum of the gradients of the alternatives' log probabilities
  __device__ __forceinline__ void Set(const ClassScoresArgs& s, const ClassGradArgs& g, long long row, float top) {
    const float log_norm = s.log_norm[row];
    const long long y = LabelOf(s, row);
    const float g_norm = g.g_log_norm ? g.g_log_norm[row] : 0.f, g_prob = g.g_log_prob ? g.g_log_prob[row] : 0.f, entropy = s.entropy[row];
    h = g.g_entropy ? g.g_entropy[row] : 0.f;
    none = log_norm == -INFINITY; bad = (!none && !(fabsf(log_norm) < InfF())) || y >= s.classes;
    again = !none && !bad && fabsf(log_norm) > kTrustedLogNorm;
    m = none ? 0.f : log_norm; log_sum = 0.f;
    label = y >= 0 && y < s.classes ? static_cast<int>(y) : -1;
    g_label = label >= 0 ? g_prob : 0.f;
    a = g_norm - g_label - h * entropy - top;
    if (none) { a = h = g_label = 0.f; }
    if (bad) a = NanF();
  }
  __device__ __forceinline__ float Soft(float v) const { const float lp = MaxNan((v - m) - log_sum, kLowestExponent); return Exp2(lp * kLog2E) * fmaf(-h, lp, a); }
  // with the label's own gradient
  __device__ __forceinline__ float At(float v, int j) const { const float d = Soft(v); return none ? 0.f : j == label ? d + g_label : d; }
  // log sum e^(s - m)
  __device__ __forceinline__ static float AgainLog(const Sums& r) { return (log2f(r.s) - Shift(r.m)) * kLn2; }
  // one thread walks the row, in sums of 64 terms: 60000 equal terms one by one gave p up to 7e-4 off
  template <typename T>
  __device__ __forceinline__ void TakeAgain(const ClassScoresArgs& s, const T* row) {
    Sums r;
    for (long long j0 = 0; j0 < s.classes; j0 += 64) {
      Sums part;
      for (long long j = j0; j < min(s.classes, j0 + 64); ++j) part.AddOne(ToFloat(row[j * s.class_stride]));
      r.Join(part.m, part.s, part.t);
    }
    m = r.m; log_sum = AgainLog(r);
  }
};
// The whole gradient of an alternative's class: an index that is named several times gets all its gradients.
template <typename T>
__device__ __forceinline__ void PatchTop(const ClassScoresArgs& a, const ClassGradArgs& g, const RowGrad& r, long long row, int t, int lo, int hi) {
  const int c = a.top_class[row * a.top_k + t];
  if (c < lo || c >= hi || r.none) return;
  float add = 0.f;
  for (int o = 0; o < a.top_k; ++o) if (a.top_class[row * a.top_k + o] == c) add += g.g_top[row * a.top_k + o];
  static_cast<T*>(g.grad)[row * g.grad_row_stride + c * g.grad_class_stride] =
      FromFloat<T>(r.At(ToFloat(static_cast<const T*>(a.scores)[row * a.row_stride + c * a.class_stride]), c) + add);
}

// Rows of few classes: the block's rows are one after the other in memory, its threads walk their elements.
constexpr int kGradThreads = 256, kGradRows = 64, kGradVectors = 4;      // kGradVectors: 16-byte loads of a thread and chunk
template <typename T>
__global__ void __launch_bounds__(kGradThreads) ClassGradFewKernel(ClassScoresArgs a, ClassGradArgs g) {
  __shared__ RowGrad s_row[kGradRows];
  const long long row0 = static_cast<long long>(blockIdx.x) * kGradRows;
  const int rows = static_cast<int>(min(static_cast<long long>(kGradRows), a.rows - row0)), K = static_cast<int>(a.classes);
  const T* in = static_cast<const T*>(a.scores) + row0 * a.row_stride;
  T* out = static_cast<T*>(g.grad) + row0 * g.grad_row_stride;
  if (threadIdx.x < rows) {
    RowGrad r(a, g, row0 + threadIdx.x);
    if (r.again) r.TakeAgain(a, in + threadIdx.x * a.row_stride);
    s_row[threadIdx.x] = r;
  }
  __syncthreads();
  int r = threadIdx.x / K, j = threadIdx.x - r * K;
  const int dr = kGradThreads / K, dj = kGradThreads - dr * K;
  while (r < rows) {
    out[r * g.grad_row_stride + j] = FromFloat<T>(s_row[r].At(ToFloat(in[r * a.row_stride + j * a.class_stride]), j));
    r += dr; j += dj;
    if (j >= K) { j -= K; ++r; }
  }
  if (a.top_k > 0) {
    __syncthreads();
    for (int e = threadIdx.x; e < rows * a.top_k; e += kGradThreads) PatchTop<T>(a, g, s_row[e / a.top_k], row0 + e / a.top_k, e % a.top_k, 0, K);
  }
}

// A block per row and chunk of classes. ALIGNED: scores and gradient of a row reach a 16-byte boundary together.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kGradThreads) ClassGradRowKernel(ClassScoresArgs a, ClassGradArgs g, int chunk, int chunks) {
  constexpr int N = Pack<T>::N;
  __shared__ RowGrad s_row; __shared__ float s_m[8], s_s[8], s_t[8];
  const long long row = blockIdx.x / chunks;
  const int K = static_cast<int>(a.classes);
  const int head = ALIGNED ? min(K, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(static_cast<const T*>(a.scores) + row * a.row_stride) & 15)) & 15) / static_cast<int>(sizeof(T))) : 0;
  const T* in = static_cast<const T*>(a.scores) + row * a.row_stride;
  T* out = static_cast<T*>(g.grad) + row * g.grad_row_stride;
  const T* type = nullptr;
  // chunk c: the classes from head + c * chunk (chunk 0: from 0) to the next one's start. Its scores are asked for before the row's
  // values, on which everything else waits.
  const int c = blockIdx.x % chunks;
  const int lo = c == 0 ? 0 : min(K, head + c * chunk), hi = c == chunks - 1 ? K : min(K, head + (c + 1) * chunk);
  const int first = min(K, head + c * chunk), vectors = ALIGNED ? (hi - first) / N : 0, rest = first + vectors * N;
  const uint4* from = reinterpret_cast<const uint4*>(in + first); uint4* to = reinterpret_cast<uint4*>(out + first);
  uint4 q[kGradVectors];
#pragma unroll
  for (int u = 0; u < kGradVectors; ++u) { const int i = threadIdx.x + u * kGradThreads; if (i < vectors) q[u] = __ldg(from + i); }
  if (threadIdx.x < 32) {
    float top = threadIdx.x < a.top_k ? RowGrad::Top(a, g, row, threadIdx.x) : 0.f;
    for (int o = 16; o > 0; o >>= 1) top += __shfl_xor_sync(0xffffffffu, top, o);
    RowGrad r;
    r.Set(a, g, row, top);
    if (threadIdx.x == 0) s_row = r;
  }
  __syncthreads();
  if (s_row.again) {
    Sums r;
    for (int j = threadIdx.x; j < K; j += kGradThreads) r.AddOne(ToFloat(in[j]));
    r.JoinLanes();
    if ((threadIdx.x & 31) == 0) { s_m[threadIdx.x >> 5] = r.m; s_s[threadIdx.x >> 5] = r.s; s_t[threadIdx.x >> 5] = r.t; }
    __syncthreads();
    if (threadIdx.x == 0) { Sums all; for (int w = 0; w < kGradThreads / 32; ++w) all.Join(s_m[w], s_s[w], s_t[w]); s_row.m = all.m; s_row.log_sum = RowGrad::AgainLog(all); }
    __syncthreads();
  }
  const RowGrad r = s_row;
  if constexpr (ALIGNED) {
    for (int j = lo + threadIdx.x; j < first; j += kGradThreads) out[j] = FromFloat<T>(r.At(ToFloat(in[j]), j));
#pragma unroll
    for (int u = 0; u < kGradVectors; ++u) {
      const int i = threadIdx.x + u * kGradThreads;
      if (i >= vectors) break;
      float v[N]; Unpack(q[u], v, type);
      union { uint4 q; T t[N]; } o;
#pragma unroll
      for (int k = 0; k < N; ++k) o.t[k] = FromFloat<T>(r.At(v[k], first + i * N + k));
      to[i] = o.q;
    }
  }
  for (int j = rest + threadIdx.x; j < hi; j += kGradThreads) out[j] = FromFloat<T>(r.At(ToFloat(in[j]), j));
  if (a.top_k > 0) {
    __syncthreads();
    if (threadIdx.x < a.top_k) PatchTop<T>(a, g, r, row, threadIdx.x, lo, hi);
  }
}

constexpr int kGradClasses = 12;      // scores of a thread in flight
// A thread per row (class-major scores, or any strides); the classes in slices over the grid's second dimension.
template <typename T>
__global__ void __launch_bounds__(kGradThreads) ClassGradColumnKernel(ClassScoresArgs a, ClassGradArgs g, int slice) {
  const long long row = static_cast<long long>(blockIdx.x) * kGradThreads + threadIdx.x;
  if (row >= a.rows) return;
  const int K = static_cast<int>(a.classes), lo = blockIdx.y * slice, hi = min(K, lo + slice);
  const T* in = static_cast<const T*>(a.scores) + row * a.row_stride;
  T* out = static_cast<T*>(g.grad) + row * g.grad_row_stride;
  float v[kGradClasses];
#pragma unroll
  for (int u = 0; u < kGradClasses; ++u) v[u] = lo + u < hi ? ToFloat(in[(lo + u) * a.class_stride]) : 0.f;      // before the row's values
  RowGrad r(a, g, row);
  if (r.again) r.TakeAgain(a, in);
  for (int j = lo; j < hi; j += kGradClasses) {
    if (j > lo) {
#pragma unroll
      for (int u = 0; u < kGradClasses; ++u) v[u] = j + u < hi ? ToFloat(in[(j + u) * a.class_stride]) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kGradClasses; ++u) if (j + u < hi) out[(j + u) * g.grad_class_stride] = FromFloat<T>(r.At(v[u], j + u));
  }
  for (int t = 0; t < a.top_k; ++t) PatchTop<T>(a, g, r, row, t, lo, hi);
}

template <typename F> void DispatchType(int dtype, F&& f) {
  switch (dtype) {
    case kOpFloat32: f(static_cast<float*>(nullptr)); return;
    case kOpFloat16: f(static_cast<__half*>(nullptr)); return;
    case kOpBFloat16: f(static_cast<__nv_bfloat16*>(nullptr)); return;
    default: Log::Fatal("class scores: unknown type code %d", dtype);
  }
}

constexpr int kSms = 148;

template <typename T, int MOST>
void LaunchFew(const ClassScoresArgs& a, bool by_class, cudaStream_t s) {
  constexpr int kRows = MOST <= 16 ? 2 : 1;      // two rows' scores in flight per thread while they fit the registers
  if (by_class) ClassLogProbsFewKernel<T, MOST, true, kRows><<<static_cast<unsigned int>((a.rows + kFewThreads * kRows - 1) / (kFewThreads * kRows)), kFewThreads, 0, s>>>(a);
  else ClassLogProbsFewKernel<T, MOST, false, 1><<<static_cast<unsigned int>((a.rows + kFewThreads - 1) / kFewThreads), kFewThreads, 0, s>>>(a);
}
template <typename T>
void LaunchFew(const ClassScoresArgs& a, cudaStream_t s) {
  // lanes walk rows: right where neighbouring rows are nearer to each other than neighbouring classes
  const bool by_class = a.row_stride < a.class_stride;
  if (a.classes <= 4) LaunchFew<T, 4>(a, by_class, s);
  else if (a.classes <= 8) LaunchFew<T, 8>(a, by_class, s);
  else if (a.classes <= 12) LaunchFew<T, 12>(a, by_class, s);
  else if (a.classes <= 16) LaunchFew<T, 16>(a, by_class, s);
  else if (a.classes <= 32) LaunchFew<T, 32>(a, by_class, s);
  else LaunchFew<T, kFewClasses>(a, by_class, s);
}

// as many blocks as are resident at once, each with several rows
template <typename T, bool TOP>
void LaunchWarps(const ClassScoresArgs& a, cudaStream_t s) {
  constexpr int kBytes = kWarpRing * kUnroll * 256 * 16;
  static PerDevice allowed;
  AllowSharedMemory(ClassLogProbsWarpKernel<T, TOP>, kBytes, &allowed);
  ClassLogProbsWarpKernel<T, TOP><<<static_cast<unsigned int>(std::min<long long>((a.rows + 7) / 8, kSms * 4)), 256, kBytes, s>>>(a);
}
template <typename T, bool TOP>
void LaunchBlocks(const ClassScoresArgs& a, int cluster, cudaStream_t s) {
  constexpr int kBytes = kBlockRing * kUnroll * 256 * 16;
  static PerDevice allowed;
  AllowSharedMemory(ClassLogProbsBlockKernel<T, TOP>, kBytes, &allowed);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned int>(std::min<long long>(a.rows, kSms * 4 / cluster) * cluster)); cfg.blockDim = dim3(kBlockThreads);
  cfg.dynamicSmemBytes = kBytes; cfg.stream = s; cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 1 : 0;
  FB_CUDA(cudaLaunchKernelEx(&cfg, ClassLogProbsBlockKernel<T, TOP>, a));
}

// an odd number of 16-byte pieces: rows of a tile start in different banks
template <typename T> long long TilePitch(long long classes) { return 16 * (((classes * static_cast<long long>(sizeof(T)) + 15) / 16) | 1); }
template <typename T, bool TOP, int PER>
void LaunchTiles(const ClassScoresArgs& a, int rows, int pitch, cudaStream_t s) {
  static PerDevice allowed;
  AllowSharedMemory(ClassLogProbsTileKernel<T, TOP, PER>, kTileMostBytes, &allowed);
  ClassLogProbsTileKernel<T, TOP, PER><<<static_cast<unsigned int>((a.rows + rows - 1) / rows), 256, static_cast<size_t>(rows) * pitch, s>>>(a, rows, pitch);
}

}  // namespace

void LaunchClassLogProbs(const ClassScoresArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return;
  DispatchType(a.dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    if (a.class_stride == 1 && a.classes > 32 && a.classes <= kSomeClasses) {
      const unsigned int blocks = static_cast<unsigned int>((a.rows + 15) / 16);
      if (a.classes <= 64) ClassLogProbsSomeKernel<T, 8><<<blocks, 128, 0, s>>>(a);
      else if (a.classes <= 128) ClassLogProbsSomeKernel<T, 16><<<blocks, 128, 0, s>>>(a);
      else ClassLogProbsSomeKernel<T, 32><<<blocks, 128, 0, s>>>(a);
    } else if (a.classes <= kFewClasses) {
      LaunchFew<T>(a, s);
    } else if (a.class_stride == 1) {
      // A warp per row as long as that fills the machine and a warp's walk stays short; else a block, and a cluster of blocks while
      // there are fewer blocks than two per SM and every block has a full chunk.
      const long long chunk = 256LL * kUnroll * Pack<T>::N;
      if (a.classes <= chunk / 8 || (a.classes <= chunk && a.rows >= kSms * 16)) {
        if (a.top_k > 0) LaunchWarps<T, true>(a, s); else LaunchWarps<T, false>(a, s);
      } else {
        int cluster = 1;
        while (cluster < 8 && a.rows * cluster < 2 * kSms && a.classes >= 2 * cluster * chunk / kUnroll) cluster *= 2;
        if (a.top_k > 0) LaunchBlocks<T, true>(a, cluster, s); else LaunchBlocks<T, false>(a, cluster, s);
      }
    } else if (TilePitch<T>(a.classes) * 8 <= kTileMostBytes) {
      const int pitch = static_cast<int>(TilePitch<T>(a.classes));
      int rows = 32;      // per tile: as many as leave room for three blocks on an SM, and no fewer than fill a 32-byte sector
      while (rows > 32 / static_cast<int>(sizeof(T)) && rows * pitch > kTileBytes) rows /= 2;
      while (rows > 8 && rows * pitch > kTileMostBytes) rows /= 2;
      if (a.classes <= 128) LaunchTiles<T, false, 16>(a, rows, pitch, s);
      else if (a.classes <= kSomeClasses) LaunchTiles<T, false, 32>(a, rows, pitch, s);
      else if (a.top_k > 0) LaunchTiles<T, true, 0>(a, rows, pitch, s);
      else LaunchTiles<T, false, 0>(a, rows, pitch, s);
    } else {
      int warps = 8;
      while (warps < 32 && (a.rows + 31) / 32 * warps < kSms * 32 && a.classes > 2LL * warps * kColumnUnroll) warps *= 2;
      while (warps > 8 && static_cast<size_t>(warps) * a.top_k * 32 * sizeof(Entry) > 128 * 1024) warps /= 2;
      const size_t smem = static_cast<size_t>(warps) * a.top_k * 32 * sizeof(Entry);
      static PerDevice allowed;      // one per type
      AllowSharedMemory(ClassLogProbsColumnKernel<T>, 128 * 1024, &allowed);
      ClassLogProbsColumnKernel<T><<<static_cast<unsigned int>((a.rows + 31) / 32), warps * 32, smem, s>>>(a);
    }
  });
  FB_LAUNCHED(); FB_KERNEL_CHECK();
}

void LaunchClassLogProbsGrad(const ClassScoresArgs& a, const ClassGradArgs& g, cudaStream_t s) {
  if (a.rows <= 0) return;
  DispatchType(a.dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    constexpr int N = Pack<T>::N;
    if (g.grad_class_stride != 1 || a.class_stride != 1) {
      // slices long enough to be worth the row's set-up, short enough to fill the machine
      const long long blocks = (a.rows + kGradThreads - 1) / kGradThreads;
      long long slices = std::max(1LL, std::min((a.classes + 31) / 32, (4LL * kSms + blocks - 1) / blocks));
      const int slice = static_cast<int>((a.classes + slices - 1) / slices);
      slices = (a.classes + slice - 1) / slice;
      if (slices > 65535) Log::Fatal("class scores: too many classes");
      ClassGradColumnKernel<T><<<dim3(static_cast<unsigned int>(blocks), static_cast<unsigned int>(slices)), kGradThreads, 0, s>>>(a, g, slice);
    } else if (a.classes < 2 * kGradThreads) {
      ClassGradFewKernel<T><<<static_cast<unsigned int>((a.rows + kGradRows - 1) / kGradRows), kGradThreads, 0, s>>>(a, g);
    } else {
      const int chunk = kGradThreads * N * kGradVectors;
      const long long chunks = (a.classes + chunk - 1) / chunk;
      if (a.rows * chunks > 0x7fffffffLL) Log::Fatal("class scores: %lld rows x %lld classes are not covered", a.rows, a.classes);
      const bool aligned = (reinterpret_cast<uintptr_t>(a.scores) & 15) == (reinterpret_cast<uintptr_t>(g.grad) & 15) && ((a.row_stride - g.grad_row_stride) * sizeof(T)) % 16 == 0;
      const unsigned int blocks = static_cast<unsigned int>(a.rows * chunks);
      if (aligned) ClassGradRowKernel<T, true><<<blocks, kGradThreads, 0, s>>>(a, g, chunk, static_cast<int>(chunks));
      else ClassGradRowKernel<T, false><<<blocks, kGradThreads, 0, s>>>(a, g, chunk, static_cast<int>(chunks));
    }
  });
  FB_LAUNCHED(); FB_KERNEL_CHECK();
}

}  // namespace fb
