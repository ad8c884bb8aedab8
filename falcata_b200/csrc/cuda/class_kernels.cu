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
// All kernels read every score once from memory, the gradient kernels write every value once: they are bound by bandwidth.
// (S, T) are kept relative to a running maximum and rescaled when it grows, so partial results of any split of a row can be
// joined. Which threads share a row goes by the number of classes and by what is contiguous:
//   few classes                 a thread per row, the row in registers           (ClassLogProbsFewKernel)
//   contiguous rows             a warp per row, or a block or cluster per row    (ClassLogProbsRowKernel)
//   contiguous columns, others  32 rows per block, the classes over its warps    (ClassLogProbsColumnKernel)
#include "kernels.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace cg = cooperative_groups;

namespace fb {

namespace {

// log_norm in fp32 gives p to a relative 2^-24 |log_norm|: beyond this size the gradient takes the row's maximum and sum again.
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
// of B shifts all x alike, and the results are put together from the same x and B, so it drops out (scores far from 0 lose
// nothing). Where B overflows (|m| > kHugeScore: scores that differ at all differ by more than e^x can hold) x = (s_j - m) log2 e.
constexpr float kHugeScore = 1e36f;
__device__ __forceinline__ bool Huge(float m) { return !(fabsf(m) <= kHugeScore); }
__device__ __forceinline__ float Exponent(float v, float m) { return Huge(m) ? (v - m) * kLog2E : fmaf(v, kLog2E, -(m * kLog2E)); }
// how much lower the exponents are when the maximum goes from m to `to` (> m)
__device__ __forceinline__ float Lower(float m, float to) { return fmaxf(Huge(m) || Huge(to) ? (m - to) * kLog2E : __fsub_rn(__fmul_rn(m, kLog2E), __fmul_rn(to, kLog2E)), kLowestExponent); }

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
// per instruction. That is exact as long as the maximum is far above that value; elsewhere every exponent is clamped by itself.
template <typename T> struct FarBelow;
template <> struct FarBelow<float> { static constexpr float kFar = INFINITY; };
template <> struct FarBelow<__half> { static constexpr unsigned int kLow = 0xfbfffbffu; static constexpr float kFar = -60000.f; };               // -65504
template <> struct FarBelow<__nv_bfloat16> { static constexpr unsigned int kLow = 0xf14af14au; static constexpr float kFar = -1e29f; };          // -1.0e30
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
      if (base > FarBelow<T>::kFar && base <= kHugeScore) {
        const unsigned int low = FarBelow<T>::kLow;
        const float minus_b = -(base * kLog2E);
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
  float m, log_sum, entropy; bool none, bad;      // log_sum: to base 2
  __device__ explicit RowResult(const Sums& r) {
    none = r.m == -INFINITY && !(r.s != r.s); bad = !none && !(fabsf(r.m) < InfF() && r.s < InfF());   // a NaN sum fails the comparison
    m = r.m; log_sum = log2f(r.s); entropy = none ? 0.f : bad ? NanF() : fmaxf((log_sum - r.t / r.s) * kLn2, 0.f);
  }
  __device__ __forceinline__ float LogProb(float v) const { return none || v == -INFINITY ? (bad ? NanF() : -INFINITY) : bad ? NanF() : Huge(m) || Huge(v) ? (v - m) - log_sum * kLn2 : fminf((Exponent(v, m) - log_sum) * kLn2, 0.f); }
  // m + the rest: what B lacks of m log2 e is put back
  __device__ __forceinline__ float LogNorm() const { return none ? -INFINITY : bad ? NanF() : m + (log_sum + (Huge(m) ? 0.f : fmaf(-m, kLog2E, __fmul_rn(m, kLog2E)))) * kLn2; }
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
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const long long row = row0 + i * kFewThreads + threadIdx.x;
    if (row >= a.rows) return;
    Sums sums;
    float m = v[i][0];
#pragma unroll
    for (int j = 1; j < MOST; ++j) m = MaxNan(m, v[i][j]);
    sums.m = m;
    const float b = sums.Base();
#pragma unroll
    for (int j = 0; j < MOST; ++j) sums.Add(v[i][j], b);
    const RowResult res(sums);
    float given = 0.f;
#pragma unroll
    for (int j = 0; j < MOST; ++j) if (j == y[i]) given = v[i][j];
    res.Store(a, row, y[i], given);
    for (int t = 0; t < a.top_k; ++t) {
      float best = -INFINITY; int cls = -1;
#pragma unroll
      for (int j = 0; j < MOST; ++j) if (v[i][j] > best) { best = v[i][j]; cls = j; }
#pragma unroll
      for (int j = 0; j < MOST; ++j) if (j == cls) v[i][j] = -INFINITY;
      res.StoreTop(a, row * a.top_k + t, best, cls);
    }
  }
}

// -------------------------------------------------------------------------------------------- contiguous rows ----
// GROUP threads (a warp or a block) walk a row, or a block cluster's share of one, kUnroll 16-byte pieces per thread at a time. The
// pieces come by asynchronous copies through a ring of kWalkRing chunks, every thread its own pieces, so that a thread waits only for
// itself; the copies run ahead into the group's next row, which covers the end of a row (sums joined, alternatives found).
// Scores before the first 16-byte boundary and behind the last come one by one.
// Alternatives: every thread knows the maximum of the scores that it has seen. With V the top_k-th largest of these maxima, only
// the threads whose maximum reaches V can hold one of the top_k best scores: about top_k of them, so the group reads only
// those threads' share of the row again (from L2, 1 / 12 of it for 20 alternatives and 256 threads), lists the scores that
// reach V and ranks that short list by counting. Nothing is done for the alternatives during the walk itself.
constexpr int kUnroll = 4, kWalkRing = 3, kWalkBytes = kWalkRing * kUnroll * 256 * 16;
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

template <int GROUP>
struct RowShared {
  static constexpr int kFlagged = 64, kCandidates = GROUP == 32 ? 128 : 512;
  Entry list[kMaxTopClasses], cand[kCandidates];
  unsigned int key[GROUP];
  float part_m[GROUP / 32], part_s[GROUP / 32], part_t[GROUP / 32];
  int flagged[kFlagged];
  int num_flagged, num_cand, last, have; unsigned int limit;
};

template <int GROUP> __device__ __forceinline__ void GroupSync() { if constexpr (GROUP == 32) __syncwarp(); else __syncthreads(); }

// The `rank`-th largest (1-based) of GROUP numbers of `bits` bits, GROUP / 32 per lane: bit by bit, the largest value that at least
// `rank` numbers reach (0: there are fewer). Run by one warp.
template <int PER>
__device__ __forceinline__ unsigned int KthLargest(const unsigned int (&mine)[PER], int rank, int bits) {
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

// A group's share of a row.
template <typename T>
struct RowShare {
  const T* s; const uint4* body; int K, head, tail, v_begin, v_end; bool first, last_part;
  __device__ __forceinline__ RowShare(const ClassScoresArgs& a, long long row, int part, int parts, int group) {
    constexpr int N = Pack<T>::N;
    s = static_cast<const T*>(a.scores) + row * a.row_stride; K = static_cast<int>(a.classes);
    head = min(K, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(s) & 15)) & 15) / static_cast<int>(sizeof(T)));
    const int vectors = (K - head) / N;
    tail = head + vectors * N; body = reinterpret_cast<const uint4*>(s + head);
    const int each = ((vectors + parts - 1) / parts + group - 1) / group * group;      // whole rounds of the group
    v_begin = min(vectors, part * each); v_end = min(vectors, v_begin + each);
    first = part == 0; last_part = part == parts - 1;
  }
};

template <int GROUP, typename T>
struct Alternatives {
  static constexpr int N = Pack<T>::N;
  RowShared<GROUP>& sh; const RowShare<T>& r; int top_k, tid;
  // f(score, class) for the scores of the flagged threads and the ends of the row, dealt out over the group
  template <typename F>
  __device__ __forceinline__ void Scores(int num_flagged, float head_v, float tail_v, F&& f) const {
    if (r.first && tid < r.head) f(head_v, tid);
    if (r.last_part && tid < r.K - r.tail) f(tail_v, r.tail + tid);
    const int rounds = (r.v_end - r.v_begin + GROUP - 1) / GROUP;
    for (int e = tid; e < num_flagged * rounds; e += GROUP) {
      const int i = r.v_begin + (e / num_flagged) * GROUP + sh.flagged[e % num_flagged];
      if (i >= r.v_end) continue;
      const uint4 q = __ldg(r.body + i);
      float v[N];
      Unpack(q, v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int k = 0; k < N; ++k) f(v[k], r.head + i * N + k);
    }
  }
  // Ranks the first `count` candidates into the list; returns how many that leaves.
  __device__ __forceinline__ int Rank(int count) {
    for (int i = tid; i < count; i += GROUP) {
      const Entry e = sh.cand[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += Before(sh.cand[j], e) ? 1 : 0;
      if (rank < top_k) sh.list[rank] = e;
    }
    GroupSync<GROUP>();
    return min(count, top_k);
  }
  // most: this thread's maximum. All threads; the list is complete on return.
  __device__ __forceinline__ int Find(float most, float head_v, float tail_v) {
    constexpr int PER = GROUP / 32;
    sh.key[tid] = OrderKey<T>(most);
    GroupSync<GROUP>();
    if (tid < 32) {
      unsigned int mine[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) mine[i] = sh.key[tid + 32 * i];
      unsigned int limit;
      if (top_k == 1) {
        unsigned int best = mine[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) best = max(best, mine[i]);
        limit = __reduce_max_sync(0xffffffffu, best);
      } else {
        limit = KthLargest<PER>(mine, top_k, KeyBits<T>::kBits);
      }
      limit = max(1u, limit);      // key 0: a thread without a score
      int n = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const unsigned int in = __ballot_sync(0xffffffffu, mine[i] >= limit);
        const int at = n + __popc(in & ((1u << tid) - 1u));
        if (mine[i] >= limit && at < RowShared<GROUP>::kFlagged) sh.flagged[at] = tid + 32 * i;
        n += __popc(in);
      }
      if (tid == 0) { sh.limit = limit; sh.num_flagged = n; sh.num_cand = 0; sh.last = 0x7fffffff; }
    }
    GroupSync<GROUP>();
    const unsigned int limit = sh.limit;
    if (GROUP > 32 && sh.num_flagged > RowShared<GROUP>::kFlagged) Ties(limit);
    const int last = sh.last, num_flagged = sh.num_flagged;
    Scores(num_flagged, head_v, tail_v, [&](float v, int cls) {
      const unsigned int k = OrderKey<T>(v);
      if (k > limit || (k == limit && cls <= last)) { const int at = atomicAdd(&sh.num_cand, 1); if (at < RowShared<GROUP>::kCandidates) { sh.cand[at].v = v; sh.cand[at].cls = cls; } }
    });
    GroupSync<GROUP>();
    const int count = sh.num_cand;
    if (count <= RowShared<GROUP>::kCandidates) return Rank(count);
    return OneByOne(num_flagged, head_v, tail_v);
  }
  // Very many equal maxima: of the threads with maximum `limit` only those count that reach it at the lowest classes.
  __device__ void Ties(unsigned int limit) {
    constexpr int PER = GROUP / 32;
    unsigned int order = 0u;
    const unsigned int mine = sh.key[tid];
    if (mine == limit) {
      int at = 0x7fffffff;
      if (r.first && tid < r.head && OrderKey<T>(ToFloat(r.s[tid])) == limit) at = tid;
      for (int i = r.v_begin + tid; i < r.v_end && at == 0x7fffffff; i += GROUP) {
        float v[N];
        Unpack(__ldg(r.body + i), v, static_cast<const T*>(nullptr));
#pragma unroll
        for (int k = N - 1; k >= 0; --k) if (OrderKey<T>(v[k]) == limit) at = r.head + i * N + k;
      }
      if (at == 0x7fffffff) at = r.tail + tid;      // its last score
      order = 0x80000000u - static_cast<unsigned int>(at);
    }
    const int higher = __syncthreads_count(mine > limit);
    sh.key[tid] = order;
    const bool above = mine > limit;
    if (tid == 0) sh.num_flagged = 0;
    __syncthreads();
    if (tid < 32) {
      unsigned int all[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) all[i] = sh.key[tid + 32 * i];
      const unsigned int kth = KthLargest<PER>(all, top_k - higher, 32);
      if (tid == 0) sh.last = static_cast<int>(0x80000000u - kth);
    }
    __syncthreads();
    if (above || (mine == limit && order >= 0x80000000u - static_cast<unsigned int>(sh.last))) sh.flagged[atomicAdd(&sh.num_flagged, 1)] = tid;
    __syncthreads();
  }
  // More candidates than the list holds (few threads own very many of the best scores): one alternative per pass.
  __device__ int OneByOne(int num_flagged, float head_v, float tail_v) {
    Entry before; before.v = INFINITY; before.cls = -1;
    int t = 0;
    for (; t < top_k; ++t) {
      Entry best; best.v = -INFINITY; best.cls = 0x7fffffff;
      Scores(num_flagged, head_v, tail_v, [&](float v, int cls) { Entry e; e.v = v; e.cls = cls; if (v > -INFINITY && Before(before, e) && Before(e, best)) best = e; });
      for (int o = 16; o > 0; o >>= 1) {
        Entry e; e.v = __shfl_xor_sync(0xffffffffu, best.v, o); e.cls = __shfl_xor_sync(0xffffffffu, best.cls, o);
        if (Before(e, best)) best = e;
      }
      if constexpr (GROUP > 32) {
        if ((tid & 31) == 0) sh.cand[tid >> 5] = best;
        __syncthreads();
        best = sh.cand[0];
        for (int w = 1; w < GROUP / 32; ++w) if (Before(sh.cand[w], best)) best = sh.cand[w];
        __syncthreads();
      }
      if (best.cls == 0x7fffffff) break;
      if (tid == 0) sh.list[t] = best;
      before = best;
    }
    GroupSync<GROUP>();
    return t;
  }
};

// TOP: alternatives are wanted. Groups walk the rows with the grid's stride; a row belongs to a warp, a block or a cluster.
template <typename T, int GROUP, bool TOP>
__global__ void __launch_bounds__(256, 4) ClassLogProbsRowKernel(ClassScoresArgs a) {
  constexpr int kGroups = 256 / GROUP;
  __shared__ RowShared<GROUP> s_all[TOP ? kGroups : 1];
  __shared__ float s_m[8], s_s[8], s_t[8];
  RowShared<GROUP>& sh = s_all[TOP && GROUP == 32 ? threadIdx.x / 32 : 0];
  const int tid = threadIdx.x % GROUP;
  const T* type = nullptr;
  const int parts = GROUP == 32 ? 1 : static_cast<int>(cg::this_cluster().num_blocks()), part = GROUP == 32 ? 0 : static_cast<int>(cg::this_cluster().block_rank());
  const long long stride = GROUP == 32 ? static_cast<long long>(gridDim.x) * kGroups : gridDim.x / parts;
  long long row = GROUP == 32 ? static_cast<long long>(blockIdx.x) * kGroups + threadIdx.x / 32 : blockIdx.x / parts;
  if (row >= a.rows) return;                     // whole groups
  extern __shared__ __align__(16) uint4 s_ring[];      // [kWalkRing][kUnroll][256]
  uint4* mine = s_ring + threadIdx.x;
  RowShare<T> r(a, row, part, parts, GROUP);
  // what is copied next
  long long ahead_row = row;
  const uint4* ahead_body = r.body; int ahead_at = r.v_begin, ahead_end = r.v_end, ahead_slot = 0;
  auto copy_ahead = [&]() {
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
    ahead_slot = ahead_slot == kWalkRing - 1 ? 0 : ahead_slot + 1;
  };
#pragma unroll
  for (int i = 0; i < kWalkRing - 1; ++i) copy_ahead();
  int slot = 0;
  long long y = LabelOf(a, row);
  for (;;) {
    const long long next_row = row + stride;
    const bool more = next_row < a.rows;
    const float head_v = r.first && tid < r.head ? ToFloat(r.s[tid]) : -INFINITY, tail_v = r.last_part && tid < r.K - r.tail ? ToFloat(r.s[r.tail + tid]) : -INFINITY;
    const float given = tid == 0 && y >= 0 && y < r.K ? ToFloat(r.s[y]) : 0.f;
    const long long y_next = more ? LabelOf(a, next_row) : -1;
    PairSums<T> pairs;
    int at = r.v_begin;
    do {                                         // a share without pieces takes one empty step
      copy_ahead();
      asm volatile("cp.async.wait_group %0;" ::"n"(kWalkRing - 1) : "memory");
      uint4 q[kUnroll];
      if (at + GROUP * kUnroll <= r.v_end) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) q[u] = mine[slot * (kUnroll * 256) + u * 256];
        const float most = MaxOf(q, type);
        if (most > pairs.m) pairs.Raise(most);
        pairs.Add16(q);
      } else {                                   // the last chunk, piece by piece
#pragma unroll 1
        for (int u = 0; u < kUnroll && (u == 0 || at + u * GROUP + (tid & ~31) < r.v_end); ++u) {
          const uint4 one[1] = {at + u * GROUP + tid < r.v_end ? mine[slot * (kUnroll * 256) + u * 256] : AllRuledOut(type)};
          const float most = MaxOf(one, type);
          if (most > pairs.m) pairs.Raise(most);
          pairs.Add16(one);
        }
      }
      at += GROUP * kUnroll;
      slot = slot == kWalkRing - 1 ? 0 : slot + 1;
    } while (at < r.v_end);
    Sums sums = pairs.Total();
    if (head_v != -INFINITY) sums.AddOne(head_v);
    if (tail_v != -INFINITY) sums.AddOne(tail_v);
    const float most = sums.m;
    sums.JoinLanes();
    if constexpr (GROUP == 32) {
      const RowResult res(sums);
      if (tid == 0) res.Store(a, row, y, given);
      if constexpr (TOP) {
        Alternatives<GROUP, T> alt{sh, r, a.top_k, tid};
        const int have = alt.Find(most, head_v, tail_v);
        if (tid < a.top_k) { const Entry e = sh.list[tid]; res.StoreTop(a, row * a.top_k + tid, tid < have ? e.v : -INFINITY, e.cls); }
        __syncwarp();
      }
    } else {
      if ((tid & 31) == 0) { s_m[tid >> 5] = sums.m; s_s[tid >> 5] = sums.s; s_t[tid >> 5] = sums.t; }
      int have = 0;
      if constexpr (TOP) { Alternatives<GROUP, T> alt{sh, r, a.top_k, tid}; have = alt.Find(most, head_v, tail_v); } else __syncthreads();
      if (tid < 32) {
        sums = Sums();
        if (tid < GROUP / 32) { sums.m = s_m[tid]; sums.s = s_s[tid]; sums.t = s_t[tid]; }
        sums.JoinLanes();
      }
      if (parts > 1) {
        // the cluster's first block joins the others' sums and lists, read from their shared memory
        __syncthreads();
        if (tid == 0) { s_m[0] = sums.m; s_s[0] = sums.s; s_t[0] = sums.t; if constexpr (TOP) sh.have = have; }
        cg::this_cluster().sync();
        if (part == 0) {
          int count = have;
          if constexpr (TOP) { if (tid < have) sh.cand[tid] = sh.list[tid]; if (tid == 0) { sh.flagged[0] = 0; sh.flagged[1] = have; } }
          for (int p = 1; p < parts; ++p) {
            if (tid < 32) sums.Join(*cg::this_cluster().map_shared_rank(&s_m[0], p), *cg::this_cluster().map_shared_rank(&s_s[0], p), *cg::this_cluster().map_shared_rank(&s_t[0], p));
            if constexpr (TOP) {
              const RowShared<GROUP>* o = cg::this_cluster().map_shared_rank(&sh, p);
              const int n = o->have;
              if (tid < n) sh.cand[count + tid] = o->list[tid];
              count += n;
              if (tid == 0) sh.flagged[p + 1] = count;
            }
          }
          if constexpr (TOP) {
            // the lists are sorted: an entry's rank is its place in its own list and, by bisection, how many of each other come before it
            __syncthreads();
            if (tid < count) {
              const Entry e = sh.cand[tid];
              int rank = 0;
              for (int p = 0; p < parts; ++p) {
                const int begin = sh.flagged[p];
                int lo = begin, hi = sh.flagged[p + 1];
                while (lo < hi) { const int mid = (lo + hi) >> 1; if (Before(sh.cand[mid], e)) lo = mid + 1; else hi = mid; }
                rank += lo - begin;
              }
              if (rank < a.top_k) sh.list[rank] = e;
            }
            __syncthreads();
            have = min(count, a.top_k);
          }
        }
        cg::this_cluster().sync();         // no block goes on while its shared memory is read
      }
      if (part == 0 && tid < 32) {
        const RowResult res(sums);
        if (tid == 0) res.Store(a, row, y, given);
        if constexpr (TOP) if (tid < a.top_k) { const Entry e = sh.list[tid]; res.StoreTop(a, row * a.top_k + tid, tid < have ? e.v : -INFINITY, e.cls); }
      }
      __syncthreads();                     // the next row writes the shared parts again
    }
    if (!more) return;
    row = next_row; r = RowShare<T>(a, row, part, parts, GROUP); y = y_next;
  }
}

// ----------------------------------------------------------------------------------------- contiguous columns ----
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
  // log sum e^(s - m), with what B lacks of m log2 e
  __device__ __forceinline__ static float AgainLog(const Sums& r) { return (log2f(r.s) + (Huge(r.m) ? 0.f : fmaf(-r.m, kLog2E, __fmul_rn(r.m, kLog2E)))) * kLn2; }
  // one thread walks the row
  template <typename T>
  __device__ __forceinline__ void TakeAgain(const ClassScoresArgs& s, const T* row) {
    Sums r;
    for (long long j = 0; j < s.classes; ++j) r.AddOne(ToFloat(row[j * s.class_stride]));
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

template <typename T, int GROUP, bool TOP>
void LaunchRows(const ClassScoresArgs& a, int cluster, cudaStream_t s) {
  // as many groups as are resident at once, each with several rows
  static PerDevice allowed;
  AllowSharedMemory(ClassLogProbsRowKernel<T, GROUP, TOP>, kWalkBytes, &allowed);
  const long long groups = GROUP == 32 ? (a.rows + 7) / 8 : a.rows, most = static_cast<long long>(kSms) * 4 * (GROUP == 32 ? 2 : 1) / cluster;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned int>(std::min(groups, most) * cluster)); cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = kWalkBytes; cfg.stream = s; cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 1 : 0;
  FB_CUDA(cudaLaunchKernelEx(&cfg, ClassLogProbsRowKernel<T, GROUP, TOP>, a));
}
template <typename T, int GROUP>
void LaunchRows(const ClassScoresArgs& a, int cluster, cudaStream_t s) {
  if (a.top_k > 0) LaunchRows<T, GROUP, true>(a, cluster, s); else LaunchRows<T, GROUP, false>(a, cluster, s);
}

}  // namespace

void LaunchClassLogProbs(const ClassScoresArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return;
  DispatchType(a.dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    if (a.classes <= kFewClasses) {
      LaunchFew<T>(a, s);
    } else if (a.class_stride == 1) {
      // A warp per row as long as that fills the machine and a warp's walk stays short; else a block, and a cluster of blocks while
      // there are fewer blocks than two per SM and every block has a full chunk.
      const long long chunk = 256LL * kUnroll * Pack<T>::N;
      if (a.classes <= chunk / 8 || (a.classes <= chunk && a.rows >= kSms * 16)) { LaunchRows<T, 32>(a, 1, s); }
      else {
        int cluster = 1;
        while (cluster < 8 && a.rows * cluster < 2 * kSms && a.classes >= 2 * cluster * chunk / kUnroll) cluster *= 2;
        LaunchRows<T, 256>(a, cluster, s);
      }
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
