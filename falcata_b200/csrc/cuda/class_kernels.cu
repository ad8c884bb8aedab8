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
#include "kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace fb {

namespace {

constexpr float kLog2E = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kThreads = 256;
constexpr float kTrustedLogNorm = 64.f;

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float NanF() { return __int_as_float(0x7fc00000); }
__device__ __forceinline__ float MaxNan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

__device__ __forceinline__ long long LabelOf(const ClassScoresArgs& a, long long row) {
  if (a.label_bits == 0) return -1;
  return a.label_bits == 32 ? static_cast<const int*>(a.labels)[row] : static_cast<const long long*>(a.labels)[row];
}

// log p of a class with score s, given the row's maximum and log S
__device__ __forceinline__ float LogProb(float s, float m, float log_sum) { return (s - m) - log_sum; }

// A row with a NaN / +inf (m NaN or +inf) or without any class (m -inf): the values its definition gives.
__device__ __forceinline__ bool Degenerate(float m) { return !(fabsf(m) < __int_as_float(0x7f800000)); }

// One block per row, any strides: maximum, sums, then one pass per alternative.
template <typename T>
__global__ void __launch_bounds__(kThreads) ClassLogProbsKernel(ClassScoresArgs a) {
  __shared__ float s_f[kThreads]; __shared__ float s_g[kThreads]; __shared__ int s_i[kThreads];
  const long long row = blockIdx.x;
  const T* s = static_cast<const T*>(a.scores) + row * a.row_stride;
  const int K = static_cast<int>(a.classes);
  float m = -INFINITY;
  for (int j = threadIdx.x; j < K; j += kThreads) m = MaxNan(m, ToFloat(s[j * a.class_stride]));
  s_f[threadIdx.x] = m; __syncthreads();
  for (int o = kThreads / 2; o > 0; o >>= 1) { if (threadIdx.x < o) s_f[threadIdx.x] = MaxNan(s_f[threadIdx.x], s_f[threadIdx.x + o]); __syncthreads(); }
  m = s_f[0]; __syncthreads();
  const bool bad = Degenerate(m), none = m == -INFINITY;
  float sum = 0.f, tsum = 0.f;
  if (!bad)
    for (int j = threadIdx.x; j < K; j += kThreads) { const float x = fmaxf(ToFloat(s[j * a.class_stride]) - m, -200.f), e = expf(x); sum += e; tsum = fmaf(e, x, tsum); }
  s_f[threadIdx.x] = sum; s_g[threadIdx.x] = tsum; __syncthreads();
  for (int o = kThreads / 2; o > 0; o >>= 1) { if (threadIdx.x < o) { s_f[threadIdx.x] += s_f[threadIdx.x + o]; s_g[threadIdx.x] += s_g[threadIdx.x + o]; } __syncthreads(); }
  sum = s_f[0]; tsum = s_g[0]; __syncthreads();
  const float log_sum = logf(sum);
  if (threadIdx.x == 0) {
    const long long y = LabelOf(a, row);
    a.log_norm[row] = none ? -INFINITY : bad ? NanF() : m + log_sum;
    a.entropy[row] = none ? 0.f : bad ? NanF() : log_sum - tsum / sum;
    if (a.log_prob != nullptr) a.log_prob[row] = y < 0 ? 0.f : y >= K ? NanF() : none ? -INFINITY : bad ? NanF() : LogProb(ToFloat(s[y * a.class_stride]), m, log_sum);
  }
  float before = INFINITY; int before_class = -1;   // the alternative found last
  for (int t = 0; t < a.top_k; ++t) {
    float best = -INFINITY; int cls = K;
    if (!bad)
      for (int j = threadIdx.x; j < K; j += kThreads) {
        const float v = ToFloat(s[j * a.class_stride]);
        if ((v < before || (v == before && j > before_class)) && v > best) { best = v; cls = j; }
      }
    s_f[threadIdx.x] = best; s_i[threadIdx.x] = cls; __syncthreads();
    for (int o = kThreads / 2; o > 0; o >>= 1) {
      if (threadIdx.x < o) {
        const float v = s_f[threadIdx.x + o]; const int c = s_i[threadIdx.x + o];
        if (v > s_f[threadIdx.x] || (v == s_f[threadIdx.x] && c < s_i[threadIdx.x])) { s_f[threadIdx.x] = v; s_i[threadIdx.x] = c; }
      }
      __syncthreads();
    }
    before = s_f[0]; before_class = s_i[0]; __syncthreads();
    if (threadIdx.x == 0) {
      a.top_log_prob[row * a.top_k + t] = before == -INFINITY ? (bad && !none ? NanF() : -INFINITY) : LogProb(before, m, log_sum);
      a.top_class[row * a.top_k + t] = before == -INFINITY ? -1 : before_class;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) ClassLogProbsGradKernel(ClassScoresArgs a, ClassGradArgs g) {
  const long long row = blockIdx.x;
  const T* s = static_cast<const T*>(a.scores) + row * a.row_stride;
  T* out = static_cast<T*>(g.grad) + row * g.grad_row_stride;
  const long long K = a.classes, y = LabelOf(a, row);
  const float log_norm = a.log_norm[row];
  const bool none = log_norm == -INFINITY, bad = (!none && Degenerate(log_norm)) || y >= K;
  const float gh = g.g_entropy ? g.g_entropy[row] : 0.f, glp = (g.g_log_prob && y >= 0) ? g.g_log_prob[row] : 0.f;
  // log_norm in fp32 gives p to a relative 2^-24 |log_norm|: beyond kTrustedLogNorm the row's maximum and sum are taken again
  float m = log_norm, log_sum = 0.f;
  if (!none && !bad && fabsf(log_norm) > kTrustedLogNorm) {
    __shared__ float s_f[kThreads];
    float t = -INFINITY;
    for (long long j = threadIdx.x; j < K; j += kThreads) t = fmaxf(t, ToFloat(s[j * a.class_stride]));
    s_f[threadIdx.x] = t; __syncthreads();
    for (int o = kThreads / 2; o > 0; o >>= 1) { if (threadIdx.x < o) s_f[threadIdx.x] = fmaxf(s_f[threadIdx.x], s_f[threadIdx.x + o]); __syncthreads(); }
    m = s_f[0]; __syncthreads();
    t = 0.f;
    for (long long j = threadIdx.x; j < K; j += kThreads) t += expf(ToFloat(s[j * a.class_stride]) - m);
    s_f[threadIdx.x] = t; __syncthreads();
    for (int o = kThreads / 2; o > 0; o >>= 1) { if (threadIdx.x < o) s_f[threadIdx.x] += s_f[threadIdx.x + o]; __syncthreads(); }
    log_sum = logf(s_f[0]);
  }
  float ca = (g.g_log_norm ? g.g_log_norm[row] : 0.f) - glp - gh * a.entropy[row];
  for (int t = 0; t < a.top_k; ++t) { const int c = a.top_class[row * a.top_k + t]; if (c >= 0 && c < K) ca -= g.g_top[row * a.top_k + t]; }
  for (long long j = threadIdx.x; j < K; j += kThreads) {
    const float lp = fmaxf(LogProb(ToFloat(s[j * a.class_stride]), m, log_sum), -200.f);
    float v = expf(lp) * (ca - gh * lp);
    if (j == y) v += glp;
    for (int t = 0; t < a.top_k; ++t) if (a.top_class[row * a.top_k + t] == j) v += g.g_top[row * a.top_k + t];
    out[j * g.grad_class_stride] = FromFloat<T>(none ? 0.f : bad ? NanF() : v);
  }
}

template <typename F> void DispatchType(int dtype, F&& f) {
  switch (dtype) {
    case kOpFloat32: f(static_cast<float*>(nullptr)); return;
    case kOpFloat16: f(static_cast<__half*>(nullptr)); return;
    case kOpBFloat16: f(static_cast<__nv_bfloat16*>(nullptr)); return;
    default: Log::Fatal("class scores: unknown type code %d", dtype);
  }
}

}  // namespace

void LaunchClassLogProbs(const ClassScoresArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return;
  DispatchType(a.dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    ClassLogProbsKernel<T><<<static_cast<unsigned int>(a.rows), kThreads, 0, s>>>(a);
  });
  FB_LAUNCHED(); FB_KERNEL_CHECK();
}

void LaunchClassLogProbsGrad(const ClassScoresArgs& a, const ClassGradArgs& g, cudaStream_t s) {
  if (a.rows <= 0) return;
  DispatchType(a.dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    ClassLogProbsGradKernel<T><<<static_cast<unsigned int>(a.rows), kThreads, 0, s>>>(a, g);
  });
  FB_LAUNCHED(); FB_KERNEL_CHECK();
}

}  // namespace fb
