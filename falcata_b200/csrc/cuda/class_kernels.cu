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
constexpr float kLowestExponent = -200.f;     // e^x is 0 in fp32 from here on; keeps 0 * (-inf) out of T

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

// The running sums of a part of a row, relative to its maximum m (-inf: nothing yet; a NaN or +inf among the scores makes s NaN).
struct Sums {
  float m = -INFINITY, s = 0.f, t = 0.f;
  __device__ __forceinline__ void Raise(float to) {     // to > m
    const float d = fmaxf(m - to, kLowestExponent), f = __expf(d);
    t = (t + s * d) * f; s *= f; m = to;
  }
  __device__ __forceinline__ float Base() const { return m == -INFINITY ? 0.f : m; }
  __device__ __forceinline__ void Add(float v, float base) { const float x = MaxNan(v - base, kLowestExponent), e = __expf(x); s += e; t = fmaf(e, x, t); }
  __device__ __forceinline__ void AddOne(float v) { if (v > m) Raise(v); Add(v, Base()); }
  __device__ __forceinline__ void Join(float m2, float s2, float t2) {
    if (m2 > m) { Sums o; o.m = m2; o.s = s2; o.t = t2; const float m1 = m, s1 = s, t1 = t; *this = o; m2 = m1; s2 = s1; t2 = t1; }
    const float d = m2 == -INFINITY ? kLowestExponent : fmaxf(m2 - m, kLowestExponent), f = __expf(d);
    t += (t2 + s2 * d) * f; s += s2 * f;
  }
  __device__ __forceinline__ void JoinLanes() {
    for (int o = 16; o > 0; o >>= 1) Join(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o), __shfl_xor_sync(0xffffffffu, t, o));
  }
};

// The results of a row from its sums.
struct RowResult {
  float m, log_sum, entropy; bool none, bad;
  __device__ explicit RowResult(const Sums& r) {
    none = r.m == -INFINITY && !(r.s != r.s); bad = !none && !(fabsf(r.m) < InfF() && r.s < InfF());   // a NaN sum fails the comparison
    m = r.m; log_sum = logf(r.s); entropy = none ? 0.f : bad ? NanF() : log_sum - r.t / r.s;
  }
  __device__ __forceinline__ float LogProb(float v) const { return none ? -INFINITY : bad ? NanF() : (v - m) - log_sum; }
  __device__ __forceinline__ float LogNorm() const { return none ? -INFINITY : bad ? NanF() : m + log_sum; }
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
// A thread per row, the row's scores in MOST registers. Class-major scores are read straight into them, 32 rows per instruction;
// rows go through shared memory (an odd row pitch there, so that neither side meets bank conflicts).
constexpr int kFewThreads = 128, kFewClasses = 64;
template <typename T, int MOST, bool BY_CLASS>
__global__ void __launch_bounds__(kFewThreads) ClassLogProbsFewKernel(ClassScoresArgs a) {
  __shared__ float s_rows[BY_CLASS ? 1 : kFewThreads * (MOST + 1)];
  const int K = static_cast<int>(a.classes);
  const long long row0 = static_cast<long long>(blockIdx.x) * kFewThreads, row = row0 + threadIdx.x;
  const T* base = static_cast<const T*>(a.scores);
  float v[MOST];
  if constexpr (BY_CLASS) {
    if (row >= a.rows) return;
#pragma unroll
    for (int j = 0; j < MOST; ++j) v[j] = j < K ? ToFloat(base[row * a.row_stride + j * a.class_stride]) : -INFINITY;
  } else {
    const int rows = static_cast<int>(min(static_cast<long long>(kFewThreads), a.rows - row0)), pitch = K | 1;
    for (int e = threadIdx.x, r = e / K, j = e - r * K; e < rows * K; e += kFewThreads) {
      s_rows[r * pitch + j] = ToFloat(base[(row0 + r) * a.row_stride + j * a.class_stride]);
      j += kFewThreads % K; r += kFewThreads / K;
      if (j >= K) { j -= K; ++r; }
    }
    __syncthreads();
    if (row >= a.rows) return;
#pragma unroll
    for (int j = 0; j < MOST; ++j) v[j] = j < K ? s_rows[threadIdx.x * pitch + j] : -INFINITY;
  }
  Sums sums;
  float m = v[0];
#pragma unroll
  for (int j = 1; j < MOST; ++j) m = MaxNan(m, v[j]);
  sums.m = m;
  const float b = sums.Base();
#pragma unroll
  for (int j = 0; j < MOST; ++j) sums.Add(v[j], b);
  const RowResult res(sums);
  const long long y = LabelOf(a, row);
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

// -------------------------------------------------------------------------------------------- contiguous rows ----
// GROUP threads (a warp or a block) walk a row, or a block cluster's share of one, in chunks of kUnroll 16-byte loads per thread;
// the next chunk's loads are in flight while one is worked on. Scores before the first 16-byte boundary and behind the last come
// one by one.
// Alternatives: the group keeps the list of the best so far and its last score as a threshold. A chunk in which some thread's
// maximum passes it is looked at again (it is still in registers): the threads that matter are those with one of the top_k
// largest maxima - no other can hold one of the best - so at most top_k threads add their scores above the threshold to the
// list, which is then ranked by counting. Work and space are bounded whatever the order of the scores; in random order a
// chunk adds top_k / (chunks so far) entries.
constexpr int kUnroll = 4;
struct Entry { float v; int cls; };
__device__ __forceinline__ bool Before(const Entry& a, const Entry& b) { return a.v > b.v || (a.v == b.v && a.cls < b.cls); }
// unsigned order of floats; zeros of both signs alike
__device__ __forceinline__ unsigned int OrderKey(float v) { const unsigned int u = __float_as_uint(v + 0.f); return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u; }
__device__ __forceinline__ float KeyValue(unsigned int k) { return __uint_as_float((k & 0x80000000u) != 0 ? k & 0x7fffffffu : ~k); }

template <int GROUP>
struct RowShared {
  Entry list[2][kMaxTopClasses];      // the best so far (in the buffer that is `live`)
  unsigned int key[GROUP]; int first[GROUP];
  float part_m[GROUP / 32], part_s[GROUP / 32], part_t[GROUP / 32];
  int cand_count; unsigned int limit_key; int limit_first, pad;
  Entry cand[1];                      // top_k threads' scores and the list
};
template <int GROUP, typename T>
constexpr int RowSharedBytes(int top_k) { return static_cast<int>(sizeof(RowShared<GROUP>)) + top_k * (kUnroll * Pack<T>::N + 1) * static_cast<int>(sizeof(Entry)); }

template <int GROUP> __device__ __forceinline__ void GroupSync() { if constexpr (GROUP == 32) __syncwarp(); else __syncthreads(); }
template <int GROUP> __device__ __forceinline__ int GroupCount(bool p) { if constexpr (GROUP == 32) return __popc(__ballot_sync(0xffffffffu, p)); else return __syncthreads_count(p); }

// The `rank`-th largest (1-based) of the group's keys: bit by bit, the largest value that at least `rank` keys reach. Run by one warp.
template <int GROUP>
__device__ __forceinline__ unsigned int KthKey(const unsigned int* key, int rank, int lane) {
  unsigned int mine[GROUP / 32];
#pragma unroll
  for (int i = 0; i < GROUP / 32; ++i) mine[i] = key[lane + 32 * i];
  unsigned int found = 0u;
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned int probe = found | (1u << bit);
    int c = 0;
#pragma unroll
    for (int i = 0; i < GROUP / 32; ++i) c += mine[i] >= probe ? 1 : 0;
    if (static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned int>(c))) >= rank) found = probe;
  }
  return found;
}

template <int GROUP>
struct TopList {
  RowShared<GROUP>* sh; int top_k, live, have; float threshold;
  __device__ __forceinline__ TopList(RowShared<GROUP>* shared, int k) : sh(shared), top_k(k), live(0), have(0), threshold(-INFINITY) {}
  // Every thread of the group calls it with the maximum of its scores of the chunk; each(f) calls f(score, class) for all of them,
  // by rising class.
  template <typename E>
  __device__ __forceinline__ void Chunk(float most, int tid, E&& each) {
    float limit = threshold;                    // only scores above it matter
    bool in = most > threshold;                 // later classes lose against equal earlier ones
    const int above = GroupCount<GROUP>(in);
    if (above == 0) return;
    if (tid == 0) sh->cand_count = have;
    for (int i = tid; i < have; i += GROUP) sh->cand[i] = sh->list[live][i];
    if (above > top_k) {
      int first = 0x7fffffff;
      if (in) each([&](float v, int cls) { if (v == most) first = min(first, cls); });
      sh->key[tid] = in ? OrderKey(most) : 0u; sh->first[tid] = first;
      GroupSync<GROUP>();
      if (tid < 32) {
        const unsigned int kth = KthKey<GROUP>(sh->key, top_k, tid);
        int higher = 0, equal = 0;
#pragma unroll
        for (int i = 0; i < GROUP / 32; ++i) { const unsigned int k = sh->key[tid + 32 * i]; higher += k > kth ? 1 : 0; equal += k == kth ? 1 : 0; }
        higher = __reduce_add_sync(0xffffffffu, static_cast<unsigned int>(higher)); equal = __reduce_add_sync(0xffffffffu, static_cast<unsigned int>(equal));
        int last = 0x7fffffff;
        if (higher + equal > top_k) {           // equal maxima: those of the lowest classes
          unsigned int order[GROUP / 32];
#pragma unroll
          for (int i = 0; i < GROUP / 32; ++i) order[i] = sh->key[tid + 32 * i] == kth ? ~static_cast<unsigned int>(sh->first[tid + 32 * i]) : 0u;
          unsigned int found = 0u;
          for (int bit = 31; bit >= 0; --bit) {
            const unsigned int probe = found | (1u << bit);
            int c = 0;
#pragma unroll
            for (int i = 0; i < GROUP / 32; ++i) c += order[i] >= probe ? 1 : 0;
            if (static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned int>(c))) >= top_k - higher) found = probe;
          }
          last = static_cast<int>(~found);
        }
        if (tid == 0) { sh->limit_key = kth; sh->limit_first = last; }
      }
      GroupSync<GROUP>();
      const unsigned int mine = OrderKey(most);
      in = in && (mine > sh->limit_key || (mine == sh->limit_key && first <= sh->limit_first));
      limit = nextafterf(KeyValue(sh->limit_key), -INFINITY);
    } else {
      GroupSync<GROUP>();
    }
    if (in) each([&](float v, int cls) { if (v > limit) { const int at = atomicAdd(&sh->cand_count, 1); sh->cand[at].v = v; sh->cand[at].cls = cls; } });
    GroupSync<GROUP>();
    const int count = sh->cand_count;
    for (int i = tid; i < count; i += GROUP) {
      const Entry e = sh->cand[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += Before(sh->cand[j], e) ? 1 : 0;
      if (rank < top_k) sh->list[live ^ 1][rank] = e;
    }
    GroupSync<GROUP>();
    live ^= 1; have = min(count, top_k);
    if (have == top_k) threshold = sh->list[live][top_k - 1].v;
  }
};

// TOP: alternatives are wanted. A warp per row: 8 rows per block. A block per row: gridDim.x = rows * cluster size.
template <typename T, int GROUP, bool TOP>
__global__ void __launch_bounds__(256, 3) ClassLogProbsRowKernel(ClassScoresArgs a) {
  constexpr int N = Pack<T>::N;
  extern __shared__ __align__(16) unsigned char s_rows_raw[];
  RowShared<GROUP>& sh = *reinterpret_cast<RowShared<GROUP>*>(s_rows_raw + (GROUP == 32 ? threadIdx.x / 32 * RowSharedBytes<GROUP, T>(a.top_k) : 0));
  const int tid = threadIdx.x % GROUP;
  const int parts = GROUP == 32 ? 1 : static_cast<int>(cg::this_cluster().num_blocks()), part = GROUP == 32 ? 0 : static_cast<int>(cg::this_cluster().block_rank());
  const long long row = GROUP == 32 ? static_cast<long long>(blockIdx.x) * (256 / GROUP) + threadIdx.x / 32 : blockIdx.x / parts;
  if (GROUP == 32 && row >= a.rows) return;                     // whole warps
  const T* s = static_cast<const T*>(a.scores) + row * a.row_stride;
  const T* type = nullptr;
  const int K = static_cast<int>(a.classes);
  const int head = min(K, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(s) & 15)) & 15) / static_cast<int>(sizeof(T)));
  const int vectors = (K - head) / N, tail = head + vectors * N;
  const int each = ((vectors + parts - 1) / parts + GROUP - 1) / GROUP * GROUP;      // whole rounds of the group
  const int v_begin = min(vectors, part * each), v_end = min(vectors, v_begin + each);
  const uint4* body = reinterpret_cast<const uint4*>(s + head);
  Sums sums;
  TopList<GROUP> top(&sh, a.top_k);
  if (part == 0 && head > 0) {
    const float v = tid < head ? ToFloat(s[tid]) : -INFINITY;
    if (tid < head) sums.AddOne(v);
    if constexpr (TOP) top.Chunk(v, tid, [&](auto&& f) { f(v, tid); });
  }
  uint4 q[kUnroll], next[kUnroll];
  auto load = [&](uint4 (&to)[kUnroll], int at) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) { const int i = at + u * GROUP + tid; to[u] = i < v_end ? __ldg(body + i) : AllRuledOut(type); }
  };
  load(q, v_begin);
  for (int at = v_begin; at < v_end; at += GROUP * kUnroll) {
    load(next, at + GROUP * kUnroll);
    float most = Max(q[0], type);
#pragma unroll
    for (int u = 1; u < kUnroll; ++u) most = MaxNan(most, Max(q[u], type));
    if (most > sums.m) sums.Raise(most);
    const float base = sums.Base();
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float v[N];
      Unpack(q[u], v, type);
#pragma unroll
      for (int i = 0; i < N; ++i) sums.Add(v[i], base);
    }
    if constexpr (TOP) {
      top.Chunk(most, tid, [&](auto&& f) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          float v[N];
          Unpack(q[u], v, type);
#pragma unroll
          for (int i = 0; i < N; ++i) f(v[i], head + (at + u * GROUP + tid) * N + i);
        }
      });
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) q[u] = next[u];
  }
  if (part == parts - 1 && tail < K) {
    const float v = tid < K - tail ? ToFloat(s[tail + tid]) : -INFINITY;
    if (tid < K - tail) sums.AddOne(v);
    if constexpr (TOP) top.Chunk(v, tid, [&](auto&& f) { f(v, tail + tid); });
  }
  sums.JoinLanes();
  const long long y = LabelOf(a, row);
  if constexpr (GROUP == 32) {
    const RowResult res(sums);
    if (tid == 0) res.Store(a, row, y, y >= 0 && y < K ? ToFloat(s[y]) : 0.f);
    if constexpr (TOP) if (tid < a.top_k) { const Entry e = sh.list[top.live][tid]; res.StoreTop(a, row * a.top_k + tid, tid < top.have ? e.v : -INFINITY, e.cls); }
  } else {
    if ((tid & 31) == 0) { sh.part_m[tid >> 5] = sums.m; sh.part_s[tid >> 5] = sums.s; sh.part_t[tid >> 5] = sums.t; }
    __syncthreads();
    sums = Sums();
    for (int w = 0; w < GROUP / 32; ++w) sums.Join(sh.part_m[w], sh.part_s[w], sh.part_t[w]);
    if (parts > 1) {
      // the cluster's first block joins the others' sums and lists, read from their shared memory
      __syncthreads();
      if (tid == 0) { sh.part_m[0] = sums.m; sh.part_s[0] = sums.s; sh.part_t[0] = sums.t; sh.cand_count = top.have; sh.limit_first = top.live; }
      cg::this_cluster().sync();
      if (part == 0) {
        int others = 0;
        for (int p = 1; p < parts; ++p) {
          const RowShared<GROUP>* o = cg::this_cluster().map_shared_rank(&sh, p);
          sums.Join(o->part_m[0], o->part_s[0], o->part_t[0]);
          if constexpr (TOP) {
            const int n = o->cand_count, from = o->limit_first;
            for (int i = tid; i < n; i += GROUP) sh.cand[top.have + others + i] = o->list[from][i];
            others += n;
          }
        }
        if constexpr (TOP) {
          for (int i = tid; i < top.have; i += GROUP) sh.cand[i] = sh.list[top.live][i];
          __syncthreads();
          const int count = top.have + others;
          for (int i = tid; i < count; i += GROUP) {
            const Entry e = sh.cand[i];
            int rank = 0;
            for (int j = 0; j < count; ++j) rank += Before(sh.cand[j], e) ? 1 : 0;
            if (rank < a.top_k) sh.list[top.live ^ 1][rank] = e;
          }
          __syncthreads();
          top.live ^= 1; top.have = min(count, a.top_k);
        }
      }
      cg::this_cluster().sync();         // no block leaves while its shared memory is read
      if (part != 0) return;
    }
    const RowResult res(sums);
    if (tid == 0) res.Store(a, row, y, y >= 0 && y < K ? ToFloat(s[y]) : 0.f);
    if constexpr (TOP) if (tid < a.top_k) { const Entry e = sh.list[top.live][tid]; res.StoreTop(a, row * a.top_k + tid, tid < top.have ? e.v : -INFINITY, e.cls); }
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
    const float log_norm = s.log_norm[row];
    const long long y = LabelOf(s, row);
    none = log_norm == -INFINITY; bad = (!none && !(fabsf(log_norm) < InfF())) || y >= s.classes;
    again = !none && !bad && fabsf(log_norm) > kTrustedLogNorm;
    m = none ? 0.f : log_norm; log_sum = 0.f;
    label = y >= 0 && y < s.classes ? static_cast<int>(y) : -1;
    h = g.g_entropy ? g.g_entropy[row] : 0.f; g_label = g.g_log_prob && label >= 0 ? g.g_log_prob[row] : 0.f;
    a = (g.g_log_norm ? g.g_log_norm[row] : 0.f) - g_label - h * s.entropy[row];
    for (int t = 0; t < s.top_k; ++t) { const int c = s.top_class[row * s.top_k + t]; if (c >= 0 && c < s.classes) a -= g.g_top[row * s.top_k + t]; }
    if (none) { a = h = g_label = 0.f; }
    if (bad) a = NanF();
  }
  __device__ __forceinline__ float Soft(float v) const { const float lp = MaxNan((v - m) - log_sum, kLowestExponent); return __expf(lp) * fmaf(-h, lp, a); }
  // with the label's own gradient
  __device__ __forceinline__ float At(float v, int j) const { const float d = Soft(v); return none ? 0.f : j == label ? d + g_label : d; }
  // one thread walks the row
  template <typename T>
  __device__ __forceinline__ void TakeAgain(const ClassScoresArgs& s, const T* row) {
    Sums r;
    for (long long j = 0; j < s.classes; ++j) r.AddOne(ToFloat(row[j * s.class_stride]));
    m = r.m; log_sum = logf(r.s);
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
constexpr int kGradThreads = 256, kGradRows = 64;
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
  if (threadIdx.x == 0) s_row = RowGrad(a, g, row);
  __syncthreads();
  if (s_row.again) {
    Sums r;
    for (int j = threadIdx.x; j < K; j += kGradThreads) r.AddOne(ToFloat(in[j]));
    r.JoinLanes();
    if ((threadIdx.x & 31) == 0) { s_m[threadIdx.x >> 5] = r.m; s_s[threadIdx.x >> 5] = r.s; s_t[threadIdx.x >> 5] = r.t; }
    __syncthreads();
    if (threadIdx.x == 0) { Sums all; for (int w = 0; w < kGradThreads / 32; ++w) all.Join(s_m[w], s_s[w], s_t[w]); s_row.m = all.m; s_row.log_sum = logf(all.s); }
    __syncthreads();
  }
  const RowGrad r = s_row;
  // chunk c: the classes from head + c * chunk (chunk 0: from 0) to the next one's start
  const int c = blockIdx.x % chunks;
  const int lo = c == 0 ? 0 : min(K, head + c * chunk), hi = c == chunks - 1 ? K : min(K, head + (c + 1) * chunk);
  if constexpr (ALIGNED) {
    const int first = min(K, head + c * chunk), vectors = (hi - first) / N, rest = first + vectors * N;
    for (int j = lo + threadIdx.x; j < first; j += kGradThreads) out[j] = FromFloat<T>(r.At(ToFloat(in[j]), j));
    const uint4* from = reinterpret_cast<const uint4*>(in + first); uint4* to = reinterpret_cast<uint4*>(out + first);
    for (int i = threadIdx.x; i < vectors; i += 2 * kGradThreads) {
      const bool two = i + kGradThreads < vectors;
      const uint4 q0 = __ldg(from + i), q1 = two ? __ldg(from + i + kGradThreads) : q0;
      auto one = [&](const uint4& q, int at) {
        float v[N]; Unpack(q, v, type);
        union { uint4 q; T t[N]; } o;
#pragma unroll
        for (int k = 0; k < N; ++k) o.t[k] = FromFloat<T>(r.At(v[k], first + at * N + k));
        to[at] = o.q;
      };
      one(q0, i);
      if (two) one(q1, i + kGradThreads);
    }
    for (int j = rest + threadIdx.x; j < hi; j += kGradThreads) out[j] = FromFloat<T>(r.At(ToFloat(in[j]), j));
  } else {
    for (int j = lo + threadIdx.x; j < hi; j += kGradThreads) out[j] = FromFloat<T>(r.At(ToFloat(in[j]), j));
  }
  if (a.top_k > 0) {
    __syncthreads();
    if (threadIdx.x < a.top_k) PatchTop<T>(a, g, r, row, threadIdx.x, lo, hi);
  }
}

// A thread per row (class-major scores, or any strides); the classes in slices over the grid's second dimension.
template <typename T>
__global__ void __launch_bounds__(kGradThreads) ClassGradColumnKernel(ClassScoresArgs a, ClassGradArgs g, int slice) {
  const long long row = static_cast<long long>(blockIdx.x) * kGradThreads + threadIdx.x;
  if (row >= a.rows) return;
  const int K = static_cast<int>(a.classes), lo = blockIdx.y * slice, hi = min(K, lo + slice);
  const T* in = static_cast<const T*>(a.scores) + row * a.row_stride;
  T* out = static_cast<T*>(g.grad) + row * g.grad_row_stride;
  RowGrad r(a, g, row);
  if (r.again) r.TakeAgain(a, in);
  int j = lo;
  for (; j + 8 <= hi; j += 8) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = ToFloat(in[(j + u) * a.class_stride]);
#pragma unroll
    for (int u = 0; u < 8; ++u) out[(j + u) * g.grad_class_stride] = FromFloat<T>(r.At(v[u], j + u));
  }
  for (; j < hi; ++j) out[j * g.grad_class_stride] = FromFloat<T>(r.At(ToFloat(in[j * a.class_stride]), j));
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

template <typename T, bool BY_CLASS>
void LaunchFew(const ClassScoresArgs& a, cudaStream_t s) {
  const unsigned int blocks = static_cast<unsigned int>((a.rows + kFewThreads - 1) / kFewThreads);
  if (a.classes <= 4) ClassLogProbsFewKernel<T, 4, BY_CLASS><<<blocks, kFewThreads, 0, s>>>(a);
  else if (a.classes <= 8) ClassLogProbsFewKernel<T, 8, BY_CLASS><<<blocks, kFewThreads, 0, s>>>(a);
  else if (a.classes <= 16) ClassLogProbsFewKernel<T, 16, BY_CLASS><<<blocks, kFewThreads, 0, s>>>(a);
  else if (a.classes <= 32) ClassLogProbsFewKernel<T, 32, BY_CLASS><<<blocks, kFewThreads, 0, s>>>(a);
  else ClassLogProbsFewKernel<T, kFewClasses, BY_CLASS><<<blocks, kFewThreads, 0, s>>>(a);
}

template <typename T, int GROUP, bool TOP>
void LaunchRows(const ClassScoresArgs& a, int cluster, cudaStream_t s) {
  static PerDevice allowed;
  constexpr int kGroups = 256 / GROUP, kMost = kGroups * RowSharedBytes<GROUP, T>(kMaxTopClasses);
  if (kMost > 48 * 1024) AllowSharedMemory(ClassLogProbsRowKernel<T, GROUP, TOP>, kMost, &allowed);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned int>(GROUP == 32 ? (a.rows + kGroups - 1) / kGroups : a.rows * cluster)); cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = kGroups * RowSharedBytes<GROUP, T>(a.top_k); cfg.stream = s; cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 1 : 0;
  FB_CUDA(cudaLaunchKernelEx(&cfg, ClassLogProbsRowKernel<T, GROUP, TOP>, a));
}
template <typename T, int GROUP>
void LaunchRows(const ClassScoresArgs& a, int cluster, cudaStream_t s) {
  if (a.top_k > 0) LaunchRows<T, GROUP, true>(a, cluster, s); else LaunchRows<T, GROUP, false>(a, cluster, s);
}

constexpr int kSms = 148;

}  // namespace

void LaunchClassLogProbs(const ClassScoresArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return;
  DispatchType(a.dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    if (a.classes <= kFewClasses) {
      // lanes walk rows: right where neighbouring rows are nearer to each other than neighbouring classes
      if (a.row_stride < a.class_stride) LaunchFew<T, true>(a, s); else LaunchFew<T, false>(a, s);
    } else if (a.class_stride == 1) {
      // A warp per row as long as that fills the machine and a warp's walk stays short; else a block, and a cluster of blocks while
      // there are fewer blocks than two per SM and every block has a full chunk.
      const long long chunk = 256LL * kUnroll * Pack<T>::N;
      if (a.classes <= chunk / 8 || (a.classes <= chunk && a.rows >= kSms * 16)) { LaunchRows<T, 32>(a, 1, s); }
      else {
        int cluster = 1;
        while (cluster < 8 && a.rows * cluster < 2 * kSms && a.classes >= 2 * cluster * chunk / kUnroll) cluster *= 2;
        if (a.rows * cluster > 0x7fffffffLL) Log::Fatal("class scores: too many rows");
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
      const int chunk = kGradThreads * N * 4;
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
