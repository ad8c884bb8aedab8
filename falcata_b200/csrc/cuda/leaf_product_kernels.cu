// Products of rows grouped by leaf: every leaf g owns the rows [begin[g], begin[g + 1]) and a linear map W_g [P x F].
//   leaf products:  y_i = W_g x_i                       for the rows i of leaf g
//   leaf Gram:      P_g = sum over the rows i of leaf g of a_i b_i^T
// The first is the linear part of leaves with several outputs; its gradient in x is the same product with the transposed maps,
// its gradient in W the second, which also gives the normal equations X^T H X of linear leaves (a = h x).
// Sums are held in fp32 and rounded once to the output's type.
#include "kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace fb {

namespace {

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Window of leaf g inside [0, rows): whatever the caller's boundaries hold, no access leaves the arrays.
__device__ __forceinline__ void LeafWindow(const LeafWindows& w, int g, long long* begin, long long* end) {
  const long long b = w.begin_bits == 32 ? static_cast<const int*>(w.begin)[g] : static_cast<const long long*>(w.begin)[g];
  const long long e = w.begin_bits == 32 ? static_cast<const int*>(w.begin)[g + 1] : static_cast<const long long*>(w.begin)[g + 1];
  *begin = min(max(b, 0LL), w.rows); *end = min(max(e, *begin), w.rows);
}

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

template <typename F> void DispatchType(int dtype, F&& f) {
  switch (dtype) {
    case kOpFloat32: f(static_cast<float*>(nullptr)); return;
    case kOpFloat16: f(static_cast<__half*>(nullptr)); return;
    case kOpBFloat16: f(static_cast<__nv_bfloat16*>(nullptr)); return;
    default: Log::Fatal("leaf products: unknown type code %d", dtype);
  }
}

inline unsigned int Tiles(long long n, long long most) { return static_cast<unsigned int>(std::max(1LL, std::min(most, (n + kTile - 1) / kTile))); }

}  // namespace

void LaunchLeafProducts(const LeafProductsArgs& a, cudaStream_t s) {
  if (a.leaves.rows <= 0 || a.outputs <= 0 || a.leaves.leaves <= 0) return;
  DispatchType(a.dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    LeaflessRowsKernel<T><<<64, 256, 0, s>>>(a);
    FB_LAUNCHED(); FB_KERNEL_CHECK();
    LeafProductsKernel<T><<<dim3(Tiles(a.outputs, 64), Tiles(a.leaves.rows, 64), std::min(a.leaves.leaves, 1024)), kTile * kTile, 0, s>>>(a);
  });
  FB_LAUNCHED(); FB_KERNEL_CHECK();
}

void LaunchLeafGram(const LeafGramArgs& a, cudaStream_t s) {
  if (a.leaves.leaves <= 0 || a.a_cols <= 0 || a.b_cols <= 0) return;
  const dim3 grid(Tiles(a.b_cols, 64), Tiles(a.a_cols, 64), std::min(a.leaves.leaves, 1024));
  DispatchType(a.dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    if (a.out_dtype == a.dtype) LeafGramKernel<T, T><<<grid, kTile * kTile, 0, s>>>(a);
    else if (a.out_dtype == kOpFloat32) LeafGramKernel<T, float><<<grid, kTile * kTile, 0, s>>>(a);
    else Log::Fatal("leaf Gram: sums of type code %d as type code %d", a.dtype, a.out_dtype);
  });
  FB_LAUNCHED(); FB_KERNEL_CHECK();
}

}  // namespace fb
