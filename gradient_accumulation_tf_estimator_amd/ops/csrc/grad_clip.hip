// Global norm over many tensors, and clipping by it (gfx950).
//
//   norm = sqrt(sum over tensors of sum g^2),  coef = min(1, clip / norm),
//   out = g * coef;  where norm is not finite coef is NaN, so that every output
//   says so (tf.clip_by_global_norm does the same).
//
// Bound by memory: the gradients are read twice and written once, since the
// factor needs them all first. A tensor is cut into chunks, one block each; the
// tensors' addresses travel by value with the launch (up to 128 a launch), so
// nothing is copied to the device, nothing is kept between calls, and a
// captured graph holds all that it needs. 335M fp32 elements in 391 tensors: 802 us
// for 4.0 GB (5.0 TB/s), 251 us of it the norm's pass; 28.7M bf16: 34 us (13 the
// norm, 4 its end, 19 the scaling).
//
// Squares are taken and summed in 64 bits: a bf16 or fp32 gradient's square
// passes the range of 32 bits long before its norm does, the chip's 64-bit rate
// (two operations an element) is far above what memory delivers, and a block's
// sum no longer depends on its size. Block sums are added in a fixed order.

#include <hip/hip_runtime.h>

#include "ga_ops.h"

namespace {

typedef __attribute__((ext_vector_type(4))) float f4;

// the tensor that block b works on: last t with first[t] <= b
__device__ __forceinline__ int tensor_of(const ClipArgs& a, int b) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.first[mid] <= b) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename E>
__device__ double sum_squares(const E* p, long long n, bool vec) {
  constexpr int V = 16 / sizeof(E);
  typedef __attribute__((ext_vector_type(V))) E ev;
  double s0 = 0, s1 = 0;
  long long i = threadIdx.x;
  if (vec) {
    const long long nv = n / V;
    const ev* q = (const ev*)p;
    for (; i + 768 < nv; i += 1024) {
      ev v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = q[i + 256 * k];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const double x = (double)(float)v[k][e], y = (double)(float)v[k][e + 1];
          s0 = fma(x, x, s0);
          s1 = fma(y, y, s1);
        }
    }
    for (; i < nv; i += 256) {
      const ev v = q[i];
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const double x = (double)(float)v[e], y = (double)(float)v[e + 1];
        s0 = fma(x, x, s0);
        s1 = fma(y, y, s1);
      }
    }
    i = nv * V + threadIdx.x;
  }
  for (; i < n; i += 256) {
    const double x = (double)(float)p[i];
    s0 = fma(x, x, s0);
  }
  return s0 + s1;
}

__device__ __forceinline__ double over_block(double s, double* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) s += lds[w];
  return s;
}

__global__ __launch_bounds__(256) void k_clip_sums(ClipArgs a, double* sums) {
  __shared__ double lds[4];
  const int t = tensor_of(a, blockIdx.x);
  const long long at = (long long)(blockIdx.x - a.first[t]) * a.chunk;
  const long long left = a.n[t] - at, n = left < a.chunk ? left : a.chunk;
  double s;
  if (a.type[t] == GA_FP32) s = sum_squares((const float*)a.in[t] + at, n, a.vec[t]);
  else if (a.type[t] == GA_BF16) s = sum_squares((const __bf16*)a.in[t] + at, n, a.vec[t]);
  else s = sum_squares((const _Float16*)a.in[t] + at, n, a.vec[t]);
  s = over_block(s, lds);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

__global__ __launch_bounds__(1024) void k_clip_finish(const double* sums, int n, double clip, float* norm, float* coef) {
  __shared__ double lds[16];
  double s = 0;
  for (int i = threadIdx.x; i < n; i += 1024) s += sums[i];
  s = over_block(s, lds);
  if (threadIdx.x == 0) {
    const double r = sqrt(s);
    *norm = (float)r;
    if (coef) *coef = !(r < __builtin_inf()) ? __builtin_nanf("") : r <= clip ? 1.f : (float)(clip / r);
  }
}

template <typename E>
__device__ void scale(const E* in, E* out, long long n, float c, bool vec) {
  constexpr int V = 16 / sizeof(E);
  typedef __attribute__((ext_vector_type(V))) E ev;
  long long i = threadIdx.x;
  if (vec) {
    const long long nv = n / V;
    const ev* q = (const ev*)in;
    ev* o = (ev*)out;
    for (; i + 768 < nv; i += 1024) {
      ev v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = q[i + 256 * k];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[k][e] = (E)((float)v[k][e] * c);
        __builtin_nontemporal_store(v[k], o + i + 256 * k);
      }
    }
    for (; i < nv; i += 256) {
      ev v = q[i];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = (E)((float)v[e] * c);
      o[i] = v;
    }
    i = nv * V + threadIdx.x;
  }
  for (; i < n; i += 256) out[i] = (E)((float)in[i] * c);
}

// Blocks run from the last chunk to the first: what the norm's pass read last is
// still in the 256 MB cache (335M fp32 elements, 1.3 GB: 852 -> 839 us in all, 802 us
// with stores that do not push it out).
__global__ __launch_bounds__(256) void k_clip_scale(ClipArgs a, const float* coef) {
  const float c = *coef;
  const int b = gridDim.x - 1 - blockIdx.x, t = tensor_of(a, b);
  if (c == 1.f && a.in[t] == a.out[t]) return;  // in place and nothing to clip
  const long long at = (long long)(b - a.first[t]) * a.chunk;
  const long long left = a.n[t] - at, n = left < a.chunk ? left : a.chunk;
  if (a.type[t] == GA_FP32) scale((const float*)a.in[t] + at, (float*)a.out[t] + at, n, c, a.vec[t]);
  else if (a.type[t] == GA_BF16) scale((const __bf16*)a.in[t] + at, (__bf16*)a.out[t] + at, n, c, a.vec[t]);
  else scale((const _Float16*)a.in[t] + at, (_Float16*)a.out[t] + at, n, c, a.vec[t]);
}

}  // namespace

hipError_t clip_sums(const ClipArgs& a, double* sums, hipStream_t s) {
  hipLaunchKernelGGL(k_clip_sums, dim3(a.first[a.count]), dim3(256), 0, s, a, sums);
  return hipGetLastError();
}
hipError_t clip_finish(const double* sums, int n, double clip, float* norm, float* coef, hipStream_t s) {
  hipLaunchKernelGGL(k_clip_finish, dim3(1), dim3(1024), 0, s, sums, n, clip, norm, coef);
  return hipGetLastError();
}
hipError_t clip_scale(const ClipArgs& a, const float* coef, hipStream_t s) {
  hipLaunchKernelGGL(k_clip_scale, dim3(a.first[a.count]), dim3(256), 0, s, a, coef);
  return hipGetLastError();
}
