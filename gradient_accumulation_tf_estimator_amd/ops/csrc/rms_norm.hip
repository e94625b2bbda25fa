// Root-mean-square norm with the residual's addition (gfx950).
//
//   h = x + r            y = h * rstd * w,   rstd = 1 / sqrt(mean(h^2) + eps)
//   dx = rstd * (w dy - n * mean(w dy n)) + dh,   n = h * rstd   (dr = dx)
//   dw = sum over rows of dy n
//   8-bit form: s = max|y| / 448 over a group of columns (1 where that is 0;
//               at least 2^-126, or s itself would be rounded to a few bits or
//               to zero), q = e4m3(y / s)
//
// Every form is bound by memory: one pass that keeps its row in registers,
// 16-byte loads, one wave64 a row up to 1024 columns (statistics by lane
// exchange, no barrier) and one 256-thread block a row above (one barrier a
// statistic). The next row's loads are issued before this row's reduction.
// 32768 rows of 4096 bf16: forward with a residual 182 us (1.07 GB, 5.9 TB/s, the
// last level cache helping), backward 235 us (1.07 GB, 4.6 TB/s) and 7 us for dw's
// sum; a large copy reaches 4.9. 16384 rows to 8 bits: 93 us a call (472 MB, 5.1
// TB/s, that cache helping here too). 1024 rows of 512: 3.3, 3.9 and 2.5 us, which
// is the latency of a launch.
//
// Sums, statistics and the norm itself are held in 32 bits. The forward norms
// the sum before it is rounded to the stream's type, so y carries one rounding;
// the backward reads the rounded h that the forward wrote (2^-9 of h in bf16,
// which enters dx only through n * mean(...)), and so needs one stream instead
// of x and r. dw is summed over a block's rows in registers, written as one
// fp32 slab a block, and the slabs are added in a fixed order: the result does
// not depend on timing.

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "ga_ops.h"

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 b8;
typedef __attribute__((ext_vector_type(8))) _Float16 h8;
typedef __attribute__((ext_vector_type(4))) float f4;

struct Bf16 { typedef __bf16 t; };
struct Fp16 { typedef _Float16 t; };
struct Fp32 { typedef float t; };

template <typename E>
__device__ __forceinline__ void store8(E* p, const float* f) {
  typedef __attribute__((ext_vector_type(8))) E e8;
  e8 v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = (E)f[k];
  *(e8*)p = v;
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float* f) {
  f4 a, b;
#pragma unroll
  for (int k = 0; k < 4; ++k) { a[k] = f[k]; b[k] = f[4 + k]; }
  *(f4*)p = a;
  *(f4*)(p + 4) = b;
}

// Column of element e of a thread's vector v. VEC: eight neighbours a thread,
// one 16-byte access (H and every row start a multiple of 8). SCALAR: odd H or
// alignment, element by element with the threads next to each other. RUN:
// the VEC columns with scalar accesses (8-bit groups on unaligned rows).
enum Mode { VEC = 0, SCALAR = 1, RUN = 2 };
template <int NT, int MODE>
__device__ __forceinline__ int column(int v, int e, int t) {
  return MODE == SCALAR ? (v * 8 + e) * NT + t : (v * NT + t) * 8 + e;
}

// A thread's part of a row as it lies in memory; converted where it is used, so
// that the next row can wait in few registers.
template <typename E, int NT, int NV, int MODE>
struct Row {
  typedef __attribute__((ext_vector_type(8))) E e8;
  e8 x[NV];
  __device__ __forceinline__ void load(const void* base, long long at, int H, int t) {
    const E* row = (const E*)base + at;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (MODE == VEC) {
        const int c = column<NT, MODE>(v, 0, t);
        x[v] = c < H ? *(const e8*)(row + c) : (e8){};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = column<NT, MODE>(v, e, t);
          x[v][e] = c < H ? row[c] : (E)0.f;
        }
      }
    }
  }
  __device__ __forceinline__ float at(int v, int e) const { return (float)x[v][e]; }
};
template <typename E, int NT, int NV, int MODE>
__device__ __forceinline__ void store_row(E* row, int H, int t, const float (*f)[8]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (MODE == VEC) {
      const int c = column<NT, MODE>(v, 0, t);
      if (c < H) store8<E>(row + c, f[v]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = column<NT, MODE>(v, e, t);
        if (c < H) row[c] = (E)f[v][e];
      }
    }
  }
}

struct Sum { static __device__ float of(float a, float b) { return a + b; } };
// a NaN stays: fmaxf alone would drop it
struct Max {
  static __device__ float of(float a, float b) { return (a > b || a != a) ? a : b; }
};

// Reduction over the NT threads of a row; `lds` holds NT / 64 floats for each
// call in flight. Every thread of the block calls it.
template <int NT, typename Op>
__device__ __forceinline__ float over_row(float s, float* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s = Op::of(s, __shfl_xor(s, o, 64));
  if (NT > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    s = lds[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) s = Op::of(s, lds[w]);
  }
  return s;
}

// A block holds 256 / NT rows; grid-stride over the rows, the next one's loads
// issued before this one's reduction. The reduction's floats alternate between
// two halves, so one barrier a row is enough.
template <typename E, int NT, int NV, int MODE>
__global__ __launch_bounds__(256) void k_rms_fwd(RmsArgs a) {
  constexpr int RB = 256 / NT;
  __shared__ float lds[2][4];
  const int t = threadIdx.x % NT;
  const long long first = (long long)blockIdx.x * RB + threadIdx.x / NT, step = (long long)gridDim.x * RB;
  typedef Row<E, NT, NV, MODE> R;
  R w, x, r;
  w.load(a.w, 0, a.H, t);
  auto fetch = [&](long long row) {
    x.load(a.x, row * a.x_stride, a.H, t);
    if (a.res) r.load(a.res, row * a.res_stride, a.H, t);
  };
  if (first < a.R) fetch(first);
  int turn = 0;
  for (long long row = first; row < a.R; row += step, turn ^= 1) {
    float h[NV][8], s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[v][e] = a.res ? x.at(v, e) + r.at(v, e) : x.at(v, e);
    if (row + step < a.R) fetch(row + step);
    if (a.res) store_row<E, NT, NV, MODE>((E*)a.h + row * a.H, a.H, t, h);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(h[v][e], h[v][e], s);
    s = over_row<NT, Sum>(s, lds[turn]);
    const float rstd = 1.f / sqrtf(s / (float)a.H + a.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[v][e] = h[v][e] * rstd * w.at(v, e);
    store_row<E, NT, NV, MODE>((E*)a.y + row * a.H, a.H, t, h);
    if (t == 0) a.rstd[row] = rstd;
  }
}

template <typename E, int NT, int NV, int MODE>
__global__ __launch_bounds__(256) void k_rms_bwd(RmsArgs a) {
  constexpr int RB = 256 / NT;
  __shared__ float lds[2][4];
  const int t = threadIdx.x % NT;
  const long long first = (long long)blockIdx.x * RB + threadIdx.x / NT, step = (long long)gridDim.x * RB;
  typedef Row<E, NT, NV, MODE> R;
  R w, x, dy, dh;
  float dw[NV][8], rs = 0.f;
  w.load(a.w, 0, a.H, t);
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[v][e] = 0.f;
  auto fetch = [&](long long row) {
    x.load(a.x, row * a.x_stride, a.H, t);
    dy.load(a.dy, row * a.dy_stride, a.H, t);
    rs = a.rstd[row];
  };
  if (first < a.R) fetch(first);
  int turn = 0;
  for (long long row = first; row < a.R; row += step, turn ^= 1) {
    float n[NV][8], g[NV][8], s = 0.f;
    const float rstd = rs;
    if (a.dh) dh.load(a.dh, row * a.dh_stride, a.H, t);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        n[v][e] = x.at(v, e) * rstd;
        dw[v][e] = fmaf(dy.at(v, e), n[v][e], dw[v][e]);
        g[v][e] = dy.at(v, e) * w.at(v, e);
        s = fmaf(g[v][e], n[v][e], s);
      }
    if (row + step < a.R) fetch(row + step);
    s = over_row<NT, Sum>(s, lds[turn]) / (float)a.H;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g[v][e] = rstd * fmaf(-n[v][e], s, g[v][e]);
        if (a.dh) g[v][e] += dh.at(v, e);
      }
    store_row<E, NT, NV, MODE>((E*)a.y + row * a.H, a.H, t, g);
  }
  // one slab a block: [gridDim.x][H]; the block's waves add theirs up in order
  if (RB > 1) {
    __shared__ float join[RB > 1 ? RB - 1 : 1][NT * NV * 8];
    const int w = threadIdx.x / NT;
    if (w > 0)
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) join[w - 1][(v * 8 + e) * NT + t] = dw[v][e];
    __syncthreads();
    if (w > 0) return;
#pragma unroll
    for (int i = 0; i < RB - 1; ++i)
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[v][e] += join[i][(v * 8 + e) * NT + t];
  }
  store_row<float, NT, NV, MODE>(a.slabs + (long long)blockIdx.x * a.H, a.H, t, dw);
}

// dw[c] = sum over slabs; 16 columns x 16 slab groups a block, joined in LDS in
// a fixed order. acc: add into the fp32 accumulation slice instead.
template <typename E>
__global__ __launch_bounds__(256) void k_rms_dw(const float* slabs, int n, int H, E* dw, float* acc) {
  __shared__ float lds[16][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), g = threadIdx.x >> 4;
  float s = 0.f;
  if (c < H) {
#pragma unroll 16
    for (int i = g; i < n; i += 16) s += slabs[(long long)i * H + c];
  }
  lds[g][threadIdx.x & 15] = s;
  __syncthreads();
  if (g == 0 && c < H) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += lds[i][threadIdx.x];
    if (acc) acc[c] += t;
    else dw[c] = (E)t;
  }
}

// 8-bit form. A group's maximum is taken over its lanes (a group of 32 / 64 /
// 128 columns is 4 / 8 / 16 lanes of one vector) or over the row. y is divided
// by the scale, not multiplied by its inverse: one rounding less before the
// 8-bit one.
template <typename E, int NT, int NV, int MODE>
__global__ __launch_bounds__(256) void k_rms_fp8(RmsArgs a) {
  constexpr int RB = 256 / NT;
  __shared__ float lds[4][4];
  const int t = threadIdx.x % NT;
  const long long first = (long long)blockIdx.x * RB + threadIdx.x / NT, step = (long long)gridDim.x * RB;
  typedef Row<E, NT, NV, MODE> R;
  R w, x, r;
  w.load(a.w, 0, a.H, t);
  auto fetch = [&](long long row) {
    x.load(a.x, row * a.x_stride, a.H, t);
    if (a.res) r.load(a.res, row * a.res_stride, a.H, t);
  };
  if (first < a.R) fetch(first);
  int turn = 0;
  for (long long row = first; row < a.R; row += step, turn ^= 2) {
    float h[NV][8], s = 0.f, m[NV], all = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[v][e] = a.res ? x.at(v, e) + r.at(v, e) : x.at(v, e);
    if (row + step < a.R) fetch(row + step);
    if (a.res) store_row<E, NT, NV, MODE>((E*)a.h + row * a.H, a.H, t, h);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(h[v][e], h[v][e], s);
    s = over_row<NT, Sum>(s, lds[turn]);
    const float rstd = 1.f / sqrtf(s / (float)a.H + a.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      m[v] = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[v][e] = h[v][e] * rstd * w.at(v, e);
        m[v] = Max::of(m[v], fabsf(h[v][e]));
      }
      all = Max::of(all, m[v]);
    }
    const int lanes = a.group >> 3;  // 0: the whole row
    if (lanes == 0) all = over_row<NT, Max>(all, lds[turn + 1]);
    const long long scales = a.group ? a.H / a.group : 1;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float top = all;
      if (lanes) {
        top = m[v];
        for (int o = lanes >> 1; o > 0; o >>= 1) top = Max::of(top, __shfl_xor(top, o, 64));
      }
      const float part = top / 448.f, scale = top == 0.f ? 1.f : part < 0x1p-126f ? 0x1p-126f : part;
      if (lanes) {
        const int c = column<NT, MODE>(v, 0, t);
        if (c < a.H && (t % lanes) == 0) a.scales[row * scales + c / a.group] = scale;
      } else if (v == 0 && t == 0) {
        a.scales[row] = scale;
      }
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = h[v][e] / scale;
      int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
      lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
      int hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], 0, false);
      hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], hi, true);
      unsigned char* q = a.q + row * a.H;
      if (MODE == VEC) {
        const int c = column<NT, MODE>(v, 0, t);
        if (c < a.H) *(int2*)(q + c) = make_int2(lo, hi);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = column<NT, MODE>(v, e, t);
          if (c < a.H) q[c] = (unsigned char)((e < 4 ? lo : hi) >> (8 * (e & 3)));
        }
      }
    }
  }
}

enum What { FWD, BWD, FP8 };

template <typename E, int NT, int NV, int MODE>
void launch(int what, const RmsArgs& a, int blocks, hipStream_t s) {
  if (what == FWD) hipLaunchKernelGGL((k_rms_fwd<E, NT, NV, MODE>), dim3(blocks), dim3(256), 0, s, a);
  if (what == BWD) hipLaunchKernelGGL((k_rms_bwd<E, NT, NV, MODE>), dim3(blocks), dim3(256), 0, s, a);
  if (what == FP8) hipLaunchKernelGGL((k_rms_fp8<E, NT, NV, MODE>), dim3(blocks), dim3(256), 0, s, a);
}

template <typename E, int NT, int NV>
void by_mode(int what, int mode, const RmsArgs& a, int blocks, hipStream_t s) {
  if (mode == VEC) return launch<E, NT, NV, VEC>(what, a, blocks, s);
  if (mode == SCALAR) return launch<E, NT, NV, SCALAR>(what, a, blocks, s);
  hipLaunchKernelGGL((k_rms_fp8<E, NT, NV, RUN>), dim3(blocks), dim3(256), 0, s, a);
}

template <typename E>
void by_width(int what, int mode, const RmsArgs& a, int blocks, hipStream_t s) {
  if (a.H <= 512) return by_mode<E, 64, 1>(what, mode, a, blocks, s);
  if (a.H <= 1024) return by_mode<E, 64, 2>(what, mode, a, blocks, s);
  if (a.H <= 2048) return by_mode<E, 256, 1>(what, mode, a, blocks, s);
  if (a.H <= 4096) return by_mode<E, 256, 2>(what, mode, a, blocks, s);
  by_mode<E, 256, 4>(what, mode, a, blocks, s);
}

hipError_t by_type(int what, int type, int mode, const RmsArgs& a, int blocks, hipStream_t s) {
  if (type == GA_BF16) by_width<__bf16>(what, mode, a, blocks, s);
  else if (type == GA_FP16) by_width<_Float16>(what, mode, a, blocks, s);
  else by_width<float>(what, mode, a, blocks, s);
  return hipGetLastError();
}

inline int rows_a_block(int H) { return H <= 1024 ? 4 : 1; }

}  // namespace

int rms_blocks(long long R, int H, bool backward) {
  const long long need = (R + rows_a_block(H) - 1) / rows_a_block(H);
  const long long most = backward ? 1024 : 4096;
  return (int)(need < most ? need : most);
}
int rms_slabs(long long R, int H) { return rms_blocks(R, H, true); }

hipError_t rms_forward(int type, bool vec, const RmsArgs& a, hipStream_t s) {
  return by_type(FWD, type, vec ? VEC : SCALAR, a, rms_blocks(a.R, a.H, false), s);
}
hipError_t rms_fp8(int type, bool vec, const RmsArgs& a, hipStream_t s) {
  return by_type(FP8, type, vec ? VEC : a.group ? RUN : SCALAR, a, rms_blocks(a.R, a.H, false), s);
}
hipError_t rms_backward(int type, bool vec, const RmsArgs& a, void* dw, float* acc, hipStream_t s) {
  const hipError_t e = by_type(BWD, type, vec ? VEC : SCALAR, a, rms_blocks(a.R, a.H, true), s);
  if (e != hipSuccess) return e;
  const int n = rms_slabs(a.R, a.H), grid = (a.H + 15) / 16;
  if (type == GA_BF16)
    hipLaunchKernelGGL((k_rms_dw<__bf16>), dim3(grid), dim3(256), 0, s, a.slabs, n, a.H, (__bf16*)dw, acc);
  else if (type == GA_FP16)
    hipLaunchKernelGGL((k_rms_dw<_Float16>), dim3(grid), dim3(256), 0, s, a.slabs, n, a.H, (_Float16*)dw, acc);
  else
    hipLaunchKernelGGL((k_rms_dw<float>), dim3(grid), dim3(256), 0, s, a.slabs, n, a.H, (float*)dw, acc);
  return hipGetLastError();
}
