// Launchers of the norm, clipping and relative-attention kernels: plain
// arguments in, a HIP error out. Shapes and types are checked by the bindings.
#pragma once

#include <hip/hip_runtime.h>

enum GaType { GA_FP32 = 0, GA_BF16 = 1, GA_FP16 = 2 };

// ---- root-mean-square norm (rms_norm.hip); strides in elements ----
struct RmsArgs {
  const void* x;    // backward: the saved h
  const void* res;  // or null
  const void* w;
  const void* dy;
  const void* dh;   // or null
  void* y;          // backward: dx
  void* h;          // x + res, written where res is given
  float* rstd;
  float* slabs;     // [rms_slabs][H] fp32, backward
  float* scales;
  unsigned char* q;
  long long R, x_stride, res_stride, dy_stride, dh_stride;
  int H, group;
  float eps;
};
int rms_slabs(long long R, int H);
hipError_t rms_forward(int type, bool vec, const RmsArgs& a, hipStream_t s);
hipError_t rms_fp8(int type, bool vec, const RmsArgs& a, hipStream_t s);
hipError_t rms_backward(int type, bool vec, const RmsArgs& a, void* dw, float* acc, hipStream_t s);

// ---- global norm over many tensors, and clipping (grad_clip.hip) ----
#define GA_CLIP_TENSORS 128  // a launch's tensors travel as one by-value argument
struct ClipArgs {
  const void* in[GA_CLIP_TENSORS];
  void* out[GA_CLIP_TENSORS];
  long long n[GA_CLIP_TENSORS];
  int first[GA_CLIP_TENSORS + 1];  // a tensor's first block of the launch
  unsigned char type[GA_CLIP_TENSORS];
  unsigned char vec[GA_CLIP_TENSORS];
  int count;
  int chunk;  // elements a block, a multiple of 2048
};
hipError_t clip_sums(const ClipArgs& a, double* sums, hipStream_t s);
hipError_t clip_finish(const double* sums, int n, double clip, float* norm, float* coef, hipStream_t s);
hipError_t clip_scale(const ClipArgs& a, const float* coef, hipStream_t s);
