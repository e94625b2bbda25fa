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

// ---- attention with a relative position bias (rel_attn.hip); strides in elements ----
#define GA_REL_MAX_DISTANCE 512
#define GA_REL_MAX_BUCKETS 256
struct RelArgs {
  const __bf16* qkv;          // [B][S][width], width = (NH + 2 NKV) * D
  const __bf16* table;        // [buckets][NH]
  const int* map;             // [2 * far + 1], the bucket of each offset
  const unsigned char* mask;  // [B][S], 1 = attend, or null
  __bf16* out;                // [B][S][NH][D]
  float* lse;                 // [2][B][NH][S]: base 2, +inf for a row with nothing allowed; a factor of P, 1 for
                              // ordinary rows
  float* split;               // [spans][B][NH][S] of D outputs, then of maximum and sum, where spans > 1
  // backward
  const __bf16* dout;         // [B][S][NH][D]
  float* dsum;                // [B][NH][S]
  __bf16* dqkv;               // like qkv
  float* dq;                  // [q_spans][B][NH][S] of D, then of the row's four sums, where q_spans > 1
  float* doff;                // [NH][B][rel_doff_rows][2 * far + 1]
  __bf16* dtable;             // [buckets][NH]
  float* dkv;                 // [parts][B][NKV][S][dK, dV] where parts > 1
  int B, S, NH, NKV, D, width, buckets, far, causal;
  int parts, spans;           // backward: workgroups for a tile of keys, spans of the queries among them;
                              // forward: spans of the keys
  int q_spans;                // backward: spans of the keys in dQ
  float scale;
};
#define GA_REL_TILE 128  // queries a workgroup
__host__ __device__ inline int rel_tiles(int S) { return (S + GA_REL_TILE - 1) / GA_REL_TILE; }
// a row of offsets' sums for each tile and span, and one for what joining the spans adds
__host__ __device__ inline int rel_doff_rows(int S, int q_spans) { return rel_tiles(S) * (q_spans > 1 ? q_spans + 1 : 1); }
int rel_spans(int B, int S, int NH);
void rel_parts(int B, int S, int NH, int NKV, int D, int* parts, int* spans);
hipError_t rel_forward(const RelArgs& a, hipStream_t s);
hipError_t rel_backward(const RelArgs& a, hipStream_t s);

struct RelTokenArgs {
  const __bf16 *q, *k, *v;
  long long q_b, q_s, q_h, k_b, k_s, k_h, v_b, v_s, v_h;
  const __bf16* table;
  const int* map;
  const int* lengths;  // [B]
  __bf16* out;         // [B][Sq][NH][D]
  float* parts;        // [B * NKV * row tiles][splits][32][D + 2]
  int B, Sq, S, NH, NKV, D, buckets, far, splits;
  float scale;
};
int rel_token_splits(int B, int Sq, int S, int NH, int NKV);
hipError_t rel_token(const RelTokenArgs& a, hipStream_t s);
