// Host launchers of the root-mean-square norm.
#pragma once
#include <cuda_runtime.h>

namespace b200ep {

enum ElemType : int { ELEM_BF16 = 0, ELEM_F16 = 1, ELEM_F32 = 2 };

constexpr int kNormMaxHidden = 32768;
constexpr int kNormScaleBlock = 128;     // channels that share one scale of the fp8 output

// Row r of a [T, H] tensor starts at r * ld elements. All of a call's rows lie alike within 16 bytes: base addresses are
// multiples of 16, and row strides in bytes are equal modulo 16.
struct NormFwdParams {
  int type, wtype;            // of the rows; of the weight (the rows' type or f32)
  int T, H;
  const void* x;
  long long x_ld;
  const void* residual;       // or null
  long long res_ld;
  const void* w;              // [H]
  float eps;
  void* y;                    // [T, H] contiguous, or null (fp8 output only)
  void* h;                    // x + residual, [T, H] contiguous; null without a residual
  float* rstd;                // [T] or null
  void* q;                    // e4m3 [T, H] contiguous, or null
  float* scales;              // f32 [T, H / 128]
};
int launch_rms_norm_fwd(const NormFwdParams& p, cudaStream_t st);

struct NormBwdParams {
  int type, wtype;
  int T, H;
  const void* dy;             // gradient of y
  long long dy_ld;
  const void* dh;             // gradient of x + residual, or null
  long long dh_ld;
  const void* h;              // what was normalised, or one part of it
  long long h_ld;
  const void* res;            // the other part, added in f32, or null
  long long res_ld;
  const void* w;
  const float* rstd;          // [T]
  void* dx;                   // [T, H] contiguous
  float* part;                // f32 [rms_norm_bwd_parts(...), H]: parts of the weight's gradient; null: not wanted
  void* dw;                   // [H] in the weight's type
  int parts;                  // what rms_norm_bwd_parts said
};
// CTAs of the backward pass, each of which leaves one part of the weight's gradient. -1: arguments that it refuses.
int rms_norm_bwd_parts(const NormBwdParams& p);
int launch_rms_norm_bwd(const NormBwdParams& p, cudaStream_t st);

}  // namespace b200ep
