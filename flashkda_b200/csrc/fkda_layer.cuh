// Parameter blocks and host checks that the operators round the recurrence share (short convolution, selective scan, norms).
#pragma once
#include "fkda_common.cuh"

namespace fkda {

// A [B][T][...] tensor whose tokens are `token` elements apart and whose batch rows `batch`.
struct Rows {
  int64_t batch, token;
};

struct ConvParams {
  const __nv_bfloat16* x;
  const void* weight;
  const void* bias;
  __nv_bfloat16* out;
  const __nv_bfloat16* initial_state;
  __nv_bfloat16* final_state;
  const int64_t* cu_seqlens;
  Rows xs, os;
  int64_t T;                // tokens of a sequence, or of the packed batch
  int C;
  int N;
  int tile;                 // tokens of a block
  int tiles;                // ... of a sequence, or of the packed batch
  int silu;
};
cudaError_t launch_short_conv(ConvParams p, int width, bool weight_fp32, cudaStream_t stream);

struct SsmParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* dt;
  const __nv_bfloat16* Bm;
  const __nv_bfloat16* Cm;
  __nv_bfloat16* out;
  const float* A_log;
  const float* dt_bias;
  const float* D;
  const void* initial_state;
  void* final_state;
  const int64_t* cu_seqlens;
  Rows xs, dts, bs, cs, os;
  int64_t T;
  int H, P, G, Ns, N;
  int state_fp32;
};
// `most`: packed batches, only sequences of at most so many tokens (0: all).  `status`: the call's status word, or NULL: not written.
cudaError_t launch_ssm_step(const SsmParams& p, int most, int* status, cudaStream_t stream);

struct GatedNormParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* gate;
  const void* weight;
  __nv_bfloat16* out;
  Rows xs, gs, os;
  int64_t rows;             // B T H, below 2^31
  int64_t T;                // tokens of a batch row, or more than there are: batch rows follow one another
  int H, D;
  float eps;
  int per_head;
};
cudaError_t launch_gated_norm(const GatedNormParams& p, bool weight_fp32, bool silu, bool gate_first, cudaStream_t stream);

struct AddNormParams {
  const __nv_bfloat16* x;
  const void* residual;
  const void* weight;
  __nv_bfloat16* out;
  void* residual_out;
  Rows xs, rs, os, ros;
  int64_t rows;             // B T, below 2^31
  int64_t T;                // as above
  int D;
  float scale, eps;
};
cudaError_t launch_add_norm(const AddNormParams& p, bool weight_fp32, bool residual_fp32, cudaStream_t stream);

// The library's error message of this thread (fkda_last_error); returns `code`.
int set_error(int code, const char* fmt, ...);

// Eight consecutive weights as fp32.
template <bool kFp32>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&w)[8]) {
  if constexpr (kFp32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    const float4 a = __ldg(q), b = __ldg(q + 1);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
    unpack8(__ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(base) + at)), w);
  }
}
// Four consecutive weights as fp32.
template <bool kFp32>
__device__ __forceinline__ float4 load4(const void* base, int64_t at) {
  if constexpr (kFp32) return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + at));
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + at));
  return make_float4(bf_lo(v.x), bf_hi(v.x), bf_lo(v.y), bf_hi(v.y));
}
__device__ __forceinline__ float rcpf(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// max(x, 0) + log(1 + e^-|x|) to fp32 accuracy.  log(1 + u) = 2 atanh(z) with z = u / (2 + u) <= 1/3, by the series of atanh to z^13: what is
// left out is below 2^-26 of the sum.
__device__ __forceinline__ float softplus(float x) {
  const float u = ex2f(-kLog2e * fabsf(x)), z = __fdividef(u, 2.f + u), q = z * z;
  float s = fmaf(q, 1.f / 13.f, 1.f / 11.f);
  s = fmaf(q, s, 1.f / 9.f);
  s = fmaf(q, s, 1.f / 7.f);
  s = fmaf(q, s, 1.f / 5.f);
  s = fmaf(q, s, 1.f / 3.f);
  s = fmaf(q, s, 1.f);
  return fmaf(2.f * z, s, fmaxf(x, 0.f));
}

}  // namespace fkda
