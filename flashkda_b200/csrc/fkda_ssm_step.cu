// Selective state space scan token by token, in fp32 throughout: decode and speculative steps.
//
//   delta = softplus(dt + dt_bias[h]),  S <- exp(-exp(A_log[h]) delta) S + delta x B^T,  out = S C + D[h] x      (S is [P][Ns])
//
// A block holds 32 (Ns = 128) or 64 (Ns = 64) rows of one chain's state in registers: the lanes of half a warp, or a quarter, share
// four rows with eight columns each, so that a row's product with C folds through four or three shuffles, and B and C are eight
// registers of a lane.  Rows never meet, so the rows of a state are as many blocks, and a single sequence spreads over the chip.
//
// A step is bound by the states, which are read and written: 256 sequences x 32 heads of 64 x 128 in fp32 take 89 us, 6.0 TB/s.  More tokens are bound by
// arithmetic, some 0.5 us a token of an SM's rows, and by what one token takes behind the other, 0.27 us: fkda_ssm.cuh has where the blocks begin.
#include "fkda_elem.cuh"
#include "fkda_layer.cuh"

namespace fkda {
namespace ssm_step {

using elem::f2;
using elem::fma2;
using elem::mul;
using elem::pk;

constexpr int kThreads = 128;

template <int kNs, bool kFp32, bool kPacked>
__global__ void __launch_bounds__(kThreads) ssm_step_kernel(const SsmParams p, int most, int* status) {
  constexpr int kLanes = kNs / 8, kRows = 4 * (32 / kLanes) * (kThreads / 32);
  grid_dependency_wait();
  if (status != nullptr && blockIdx.x == 0) {
    // (the call's status word: one block looks at all borders, so that the word is written once and no launch has to clear it before)
    int bad = 0;
    if constexpr (kPacked)
      for (int i = threadIdx.x; i < p.N; i += kThreads) bad |= p.cu_seqlens[i] < 0 || p.cu_seqlens[i + 1] < p.cu_seqlens[i] || p.cu_seqlens[i + 1] > p.T;
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) *status = bad ? kStatusBadCuSeqlens : kStatusOk;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = lane % kLanes;
  const int parts = p.P / kRows;
  const int chain = static_cast<int>(blockIdx.x) / parts, part = static_cast<int>(blockIdx.x) - chain * parts;
  const int n = chain / p.H, h = chain - n * p.H, group = h / (p.H / p.G);
  const int row = part * kRows + (warp * (32 / kLanes) + lane / kLanes) * 4;       // this thread's rows: row .. row + 3
  int64_t bos = 0, len = p.T, b = n;
  if constexpr (kPacked) {
    bos = p.cu_seqlens[n];
    int64_t eos = p.cu_seqlens[n + 1];
    bos = bos < 0 ? 0 : bos > p.T ? p.T : bos;
    eos = eos < bos ? bos : eos > p.T ? p.T : eos;
    len = eos - bos;
    if (most > 0 && len > most) return;
    b = 0;
  }
  const int64_t state = (static_cast<int64_t>(chain) * p.P + row) * kNs + 4 * j;
  f2 S[4][4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p.initial_state != nullptr) {
        const int64_t at = state + r * kNs + i * (kNs / 2);
        if constexpr (kFp32) {
          v = *reinterpret_cast<const float4*>(static_cast<const float*>(p.initial_state) + at);
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.initial_state) + at);
          v = make_float4(bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y));
        }
      }
      S[r][2 * i] = pk(v.x, v.y);
      S[r][2 * i + 1] = pk(v.z, v.w);
    }
  const float A = -kLog2e * ex2f(kLog2e * __ldg(p.A_log + h)), bias = __ldg(p.dt_bias + h);
  const float D = p.D != nullptr ? __ldg(p.D + h) : 0.f;
  const __nv_bfloat16* x = p.x + b * p.xs.batch + bos * p.xs.token + static_cast<int64_t>(h) * p.P + row;
  const __nv_bfloat16* dt = p.dt + b * p.dts.batch + bos * p.dts.token + h;
  const __nv_bfloat16* B = p.Bm + b * p.bs.batch + bos * p.bs.token + static_cast<int64_t>(group) * kNs + 4 * j;
  const __nv_bfloat16* C = p.Cm + b * p.cs.batch + bos * p.cs.token + static_cast<int64_t>(group) * kNs + 4 * j;
  __nv_bfloat16* out = p.out + b * p.os.batch + bos * p.os.token + static_cast<int64_t>(h) * p.P + row;

  struct Token {
    uint2 x, b[2], c[2];
    float dt;
  };
  auto load = [&](int64_t t) {
    Token k;
    k.x = __ldg(reinterpret_cast<const uint2*>(x + t * p.xs.token));
    k.dt = __bfloat162float(dt[t * p.dts.token]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      k.b[i] = __ldg(reinterpret_cast<const uint2*>(B + t * p.bs.token + i * (kNs / 2)));
      k.c[i] = __ldg(reinterpret_cast<const uint2*>(C + t * p.cs.token + i * (kNs / 2)));
    }
    return k;
  };
  Token next;
  if (len > 0) next = load(0);
  for (int64_t t = 0; t < len; ++t) {
    const Token k = next;
    if (t + 1 < len) next = load(t + 1);
    const float delta = softplus(k.dt + bias), decay = ex2f(A * delta);
    const float xr[4] = {bf_lo(k.x.x), bf_hi(k.x.x), bf_lo(k.x.y), bf_hi(k.x.y)};
    const f2 d2 = pk(decay, decay);
    float y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float dx = delta * xr[r];
      const f2 dx2 = pk(dx, dx);
      f2 acc = pk(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        S[r][2 * i] = fma2(S[r][2 * i], d2, mul(dx2, pk(bf_lo(k.b[i].x), bf_hi(k.b[i].x))));
        S[r][2 * i + 1] = fma2(S[r][2 * i + 1], d2, mul(dx2, pk(bf_lo(k.b[i].y), bf_hi(k.b[i].y))));
        acc = fma2(S[r][2 * i], pk(bf_lo(k.c[i].x), bf_hi(k.c[i].x)), acc);
        acc = fma2(S[r][2 * i + 1], pk(bf_lo(k.c[i].y), bf_hi(k.c[i].y)), acc);
      }
      float lo, hi;
      elem::upk(acc, lo, hi);
      y[r] = lo + hi;
    }
#pragma unroll
    for (int d = kLanes >> 1; d > 0; d >>= 1)
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] += __shfl_xor_sync(0xffffffffu, y[r], d);
    if (j == 0)
      *reinterpret_cast<uint2*>(out + t * p.os.token) =
          make_uint2(pack_bf16(fmaf(D, xr[0], y[0]), fmaf(D, xr[1], y[1])), pack_bf16(fmaf(D, xr[2], y[2]), fmaf(D, xr[3], y[3])));
  }
  if (p.final_state == nullptr) return;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t at = state + r * kNs + i * (kNs / 2);
      float a, c, e, f;
      elem::upk(S[r][2 * i], a, c);
      elem::upk(S[r][2 * i + 1], e, f);
      if constexpr (kFp32) *reinterpret_cast<float4*>(static_cast<float*>(p.final_state) + at) = make_float4(a, c, e, f);
      else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.final_state) + at) = make_uint2(pack_bf16(a, c), pack_bf16(e, f));
    }
}

template <int kNs>
cudaError_t launch(const SsmParams& p, int most, int* status, cudaStream_t stream) {
  const int64_t blocks = static_cast<int64_t>(p.N) * p.H * (p.P / (kNs == 128 ? 32 : 64));
  auto kernel = p.cu_seqlens != nullptr ? (p.state_fp32 ? ssm_step_kernel<kNs, true, true> : ssm_step_kernel<kNs, false, true>)
                                        : (p.state_fp32 ? ssm_step_kernel<kNs, true, false> : ssm_step_kernel<kNs, false, false>);
  return launch_after(kernel, dim3(static_cast<unsigned>(blocks)), kThreads, 0, stream, p, most, status);
}

}  // namespace ssm_step

cudaError_t launch_ssm_step(const SsmParams& p, int most, int* status, cudaStream_t stream) {
  return p.Ns == 128 ? ssm_step::launch<128>(p, most, status, stream) : ssm_step::launch<64>(p, most, status, stream);
}

}  // namespace fkda
