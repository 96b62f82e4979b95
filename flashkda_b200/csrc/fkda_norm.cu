// Root-mean-square norms before and after the recurrence's block: with its gate, and with the residual stream.
//
//   gated_norm   out = x / rms(x) w a(g)  or  (x a) / rms(x a) w,  a = sigmoid(g) or g sigmoid(g)
//   add_norm     h = residual + scale x -> residual_out;  out = h / rms(h) w
//
// One pass: a row lives in the registers of the threads that share it, eight elements (16 bytes of bf16) at a time, from its loads to its
// stores; the sum of squares is fp32.  Rows of up to 1024 elements are shared by 8 to 32 lanes of a warp, longer ones by a block.
//
// Bound by memory: 6 bytes an element (gated), 8 or 12 (residual stream in bf16 or fp32).  4 x 8192 rows of 32 x 128 with their gate take 142 us, 5.7 TB/s:
// arithmetic on pairs, and four of these short rows a thread, without which there were too few loads on the way (185 us); 4 x 8192 rows of 4096 with an
// fp32 residual stream 234 us, 6.9 TB/s.  A step of 64 rows takes 3.3 us, the launch.
#include "fkda_elem.cuh"
#include "fkda_layer.cuh"

namespace fkda {
namespace norm {

// Sum over the `lanes` threads that share a row (a power of two up to 32), or over the block.
template <bool kBlock>
__device__ __forceinline__ float row_sum(float x, int lanes, float* scratch) {
  const int width = kBlock ? 32 : lanes;
  for (int d = width >> 1; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  if constexpr (kBlock) {
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0.f;
    for (int i = 0; i < warps; ++i) x += scratch[i];
  }
  return x;
}

// Where the row that this thread works on starts, and which eight-element pieces of it are its own: lane, lane + lanes, ...
struct Place {
  int64_t row;
  int lane, lanes;
  bool live;
};
template <bool kBlock>
__device__ __forceinline__ Place place(int64_t rows, int lanes) {
  Place w;
  if constexpr (kBlock) {
    w.row = blockIdx.x;
    w.lane = threadIdx.x;
    w.lanes = blockDim.x;
  } else {
    const int per = blockDim.x / lanes;
    w.row = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / lanes;
    w.lane = threadIdx.x % lanes;
    w.lanes = lanes;
  }
  w.live = w.row < rows;
  if (!w.live) w.row = rows - 1;               // (takes part in the sums, stores nothing)
  return w;
}
__device__ __forceinline__ int64_t at_token(const Rows& s, unsigned token, int64_t T) {
  if (T > 0x7fffffff) return token * s.token;                      // (one row of tokens)
  const unsigned b = token / static_cast<unsigned>(T);
  return b * s.batch + (token - b * static_cast<unsigned>(T)) * s.token;
}

using elem::f2;
using elem::fma2;
using elem::mul;
using elem::pk;
__device__ __forceinline__ void unpack(const uint4& v, f2 (&x)[4]) {
  x[0] = pk(bf_lo(v.x), bf_hi(v.x));
  x[1] = pk(bf_lo(v.y), bf_hi(v.y));
  x[2] = pk(bf_lo(v.z), bf_hi(v.z));
  x[3] = pk(bf_lo(v.w), bf_hi(v.w));
}
// u a(g).  (a first: where it is 0, u g may be beyond the largest number already)
template <bool kSilu>
__device__ __forceinline__ f2 gated(f2 u, f2 g) {
  float a, b;
  elem::upk(mul(g, pk(-kLog2e, -kLog2e)), a, b);
  elem::upk(elem::add2(pk(ex2f(a), ex2f(b)), pk(1.f, 1.f)), a, b);
  f2 act = pk(rcpf(a), rcpf(b));
  if constexpr (kSilu) act = mul(act, g);
  return mul(u, act);
}

// kBatch: rows of a thread, whose loads are in flight together (rows of a head of 128 channels are 16 bytes a lane each).
template <bool kBlock, int V, bool kWFp32, bool kSilu, bool kFirst, int kBatch>
__global__ void gated_norm_kernel(const GatedNormParams p, int lanes) {
  __shared__ float scratch[kBatch][32];
  grid_dependency_wait();
  const int pieces = p.D / 8, per = kBlock ? 1 : blockDim.x / lanes;
  const int lane = kBlock ? threadIdx.x : threadIdx.x % lanes, step = kBlock ? blockDim.x : lanes;
  uint4 xw[kBatch][V], gw[kBatch][V];
  unsigned token[kBatch], h[kBatch];
  bool live[kBatch];
#pragma unroll
  for (int r = 0; r < kBatch; ++r) {
    unsigned row = (blockIdx.x * kBatch + r) * per + (kBlock ? 0 : threadIdx.x / lanes);
    live[r] = row < p.rows;
    if (!live[r]) row = static_cast<unsigned>(p.rows) - 1;         // (takes part in the sums, stores nothing)
    token[r] = row / static_cast<unsigned>(p.H);
    h[r] = row - token[r] * static_cast<unsigned>(p.H);
    const __nv_bfloat16* x = p.x + at_token(p.xs, token[r], p.T) + static_cast<int64_t>(h[r]) * p.D;
    const __nv_bfloat16* g = p.gate + at_token(p.gs, token[r], p.T) + static_cast<int64_t>(h[r]) * p.D;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = lane + i * step;
      xw[r][i] = gw[r][i] = make_uint4(0u, 0u, 0u, 0u);
      if (c < pieces) {
        xw[r][i] = *reinterpret_cast<const uint4*>(x + 8 * c);
        gw[r][i] = *reinterpret_cast<const uint4*>(g + 8 * c);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kBatch; ++r) {
    f2 u[V][4], sum = pk(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      f2 g[4];
      unpack(xw[r][i], u[i]);
      unpack(gw[r][i], g);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (kFirst) u[i][e] = gated<kSilu>(u[i][e], g[e]);
        sum = fma2(u[i][e], u[i][e], sum);
      }
    }
    float lo, hi;
    elem::upk(sum, lo, hi);
    const float root = rsqrtf(row_sum<kBlock>(lo + hi, lanes, scratch[r]) / static_cast<float>(p.D) + p.eps);
    if (!live[r]) continue;
    __nv_bfloat16* out = p.out + at_token(p.os, token[r], p.T) + static_cast<int64_t>(h[r]) * p.D;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = lane + i * step;
      if (c >= pieces) break;
      float w[8];
      load8<kWFp32>(p.weight, (p.per_head ? static_cast<int64_t>(h[r]) * p.D : 0) + 8 * c, w);
      f2 g[4];
      unpack(gw[r][i], g);
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f2 y = mul(u[i][e], mul(pk(root, root), pk(w[2 * e], w[2 * e + 1])));
        if constexpr (!kFirst) y = gated<kSilu>(y, g[e]);
        o[e] = elem::round_bf(y);
      }
      *reinterpret_cast<uint4*>(out + 8 * c) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

template <bool kBlock, int V, bool kWFp32, bool kRFp32>
__global__ void add_norm_kernel(const AddNormParams p, int lanes) {
  __shared__ float scratch[32];
  grid_dependency_wait();
  const Place at = place<kBlock>(p.rows, lanes);
  const int pieces = p.D / 8;
  const __nv_bfloat16* x = p.x + at_token(p.xs, static_cast<unsigned>(at.row), p.T);
  const int64_t from = at_token(p.rs, static_cast<unsigned>(at.row), p.T);
  uint4 xw[V];
  float u[V][8], sum = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = at.lane + i * at.lanes;
    xw[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int e = 0; e < 8; ++e) u[i][e] = 0.f;
    if (c < pieces) {
      xw[i] = *reinterpret_cast<const uint4*>(x + 8 * c);
      if constexpr (kRFp32) {
        const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p.residual) + from + 8 * c);
        const float4 a = q[0], b = q[1];
        u[i][0] = a.x; u[i][1] = a.y; u[i][2] = a.z; u[i][3] = a.w; u[i][4] = b.x; u[i][5] = b.y; u[i][6] = b.z; u[i][7] = b.w;
      } else {
        unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.residual) + from + 8 * c), u[i]);
      }
    }
  }
  const int64_t to = at_token(p.ros, static_cast<unsigned>(at.row), p.T);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = at.lane + i * at.lanes;
    float xf[8];
    unpack8(xw[i], xf);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      u[i][e] = fmaf(p.scale, xf[e], u[i][e]);
      sum = fmaf(u[i][e], u[i][e], sum);
    }
    if (c < pieces && at.live) {
      if constexpr (kRFp32) {
        float4* q = reinterpret_cast<float4*>(static_cast<float*>(p.residual_out) + to + 8 * c);
        q[0] = make_float4(u[i][0], u[i][1], u[i][2], u[i][3]);
        q[1] = make_float4(u[i][4], u[i][5], u[i][6], u[i][7]);
      } else {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.residual_out) + to + 8 * c) = pack8(u[i]);
      }
    }
  }
  const float r = rsqrtf(row_sum<kBlock>(sum, lanes, scratch) / static_cast<float>(p.D) + p.eps);
  if (!at.live) return;
  __nv_bfloat16* out = p.out + at_token(p.os, static_cast<unsigned>(at.row), p.T);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = at.lane + i * at.lanes;
    if (c >= pieces) break;
    float w[8];
    load8<kWFp32>(p.weight, 8 * c, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) u[i][e] *= r * w[e];
    *reinterpret_cast<uint4*>(out + 8 * c) = pack8(u[i]);
  }
}

// How a row of D elements is shared: lanes per row and pieces per lane, or a block of `threads`.
struct Split {
  bool block;
  int v, lanes, threads;
};
inline Split split_of(int D) {
  const int pieces = D / 8;
  if (pieces <= 128) {
    int lanes = 8;
    while (lanes < 32 && lanes < pieces) lanes <<= 1;
    return Split{false, pieces <= lanes ? 1 : pieces <= 2 * lanes ? 2 : 4, lanes, 256};
  }
  int threads = 128;
  while (threads < 512 && threads * 2 < pieces) threads <<= 1;      // two pieces a thread up to 8192 elements, four beyond
  return Split{true, pieces <= 2 * threads ? 2 : 4, 0, threads};
}

}  // namespace norm

// (kernel template of norm with <kBlock, V> resolved from a Split)
#define FKDA_NORM_PICK(name, s, ...)                                                                                       \
  ((s).block ? ((s).v == 2 ? norm::name<true, 2, __VA_ARGS__> : norm::name<true, 4, __VA_ARGS__>)                          \
             : ((s).v == 1 ? norm::name<false, 1, __VA_ARGS__> : (s).v == 2 ? norm::name<false, 2, __VA_ARGS__> : norm::name<false, 4, __VA_ARGS__>))

namespace norm {
template <bool kWFp32, bool kSilu, bool kFirst>
void (*pick_gated(const Split& s, bool four))(GatedNormParams, int) {
  if (four) return gated_norm_kernel<false, 1, kWFp32, kSilu, kFirst, 4>;
  return FKDA_NORM_PICK(gated_norm_kernel, s, kWFp32, kSilu, kFirst, 1);
}
}  // namespace norm

cudaError_t launch_gated_norm(const GatedNormParams& p, bool weight_fp32, bool silu, bool gate_first, cudaStream_t stream) {
  if (p.rows == 0) return cudaSuccess;
  const norm::Split s = norm::split_of(p.D);
  // Four short rows a thread once there are enough rows for that to leave every SM two thousand threads.
  const bool four = !s.block && s.v == 1 && p.rows * s.lanes >= 4 * 2048ll * device_sm_count();
  const int64_t per = s.block ? 1 : s.threads / s.lanes * (four ? 4 : 1);
  const dim3 grid(static_cast<unsigned>((p.rows + per - 1) / per));
  void (*kernel)(GatedNormParams, int);
  if (weight_fp32) kernel = silu ? (gate_first ? norm::pick_gated<true, true, true>(s, four) : norm::pick_gated<true, true, false>(s, four))
                                 : (gate_first ? norm::pick_gated<true, false, true>(s, four) : norm::pick_gated<true, false, false>(s, four));
  else kernel = silu ? (gate_first ? norm::pick_gated<false, true, true>(s, four) : norm::pick_gated<false, true, false>(s, four))
                     : (gate_first ? norm::pick_gated<false, false, true>(s, four) : norm::pick_gated<false, false, false>(s, four));
  return launch_after(kernel, grid, static_cast<unsigned>(s.threads), 0, stream, p, s.lanes);
}

cudaError_t launch_add_norm(const AddNormParams& p, bool weight_fp32, bool residual_fp32, cudaStream_t stream) {
  if (p.rows == 0) return cudaSuccess;
  const norm::Split s = norm::split_of(p.D);
  const int64_t per = s.block ? 1 : s.threads / s.lanes;
  const dim3 grid(static_cast<unsigned>((p.rows + per - 1) / per));
  void (*kernel)(AddNormParams, int) = weight_fp32 ? (residual_fp32 ? FKDA_NORM_PICK(add_norm_kernel, s, true, true) : FKDA_NORM_PICK(add_norm_kernel, s, true, false))
                                                   : (residual_fp32 ? FKDA_NORM_PICK(add_norm_kernel, s, false, true) : FKDA_NORM_PICK(add_norm_kernel, s, false, false));
  return launch_after(kernel, grid, static_cast<unsigned>(s.threads), 0, stream, p, s.lanes);
}

}  // namespace fkda
