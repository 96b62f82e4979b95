// Depthwise causal convolution of 2 to 4 taps with bias and SiLU, over prompts, packed batches and single tokens.
//
// y[t][c] = act(bias[c] + sum_k w[c][k] x[t - (W-1) + k][c]).  A thread owns four channels (8 bytes) and walks a tile of tokens with
// the last W-1 inputs in registers, so that every input is read from memory once, but for the W-1 rows before each tile.
//
// Bound by memory: a read and a write an element, against some 30 instructions for four (two of them on the special function unit an
// element).  What is worked on fills 96 registers, so that an SM holds 640 threads, and one group of four rows each on its way in
// registers was 20 KB an SM, far from enough: 4 x 8192 x 4352 took 121 us.  Rows come by asynchronous copies through shared memory instead,
// each thread its own, four groups ahead, without a barrier: 92 us on the same tensors over and over, 6.2 TB/s read and written, and 105 on other ones
// each time, 5.4 TB/s.  (Over and over: three groups ahead 94, six 92; fewer registers - 72, seven blocks an SM - cost spills, 100; groups of two rows 106;
// prefetches into L2 in place of the copies 104.)
// Packed sequences of 1 to 300 tokens (30 thousand x 2048 with states) take 52 us, 4.9 TB/s: a sequence's start asks memory for its borders, then for
// its state and its last rows.
//
// States: the last W-1 inputs of a sequence.  Only the thread that owns a sequence's first token reads the initial state, and it
// writes the final one behind that (from the sequence's last rows), so the two may be one tensor; for that it also walks the tokens
// behind its tile that still see the initial state, which the next tile leaves out.
#include "fkda_elem.cuh"
#include "fkda_layer.cuh"

namespace fkda {
namespace conv {

using elem::f2;
using elem::fma2;
using elem::mul;
using elem::pk;

constexpr int kThreads = 128;
constexpr int kOwn = 4;            // channels of a thread
constexpr int kGroup = 4;          // tokens that are worked on together
constexpr int kAhead = 4;          // groups on their way meanwhile

__device__ __forceinline__ void cp_async8(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

__device__ __forceinline__ void unpack(const uint2& v, f2 (&x)[2]) {
  x[0] = pk(bf_lo(v.x), bf_hi(v.x));
  x[1] = pk(bf_lo(v.y), bf_hi(v.y));
}
__device__ __forceinline__ f2 silu(f2 y) {
  float a, b;
  elem::upk(mul(y, pk(-kLog2e, -kLog2e)), a, b);
  elem::upk(elem::add2(pk(ex2f(a), ex2f(b)), pk(1.f, 1.f)), a, b);
  return mul(y, pk(rcpf(a), rcpf(b)));
}

template <int W, bool kWFp32, bool kPacked, bool kSilu>
__global__ void __launch_bounds__(kThreads, 5) conv_kernel(const ConvParams p) {
  __shared__ uint2 ring[kAhead + 1][kGroup][kThreads];
  grid_dependency_wait();
  const unsigned vecs = static_cast<unsigned>(p.C) / kOwn;
  const int64_t flat = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t item = flat / vecs;
  const int c = static_cast<int>(flat - item * vecs) * kOwn;
  const int64_t items = static_cast<int64_t>(kPacked ? 1 : p.N) * p.tiles;
  if (item >= items) {
    // one more thread per sequence and channel vector, where there may be sequences without tokens: hands their state on
    const int64_t n = item - items;
    if (p.final_state == nullptr || n >= p.N || (kPacked ? p.cu_seqlens[n + 1] > p.cu_seqlens[n] : p.T > 0)) return;
    for (int j = 0; j < W - 1; ++j) {
      const int64_t at = (n * (W - 1) + j) * p.C + c;
      uint2 v = make_uint2(0u, 0u);
      if (p.initial_state != nullptr) v = *reinterpret_cast<const uint2*>(p.initial_state + at);
      *reinterpret_cast<uint2*>(p.final_state + at) = v;
    }
    return;
  }
  int64_t n = 0, t, bos = 0, eos = p.T;           // sequence, token, the sequence's first token and end (equal lengths: within it)
  const __nv_bfloat16* x = p.x + c;
  __nv_bfloat16* out = p.out + c;
  if constexpr (kPacked) {
    t = item * p.tile;
    int64_t lo = 0, hi = p.N;                     // the last sequence that starts at or before t
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (p.cu_seqlens[mid] <= t) lo = mid; else hi = mid;
    }
    n = lo;
    bos = p.cu_seqlens[n];
    eos = p.cu_seqlens[n + 1];
    if (bos < 0) bos = 0;
    if (eos > p.T) eos = p.T;
  } else {
    n = item / p.tiles;
    t = (item - n * p.tiles) * p.tile;
    x += n * p.xs.batch;
    out += n * p.os.batch;
  }
  const int64_t t0 = t, end = t + p.tile < p.T ? t + p.tile : p.T;
  if (bos > t) t = bos;                           // (rows before the first sequence)
  if (bos < t0 && t < bos + W - 1) t = bos + W - 1 < eos ? bos + W - 1 : eos;

  f2 w[W][2], b[2];                               // pairs of channels
  {
    float all[kOwn * W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float4 v = load4<kWFp32>(p.weight, static_cast<int64_t>(c) * W + 4 * i);
      all[4 * i] = v.x;
      all[4 * i + 1] = v.y;
      all[4 * i + 2] = v.z;
      all[4 * i + 3] = v.w;
    }
    const float4 v = p.bias != nullptr ? load4<kWFp32>(p.bias, c) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float bias[kOwn] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      b[e] = pk(bias[2 * e], bias[2 * e + 1]);
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][e] = pk(all[2 * e * W + j], all[(2 * e + 1) * W + j]);
    }
  }
  f2 u[W - 1 + kGroup][2];                        // the inputs that reach back, then a group's own
  auto result = [&](int i) {
    f2 y[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      y[e] = b[e];
#pragma unroll
      for (int j = 0; j < W; ++j) y[e] = fma2(w[j][e], u[i + j][e], y[e]);
      if constexpr (kSilu) y[e] = silu(y[e]);
    }
    return make_uint2(elem::round_bf(y[0]), elem::round_bf(y[1]));
  };
  while (true) {
    if (t >= eos) {
      if constexpr (!kPacked) break;
      int64_t next = eos;
      while (++n < p.N) {                         // on to the next sequence with tokens
        bos = p.cu_seqlens[n];
        next = p.cu_seqlens[n + 1];
        if (next > p.T) next = p.T;
        if (next > bos && next > t) break;
      }
      if (n >= p.N) break;
      if (bos < t) bos = t;                       // (only where cu_seqlens is not monotone)
      t = bos;
      eos = next;
    }
    const int64_t limit = bos >= t0 && bos + W - 1 > end ? (bos + W - 1 < eos ? bos + W - 1 : eos) : (end < eos ? end : eos);
    if (t >= limit || (bos >= end && t >= end)) break;
    const __nv_bfloat16* from = x + t * p.xs.token;
    __nv_bfloat16* to = out + t * p.os.token;
    int left = static_cast<int>(limit - t);
    // groups on the way to shared memory, each thread's own
    auto ask = [&](int ahead, int slot) {          // (`ahead` groups from `from`)
      if (left >= (ahead + 1) * kGroup) {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) cp_async8(smem_u32(&ring[slot][i][threadIdx.x]), from + (ahead * kGroup + i) * p.xs.token);
      }
      cp_async_commit();
    };
    int slot = 0;
#pragma unroll
    for (int g = 0; g < kAhead; ++g) ask(g, g);
    {
      auto row_at = [&](int64_t at) {             // (rows before the sequence: of its initial state)
        if (at >= bos) return *reinterpret_cast<const uint2*>(x + at * p.xs.token);
        if (p.initial_state != nullptr) return *reinterpret_cast<const uint2*>(p.initial_state + (n * (W - 1) + (W - 1) + at - bos) * p.C + c);
        return make_uint2(0u, 0u);
      };
      const bool leave = t == bos && p.final_state != nullptr;
      uint2 back[W - 1], last[W - 1];
#pragma unroll
      for (int j = 0; j < W - 1; ++j) back[j] = row_at(t - (W - 1) + j);
      if (leave) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) last[j] = row_at(eos - (W - 1) + j);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) *reinterpret_cast<uint2*>(p.final_state + (n * (W - 1) + j) * p.C + c) = last[j];
      }
#pragma unroll
      for (int j = 0; j < W - 1; ++j) unpack(back[j], u[j]);
    }
    for (; left >= kGroup; left -= kGroup) {
      cp_async_wait<kAhead - 1>();
#pragma unroll
      for (int i = 0; i < kGroup; ++i) unpack(ring[slot][i][threadIdx.x], u[W - 1 + i]);
      ask(kAhead, slot == 0 ? kAhead : slot - 1);     // (into the slot of the group before, whose rows are in use no more)
      slot = slot == kAhead ? 0 : slot + 1;
      from += kGroup * p.xs.token;
#pragma unroll
      for (int i = 0; i < kGroup; ++i) *reinterpret_cast<uint2*>(to + i * p.os.token) = result(i);
      to += kGroup * p.os.token;
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) u[j][e] = u[kGroup + j][e];
    }
    if (left > 0) {                             // (what is left of a group: nothing follows on it)
      uint2 in[kGroup - 1];
#pragma unroll
      for (int i = 0; i < kGroup - 1; ++i)
        if (i < left) in[i] = *reinterpret_cast<const uint2*>(from + i * p.xs.token);
#pragma unroll
      for (int i = 0; i < kGroup - 1; ++i) {
        if (i >= left) break;
        unpack(in[i], u[W - 1 + i]);
        *reinterpret_cast<uint2*>(to + i * p.os.token) = result(i);
      }
    }
    t = limit;
    if (t >= end && t < eos) break;
  }
}

template <int W, bool kWFp32, bool kPacked>
auto pick(bool silu) { return silu ? conv_kernel<W, kWFp32, kPacked, true> : conv_kernel<W, kWFp32, kPacked, false>; }

template <int W>
cudaError_t launch(const ConvParams& p, bool weight_fp32, cudaStream_t stream) {
  const bool packed = p.cu_seqlens != nullptr;
  const int64_t items = (packed ? 1 : static_cast<int64_t>(p.N)) * p.tiles + (p.final_state != nullptr && (packed || p.T == 0) ? p.N : 0);
  const int64_t blocks = (items * (p.C / kOwn) + kThreads - 1) / kThreads;
  if (blocks == 0) return cudaSuccess;
  auto kernel = packed ? (weight_fp32 ? pick<W, true, true>(p.silu) : pick<W, false, true>(p.silu)) : (weight_fp32 ? pick<W, true, false>(p.silu) : pick<W, false, false>(p.silu));
  return launch_after(kernel, dim3(static_cast<unsigned>(blocks)), kThreads, 0, stream, p);
}

}  // namespace conv

cudaError_t launch_short_conv(ConvParams p, int width, bool weight_fp32, cudaStream_t stream) {
  const bool packed = p.cu_seqlens != nullptr;
  const int64_t vectors = static_cast<int64_t>(packed ? 1 : p.N) * p.T * (p.C / conv::kOwn);
  // Tokens per thread: as many as leave every SM a thousand threads (the rows before a tile are read again, 3 of 64, and its weights; 128 tokens took
  // 96 us where 64 take 92), but no fewer than the taps that reach back: only a sequence's first tile may see its initial state.
  int tile = 64;
  while (tile > 4 && vectors / tile < 1024ll * device_sm_count()) tile >>= 1;
  p.tile = !packed && p.T < tile ? static_cast<int>(p.T > 0 ? p.T : 1) : tile;
  p.tiles = static_cast<int>((p.T + p.tile - 1) / p.tile);
  switch (width) {
    case 2: return conv::launch<2>(p, weight_fp32, stream);
    case 3: return conv::launch<3>(p, weight_fp32, stream);
    default: return conv::launch<4>(p, weight_fp32, stream);
  }
}

}  // namespace fkda
