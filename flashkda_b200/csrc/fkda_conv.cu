// Depthwise causal convolution of 2 to 4 taps with bias and SiLU, over prompts, packed batches and single tokens.
//
// y[t][c] = act(bias[c] + sum_k w[c][k] x[t - (W-1) + k][c]).  A thread owns eight channels (16 bytes) and walks a tile of tokens with
// the last W-1 inputs in registers, so that every input is read from memory once, but for the W-1 rows before each tile.
// States: the last W-1 inputs of a sequence.  Only the thread that owns a sequence's first token reads the initial state, and it
// writes the final one behind that (from the sequence's last rows), so the two may be one tensor; for that it also walks the tokens
// behind its tile that still see the initial state, which the next tile leaves out.
#include "fkda_layer.cuh"

namespace fkda {
namespace conv {

constexpr int kThreads = 128;
constexpr int kGroup = 4;          // tokens whose loads are in flight together

template <int W, bool kWFp32, bool kPacked>
__global__ void __launch_bounds__(kThreads) conv_kernel(const ConvParams p) {
  grid_dependency_wait();
  const unsigned vecs = static_cast<unsigned>(p.C) / 8;
  const int64_t flat = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t item = flat / vecs;
  const int c = static_cast<int>(flat - item * vecs) * 8;
  const int64_t items = static_cast<int64_t>(kPacked ? 1 : p.N) * p.tiles;
  if (item >= items) {
    // one more thread per sequence and channel vector, where there may be sequences without tokens: hands their state on
    const int64_t n = item - items;
    if (p.final_state == nullptr || n >= p.N || (kPacked ? p.cu_seqlens[n + 1] > p.cu_seqlens[n] : p.T > 0)) return;
    for (int j = 0; j < W - 1; ++j) {
      const int64_t at = (n * (W - 1) + j) * p.C + c;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (p.initial_state != nullptr) v = *reinterpret_cast<const uint4*>(p.initial_state + at);
      *reinterpret_cast<uint4*>(p.final_state + at) = v;
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

  float w[8 * W], b[8];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    float part[8];
    load8<kWFp32>(p.weight, static_cast<int64_t>(c) * W + 8 * i, part);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[8 * i + e] = part[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = 0.f;
  if (p.bias != nullptr) load8<kWFp32>(p.bias, c, b);

  float past[W - 1][8];
  bool fresh = true;                              // `past` has to be loaded
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
      fresh = true;
    }
    const int64_t limit = bos >= t0 && bos + W - 1 > end ? (bos + W - 1 < eos ? bos + W - 1 : eos) : (end < eos ? end : eos);
    if (t >= limit || (bos >= end && t >= end)) break;
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        const int64_t at = t - (W - 1) + j;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (at >= bos) v = *reinterpret_cast<const uint4*>(x + at * p.xs.token);
        else if (p.initial_state != nullptr) v = *reinterpret_cast<const uint4*>(p.initial_state + (n * (W - 1) + (W - 1) + at - bos) * p.C + c);
        unpack8(v, past[j]);
      }
      if (t == bos && p.final_state != nullptr) {
        uint4 last[W - 1];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
          const int64_t at = eos - (W - 1) + j;
          last[j] = make_uint4(0u, 0u, 0u, 0u);
          if (at >= bos) last[j] = *reinterpret_cast<const uint4*>(x + at * p.xs.token);
          else if (p.initial_state != nullptr) last[j] = *reinterpret_cast<const uint4*>(p.initial_state + (n * (W - 1) + (W - 1) + at - bos) * p.C + c);
        }
#pragma unroll
        for (int j = 0; j < W - 1; ++j) *reinterpret_cast<uint4*>(p.final_state + (n * (W - 1) + j) * p.C + c) = last[j];
      }
    }
    for (; t < limit; t += kGroup) {
      uint4 in[kGroup];
#pragma unroll
      for (int i = 0; i < kGroup; ++i)
        if (t + i < limit) in[i] = *reinterpret_cast<const uint4*>(x + (t + i) * p.xs.token);
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        if (t + i >= limit) break;
        float now[8], y[8];
        unpack8(in[i], now);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] = b[e];
#pragma unroll
          for (int j = 0; j < W - 1; ++j) y[e] = fmaf(w[e * W + j], past[j][e], y[e]);
          y[e] = fmaf(w[e * W + W - 1], now[e], y[e]);
#pragma unroll
          for (int j = 0; j + 1 < W - 1; ++j) past[j][e] = past[j + 1][e];
          past[W - 2][e] = now[e];
        }
        if (p.silu) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] *= sigmoid_exact(y[e]);
        }
        *reinterpret_cast<uint4*>(out + (t + i) * p.os.token) = pack8(y);
      }
    }
    t = limit;
    if (t >= end && t < eos) break;
  }
}

template <int W>
cudaError_t launch(const ConvParams& p, bool weight_fp32, cudaStream_t stream) {
  const bool packed = p.cu_seqlens != nullptr;
  const int64_t items = (packed ? 1 : static_cast<int64_t>(p.N)) * p.tiles + (p.final_state != nullptr && (packed || p.T == 0) ? p.N : 0);
  const int64_t blocks = (items * (p.C / 8) + kThreads - 1) / kThreads;
  if (blocks == 0) return cudaSuccess;
  auto kernel = packed ? (weight_fp32 ? conv_kernel<W, true, true> : conv_kernel<W, false, true>)
                       : (weight_fp32 ? conv_kernel<W, true, false> : conv_kernel<W, false, false>);
  return launch_after(kernel, dim3(static_cast<unsigned>(blocks)), kThreads, 0, stream, p);
}

}  // namespace conv

cudaError_t launch_short_conv(ConvParams p, int width, bool weight_fp32, cudaStream_t stream) {
  const bool packed = p.cu_seqlens != nullptr;
  const int64_t vectors = static_cast<int64_t>(packed ? 1 : p.N) * p.T * (p.C / 8);
  // Tokens per thread: as many as leave every SM two thousand threads (the rows before a tile are read again, 3 of 16), but no
  // fewer than the taps that reach back: only a sequence's first tile may see its initial state.
  int tile = 16;
  while (tile > 4 && vectors / tile < 2048ll * device_sm_count()) tile >>= 1;
  p.tile = !packed && p.T < tile ? static_cast<int>(p.T > 0 ? p.T : 1) : tile;
  p.tiles = static_cast<int>((p.T + p.tile - 1) / p.tile);
  switch (width) {
    case 2: return conv::launch<2>(p, weight_fp32, stream);
    case 3: return conv::launch<3>(p, weight_fp32, stream);
    default: return conv::launch<4>(p, weight_fp32, stream);
  }
}

}  // namespace fkda
