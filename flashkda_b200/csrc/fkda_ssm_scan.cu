// Selective state space scan in blocks of 128 tokens on tcgen05: prompts.
//
// With a = -exp(A_log) delta log2(e) the log2 decay of a token, l_i its running sum from the block's start and S the state [P][Ns]
// before the block (per head),
//     G = C B^T,   M_ij = G_ij 2^(l_i - l_j) delta_j  (j <= i),   out = M X + 2^(l_i) (C S^T) + D X
//     S <- 2^(l_127) S + X'^T B,   x'_j = 2^(l_127 - l_j) delta_j x_j
// A CTA walks the blocks of 128 rows of a sequence's states: two heads of P = 64 that share B and C, or one of P = 128.  Five products a block,
// 128 x 128 x 128 each (two of them X'^T B): G, Z = C S^T, X' as hi + lo (below), Y = M X.  Nineteen warps:
//     0-7    M from G, in tensor memory over G itself (rows i = lanes; the even warpgroup takes the column blocks 0 and 2, the odd one 1 and 3), then
//            out = Y + 2^l Z + D x over the tile of x in shared memory, from where a tensor copy takes it
//     8-11   the state: fp32 in tensor memory, once a block read, rescaled and written back, and its bf16 copy for Z
//     12-15  delta and the decays of the next block; x' in steps of 16 tokens
//     16     loads of B and C       17     products       18     loads of x, stores of out
//
// Roundings: G, Y, Z and S accumulate in fp32.  M and the state's copy for Z are bf16 operands, as out is bf16.  The state is what a
// caller keeps, so X' goes into its product as hi + lo, two bf16 parts that hold 16 bits, where the state is asked for in fp32; where it is
// asked for in bf16, or not at all, as one.
// Decays: every exponent that is evaluated is a sum of terms of one sign, so that nothing cancels, but for those within 32 x 32 blocks on
// the diagonal, which are differences of sums over less than 32 tokens.
// Rows past a sequence's end are zeroed in the tiles of x and B where they are summed over; those of C only reach outputs that are not stored.
#include "fkda_elem.cuh"
#include "fkda_layer.cuh"
#include "fkda_ssm.cuh"
#include "fkda_tma.cuh"

namespace fkda {
namespace ssm_scan {

constexpr int kQ = kSsmBlock;
constexpr int kThreads = 19 * 32;
constexpr int kSlots = 3;                        // steps of x' under way
constexpr int kSlotBytes = 2 * 16 * 128 * 2;     // hi | lo, each [2 halves of 64 columns][16 tokens][128 B]
constexpr int kTileX = kQ * 128 * 2;
constexpr uint32_t kColG = 0, kColY = 128, kColZ = 256, kColS = 384;     // tensor memory; M lies over G

// Per block and head, written by warps 12-15.
struct Scalars {
  float p[2][kQ];          // running sum of a from the start of the token's 32-token block, itself included
  float lp[2][kQ];         // p - log2(delta)
  float f[2][kQ];          // delta 2^(sum of a behind the token to the end of its 32-token block)
  float w[2][kQ];          // ... to the end of the block of 128
  float tot[2][4];         // sums over the four 32-token blocks
  float decay[2];          // 2^(sum over all)
  float pad[6];
};

template <int kNs>
struct Smem {
  static constexpr int kTile = kQ * kNs * 2;
  static constexpr int kB = 0, kC = kB + 2 * kTile, kX = kC + kTile, kS = kX + 2 * kTileX, kXp = kS + 128 * kNs * 2;
  static constexpr int kScal = kXp + kSlots * kSlotBytes, kBars = kScal + 2 * static_cast<int>(sizeof(Scalars)), kMisc = kBars + 256;
  static constexpr int kBytes = kMisc + 64;
};
static_assert(Smem<128>::kBytes <= 227 * 1024, "shared memory of a CTA");

enum {
  B_FULL_B = 0 /*[2]*/, B_EMPTY_B = 2 /*[2]*/, B_FULL_C = 4, B_EMPTY_C, B_FULL_X /*[2]*/, B_EMPTY_X = 8 /*[2]*/, B_XP_FULL = 10 /*[kSlots]*/, B_XP_EMPTY = 13 /*[kSlots]*/,
  B_SCAL = 16 /*[2]*/, B_SCAL_FREE = 18 /*[2]*/, B_G = 20, B_M, B_Y, B_ZY_FREE, B_S_FULL, B_S_READY, B_OUT /*[2]*/, B_DRAIN = 28, B_MEET, B_COUNT
};
static_assert(B_COUNT * 8 <= 256, "barrier area");

// Shared-memory matrix descriptor of a tile with the 128-byte swizzle (rows of 128 bytes, 1024-byte aligned groups of eight).  K-major: `sbo`
// is the distance between groups of eight rows (M or N), 16 elements along K are 32 bytes on.  MN-major (rows along K): `sbo` is the
// distance between groups of eight rows along K, `lbo` between blocks of 64 elements of M or N.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lbo) { return umma_desc(addr, lbo, 1024) | (2ull << 61); }

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait_parked(bar, parity, abort_flag));
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// After a wait has given up: the copies under way land in this CTA's memory, which has to stay its own until then.
__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_test(bar, parity) && globaltimer_ns() - t0 < 20000000ull) {
  }
}
// 2^-|x| is at most 1, so neither branch overflows.
__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(ex2f(-kLog2e * fabsf(x))); }
using elem::f2;
using elem::fma2;
using elem::mul;
using elem::pk;
using elem::upk;
__device__ __forceinline__ f2 pk(uint32_t a, uint32_t b) { return elem::pk(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ uint32_t round2(f2 x) { return elem::round_bf(x); }

// kWide: one head of P = 128, else two of P = 64.  kFull: the outputs too, else only what a run adds to a zero state.
template <int kNs, bool kWide, bool kFull>
__global__ void __launch_bounds__(kThreads, 1) ssm_scan_kernel(const __grid_constant__ SsmMaps maps, const SsmScanParams p) {
  using L = Smem<kNs>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  auto bar = [&](int i) { return sbase + L::kBars + 8 * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc + 4);
  Scalars* scal = reinterpret_cast<Scalars*>(smem + L::kScal);

  if (tid == 0) {
    // the swizzled tiles need this alignment: report instead of computing garbage (below zero: a wait limit, test aid)
    *abort_flag = (sbase & 1023u) != 0u ? 1 : -p.wait_limit_us;
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(B_FULL_B + i), 1);
      mbar_init(bar(B_EMPTY_B + i), 1);
      mbar_init(bar(B_FULL_X + i), 1);
      mbar_init(bar(B_EMPTY_X + i), 4);
      mbar_init(bar(B_SCAL + i), 4);
      mbar_init(bar(B_SCAL_FREE + i), 8);
      mbar_init(bar(B_OUT + i), 8);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(bar(B_XP_FULL + i), 4);
      mbar_init(bar(B_XP_EMPTY + i), 1);
    }
    mbar_init(bar(B_FULL_C), 1);
    mbar_init(bar(B_EMPTY_C), 1);
    mbar_init(bar(B_G), 1);
    mbar_init(bar(B_M), 8);
    mbar_init(bar(B_Y), 1);
    mbar_init(bar(B_ZY_FREE), 8);
    mbar_init(bar(B_S_FULL), 1);
    mbar_init(bar(B_S_READY), 4);
    mbar_init(bar(B_DRAIN), 1);
    mbar_init(bar(B_MEET), 4);
    fence_mbar_init();
  }
  if (warp == 17) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  bool ok = *abort_flag <= 0;
  grid_dependency_wait();
  const SsmItem it = ssm_item(p, blockIdx.x, kFull);
  const int blocks = ok ? it.blocks : 0;

  if (warp < 8) {
    if constexpr (kFull) {
      const int q = warp >> 2, w = warp & 3;                          // column blocks q, q + 2; rows 32 w + lane
      const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * w) << 16);
      const int head = it.head0 + (kWide ? 0 : q);
      const bool mine = kWide || q == 0 || it.two;
      const float D = p.D != nullptr && mine ? __ldg(p.D + head) : 0.f;
      for (int c = 0; c < blocks; ++c) {
        const Scalars& s = scal[c & 1];
        if (!(ok = warp_wait(bar(B_SCAL + (c & 1)), (c >> 1) & 1, abort_flag))) break;
        if (!(ok = warp_wait(bar(B_G), c & 1, abort_flag))) break;
        tc_fence_after();
        float pi[2];
#pragma unroll
        for (int h = 0; h < (kWide ? 1 : 2); ++h) pi[h] = s.p[h][32 * w + lane];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int b = q + 2 * k;
          if (b > w) {
            uint32_t zero[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) zero[i] = 0u;
            tmem_st32(lanes + kColG + 32 * b, zero);
            continue;
          }
          uint32_t g[32];
          tmem_ld32(lanes + kColG + 32 * b, g);
          tmem_wait_ld();
#pragma unroll
          for (int h = 0; h < (kWide ? 1 : 2); ++h) {
            uint32_t m[16];
            if (b < w) {
              float between = 0.f;                                    // (sums over the 32-token blocks between the two)
              if (b < 1 && w > 1) between += s.tot[h][1];
              if (b < 2 && w > 2) between += s.tot[h][2];
              const float r = ex2f(pi[h] + between);
              const f2 r2 = pk(r, r);
              const float4* f = reinterpret_cast<const float4*>(s.f[h] + 32 * b);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float4 v = f[j];
                m[2 * j] = round2(mul(pk(g[4 * j], g[4 * j + 1]), mul(r2, pk(v.x, v.y))));
                m[2 * j + 1] = round2(mul(pk(g[4 * j + 2], g[4 * j + 3]), mul(r2, pk(v.z, v.w))));
              }
            } else {
              const float4* lp = reinterpret_cast<const float4*>(s.lp[h] + 32 * b);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float4 v = lp[j];
                const float e0 = 4 * j <= lane ? __uint_as_float(g[4 * j]) * ex2f(pi[h] - v.x) : 0.f;
                const float e1 = 4 * j + 1 <= lane ? __uint_as_float(g[4 * j + 1]) * ex2f(pi[h] - v.y) : 0.f;
                const float e2 = 4 * j + 2 <= lane ? __uint_as_float(g[4 * j + 2]) * ex2f(pi[h] - v.z) : 0.f;
                const float e3 = 4 * j + 3 <= lane ? __uint_as_float(g[4 * j + 3]) * ex2f(pi[h] - v.w) : 0.f;
                m[2 * j] = pack_bf16(e0, e1);
                m[2 * j + 1] = pack_bf16(e2, e3);
              }
            }
            tmem_st16(lanes + kColG + 32 * b + 16 * h, m);
          }
        }
        const int hq = kWide ? 0 : q;
        float before = 0.f;
        for (int k = 0; k < w; ++k) before += s.tot[hq][k];
        const float e = ex2f(pi[hq] + before);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar(B_M));
          mbar_arrive(bar(B_SCAL_FREE + (c & 1)));
        }

        if (!(ok = warp_wait(bar(B_Y), c & 1, abort_flag))) break;
        tc_fence_after();
        const int row = 32 * w + lane;
        const uint32_t xrow = sbase + L::kX + (c & 1) * kTileX + q * (kTileX / 2) + row * 128;
        const f2 e2 = pk(e, e), D2 = pk(D, D);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t y[32], z[32];
          tmem_ld32(lanes + kColY + 64 * q + 32 * half, y);
          tmem_ld32(lanes + kColZ + 64 * q + 32 * half, z);
          tmem_wait_ld();
          if (half == 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_ZY_FREE));
          }
          if (!mine) continue;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t at = xrow + (((4 * half + j) ^ (row & 7)) << 4);
            f2 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = fma2(pk(z[8 * j + 2 * i], z[8 * j + 2 * i + 1]), e2, pk(y[8 * j + 2 * i], y[8 * j + 2 * i + 1]));
            if (p.D != nullptr) {
              const uint4 xv = lds128(at);
              v[0] = fma2(pk(bf_lo(xv.x), bf_hi(xv.x)), D2, v[0]);
              v[1] = fma2(pk(bf_lo(xv.y), bf_hi(xv.y)), D2, v[1]);
              v[2] = fma2(pk(bf_lo(xv.z), bf_hi(xv.z)), D2, v[2]);
              v[3] = fma2(pk(bf_lo(xv.w), bf_hi(xv.w)), D2, v[3]);
            }
            sts128(at, round2(v[0]), round2(v[1]), round2(v[2]), round2(v[3]));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_OUT + (c & 1)));
      }
    }
  } else if (warp < 12) {
    // ---- the state: this thread's row of 128 --------------------------------------------------------------------------------
    const int row = 32 * (warp & 3) + lane, h = kWide ? 0 : row >> 6;
    const uint32_t at = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + kColS;
    const bool there = kWide || h == 0 || it.two;
    const int64_t state = (static_cast<int64_t>(it.n) * p.H + it.head0 + h) * (kWide ? 128 : 64) * kNs + static_cast<int64_t>(kWide ? row : row & 63) * kNs;
    const uint32_t srow = sbase + L::kS + row * 128;
    // (32 columns of the state before a block -> its copy for Z; rescaled to the block's end)
    auto copy_out = [&](const uint32_t (&v)[32], int part) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sts128(srow + (part >> 1) * 16384 + (((4 * (part & 1) + j) ^ (row & 7)) << 4), pack_bf16(__uint_as_float(v[8 * j]), __uint_as_float(v[8 * j + 1])),
               pack_bf16(__uint_as_float(v[8 * j + 2]), __uint_as_float(v[8 * j + 3])), pack_bf16(__uint_as_float(v[8 * j + 4]), __uint_as_float(v[8 * j + 5])),
               pack_bf16(__uint_as_float(v[8 * j + 6]), __uint_as_float(v[8 * j + 7])));
    };
    auto rescale = [&](uint32_t (&v)[32], float d) {
#pragma unroll
      for (int i = 0; i < 16; ++i) mul2(v[2 * i], v[2 * i + 1], make_float2(d, d));
    };
    const float* slot = it.slot >= 0 ? p.slots + (static_cast<int64_t>(it.slot) * 128 + row) * kNs : nullptr;
    for (int c = 0; blocks > 0 && c <= blocks; ++c) {
      if (c > 0) {
        if (!(ok = warp_wait(bar(B_S_FULL), (c - 1) & 1, abort_flag))) break;
        tc_fence_after();
      }
      float d = 1.f;
      if (c < blocks) {
        if (!(ok = warp_wait(bar(B_SCAL + (c & 1)), (c >> 1) & 1, abort_flag))) break;
        d = scal[c & 1].decay[h];
      }
#pragma unroll
      for (int part = 0; part < kNs / 32; ++part) {
        uint32_t v[32];
        if (c > 0) {
          tmem_ld32(at + 32 * part, v);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0u;
          if (kFull && there) {
            if (slot != nullptr) {
#pragma unroll
              for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(v + 4 * i) = *reinterpret_cast<const uint4*>(slot + 32 * part + 4 * i);
            } else if (p.initial_state != nullptr && p.state_fp32) {
              const float* src = static_cast<const float*>(p.initial_state) + state + 32 * part;
#pragma unroll
              for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(v + 4 * i) = *reinterpret_cast<const uint4*>(src + 4 * i);
            } else if (p.initial_state != nullptr) {
              const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.initial_state) + state + 32 * part;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint4 b = *reinterpret_cast<const uint4*>(src + 8 * i);
                const uint32_t word[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  v[8 * i + 2 * k] = word[k] << 16;
                  v[8 * i + 2 * k + 1] = word[k] & 0xffff0000u;
                }
              }
            }
          }
        }
        if (c < blocks) {
          if constexpr (kFull) copy_out(v, part);
          rescale(v, d);
          tmem_st32(at + 32 * part, v);
        } else if (there) {
          if (!kFull) {
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(const_cast<float*>(slot) + 32 * part + 4 * i) = *reinterpret_cast<const uint4*>(v + 4 * i);
          } else if (it.last && p.final_state != nullptr) {
            if (p.state_fp32) {
              float* dst = static_cast<float*>(p.final_state) + state + 32 * part;
#pragma unroll
              for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(dst + 4 * i) = *reinterpret_cast<const uint4*>(v + 4 * i);
            } else {
              __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.final_state) + state + 32 * part;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint4*>(dst + 8 * i) =
                    make_uint4(pack_bf16(__uint_as_float(v[8 * i]), __uint_as_float(v[8 * i + 1])), pack_bf16(__uint_as_float(v[8 * i + 2]), __uint_as_float(v[8 * i + 3])),
                               pack_bf16(__uint_as_float(v[8 * i + 4]), __uint_as_float(v[8 * i + 5])), pack_bf16(__uint_as_float(v[8 * i + 6]), __uint_as_float(v[8 * i + 7])));
            }
          }
        }
      }
      if (c < blocks) {
        tmem_wait_st();
        tc_fence_before();
        if constexpr (kFull) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_S_READY));
      }
    }
  } else if (warp < 16) {
    // ---- decays, and x' ------------------------------------------------------------------------------------------------------
    const int t = tid - 12 * 32, v = warp - 12;
    const int heads[2] = {it.head0, it.head0 + (!kWide && it.two ? 1 : 0)};
    float A[2], bias[2];
    if (blocks > 0) {
#pragma unroll
      for (int h = 0; h < (kWide ? 1 : 2); ++h) {
        A[h] = -kLog2e * ex2f(kLog2e * __ldg(p.A_log + heads[h]));
        bias[h] = __ldg(p.dt_bias + heads[h]);
      }
    }
    float dt[2] = {0.f, 0.f};
    auto load_dt = [&](int c) {
      if (c >= blocks || static_cast<int64_t>(c) * kQ + t >= it.tokens) return;
      const __nv_bfloat16* src = p.dt + it.b * p.dts.batch + (it.t0 + static_cast<int64_t>(c) * kQ + t) * p.dts.token;
#pragma unroll
      for (int h = 0; h < (kWide ? 1 : 2); ++h) dt[h] = __bfloat162float(src[heads[h]]);
    };
    // (a rendezvous of these four warps whose wait is bounded, too)
    uint32_t meetings = 0;
    auto meet = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_MEET));
      return warp_wait(bar(B_MEET), meetings++ & 1, abort_flag);
    };
    float log_decay[2] = {0.f, 0.f};                                 // of the blocks so far (thread 0)
    auto scalars = [&](int c) {
      if (c >= blocks) return true;
      Scalars& s = scal[c & 1];
      if (kFull && c >= 2 && !warp_wait(bar(B_SCAL_FREE + (c & 1)), ((c >> 1) - 1) & 1, abort_flag)) return false;
      const bool valid = static_cast<int64_t>(c) * kQ + t < it.tokens;
      float f[2], tot[2];
#pragma unroll
      for (int h = 0; h < (kWide ? 1 : 2); ++h) {
        const float delta = valid ? softplus(dt[h] + bias[h]) : 0.f;
        const float a = valid ? A[h] * delta : 0.f;
        float up = a, down = __shfl_down_sync(0xffffffffu, a, 1);
        if (lane == 31) down = 0.f;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const float u = __shfl_up_sync(0xffffffffu, up, d), e = __shfl_down_sync(0xffffffffu, down, d);
          if (lane >= d) up += u;
          if (lane + d < 32) down += e;
        }
        f[h] = delta * ex2f(down);
        tot[h] = __shfl_sync(0xffffffffu, up, 31);
        s.p[h][t] = up;
        s.lp[h][t] = up - __log2f(delta);
        s.f[h][t] = f[h];
        if (lane == 0) s.tot[h][v] = tot[h];
      }
      load_dt(c + 1);
      if (!meet()) return false;
#pragma unroll
      for (int h = 0; h < (kWide ? 1 : 2); ++h) {
        const float4 all = *reinterpret_cast<const float4*>(s.tot[h]);
        const float behind = (v < 1 ? all.y : 0.f) + (v < 2 ? all.z : 0.f) + (v < 3 ? all.w : 0.f), sum = (all.x + all.y) + (all.z + all.w);
        s.w[h][t] = f[h] * ex2f(behind);
        if (t == 0) s.decay[h] = ex2f(sum);
        log_decay[h] += sum;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_SCAL + (c & 1)));
      return meet();                                                  // (w of all tokens, for x')
    };
    load_dt(0);
    if (blocks > 0) ok = scalars(0);
    uint32_t step = 0;
    const int tok = t >> 3, chunk = t & 7;
    for (int c = 0; ok && c < blocks; ++c) {
      if (!(ok = scalars(c + 1))) break;
      const Scalars& s = scal[c & 1];
      if (!(ok = warp_wait(bar(B_FULL_X + (c & 1)), (c >> 1) & 1, abort_flag))) break;
      const uint32_t x = sbase + L::kX + (c & 1) * kTileX;
      const int64_t left = it.tokens - static_cast<int64_t>(c) * kQ;
      if (left < kQ) {
        if (!(ok = warp_wait(bar(B_FULL_B + (c & 1)), (c >> 1) & 1, abort_flag))) break;
        const uint32_t b = sbase + L::kB + (c & 1) * L::kTile;
        for (int i = t; i < (kQ - static_cast<int>(left)) * 8; i += 128) {
          const uint32_t off = (static_cast<uint32_t>(left) + i / 8) * 128 + (i % 8) * 16;
          sts128(x + off, 0u, 0u, 0u, 0u);
          sts128(x + kTileX / 2 + off, 0u, 0u, 0u, 0u);
          sts128(b + off, 0u, 0u, 0u, 0u);
          if (kNs == 128) sts128(b + L::kTile / 2 + off, 0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        if (!(ok = meet())) break;
      }
      for (int st = 0; st < 8; ++st, ++step) {
        const uint32_t sl = step % kSlots, use = step / kSlots;
        if (use > 0 && !(ok = warp_wait(bar(B_XP_EMPTY + sl), (use - 1) & 1, abort_flag))) break;
        const int tt = 16 * st + tok;
        const uint32_t dst = sbase + L::kXp + sl * kSlotBytes + tok * 128 + ((chunk ^ (tok & 7)) << 4);
        const uint32_t src = x + tt * 128 + ((chunk ^ (tt & 7)) << 4);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float w = s.w[kWide ? 0 : half][tt];
          const uint4 xv = lds128(src + half * (kTileX / 2));
          const uint32_t in[4] = {xv.x, xv.y, xv.z, xv.w};
          const f2 w2 = pk(w, w);
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f2 y = mul(pk(bf_lo(in[i]), bf_hi(in[i])), w2);
            hi[i] = round2(y);
            const f2 rest = fma2(pk(bf_lo(hi[i]), bf_hi(hi[i])), pk(-1.f, -1.f), y);
            lo[i] = round2(rest);
          }
          sts128(dst + half * 2048, hi[0], hi[1], hi[2], hi[3]);
          if (p.split) sts128(dst + kSlotBytes / 2 + half * 2048, lo[0], lo[1], lo[2], lo[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_XP_FULL + sl));
      }
      if (!ok) break;
      if (!kFull) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_EMPTY_X + (c & 1)));
      }
    }
    if (!kFull && ok && t == 0 && blocks > 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) p.decays[2 * it.slot + h] = ex2f(log_decay[kWide ? 0 : h]);
    }
  } else if (warp == 16) {
    // ---- loads of B and C ------------------------------------------------------------------------------------------------------
    int issued = 0;
    const int column = it.group * kNs;
    for (int c = 0; c < blocks && c < p.stop_loads_after; ++c) {
      const int buf = c & 1, row = static_cast<int>(it.t0) + c * kQ;
      if (c >= 2 && !(ok = warp_wait(bar(B_EMPTY_B + buf), ((c >> 1) - 1) & 1, abort_flag))) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(bar(B_FULL_B + buf), L::kTile);
#pragma unroll
        for (int i = 0; i < kNs / 64; ++i) tma_load_3d(sbase + L::kB + buf * L::kTile + i * 16384, &maps.b, column + 64 * i, row, static_cast<int>(it.b), bar(B_FULL_B + buf));
      }
      issued = c + 1;
      if constexpr (kFull) {
        if (c >= 1 && !(ok = warp_wait(bar(B_EMPTY_C), (c - 1) & 1, abort_flag))) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(bar(B_FULL_C), L::kTile);
#pragma unroll
          for (int i = 0; i < kNs / 64; ++i) tma_load_3d(sbase + L::kC + i * 16384, &maps.c, column + 64 * i, row, static_cast<int>(it.b), bar(B_FULL_C));
        }
        __syncwarp();
      }
    }
    // every copy has landed before this CTA's memory goes to another: those that nobody waited for
    if (lane == 0) {
      for (int c = issued > 2 ? issued - 2 : 0; c < issued; ++c) drain(bar(B_FULL_B + (c & 1)), (c >> 1) & 1);
      if (kFull && issued > 0 && ok) drain(bar(B_FULL_C), (issued - 1) & 1);
      if (kFull && issued > 1 && !ok) drain(bar(B_FULL_C), (issued - 2) & 1);
    }
  } else if (warp == 17) {
    // ---- products ----------------------------------------------------------------------------------------------------------------
    constexpr uint32_t idesc_g = umma_idesc_bf16(128, 128, 0, 0), idesc_s = umma_idesc_bf16(128, kNs, 1, 1), idesc_y = umma_idesc_bf16(128, kWide ? 128 : 64, 0, 1);
    const uint64_t dc = desc_sw128(sbase + L::kC, 16), ds = desc_sw128(sbase + L::kS, 16);
    uint32_t step = 0;
    for (int c = 0; c < blocks; ++c) {
      const int buf = c & 1;
      const uint32_t b = sbase + L::kB + buf * L::kTile, x = sbase + L::kX + buf * kTileX;
      if (!(ok = warp_wait(bar(B_FULL_B + buf), (c >> 1) & 1, abort_flag))) break;
      if constexpr (kFull) {
        if (!(ok = warp_wait(bar(B_FULL_C), c & 1, abort_flag))) break;
        if (c > 0 && !(ok = warp_wait(bar(B_Y), (c - 1) & 1, abort_flag))) break;       // M of the block before has been read
        tc_fence_after();
        if (elect_one()) {
          const uint64_t db = desc_sw128(b, 16);
#pragma unroll
          for (int k = 0; k < kNs / 16; ++k) umma_ss(tmem + kColG, dc + (k / 4) * 1024 + (k % 4) * 2, db + (k / 4) * 1024 + (k % 4) * 2, idesc_g, k > 0);
          umma_commit(bar(B_G));
        }
        __syncwarp();
      }
      if (!(ok = warp_wait(bar(B_S_READY), c & 1, abort_flag))) break;
      if constexpr (kFull) {
        if (c > 0 && !(ok = warp_wait(bar(B_ZY_FREE), (c - 1) & 1, abort_flag))) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kNs / 16; ++k) umma_ss(tmem + kColZ, dc + (k / 4) * 1024 + (k % 4) * 2, ds + (k / 4) * 1024 + (k % 4) * 2, idesc_g, k > 0);
          umma_commit(bar(B_EMPTY_C));
        }
        __syncwarp();
      }
      for (int st = 0; st < 8; ++st, ++step) {
        const uint32_t sl = step % kSlots, use = step / kSlots;
        if (!(ok = warp_wait(bar(B_XP_FULL + sl), use & 1, abort_flag))) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t da = desc_sw128(sbase + L::kXp + sl * kSlotBytes, 2048), db = desc_sw128(b + st * 2048, 16384);
          umma_ss(tmem + kColS, da, db, idesc_s, 1);
          if (p.split) umma_ss(tmem + kColS, da + kSlotBytes / 2 / 16, db, idesc_s, 1);
          umma_commit(bar(B_XP_EMPTY + sl));
          if (st == 7) {
            umma_commit(bar(B_EMPTY_B + buf));
            umma_commit(bar(B_S_FULL));
          }
        }
        __syncwarp();
      }
      if (!ok) break;
      if constexpr (kFull) {
        if (!(ok = warp_wait(bar(B_FULL_X + buf), (c >> 1) & 1, abort_flag))) break;
        if (!(ok = warp_wait(bar(B_M), c & 1, abort_flag))) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < (kWide ? 1 : 2); ++h) {
            const uint64_t dx = desc_sw128(x + h * (kTileX / 2), 16384);
#pragma unroll
            for (int k = 0; k < 8; ++k) umma_ts(tmem + kColY + 64 * h, tmem + kColG + 32 * (k / 2) + 16 * h + 8 * (k % 2), dx + k * 128, idesc_y, k > 0);
          }
          umma_commit(bar(B_Y));
        }
        __syncwarp();
      }
    }
    // no product may be under way when the tensor memory is given back
    if (elect_one()) umma_commit(bar(B_DRAIN));
    __syncwarp();
    if (lane == 0) drain(bar(B_DRAIN), 0);
    __syncwarp();
  } else {
    // ---- loads of x, stores of out -----------------------------------------------------------------------------------------------
    const int column = it.head0 * (kWide ? 128 : 64);
    auto store = [&](int c) {
      const int buf = c & 1;
      if (!warp_wait(bar(B_OUT + buf), (c >> 1) & 1, abort_flag)) return false;
      const uint32_t x = sbase + L::kX + buf * kTileX;
      const int64_t left = it.tokens - static_cast<int64_t>(c) * kQ;
      if (p.packed && left < kQ) {
        // rows behind the sequence's end are somebody else's
        const int pieces = kWide || it.two ? 16 : 8;
        __nv_bfloat16* dst = p.out + (it.t0 + static_cast<int64_t>(c) * kQ) * p.os.token + column;
        for (int i = lane; i < static_cast<int>(left) * pieces; i += 32) {
          const int row = i / pieces, piece = i % pieces;
          *reinterpret_cast<uint4*>(dst + row * p.os.token + piece * 8) = lds128(x + (piece >> 3) * (kTileX / 2) + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
        }
        return true;
      }
      if (lane == 0) {
        const int row = static_cast<int>(it.t0) + c * kQ;
        tma_store_3d(&maps.out, x, column, row, static_cast<int>(it.b));
        if (kWide || it.two) tma_store_3d(&maps.out, x + kTileX / 2, column + 64, row, static_cast<int>(it.b));
        bulk_commit();
        bulk_wait_read0();
      }
      __syncwarp();
      return true;
    };
    int issued = 0;
    for (int c = 0; c < blocks && c < p.stop_loads_after; ++c) {
      const int buf = c & 1;
      if (c >= 2) {
        ok = kFull ? store(c - 2) : warp_wait(bar(B_EMPTY_X + buf), ((c >> 1) - 1) & 1, abort_flag);
        if (!ok) break;
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(bar(B_FULL_X + buf), kTileX);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          tma_load_3d(sbase + L::kX + buf * kTileX + i * (kTileX / 2), &maps.x, column + 64 * i, static_cast<int>(it.t0) + c * kQ, static_cast<int>(it.b), bar(B_FULL_X + buf));
      }
      __syncwarp();
      issued = c + 1;
    }
    if (kFull && ok)
      for (int c = blocks > 2 ? blocks - 2 : 0; ok && c < blocks; ++c) ok = store(c);
    if (lane == 0) {
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      for (int c = issued > 2 ? issued - 2 : 0; c < issued; ++c) drain(bar(B_FULL_X + (c & 1)), (c >> 1) & 1);
    }
    __syncwarp();
  }
  if ((!ok || *abort_flag > 0) && p.status != nullptr) atomicCAS(p.status, kStatusOk, kStatusWaitTimeout);
  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- plan of a packed batch, and the chaining of runs -------------------------------------------------------------------------------
// Sequences of more than kSsmStepT tokens, longest first, cut into runs of the length that the costs below (in blocks of the full walk) make cheapest.
constexpr int kPlanThreads = 1024, kCandidates = 8;
__device__ __forceinline__ int candidate(int least, int i) {         // run lengths that are tried; the last one: whole sequences
  return i == kCandidates - 1 ? 0x7fffffff : (least << (i >> 1)) + ((i & 1) ? (least << (i >> 1)) / 2 : 0);
}
__global__ void __launch_bounds__(kPlanThreads) ssm_plan_kernel(const int64_t* cu, int N, int64_t T, int pairs, int sms, int least, SsmPlan* plan, int* status) {
  __shared__ int s_blocks[kSsmPlanMost];
  __shared__ int s_seq[kSsmPlanMost];
  __shared__ int s_active, s_longest, s_bad;
  __shared__ unsigned long long s_total, s_first[kCandidates];
  __shared__ int s_run;
  grid_dependency_wait();
  const int tid = threadIdx.x;
  if (tid == 0) {
    s_active = s_longest = s_bad = 0;
    s_total = 0;
    if (status != nullptr) *status = 0;
  }
  if (tid < kCandidates) s_first[tid] = 0;
  __syncthreads();
  auto blocks_of = [&](int n) {
    int64_t bos = cu[n], eos = cu[n + 1];
    if (bos < 0 || eos < bos || eos > T) s_bad = 1;
    bos = bos < 0 ? 0 : bos > T ? T : bos;
    eos = eos < bos ? bos : eos > T ? T : eos;
    return eos - bos <= kSsmStepT ? 0 : static_cast<int>((eos - bos + kQ - 1) / kQ);
  };
  // the sequences with blocks, in the order that they come in where they are too many to be sorted
  int* order = plan->order(), *prefix = plan->prefix(N), *slots = plan->slot_prefix(N);
  for (int base = 0; base < N; base += kPlanThreads) {
    const int n = base + tid;
    const int b = n < N ? blocks_of(n) : 0;
    __shared__ int s_scan[32];
    const unsigned vote = __ballot_sync(0xffffffffu, b > 0);
    if ((tid & 31) == 0) s_scan[tid >> 5] = __popc(vote);
    __syncthreads();
    int at = s_active + __popc(vote & ((1u << (tid & 31)) - 1));
    for (int i = 0; i < (tid >> 5); ++i) at += s_scan[i];
    if (b > 0) {
      if (at < N) order[at] = n;
      if (at < kSsmPlanMost) {
        s_seq[at] = n;
        s_blocks[at] = b;
      }
      atomicMax(&s_longest, b);
      atomicAdd(&s_total, static_cast<unsigned long long>(b));
      if (least > 0)
        for (int i = 0; i < kCandidates; ++i) {
          const int l = candidate(least, i);
          if (b > l) atomicAdd(&s_first[i], static_cast<unsigned long long>((b - 1) / l) * l);
        }
    }
    __syncthreads();
    if (tid == 0)
      for (int i = 0; i < 32; ++i) s_active += s_scan[i];
    __syncthreads();
  }
  // (sequences that are not monotone may overlap, and then be more than there is room for: none is walked)
  const int active = s_bad ? 0 : s_active;
  if (tid == 0 && s_bad && status != nullptr) atomicCAS(status, kStatusOk, kStatusBadCuSeqlens);
  const bool sorted = active <= kSsmPlanMost;
  if (tid == 0) {
    int run = 0x7fffffff;
    if (least > 0 && sorted) {
      long long best = -1;
      for (int i = kCandidates - 1; i >= 0; --i) {
        const int l = candidate(least, i);
        const long long even = static_cast<long long>(s_total * pairs + sms - 1) / sms, longest = s_longest < l ? s_longest : l;
        long long cost = 100 * (even > longest ? even : longest) + 30 * (even < longest ? even : longest);
        if (s_first[i] > 0) {
          const long long first = static_cast<long long>(s_first[i] * pairs + sms - 1) / sms;
          cost += kSsmFirstCost * (first > longest ? first : longest) + kSsmCutCost;
        }
        if (best < 0 || cost < best) {
          best = cost;
          run = l;
        }
      }
    }
    s_run = run;
    plan->run_blocks = run;
    plan->active = active;
  }
  __syncthreads();
  const int run = s_run;
  if (sorted) {
    for (int i = tid; i < active; i += kPlanThreads) {
      const int b = s_blocks[i];
      int rank = 0;
      for (int k = 0; k < active; ++k) rank += s_blocks[k] > b || (s_blocks[k] == b && k < i);
      order[rank] = s_seq[i];
    }
    __syncthreads();
  }
  // prefixes over the ranks: runs, and runs of the sequences that are cut (they come first)
  __shared__ int s_part[2][32];
  int done[2] = {0, 0};
  for (int base = 0; base < active; base += kPlanThreads) {
    const int i = base + tid;
    int runs = 0;
    if (i < active) {
      const int b = blocks_of(order[i]);
      runs = run == 0x7fffffff ? 1 : (b + run - 1) / run;
    }
    int a = runs, c = runs > 1 ? runs : 0;
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, a, d), v = __shfl_up_sync(0xffffffffu, c, d);
      if ((tid & 31) >= d) {
        a += u;
        c += v;
      }
    }
    if ((tid & 31) == 31) {
      s_part[0][tid >> 5] = a;
      s_part[1][tid >> 5] = c;
    }
    __syncthreads();
    int whole[2] = {0, 0};
    for (int k = 0; k < 32; ++k) {
      if (k < (tid >> 5)) {
        a += s_part[0][k];
        c += s_part[1][k];
      }
      whole[0] += s_part[0][k];
      whole[1] += s_part[1][k];
    }
    if (i < active) {
      prefix[i + 1] = done[0] + a;
      slots[i + 1] = done[1] + c;
    }
    done[0] += whole[0];
    done[1] += whole[1];
    __syncthreads();
  }
  if (tid == 0) {
    prefix[0] = slots[0] = 0;
    plan->cut = 0;
  }
  __syncthreads();
  for (int i = tid; i < active; i += kPlanThreads)
    if (slots[i + 1] > slots[i]) atomicMax(&plan->cut, i + 1);
}

// Per sequence that is cut: its runs' local states -> the state that each run starts from.
__global__ void __launch_bounds__(256) ssm_chain_kernel(const SsmScanParams p, int Ns, int pairs) {
  grid_dependency_wait();
  const int pieces = 128 * Ns / 4 / 256;                              // blocks of 256 float4
  const int piece = static_cast<int>(blockIdx.x % pieces), pair = static_cast<int>(blockIdx.x / pieces % pairs), rank = static_cast<int>(blockIdx.x / pieces / pairs);
  int n = rank, runs = p.runs, first = rank * p.runs;
  if (p.packed) {
    if (rank >= p.plan->cut) return;
    n = p.plan->order()[rank];
    first = p.plan->slot_prefix(p.N)[rank];
    runs = p.plan->slot_prefix(p.N)[rank + 1] - first;
  }
  const int at = (piece * 256 + threadIdx.x) * 4, row = at / Ns;
  const int per = p.P == 128 ? 1 : 2, in_group = p.H / p.G, group = pair / p.pairs_per_group;
  const int within = (pair - group * p.pairs_per_group) * per + (per == 2 ? row >> 6 : 0);       // head within its group
  const int h = per == 2 ? row >> 6 : 0;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (p.initial_state != nullptr && within < in_group) {
    const int64_t src = ((static_cast<int64_t>(n) * p.H + group * in_group + within) * p.P + (per == 2 ? row & 63 : row)) * Ns + at % Ns;
    if (p.state_fp32) {
      s = *reinterpret_cast<const float4*>(static_cast<const float*>(p.initial_state) + src);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.initial_state) + src);
      s = make_float4(bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y));
    }
  }
  float4 next = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int r = 0; r < runs; ++r) {
    const int64_t slot = static_cast<int64_t>(first + r) * pairs + pair;
    float4* q = reinterpret_cast<float4*>(p.slots + slot * 128 * Ns + at);
    if (r + 1 < runs) next = *q;
    *q = s;
    if (r + 1 < runs) {
      const float d = p.decays[2 * slot + h];
      s = make_float4(fmaf(d, s.x, next.x), fmaf(d, s.y, next.y), fmaf(d, s.z, next.z), fmaf(d, s.w, next.w));
    }
  }
}

bool make_tile_map(CUtensorMap* map, const void* base, int64_t columns, int64_t T, int64_t B, const Rows& s) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return false;
  const int64_t token = T > 1 ? s.token : (columns + 7) / 8 * 8, batch = B > 1 ? s.batch : token;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(T), static_cast<cuuint64_t>(B)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(token) * 2, static_cast<cuuint64_t>(batch) * 2};
  const cuuint32_t box[3] = {64, kQ, 1}, estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kNs, bool kWide, bool kFull>
cudaError_t launch_walk(const SsmMaps& maps, const SsmScanParams& p, int64_t items, cudaStream_t stream) {
  if (items == 0) return cudaSuccess;
  static SmemOptIn opt_in;
  auto kernel = ssm_scan_kernel<kNs, kWide, kFull>;
  const cudaError_t e = opt_in.ensure(kernel, Smem<kNs>::kBytes);
  if (e != cudaSuccess) return e;
  return launch_after(kernel, dim3(static_cast<unsigned>(items)), kThreads, Smem<kNs>::kBytes, stream, maps, p);
}
template <bool kFull>
cudaError_t launch_pass(const SsmMaps& maps, const SsmScanParams& p, int Ns, int64_t items, cudaStream_t stream) {
  if (Ns == 128) return p.P == 128 ? launch_walk<128, true, kFull>(maps, p, items, stream) : launch_walk<128, false, kFull>(maps, p, items, stream);
  return p.P == 128 ? launch_walk<64, true, kFull>(maps, p, items, stream) : launch_walk<64, false, kFull>(maps, p, items, stream);
}

}  // namespace ssm_scan

SsmLayout ssm_layout(int64_t T, int64_t N, int H, int P, int G, int Ns, bool packed, int sms) {
  SsmLayout L{};
  L.pairs_per_group = P == 128 ? H / G : (H / G + 1) / 2;
  L.pairs = L.pairs_per_group * G;
  const int64_t slot_bytes = 128 * Ns * 4;
  if (!packed) {
    const int64_t blocks = (T + kSsmBlock - 1) / kSsmBlock, chains = N * L.pairs;
    auto rounds = [&](int64_t ctas) { return (ctas + sms - 1) / sms; };
    int64_t best = rounds(chains) * blocks * 100;
    L.runs = 1;
    L.run_blocks = static_cast<int>(blocks);
    for (int64_t r = 2; r <= blocks && r <= 160 && chains < 4 * sms; ++r) {
      const int64_t len = (blocks + r - 1) / r;
      if ((r - 1) * len >= blocks) continue;                        // the last run would be empty
      const int64_t cost = (rounds(chains * r) * 100 + rounds(chains * (r - 1)) * kSsmFirstCost) * len + kSsmCutCost + kSsmRunCost * r;
      if (cost < best) {
        best = cost;
        L.runs = static_cast<int>(r);
        L.run_blocks = static_cast<int>(len);
      }
    }
    L.items = chains * L.runs;
    L.first_items = L.runs > 1 ? chains * (L.runs - 1) : 0;
    L.slots = L.runs > 1 ? L.items : 0;
    L.chained = L.runs > 1 ? N : 0;
    L.plan_off = 256;
    L.decay_off = 256;
  } else {
    const int64_t blocks = (T + kSsmBlock - 1) / kSsmBlock, even = (blocks * L.pairs + sms - 1) / sms;
    int64_t least = (even + 3) / 4;
    if (least < 8) least = 8;
    const bool cut = blocks > least && least < (1 << 20);
    L.least = cut ? static_cast<int>(least) : 0;
    const int64_t active = N < T / (kSsmStepT + 1) ? N : T / (kSsmStepT + 1);
    L.items = (active + (cut ? blocks / least : 0)) * L.pairs;
    L.first_items = cut ? (2 * blocks / least + 1) * L.pairs : 0;
    L.slots = L.first_items;
    L.chained = cut ? blocks / least + 1 : 0;
    L.plan_off = 256;
    L.decay_off = L.plan_off + (static_cast<int64_t>(sizeof(SsmPlan)) + (3 * N + 2) * 4 + 255) / 256 * 256;
  }
  L.slot_off = L.decay_off + (L.slots * 8 + 255) / 256 * 256;
  L.bytes = L.slot_off + L.slots * slot_bytes;
  return L;
}

cudaError_t launch_ssm_scan(const SsmParams& q, const SsmLayout& L, const SsmAid& aid, void* workspace, bool clear_status, cudaStream_t stream) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const bool packed = q.cu_seqlens != nullptr;
  const int64_t B = packed ? 1 : q.N;
  SsmMaps maps;
  if (!ssm_scan::make_tile_map(&maps.x, q.x, static_cast<int64_t>(q.H) * q.P, q.T, B, q.xs) || !ssm_scan::make_tile_map(&maps.out, q.out, static_cast<int64_t>(q.H) * q.P, q.T, B, q.os) ||
      !ssm_scan::make_tile_map(&maps.b, q.Bm, static_cast<int64_t>(q.G) * q.Ns, q.T, B, q.bs) || !ssm_scan::make_tile_map(&maps.c, q.Cm, static_cast<int64_t>(q.G) * q.Ns, q.T, B, q.cs))
    return cudaErrorInvalidValue;
  SsmScanParams p{};
  p.dt = q.dt;
  p.out = q.out;
  p.A_log = q.A_log;
  p.dt_bias = q.dt_bias;
  p.D = q.D;
  p.initial_state = q.initial_state;
  p.final_state = q.final_state;
  p.cu_seqlens = q.cu_seqlens;
  p.plan = reinterpret_cast<SsmPlan*>(ws + L.plan_off);
  p.slots = reinterpret_cast<float*>(ws + L.slot_off);
  p.decays = reinterpret_cast<float*>(ws + L.decay_off);
  p.status = reinterpret_cast<int*>(ws);
  p.dts = q.dts;
  p.os = q.os;
  p.T = q.T;
  p.H = q.H;
  p.P = q.P;
  p.G = q.G;
  p.N = q.N;
  p.pairs_per_group = L.pairs_per_group;
  p.pairs = L.pairs;
  p.runs = L.runs;
  p.run_blocks = L.run_blocks;
  p.packed = packed;
  p.state_fp32 = q.state_fp32;
  p.split = q.final_state != nullptr && q.state_fp32;
  p.wait_limit_us = aid.wait_limit_us;
  p.stop_loads_after = aid.stop_loads_after > 0 ? aid.stop_loads_after : 0x7fffffff;
  cudaError_t e = cudaSuccess;
  if (packed) e = launch_after(ssm_scan::ssm_plan_kernel, dim3(1), ssm_scan::kPlanThreads, 0, stream, q.cu_seqlens, q.N, q.T, L.pairs, device_sm_count(), L.least, p.plan, p.status);
  else if (clear_status) e = cudaMemsetAsync(ws, 0, 4, stream);
  if (e != cudaSuccess) return e;
  if (L.first_items > 0) {
    e = ssm_scan::launch_pass<false>(maps, p, q.Ns, L.first_items, stream);
    if (e != cudaSuccess) return e;
    e = launch_after(ssm_scan::ssm_chain_kernel, dim3(static_cast<unsigned>(L.chained * L.pairs * (128 * q.Ns / 1024))), 256, 0, stream, p, q.Ns, L.pairs);
    if (e != cudaSuccess) return e;
  }
  return ssm_scan::launch_pass<true>(maps, p, q.Ns, L.items, stream);
}

}  // namespace fkda
