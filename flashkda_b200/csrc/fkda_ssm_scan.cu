// Selective state space scan in blocks of 128 tokens on tcgen05: prompts.
//
// With a = -exp(A_log) delta log2(e) the log2 decay of a token, l_i its running sum from the block's start and S the state [P][Ns]
// before the block (per head),
//     G = C B^T,   M_ij = G_ij 2^(l_i - l_j) delta_j  (j <= i),   out = M X + 2^(l_i) (C S^T) + D X
//     S <- 2^(l_127) S + X'^T B,   x'_j = 2^(l_127 - l_j) delta_j x_j
// A CTA walks the blocks of 128 rows of a sequence's states: two heads of P = 64 that share B and C, or one of P = 128.  Five or six products a block,
// 128 x 128 x 128 each: G, C S^T, X'^T B in two or three parts (below), M X.  Tensor memory holds G and over it M; the output, first as C S^T,
// then rescaled by rows, then with M X on top; X'^T; and S.  Twenty warps:
//     0-15   M from G: a warp a 32 x 32 block (rows i = lanes)
//     0-7    the output's rescaling (rows i = lanes, half of the columns each warpgroup); then out = that + D x over the tile of x in shared
//            memory, from where a tensor copy takes it
//     8-15   the state: fp32 in tensor memory, once a block read, rescaled and written back, and its bf16 copy for C S^T (half the columns
//            each warpgroup); then X'^T (half the rows each), by transposing ldmatrix, whose fragments are those of tcgen05.st
//     16, 18 delta and the decays, a head each       17     products       19     tensor copies (beside the rows of M with the most to do)
//
// Roundings: all products accumulate in fp32.  M and the state's copy are bf16 operands, as out is bf16.  The state is what a
// caller keeps, so X' goes into its product in parts: three bf16 numbers, which hold fp32's 24 bits, where the caller gets an fp32 state; two (16 bits) where
// it is rounded to bf16 or not asked for.  The parts come straight from x, which is bf16, and the token's weight as w0 + w1 (+ w2), in operations on bf16 pairs:
//     h = round(x w0),  e = x w0 - h, a bf16 number itself;   two parts: h and round(e + x w1)
//     three parts: m = round(e + round(x w1));  m - e is a bf16 number too (e is a multiple of the last bit of round(x w1));  l = round(round(x w1 - (m - e)) + x w2)
// Three instructions for two elements, and seven; taken apart in fp32 it was eight and twelve.  Against 64 bits the final state of 4 x 8192 x 32 x 128 is off by 2.4e-7
// of its norm with three parts, and would be by 4.7e-6 with two (240 us for 208); a 32-bit evaluation by products of plain matrices is off by 9e-8.
// Decays: every exponent that is evaluated is a sum of terms of one sign, so that nothing cancels, but for those within 32 x 32 blocks on
// the diagonal that lose less than 2^-100: there M's factor is 2^p_i 2^-p_j delta_j, off by 2^-24 of the running sums p, 1e-5 at most.  In blocks that lose
// more each row adds up its own exponents from the diagonal backwards (a step that resets the state leaves those behind it as they are).
// Rows past a sequence's end are zeroed in the tiles of x and B where they are summed over; those of C only reach outputs that are not stored.
//
// What bounds it (4 x 8192 tokens, 32 heads of P = Ns = 128: 128 CTAs of 64 blocks, on tensors that are new each time; 86 GFLOP as 5 P Ns a token): 208 us with states
// in bf16, 2.7 TB/s, 240 in fp32.  Not memory: a block takes 5000 cycles, 5900 with three parts, at the 1.5 to 1.6 GHz that the power limit leaves.  Its chain,
// traced: X'^T B of the block before is done, the next tile of B comes (1800 cycles; there is room for one), G (700), C S^T (800 to 1000), X'^T B (1040; with three
// parts 2200, of which its products are 1540); M X (700) and the reading of the output out of tensor memory (900) go beside the way of B.  All of it goes through
// shared memory: of a block's cycles there the products take 1800 (2050), the warps 1760 (1900), the tensor copies 1000, and G and C S^T read both operands at all that it gives, so that
// the warps' accesses wait meanwhile.  Left out to see, of 180 us (two parts, the same tensors over and over): half of G 8 us, the second part 14, as much as their cycles;
// reads of x for the output 2, the state's copy and the output's rescaling 1.
// Taken: products of 128 x 128 x 128 on two heads at once, since one head of P = 64 would leave half of a product's rows empty; X'^T in tensor memory
// (in shared memory: 281 us); a warp a block of M (a table of masks, one copy of the code: unrolled for each kind of block, the kernel no
// longer fitted in the instruction caches, 10 %).  Taken back: X'^T B before C S^T (the state's warps then wait for C S^T: 186 for 180, packed 435 for 397),
// the output on warps 8-15 (236), tiles of B and C asked for in the L2 beforehand (none).  Of three parts, which tensor memory holds two thirds of at a time (242): parts
// taken apart in fp32 (250), a quarter of a block at a time (260), the first half before the state's turn (258), M of warps 8-15 between the halves (250) or before the
// last pieces (251), a token's weights in one word of 16 bytes (255).
//
// Few chains are cut into runs (fkda_ssm.cuh): a first pass leaves what each run adds to a zero state, a small launch chains these, and the
// full pass starts every run from its state.  One sequence of 131072 x 8 heads of 64 takes 167 us with states in bf16 and 188 in fp32 (67 ms token by token): in a trace
// of such calls the first pass 48 (53), its chaining until 9 behind that, the full pass 92 (103) more.  A prompt of 777 x 32 heads takes 19.1 us (20.4): there each
// launch's start counts, some 2.5 us until decays and the first tiles are there, so that the launches overlap (see the waits below).  Packed batches of 16 sequences of 256
// to 16384 tokens, 32 heads: 435 us, 2.5 TB/s (481).
#include "fkda_elem.cuh"
#include "fkda_layer.cuh"
#include "fkda_ssm.cuh"
#include "fkda_tma.cuh"

namespace fkda {
namespace ssm_scan {

constexpr int kQ = kSsmBlock;
constexpr int kThreads = 20 * 32;          // (registers are given to four warps at a time: a twenty-first would leave 80 a thread)
constexpr int kTileX = kQ * 128 * 2;
constexpr int kXs = 3;                           // tiles of x: one being read, one with its output on the way out, one on the way in
constexpr int kScals = 4;                        // blocks whose decays are at hand: they are worked out ahead
constexpr uint32_t kColG = 0, kColY = 128, kColX = 256, kColS = 384;     // tensor memory; M lies over G
// X'^T over 32 tokens (a quarter of a block) takes 16 columns a part, in the order of the products: the last part first.  The full pass has room for eight such pieces: all
// of two parts, two thirds of three.
template <int kParts, bool kFull>
__device__ __forceinline__ uint32_t piece_column(int quarter, int part) {
  const int piece = quarter * kParts + kParts - 1 - part;
  return 16 * piece + (kFull ? kColX - (piece >= 8 ? 128 : 0) : 0);
}

// Per block and head, written by warps 16 and 18.
struct Scalars {
  float p[2][kQ];          // running sum of a from the start of the token's 32-token block, itself included
  float g[2][kQ];          // delta 2^-p; where the block's sum is beyond `most` delta itself
  float f[2][kQ];          // delta 2^(sum of a behind the token to the end of its 32-token block)
  uint2 w[2][kQ / 2];      // f decayed to the end of the block of 128, two tokens a word: as bf16, and what that leaves as bf16,
  uint32_t rest[2][kQ / 2];        // and (three parts) what that leaves
  float tot[2][4];         // sums over the four 32-token blocks
  float decay[2];          // 2^(sum over all)
  float rate[2];           // a of a delta of 1
  float most[2];           // sum of a over a 32-token block up to which decays within it are products of powers
  float pad[2];
};

// Decay within a 32-token block up to which 2^(p_i - p_j) is taken as 2^p_i 2^-p_j, and sum of its deltas: both factors, with delta, stay normal numbers.
constexpr float kMostDecay = -100.f, kMostDelta = 134217728.f;
// Masks of a 32 x 32 triangle for pairs of bf16: row i, 16 words, rows 80 bytes apart (16-byte reads of eight rows then meet no bank twice).
constexpr int kMaskPitch = 80;

template <int kNs>
struct Smem {
  static constexpr int kTile = kQ * kNs * 2;
  static constexpr int kB = 0, kC = kB + kTile, kX = kC + kTile, kS = kX + kXs * kTileX;
  static constexpr int kScal = kS + 128 * kNs * 2, kBars = kScal + kScals * static_cast<int>(sizeof(Scalars)), kMisc = kBars + 256;
  static constexpr int kMask = kMisc + 64, kBytes = kMask + 32 * kMaskPitch;
};
static_assert(Smem<128>::kBytes <= 227 * 1024, "shared memory of a CTA");

enum {
  B_FULL_B = 0, B_FULL_C, B_Z /* C S^T done, C free */, B_FULL_X /*[kXs]*/, B_EMPTY_X = 6 /*[kXs]*/, B_OUT = 9 /*[kXs]*/, B_XT = 12 /*[2]*/, B_SCAL = 14 /*[kScals]*/,
  B_SCAL_FREE = 18 /*[kScals]*/, B_G = 22, B_Y, B_M, B_Y_FREE, B_S_FULL /* X'^T B done, B free */, B_S_READY, B_DRAIN, B_MEET, B_XT_FREE /*[2]*/, B_COUNT = B_XT_FREE + 2,
  B_EMPTY_B = B_G, B_XT2 = B_OUT      // of the first pass, [2] each: buffer c & 1 of B and X'^T free; X'^T of the second buffer
};
static_assert(B_COUNT <= 32, "a lane each to make them, 256 bytes");

// Arrivals that complete a phase of barrier `i`.
template <bool kFull, bool kWide>
__device__ __forceinline__ uint32_t arrivals(int i) {
  if (i >= B_SCAL && i < B_SCAL + kScals) return kWide ? 1 : 2;
  if (i >= B_EMPTY_X && i < B_XT + 2) return 8;                       // (EMPTY_X, OUT, XT)
  if (i >= B_SCAL_FREE && i < B_SCAL_FREE + kScals) return kFull ? 16 : 8;
  if (i == B_M) return 16;
  return i == B_Y_FREE || i == B_S_READY || i == B_MEET ? 8 : 1;
}
__device__ __forceinline__ void mbar_inval(uint32_t bar) { asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }

// Shared-memory matrix descriptor of a tile with the 128-byte swizzle (rows of 128 bytes, 1024-byte aligned groups of eight).  K-major: `sbo`
// is the distance between groups of eight rows (M or N), 16 elements along K are 32 bytes on.  MN-major (rows along K): `sbo` is the
// distance between groups of eight rows along K, `lbo` between blocks of 64 elements of M or N.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lbo) { return umma_desc(addr, lbo, 1024) | (2ull << 61); }

// (What follows a first attempt is kept out of line: a sub-partition's instruction cache holds some 500 instructions, which four roles share.)
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || wait_on(bar, parity, abort_flag);
}
__device__ __forceinline__ void prefetch_l2(const void* at) { asm volatile("prefetch.global.L2 [%0];" ::"l"(at) : "memory"); }
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
// Products of bf16 pairs, rounded to bf16.
__device__ __forceinline__ uint32_t mul_bf2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t add_bf2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t sub_bf2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t fma_bf2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// 16 TMEM lanes x 16 columns (the shape of tmem_st_16x128b_x8, half of it).
__device__ __forceinline__ void tmem_st_16x128b_x4(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
               "r"(r[6]), "r"(r[7])
               : "memory");
}
using elem::f2;
using elem::fma2;
using elem::mul;
using elem::pk;
__device__ __forceinline__ f2 pk(uint32_t a, uint32_t b) { return elem::pk(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ uint32_t round2(f2 x) { return elem::round_bf(x); }

// (clears what lies above the diagonal, whatever it is: row `mask` of the table)
__device__ __forceinline__ void keep_triangle(uint32_t (&m)[16], const uint8_t* mask) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 k = *reinterpret_cast<const uint4*>(mask + 16 * j);
    m[4 * j] &= k.x;
    m[4 * j + 1] &= k.y;
    m[4 * j + 2] &= k.z;
    m[4 * j + 3] &= k.w;
  }
}

// Whether a head's M of the 32 x 32 block on the diagonal has to take its exponents one by one.
__device__ __forceinline__ bool forgets(const Scalars& s, int h, int block) { return !(s.tot[h][block] >= s.most[h]); }
// (powers that are multiplied: of a row's running sum and of a column's own)
__device__ __forceinline__ void weigh_m(uint32_t (&m)[16], const uint32_t (&g)[32], float r, const float* column) {
  const float e = ex2f(r);
  const f2 r2 = pk(e, e);
  const float4* f = reinterpret_cast<const float4*>(column);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float4 v = f[j];
    m[2 * j] = round2(mul(pk(g[4 * j], g[4 * j + 1]), mul(r2, pk(v.x, v.y))));
    m[2 * j + 1] = round2(mul(pk(g[4 * j + 2], g[4 * j + 3]), mul(r2, pk(v.z, v.w))));
  }
}
// The block (w, w) where a head forgets.  Apart from make_m, which then is no longer in the instruction caches' way (in line a packed batch took 465 us where it takes 436).
template <bool kWide>
__device__ __noinline__ void make_m_one_by_one(uint32_t at, const Scalars& s, int w, const uint8_t* masks) {
  const int lane = threadIdx.x & 31;
  uint32_t g[32];
  tmem_ld32(at, g);
  tmem_wait_ld();
#pragma unroll 1
  for (int h = 0; h < (kWide ? 1 : 2); ++h) {
    uint32_t m[16];
    if (forgets(s, h, w)) {
      const float2* delta = reinterpret_cast<const float2*>(s.g[h] + 32 * w);
      const float rate = s.rate[h];
      float sum = 0.f;                                                // of a behind the column's token up to the row's
#pragma unroll
      for (int j = 15; j >= 0; --j) {
        const float2 d = delta[j];
        const float hi = __uint_as_float(g[2 * j + 1]) * (ex2f(sum) * d.y);
        if (2 * j + 1 <= lane) sum = fmaf(rate, d.y, sum);
        m[j] = pack_bf16(__uint_as_float(g[2 * j]) * (ex2f(sum) * d.x), hi);
        if (2 * j <= lane) sum = fmaf(rate, d.x, sum);
      }
    } else {
      weigh_m(m, g, s.p[h][32 * w + lane], s.g[h] + 32 * w);
    }
    keep_triangle(m, masks + lane * kMaskPitch);
    tmem_st16(at + 16 * h, m);
  }
}
// M of the 32 x 32 block (w, b) from G, over it: 16 columns a head.  (One copy for all sixteen warps that make M: see wait_on.)
template <bool kWide>
__device__ __noinline__ void make_m(uint32_t at, const Scalars& s, int b, int w, const uint8_t* masks) {
  const int lane = threadIdx.x & 31;
  uint32_t g[32];
  at += 32 * b;
  if (b > w) {
#pragma unroll
    for (int i = 0; i < 32; ++i) g[i] = 0u;
    tmem_st32(at, g);
    return;
  }
  if (b == w && (forgets(s, 0, w) || (!kWide && forgets(s, 1, w)))) return make_m_one_by_one<kWide>(at, s, w, masks);
  tmem_ld32(at, g);
  tmem_wait_ld();
#pragma unroll 1
  for (int h = 0; h < (kWide ? 1 : 2); ++h) {
    uint32_t m[16];
    const float4 tot = *reinterpret_cast<const float4*>(s.tot[h]);
    // (with the sums over the 32-token blocks between the two)
    const float r = s.p[h][32 * w + lane] + (b < 1 && w > 1 ? tot.y : 0.f) + (b < 2 && w > 2 ? tot.z : 0.f);
    weigh_m(m, g, r, (b < w ? s.f[h] : s.g[h]) + 32 * b);
    if (b == w) keep_triangle(m, masks + lane * kMaskPitch);
    tmem_st16(at + 16 * h, m);
  }
}

// 32 rows of the state, half of the columns, from tensor memory to `dst` (its first row).  By way of 32 rows of shared memory (tiles of B and C, free by
// then): 16 bytes a lane straight from a row each kept the output's warps from shared memory for 2 us.
template <int kNs, bool kFp32>
__device__ __noinline__ void leave_state(uint32_t at, uint32_t rows, void* dst) {
  constexpr int kOwn = kNs / 2, kSize = kFp32 ? 4 : 2, kPieces = kOwn * kSize / 16, kPitch = kOwn * 4;
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int part = 0; part < kOwn / 32; ++part) {
    uint32_t v[32];
    tmem_ld32(at + 32 * part, v);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 2 * kSize; ++i) {
      const uint32_t to = rows + lane * kPitch + (((2 * kSize * part + i) ^ (lane & 7)) << 4);
      if constexpr (kFp32) {
        sts128(to, v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      } else {
        uint32_t word[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) word[k] = pack_bf16(__uint_as_float(v[8 * i + 2 * k]), __uint_as_float(v[8 * i + 2 * k + 1]));
        sts128(to, word[0], word[1], word[2], word[3]);
      }
    }
  }
  __syncwarp();
#pragma unroll 4
  for (int i = lane; i < 32 * kPieces; i += 32) {
    const int row = i / kPieces, piece = i % kPieces;
    *reinterpret_cast<uint4*>(static_cast<char*>(dst) + row * (kNs * kSize) + 16 * piece) = lds128(rows + row * kPitch + ((piece ^ (row & 7)) << 4));
  }
  fence_proxy_async_smem();                       // (tensor copies write there next)
}

// kWide: one head of P = 128, else two of P = 64.  kFull: the outputs too, else only what a run adds to a zero state.  kParts: of X', two or three.
template <int kNs, bool kWide, bool kFull, int kParts>
__global__ void __launch_bounds__(kThreads, 1) ssm_scan_kernel(const __grid_constant__ SsmMaps maps, const SsmScanParams p) {
  using L = Smem<kNs>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  auto bar = [&](int i) { return sbase + L::kBars + 8 * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc + 4);
  Scalars* scal = reinterpret_cast<Scalars*>(smem + L::kScal);

  if (tid < 4) prefetch_tensormap(&maps.x + tid);
  // the swizzled tiles need this alignment: report instead of computing garbage (below zero: a wait limit, test aid)
  if (tid == 0) *abort_flag = (sbase & 1023u) != 0u ? 1 : -p.wait_limit_us;
  if (kFull && tid < 512) {
    const int i = tid >> 4, j = 2 * (tid & 15);
    *reinterpret_cast<uint32_t*>(smem + L::kMask + i * kMaskPitch + 2 * j) = (j <= i ? 0xffffu : 0u) | (j + 1 <= i ? 0xffff0000u : 0u);
  }
  if (warp == 17) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  uint32_t tmem_base = 0;
  volatile unsigned* next = reinterpret_cast<volatile unsigned*>(smem + L::kMisc + 8);
  // Packed batches read their plan to begin with.  The others know their walk, and ask for what its first block needs while barriers and tensor memory are
  // set up.  Of the full pass behind a first one that is everything but the states: what the caller's kernels wrote was there before the first pass
  // went past its own wait.  (It reads around the first-level cache.)
  if (p.packed) {
    grid_dependency_wait();
  } else if (warp == 8 || warp == 16 || warp >= 18) {
    const SsmItem it = ssm_item(p, blockIdx.x, kFull);
    if (!kFull || !p.late) grid_dependency_wait();
    const int64_t start = kFull || it.blocks == 0 ? it.t0 : it.t0 + static_cast<int64_t>(it.blocks - 1) * kQ;
    const int64_t left = it.t0 + it.tokens - start;
    if (warp == 19) {
      if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kNs / 64; ++i) {
          tma_prefetch_3d(&maps.b, it.group * kNs + 64 * i, static_cast<int>(start), static_cast<int>(it.b));
          if (kFull) tma_prefetch_3d(&maps.c, it.group * kNs + 64 * i, static_cast<int>(start), static_cast<int>(it.b));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) tma_prefetch_3d(&maps.x, it.head0 * (kWide ? 128 : 64) + 64 * i, static_cast<int>(start), static_cast<int>(it.b));
      }
    } else if (warp >= 16) {
      const __nv_bfloat16* dt = p.dt + it.b * p.dts.batch + (start + 2 * lane + (warp == 18)) * p.dts.token + it.head0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (2 * lane + (warp == 18) + 64 * i < left) prefetch_l2(dt + 64 * i * p.dts.token);
      if (lane == 0) prefetch_l2(warp == 18 ? p.A_log + it.head0 : p.dt_bias + it.head0);
    } else if (kFull && warp == 8 && lane == 0 && p.initial_state != nullptr && it.slot < 0) {
      const int size = kNs * (p.state_fp32 ? 4 : 2), P = kWide ? 128 : 64;
      bulk_prefetch_l2(static_cast<const char*>(p.initial_state) + (static_cast<int64_t>(it.n) * p.H + it.head0) * P * size, (kWide || it.two ? 128 : 64) * size);
    }
  }
  // Packed batches: as many CTAs as there are SMs take one walk after the other, the longest first.
  for (unsigned turn = 0;; ++turn) {
  if (warp == 0) {
    if (lane == 0) *next = p.queue != nullptr ? atomicAdd(p.queue, 1u) : blockIdx.x;
    if (lane < B_COUNT) {
      if (turn > 0) mbar_inval(bar(lane));
      mbar_init(bar(lane), arrivals<kFull, kWide>(lane));
    }
    fence_mbar_init();
  }
  tc_fence_before();
  __syncwarp();                                     // (every warp comes here as one: lane 0 of most has just been on its own)
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  tmem_base = tmem;
  bool ok = *abort_flag <= 0;
  const SsmItem it = ssm_item(p, *next, kFull);
  if (!kFull || !p.late) grid_dependency_wait();
  if (!kFull) grid_release_next();                  // (the launches behind this one wait in their turn)
  const int blocks = ok ? it.blocks : 0;
  if (warp < 8) {
    if constexpr (kFull) {
      const int q = warp >> 2, w = warp & 3;                          // column blocks q, q + 2; rows 32 w + lane
      const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * w) << 16);
      const bool mine = kWide || q == 0 || it.two;                    // (this warpgroup's half of the output)
      const float D = blocks > 0 && mine && p.D != nullptr ? __ldcg(p.D + it.head0 + (kWide ? 0 : q)) : 0.f;
      for (int c = 0; c < blocks; ++c) {
        const Scalars& s = scal[c % kScals];
        if (!(ok = warp_wait(bar(B_SCAL + c % kScals), (c / kScals) & 1, abort_flag))) break;
        if (!(ok = warp_wait(bar(B_G), c & 1, abort_flag))) break;
        tc_fence_after();
        make_m<kWide>(lanes + kColG, s, q, w, smem + L::kMask);
        const int hq = kWide ? 0 : q;
        float before = 0.f;
        if (w > 0) before += s.tot[hq][0];
        if (w > 1) before += s.tot[hq][1];
        if (w > 2) before += s.tot[hq][2];
        const float e = ex2f(s.p[hq][32 * w + lane] + before);
        // C S^T -> what the rows' decays leave of it
        if (!(ok = warp_wait(bar(B_Z), c & 1, abort_flag))) break;
        tc_fence_after();
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          uint32_t y[32];
          tmem_ld32(lanes + kColY + 64 * q + 32 * half, y);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) mul2(y[2 * i], y[2 * i + 1], make_float2(e, e));
          tmem_st32(lanes + kColY + 64 * q + 32 * half, y);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar(B_M));
          mbar_arrive(bar(B_SCAL_FREE + c % kScals));
        }
        // ---- out ----------------------------------------------------------------------------------------------------------------
        if (!(ok = warp_wait(bar(B_Y), c & 1, abort_flag))) break;
        tc_fence_after();
        const int row = 32 * w + lane;
        const uint32_t xrow = sbase + L::kX + (c % kXs) * kTileX + q * (kTileX / 2) + row * 128;
        const f2 D2 = pk(D, D);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          uint32_t y[32];
          uint4 x[4];
          tmem_ld32(lanes + kColY + 64 * q + 32 * half, y);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = lds128(xrow + (((4 * half + j) ^ (row & 7)) << 4));
          tmem_wait_ld();
          if (half == 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_Y_FREE));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t xv[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = round2(fma2(pk(bf_lo(xv[i]), bf_hi(xv[i])), D2, pk(y[8 * j + 2 * i], y[8 * j + 2 * i + 1])));
            if (mine) sts128(xrow + (((4 * half + j) ^ (row & 7)) << 4), o[0], o[1], o[2], o[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_OUT + c % kXs));
      }
    }
  } else if (warp < 16) {
    // ---- the state (this thread's row of 128, half of its columns), then x' (every other step) -----------------------------------
    const int g = (warp - 8) >> 2, row = 32 * (warp & 3) + lane, h = kWide ? 0 : row >> 6;
    constexpr int kOwn = kNs / 2;                                     // columns g * kOwn ..
    const uint32_t at = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + kColS + g * kOwn;
    const bool there = kWide || h == 0 || it.two;
    auto state_at = [&](int r) { return ((static_cast<int64_t>(it.n) * p.H + it.head0 + h) * (kWide ? 128 : 64) + (kWide ? r : r & 63)) * kNs + g * kOwn; };
    float4* slot = it.slot >= 0 ? p.slots + static_cast<int64_t>(it.slot) * (128 * kNs / 4) + (g * kOwn / 4) * 128 + row : nullptr;       // (four columns of a row, 128 further on the next four)
    const int t = tid - 8 * 32;
    // X'^T over 64 tokens, this warp's 16 rows of 32, 32 tokens at a time.  A transposed 8 x 8 tile of x has two tokens of a channel in a register,
    // as tensor memory wants them (register 2j | 2j + 1: lane t/4 | t/4 + 8, column 4j + t%4).
    uint32_t part[2][kParts][8];
    auto weigh = [&](uint32_t x, const Scalars& s, int half) {
      const uint32_t src = x + ((warp & 3) >> 1) * (kTileX / 2) + (64 * half + 8 * (lane >> 4) + (lane & 7)) * 128 + (((4 * (warp & 1) + 2 * g + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
      const uint2* w = s.w[kWide ? 0 : h] + 32 * half + (lane & 3);
      const uint32_t* rest = s.rest[kWide ? 0 : h] + 32 * half + (lane & 3);
      __syncwarp();
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t (&first)[8] = part[q][0];
#pragma unroll
        for (int j = 0; j < 4; j += 2) ldsm_x4_trans(src + (32 * q + 8 * j) * 128, first[2 * j], first[2 * j + 1], first[2 * j + 2], first[2 * j + 3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint2 wj = w[16 * q + 4 * j];
          const uint32_t minus = wj.x ^ 0x80008000u, rj = kParts == 3 ? rest[16 * q + 4 * j] : 0u;
#pragma unroll
          for (int i = 2 * j; i < 2 * j + 2; ++i) {
            const uint32_t xi = first[i];
            first[i] = mul_bf2(xi, minus);                              // (the first part is minus what it stands for; the products have the sign)
            const uint32_t err = fma_bf2(xi, wj.x, first[i]);
            if constexpr (kParts == 2) {
              part[q][1][i] = fma_bf2(xi, wj.y, err);
            } else {
              part[q][1][i] = add_bf2(err, mul_bf2(xi, wj.y));
              part[q][2][i] = fma_bf2(xi, rj, fma_bf2(xi, wj.y, sub_bf2(err, part[q][1][i])));
            }
          }
        }
      }
    };
    auto put = [&](int quarter, int q, int k) { tmem_st_16x128b_x4(tmem + (static_cast<uint32_t>(32 * (warp & 3) + 16 * g) << 16) + piece_column<kParts, kFull>(quarter, k), part[q][k]); };
    auto stored = [&](int done) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(done));
    };
    if constexpr (!kFull) {
      // First pass: from the run's last block to its first, with weights that decay to the run's end, so that nothing is ever rescaled.
      // Two buffers of X'^T (from column 0 on: there is no G, M or output) and of B.
      for (int c = 0; c < blocks; ++c) {
        if (!(ok = warp_wait(bar(B_SCAL + c % kScals), (c / kScals) & 1, abort_flag))) break;
        if (!(ok = warp_wait(bar(B_FULL_X + c % kXs), (c / kXs) & 1, abort_flag))) break;
        if (c >= 2) {
          if (!(ok = warp_wait(bar(B_EMPTY_B + (c & 1)), ((c >> 1) - 1) & 1, abort_flag))) break;
          tc_fence_after();
        }
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          weigh(sbase + L::kX + (c % kXs) * kTileX, scal[c % kScals], half);
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int k = 0; k < kParts; ++k) put(4 * (c & 1) + 2 * half + q, q, k);
          stored((c & 1 ? B_XT2 : B_XT) + half);
        }
        if (lane == 0) {
          mbar_arrive(bar(B_SCAL_FREE + c % kScals));
          mbar_arrive(bar(B_EMPTY_X + c % kXs));
        }
      }
      if (ok && blocks > 0 && (ok = warp_wait(bar(B_S_FULL), 0, abort_flag))) {
        tc_fence_after();
#pragma unroll 1
        for (int part = 0; part < kOwn / 32; ++part) {
          uint32_t v[32];
          tmem_ld32(at + 32 * part, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(slot + (8 * part + i) * 128) = *reinterpret_cast<const uint4*>(v + 4 * i);
        }
      }
    } else {
      if (p.late) grid_dependency_wait();
      if (blocks > 0) {
#pragma unroll 1
        for (int part = 0; part < kOwn / 32; ++part) {
          uint32_t v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0u;
          if (there) {
            if (slot != nullptr) {
#pragma unroll
              for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(v + 4 * i) = *reinterpret_cast<const uint4*>(slot + (8 * part + i) * 128);
            } else if (p.initial_state != nullptr && p.state_fp32) {
              const float* src = static_cast<const float*>(p.initial_state) + state_at(row) + 32 * part;
#pragma unroll
              for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(v + 4 * i) = *reinterpret_cast<const uint4*>(src + 4 * i);
            } else if (p.initial_state != nullptr) {
              const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.initial_state) + state_at(row) + 32 * part;
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
          tmem_st32(at + 32 * part, v);
        }
        tmem_wait_st();
      }
      for (int c = 0; c < blocks; ++c) {
        if (c > 0) {
          if (!(ok = warp_wait(bar(B_S_FULL), (c - 1) & 1, abort_flag))) break;
          tc_fence_after();
        }
        const Scalars& s = scal[c % kScals];
        if (!(ok = warp_wait(bar(B_SCAL + c % kScals), (c / kScals) & 1, abort_flag))) break;
        const float d = s.decay[h];
#pragma unroll 1
        for (int part = 0; part < kOwn / 32; ++part) {
          uint32_t v[32];
          tmem_ld32(at + 32 * part, v);
          tmem_wait_ld();
          // the copy for C S^T (that of the block before has been read: its product came before those of the state)
          const uint32_t dst = sbase + L::kS + row * 128;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int piece = g * (kOwn / 8) + 4 * part + i;
            uint32_t word[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) word[k] = pack_bf16(__uint_as_float(v[8 * i + 2 * k]), __uint_as_float(v[8 * i + 2 * k + 1]));
            sts128(dst + (piece >> 3) * 16384 + (((piece & 7) ^ (row & 7)) << 4), word[0], word[1], word[2], word[3]);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) mul2(v[2 * i], v[2 * i + 1], make_float2(d, d));
          tmem_st32(at + 32 * part, v);
        }
        tmem_wait_st();
        tc_fence_before();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_S_READY));

        if (!(ok = warp_wait(bar(B_FULL_X + c % kXs), (c / kXs) & 1, abort_flag))) break;
        const uint32_t x = sbase + L::kX + (c % kXs) * kTileX;
        const int64_t left = it.tokens - static_cast<int64_t>(c) * kQ;
        if (left < kQ) {
          // the last block: rows past the end, in the tiles whose rows are summed over
          if (!(ok = warp_wait(bar(B_FULL_B), c & 1, abort_flag))) break;
          const uint32_t b = sbase + L::kB;
          for (int i = t; i < (kQ - static_cast<int>(left)) * 8; i += 256) {
            const uint32_t off = (static_cast<uint32_t>(left) + i / 8) * 128 + (i % 8) * 16;
            sts128(x + off, 0u, 0u, 0u, 0u);
            sts128(x + kTileX / 2 + off, 0u, 0u, 0u, 0u);
            sts128(b + off, 0u, 0u, 0u, 0u);
            if (kNs == 128) sts128(b + L::kTile / 2 + off, 0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(B_MEET));
          if (!(ok = warp_wait(bar(B_MEET), 0, abort_flag))) break;
        }
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          weigh(x, s, half);
          if (kParts == 3 && half == 1) {
            // the first eight pieces are there; the last four follow the products of the first quarter, and of the second
            put(2, 0, 2);
            put(2, 0, 1);
            stored(B_XT + 1);
            if (!(ok = warp_wait(bar(B_XT_FREE), c & 1, abort_flag))) break;
            tc_fence_after();
            put(2, 0, 0);
            put(3, 1, 2);
            put(3, 1, 1);
            stored(B_XT);
            if (!(ok = warp_wait(bar(B_XT_FREE + 1), c & 1, abort_flag))) break;
            tc_fence_after();
            put(3, 1, 0);
            stored(B_XT + 1);
          } else {
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int k = 0; k < kParts; ++k) put(2 * half + q, q, k);
            stored(B_XT + half);
          }
          if (half == 1) {
            if (!(ok = warp_wait(bar(B_G), c & 1, abort_flag))) break;
            tc_fence_after();
            make_m<kWide>(tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + kColG, s, 2 + g, warp & 3, smem + L::kMask);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_M));
          }
        }
        if (!ok) break;
        if (lane == 0) mbar_arrive(bar(B_SCAL_FREE + c % kScals));
      }
      if (ok && blocks > 0 && (ok = warp_wait(bar(B_S_FULL), (blocks - 1) & 1, abort_flag)) && there && it.last && p.final_state != nullptr) {
        tc_fence_after();
        const int64_t first = state_at(row - lane);
        if (p.state_fp32) leave_state<kNs, true>(at, sbase + L::kB + (t - lane) * (kOwn * 4), static_cast<float*>(p.final_state) + first);
        else leave_state<kNs, false>(at, sbase + L::kB + (t - lane) * (kOwn * 4), static_cast<__nv_bfloat16*>(p.final_state) + first);
      }
    }
  } else if (warp == 17) {
    // ---- products ----------------------------------------------------------------------------------------------------------------
    constexpr uint32_t idesc_g = umma_idesc_bf16(128, 128, 0, 0), idesc_s = umma_idesc_bf16(128, kNs, 0, 1), idesc_y = umma_idesc_bf16(128, kWide ? 128 : 64, 0, 1);
    constexpr uint32_t kMinusA = 1u << 13;                            // (of an instruction descriptor: A with the other sign)
    // S += X'^T B over 32 tokens, the smallest parts first (sums are rounded towards zero)
    auto add_part = [&](uint32_t b, int quarter, int slot, int part, bool onto) {
      const uint64_t db = desc_sw128(b + quarter * 4096, 16384);
#pragma unroll
      for (int k = 0; k < 2; ++k) umma_ts(tmem + kColS, tmem + piece_column<kParts, kFull>(slot, part) + 8 * k, db + k * 128, idesc_s | (part == 0 ? kMinusA : 0u), onto || k > 0);
    };
    if constexpr (!kFull) {
      for (int c = 0; c < blocks; ++c) {
        if (!(ok = warp_wait(bar(B_FULL_B + (c & 1)), (c >> 1) & 1, abort_flag))) break;
        for (int th = 0; th < 2; ++th) {
          if (!(ok = warp_wait(bar((c & 1 ? B_XT2 : B_XT) + th), (c >> 1) & 1, abort_flag))) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int q = 2 * th; q < 2 * th + 2; ++q)
#pragma unroll
              for (int k = kParts - 1; k >= 0; --k) add_part(sbase + L::kB + (c & 1) * L::kTile, q, 4 * (c & 1) + q, k, c + q > 0 || k + 1 < kParts);
            if (th == 1) {
              if (c + 2 < blocks) umma_commit(bar(B_EMPTY_B + (c & 1)));
              else if (c + 1 == blocks) umma_commit(bar(B_S_FULL));
            }
          }
          __syncwarp();
        }
        if (!ok) break;
      }
    }
    const uint64_t dc = desc_sw128(sbase + L::kC, 16), ds = desc_sw128(sbase + L::kS, 16);
    for (int c = 0; kFull && c < blocks; ++c) {
      const uint32_t b = sbase + L::kB, x = sbase + L::kX + (c % kXs) * kTileX;
      if (!(ok = warp_wait(bar(B_FULL_B), c & 1, abort_flag))) break;
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
      if (!(ok = warp_wait(bar(B_S_READY), c & 1, abort_flag))) break;
      if (c > 0 && !(ok = warp_wait(bar(B_Y_FREE), (c - 1) & 1, abort_flag))) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kNs / 16; ++k) umma_ss(tmem + kColY, dc + (k / 4) * 1024 + (k % 4) * 2, ds + (k / 4) * 1024 + (k % 4) * 2, idesc_g, k > 0);
        umma_commit(bar(B_Z));
      }
      __syncwarp();
      if constexpr (kParts == 3) {
        // pieces 0 to 5, 6 and 7, 8 to 10, 11: as they come
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          if (!(ok = warp_wait(bar(B_XT + (step & 1)), step >> 1, abort_flag))) break;
          tc_fence_after();
          if (elect_one()) {
            if (step == 1) umma_commit(bar(B_XT_FREE + 1));           // (the first two quarters)
#pragma unroll
            for (int piece = step == 0 ? 0 : step == 1 ? 6 : step == 2 ? 8 : 11; piece < (step == 0 ? 6 : step == 1 ? 8 : step == 2 ? 11 : 12); ++piece) {
              add_part(b, piece / 3, piece / 3, 2 - piece % 3, true);
              if (piece == 2) umma_commit(bar(B_XT_FREE));
            }
            if (step == 3) umma_commit(bar(B_S_FULL));
          }
          __syncwarp();
        }
      } else {
        for (int th = 0; th < 2; ++th) {
          if (!(ok = warp_wait(bar(B_XT + th), c & 1, abort_flag))) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int q = 2 * th; q < 2 * th + 2; ++q)
#pragma unroll
              for (int k = kParts - 1; k >= 0; --k) add_part(b, q, q, k, true);
            if (th == 1) umma_commit(bar(B_S_FULL));
          }
          __syncwarp();
        }
      }
      if (!ok) break;
      if (!(ok = warp_wait(bar(B_FULL_X + c % kXs), (c / kXs) & 1, abort_flag))) break;
      if (!(ok = warp_wait(bar(B_M), c & 1, abort_flag))) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < (kWide ? 1 : 2); ++h) {
          const uint64_t dx = desc_sw128(x + h * (kTileX / 2), 16384);
#pragma unroll
          for (int k = 0; k < 8; ++k) umma_ts(tmem + kColY + 64 * h, tmem + kColG + 32 * (k / 2) + 16 * h + 8 * (k % 2), dx + k * 128, idesc_y, 1);
        }
        umma_commit(bar(B_Y));
      }
      __syncwarp();
    }
    // no product may be under way when the tensor memory is given back
    if (elect_one()) umma_commit(bar(B_DRAIN));
    __syncwarp();
    if (lane == 0) drain(bar(B_DRAIN), 0);
    __syncwarp();
  } else if (warp != 19) {
    // ---- delta and the decays of a head: four tokens a lane, eight lanes a 32-token block (the second head's on warp 18) ------------
    const int h = warp == 16 ? 0 : 1, head = it.head0 + (h == 1 && it.two ? 1 : 0), mine = kWide && h == 1 ? 0 : blocks;
    float log_decay = 0.f, A = 0.f, bias = 0.f;
    // dt of this block and the next two: asked for two blocks ahead, as nothing else hides the way to memory
    const int64_t pitch = p.dts.token, turn_on = (kFull ? kQ : -kQ) * pitch;
    const int64_t start = kFull || blocks == 0 ? 0 : static_cast<int64_t>(blocks - 1) * kQ;       // (the first pass goes backwards)
    const unsigned short* src = reinterpret_cast<const unsigned short*>(p.dt) + it.b * p.dts.batch + (it.t0 + start + 4 * lane) * pitch + head;
    auto load_dt = [&](int c, uint32_t (&to)[4]) {
      const int64_t left = c < mine ? it.tokens - static_cast<int64_t>(kFull ? c : blocks - 1 - c) * kQ - 4 * lane : 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) to[k] = k < left ? static_cast<uint32_t>(__ldcg(src + k * pitch)) << 16 : 0u;
      src += turn_on;
    };
    uint32_t raw[4], then[4], after_then[4];
    load_dt(0, raw);
    load_dt(1, then);
    if (mine > 0) {
      A = -kLog2e * ex2f(kLog2e * __ldcg(p.A_log + head));
      bias = __ldcg(p.dt_bias + head);
    }
#pragma unroll 1
    for (int c = 0; c < mine; ++c) {
      Scalars& s = scal[c % kScals];
      load_dt(c + 2, after_then);
      const int64_t left = it.tokens - static_cast<int64_t>(kFull ? c : blocks - 1 - c) * kQ - 4 * lane;      // this lane's tokens that are there
      float d[4], a[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        d[k] = k < left ? softplus(__uint_as_float(raw[k]) + bias) : 0.f;
        a[k] = k < left ? A * d[k] : 0.f;
        raw[k] = then[k];
        then[k] = after_then[k];
      }
      const float own = (a[0] + a[1]) + (a[2] + a[3]);
      float up = own, down = own;                                     // inclusive sums over the eight lanes, forwards and backwards
#pragma unroll
      for (int i = 1; i < 8; i <<= 1) {
        const float u = __shfl_up_sync(0xffffffffu, up, i), e = __shfl_down_sync(0xffffffffu, down, i);
        if ((lane & 7) >= i) up += u;
        if ((lane & 7) + i < 8) down += e;
      }
      const float before = __shfl_up_sync(0xffffffffu, up, 1), after = __shfl_down_sync(0xffffffffu, down, 1);
      const float head_sum = (lane & 7) == 0 ? 0.f : before, rest = (lane & 7) == 7 ? 0.f : after;
      const float t0 = __shfl_sync(0xffffffffu, up, 7), t1 = __shfl_sync(0xffffffffu, up, 15), t2 = __shfl_sync(0xffffffffu, up, 23), t3 = __shfl_sync(0xffffffffu, up, 31);
      const int block = lane >> 3;
      const float behind = (block < 1 ? t1 : 0.f) + (block < 2 ? t2 : 0.f) + (block < 3 ? t3 : 0.f);
      const float sum = (t0 + t1) + (t2 + t3), to_end = ex2f(kFull ? behind : behind + log_decay);
      log_decay += sum;
      const float s2 = rest + a[3], s1 = s2 + a[2], s0 = s1 + a[1];
      const float4 f = make_float4(d[0] * ex2f(s0), d[1] * ex2f(s1), d[2] * ex2f(s2), d[3] * ex2f(rest));
      const float w0 = f.x * to_end, w1 = f.y * to_end, w2 = f.z * to_end, w3 = f.w * to_end;
      const uint32_t h01 = pack_bf16(w0, w1), h23 = pack_bf16(w2, w3);
      const float l0 = w0 - bf_lo(h01), l1 = w1 - bf_hi(h01), l2 = w2 - bf_lo(h23), l3 = w3 - bf_hi(h23);
      const uint32_t l01 = pack_bf16(l0, l1), l23 = pack_bf16(l2, l3);
      if (c >= kScals && !(ok = warp_wait(bar(B_SCAL_FREE + c % kScals), (c / kScals - 1) & 1, abort_flag))) break;
      reinterpret_cast<uint4*>(s.w[h])[lane] = make_uint4(h01, l01, h23, l23);
      if constexpr (kParts == 3) reinterpret_cast<uint2*>(s.rest[h])[lane] = make_uint2(pack_bf16(l0 - bf_lo(l01), l1 - bf_hi(l01)), pack_bf16(l2 - bf_lo(l23), l3 - bf_hi(l23)));
      if constexpr (kFull) {
        const float whole = block == 0 ? t0 : block == 1 ? t1 : block == 2 ? t2 : t3;
        const float most = fmaxf(kMostDecay, A * kMostDelta);
        const float p0 = head_sum + a[0], p1 = p0 + a[1], p2 = p1 + a[2], p3 = p2 + a[3];
        reinterpret_cast<float4*>(s.p[h])[lane] = make_float4(p0, p1, p2, p3);
        reinterpret_cast<float4*>(s.g[h])[lane] = whole >= most ? make_float4(d[0] * ex2f(-p0), d[1] * ex2f(-p1), d[2] * ex2f(-p2), d[3] * ex2f(-p3))
                                                                      : make_float4(d[0], d[1], d[2], d[3]);
        reinterpret_cast<float4*>(s.f[h])[lane] = f;
        if (lane == 0) {
          *reinterpret_cast<float4*>(s.tot[h]) = make_float4(t0, t1, t2, t3);
          s.decay[h] = ex2f(sum);
          s.rate[h] = A;
          s.most[h] = most;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_SCAL + c % kScals));
    }
    if (!kFull && ok && mine > 0 && lane == 0) {
      p.decays[2 * it.slot + h] = ex2f(log_decay);
      if (kWide) p.decays[2 * it.slot + 1] = ex2f(log_decay);
    }
  } else {
    // ---- tensor copies ------------------------------------------------------------------------------------------------------------
    // They are worked off one behind the other, and a tile of out takes some 1400 cycles to leave.  So it goes behind the loads of B and
    // C, for which the next block's first product waits; x, of which there are three tiles, comes long before it is wanted.
    const int column = it.head0 * (kWide ? 128 : 64), bc_column = it.group * kNs, first = static_cast<int>(it.t0), batch = static_cast<int>(it.b);
    const int most = blocks < p.stop_loads_after ? blocks : p.stop_loads_after;
    int nb = 0, nc = 0, nx = 0;                                       // loads of B, C, x so far
    auto row_of = [&](int n) { return first + (kFull ? n : blocks - 1 - n) * kQ; };      // (the first pass goes backwards)
    auto load_x = [&] {
      if (lane == 0) {
        const uint32_t full = bar(B_FULL_X + nx % kXs);
        mbar_arrive_expect_tx(full, kTileX);
#pragma unroll
        for (int i = 0; i < 2; ++i) tma_load_3d(sbase + L::kX + (nx % kXs) * kTileX + i * (kTileX / 2), &maps.x, column + 64 * i, row_of(nx), batch, full);
      }
      ++nx;
      __syncwarp();
    };
    auto load_bc = [&](const CUtensorMap* map, uint32_t to, int full, int& n) {
      if (lane == 0) {
        mbar_arrive_expect_tx(bar(full), L::kTile);
#pragma unroll
        for (int i = 0; i < kNs / 64; ++i) tma_load_3d(to + i * 16384, map, bc_column + 64 * i, row_of(n), batch, bar(full));
      }
      ++n;
      __syncwarp();
    };
    auto store = [&](int c) {
      if (!warp_wait(bar(B_OUT + c % kXs), (c / kXs) & 1, abort_flag)) return false;
      const uint32_t x = sbase + L::kX + (c % kXs) * kTileX;
      const int64_t left = it.tokens - static_cast<int64_t>(c) * kQ;
      if (p.packed && left < kQ) {
        // rows behind the sequence's end are somebody else's
        const int pieces = kWide || it.two ? 16 : 8;
        __nv_bfloat16* dst = p.out + (it.t0 + static_cast<int64_t>(c) * kQ) * p.os.token + column;
        for (int i = lane; i < static_cast<int>(left) * pieces; i += 32) {
          const int row = i / pieces, piece = i % pieces;
          *reinterpret_cast<uint4*>(dst + row * p.os.token + piece * 8) = lds128(x + (piece >> 3) * (kTileX / 2) + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
        }
      } else if (lane == 0) {
        tma_store_3d(&maps.out, x, column, first + c * kQ, batch);
        if (kWide || it.two) tma_store_3d(&maps.out, x + kTileX / 2, column + 64, first + c * kQ, batch);
        bulk_commit();
      }
      __syncwarp();
      return true;
    };
    if (most > 0) {
      load_bc(&maps.b, sbase + L::kB, B_FULL_B, nb);
      if constexpr (kFull) load_bc(&maps.c, sbase + L::kC, B_FULL_C, nc);
      else if (nb < most) load_bc(&maps.b, sbase + L::kB + L::kTile, B_FULL_B + 1, nb);
      while (nx < kXs && nx < most) load_x();
    }
    for (int c = 0; c < blocks; ++c) {
      if (c + 1 >= kXs && c + 1 < most) {
        if constexpr (kFull) {
          if (lane == 0) bulk_wait_read0();                           // (the output of block c - 2, which lay there)
        } else {
          if (!(ok = warp_wait(bar(B_EMPTY_X + nx % kXs), (nx / kXs - 1) & 1, abort_flag))) break;
        }
        load_x();
      }
      if constexpr (kFull) {
        if (c + 1 < most) {
          if (!(ok = warp_wait(bar(B_Z), c & 1, abort_flag))) break;
          load_bc(&maps.c, sbase + L::kC, B_FULL_C, nc);
          if (!(ok = warp_wait(bar(B_S_FULL), c & 1, abort_flag))) break;
          load_bc(&maps.b, sbase + L::kB, B_FULL_B, nb);
        }
      } else if (c + 2 < most) {
        if (!(ok = warp_wait(bar(B_EMPTY_B + (c & 1)), (c >> 1) & 1, abort_flag))) break;
        load_bc(&maps.b, sbase + L::kB + (c & 1) * L::kTile, B_FULL_B + (c & 1), nb);
      }
      if (kFull && c > 0 && !(ok = store(c - 1))) break;
    }
    if (kFull && ok && blocks > 0) ok = store(blocks - 1);
    // every copy has landed before this CTA's memory goes to another: those that nobody waited for
    if (lane == 0) {
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      for (int c = nx > kXs ? nx - kXs : 0; c < nx; ++c) drain(bar(B_FULL_X + c % kXs), (c / kXs) & 1);
      if constexpr (kFull) {
        if (nb > 0) drain(bar(B_FULL_B), (nb - 1) & 1);
        if (nc > 0) drain(bar(B_FULL_C), (nc - 1) & 1);
      } else {
        for (int c = nb > 2 ? nb - 2 : 0; c < nb; ++c) drain(bar(B_FULL_B + (c & 1)), (c >> 1) & 1);
      }
    }
    __syncwarp();
  }
  if (!ok) *abort_flag = 1;
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (*abort_flag > 0 || p.queue == nullptr || !it.there) break;
  }
  if (kFull && p.late) grid_dependency_wait();       // (all of it: what follows in the stream waits for this launch alone)
  if (tid == 0 && *abort_flag > 0) atomicCAS(p.status, kStatusOk, kStatusWaitTimeout);
  if (warp == 17) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---- plan of a packed batch, and the chaining of runs -------------------------------------------------------------------------------
// Sequences of more than kSsmStepT tokens, longest first, cut into runs of the length that the costs below (in blocks of the full walk) make cheapest.
constexpr int kPlanThreads = 512, kPlanWarps = kPlanThreads / 32, kCandidates = 8;
__device__ __forceinline__ int candidate(int least, int i) {         // run lengths that are tried; the last one: whole sequences
  return i == kCandidates - 1 ? 0x7fffffff : (least << (i >> 1)) + ((i & 1) ? (least << (i >> 1)) / 2 : 0);
}
__global__ void __launch_bounds__(kPlanThreads) ssm_plan_kernel(const int64_t* cu, int N, int64_t T, int pairs, int sms, int least, SsmPlan* plan, int* status) {
  __shared__ int s_blocks[kSsmPlanMost], s_seq[kSsmPlanMost];
  __shared__ int s_sum[2][kPlanWarps], s_active, s_longest, s_bad, s_run, s_cut, s_total, s_first[kCandidates], s_cuts[kCandidates], s_runs[kCandidates];
  grid_dependency_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_active = s_longest = s_bad = s_cut = s_total = 0;
  if (tid < kCandidates) s_first[tid] = s_cuts[tid] = s_runs[tid] = 0;
  __syncthreads();
  auto blocks_of = [&](int n) {
    int64_t bos = cu[n], eos = cu[n + 1];
    if (bos < 0 || eos < bos || eos > T) s_bad = 1;
    bos = bos < 0 ? 0 : bos > T ? T : bos;
    eos = eos < bos ? bos : eos > T ? T : eos;
    return eos - bos <= kSsmStepT ? 0 : static_cast<int>((eos - bos + kQ - 1) / kQ);
  };
  // the sequences with blocks, in the order that they come in where they are too many to be sorted
  int *order = plan->order(), *prefix = plan->prefix(N), *slots = plan->slot_prefix(N);
  for (int base = 0; base < N; base += kPlanThreads) {
    const int n = base + tid, b = n < N ? blocks_of(n) : 0;
    const unsigned vote = __ballot_sync(0xffffffffu, b > 0);
    if (lane == 0) s_sum[0][warp] = __popc(vote);
    __syncthreads();
    int at = s_active + __popc(vote & ((1u << lane) - 1));
    for (int i = 0; i < warp; ++i) at += s_sum[0][i];
    if (b > 0) {
      if (at < N) order[at] = n;
      if (at < kSsmPlanMost) {
        s_seq[at] = n;
        s_blocks[at] = b;
      }
      atomicMax(&s_longest, b);
      atomicAdd(&s_total, b);
      for (int i = 0; i < kCandidates - 1 && least > 0; ++i) {
        const int l = candidate(least, i);
        if (b > l) {
          atomicAdd(&s_first[i], (b - 1) / l * l);
          atomicAdd(&s_cuts[i], 1);
          atomicAdd(&s_runs[i], (b - 1) / l + 1);
        }
      }
    }
    __syncthreads();
    if (tid < 32) {
      int k = lane < kPlanWarps ? s_sum[0][lane] : 0;
      for (int d = 16; d > 0; d >>= 1) k += __shfl_xor_sync(0xffffffffu, k, d);
      if (lane == 0) s_active += k;
    }
    __syncthreads();
  }
  // (sequences that are not monotone may overlap, and then be more than there is room for: none is walked)
  const int active = s_bad ? 0 : s_active;
  const bool sorted = active <= kSsmPlanMost;
  if (tid < 32) {
    // the cheapest run length: the longest walk or an even share of all, whichever takes longer, and a little of the other; the same for
    // the first pass, which takes the runs of cut sequences but their last ones; and the states between the passes
    float cost = 3e38f;
    if (lane < kCandidates && (lane == kCandidates - 1 || (least > 0 && sorted))) {
      const int l = candidate(least, lane), cuts = lane < kCandidates - 1 ? s_cuts[lane] : 0, runs = lane < kCandidates - 1 ? s_runs[lane] : 0;
      const float share = static_cast<float>(pairs) / sms, longest = s_longest < l ? s_longest : l;
      auto both = [](float a, float b) { return fmaxf(a, b) + 0.15f * fminf(a, b); };
      cost = both((100.f * s_total + kSsmStartCost * (active - cuts + runs)) * share, 100.f * longest + kSsmStartCost);
      if (cuts > 0) cost += both((kSsmFirstCost * s_first[lane] + kSsmStartCost * (runs - cuts)) * share, kSsmFirstCost * longest + kSsmStartCost) + kSsmChainCost + kSsmSlotCost * 0.01f * runs * pairs;
    }
    float best = cost;
    for (int d = 16; d > 0; d >>= 1) best = fminf(best, __shfl_xor_sync(0xffffffffu, best, d));
    const unsigned at = __ballot_sync(0xffffffffu, cost == best);
    if (lane == 0) {
      s_run = candidate(least, 31 - __clz(at));                        // (of equal ones the longest)
      plan->run_blocks = s_run;
      plan->active = active;
      plan->next[0] = plan->next[1] = 0;
      if (status != nullptr) *status = s_bad ? kStatusBadCuSeqlens : 0;
    }
  }
  if (sorted) {
    for (int i = tid; i < active; i += kPlanThreads) {
      const int b = s_blocks[i];
      int rank = 0;
      for (int k = 0; k < active; ++k) rank += s_blocks[k] > b || (s_blocks[k] == b && k < i);
      order[rank] = s_seq[i];
    }
  }
  __syncthreads();
  const int run = s_run;
  // prefixes over the ranks: runs, and runs of the sequences that are cut (they come first)
  int done[2] = {0, 0};
  for (int base = 0; base < active; base += kPlanThreads) {
    const int i = base + tid;
    int runs = 0;
    if (i < active) runs = run == 0x7fffffff ? 1 : (blocks_of(order[i]) + run - 1) / run;
    int a = runs, c = runs > 1 ? runs : 0;
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, a, d), v = __shfl_up_sync(0xffffffffu, c, d);
      if (lane >= d) {
        a += u;
        c += v;
      }
    }
    if (lane == 31) {
      s_sum[0][warp] = a;
      s_sum[1][warp] = c;
    }
    __syncthreads();
    int whole[2] = {0, 0};
    for (int k = 0; k < kPlanWarps; ++k) {
      if (k < warp) {
        a += s_sum[0][k];
        c += s_sum[1][k];
      }
      whole[0] += s_sum[0][k];
      whole[1] += s_sum[1][k];
    }
    if (i < active) {
      prefix[i + 1] = done[0] + a;
      slots[i + 1] = done[1] + c;
      if (runs > 1) atomicMax(&s_cut, i + 1);
    }
    done[0] += whole[0];
    done[1] += whole[1];
    __syncthreads();
  }
  if (tid == 0) {
    prefix[0] = slots[0] = 0;
    plan->cut = s_cut;
    plan->walks[0] = done[1];
    plan->walks[1] = done[0];
  }
}

// Per sequence that is cut: its runs' local states -> the state that each run starts from.
__global__ void __launch_bounds__(256) ssm_chain_kernel(const SsmScanParams p, int Ns, int pairs) {
  grid_release_next();
  if (p.packed) grid_dependency_wait();
  const int pieces = 128 * Ns / 4 / 256;                              // blocks of 256 float4
  const int piece = static_cast<int>(blockIdx.x % pieces), pair = static_cast<int>(blockIdx.x / pieces % pairs);
  const int stride = static_cast<int>(gridDim.x / pieces / pairs), ranks = p.packed ? p.plan->cut : p.N;
  for (int rank = static_cast<int>(blockIdx.x / pieces / pairs); rank < ranks; rank += stride) {
  int n = rank, runs = p.runs, first = rank * p.runs;
  if (p.packed) {
    n = p.plan->order()[rank];
    first = p.plan->slot_prefix(p.N)[rank];
    runs = p.plan->slot_prefix(p.N)[rank + 1] - first;
  }
  const int at = piece * 256 + threadIdx.x, row = at & 127, column = (at >> 7) * 4;      // (the order of the states' memory)
  const int per = p.P == 128 ? 1 : 2, in_group = p.H / p.G, group = pair / p.pairs_per_group;
  const int within = (pair - group * p.pairs_per_group) * per + (per == 2 ? row >> 6 : 0);       // head within its group
  const int h = per == 2 ? row >> 6 : 0;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  // (the caller's, which was there before the first pass went past its wait)
  if (p.initial_state != nullptr && within < in_group) {
    const int64_t src = ((static_cast<int64_t>(n) * p.H + group * in_group + within) * p.P + (per == 2 ? row & 63 : row)) * Ns + column;
    if (p.state_fp32) {
      s = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(p.initial_state) + src));
    } else {
      const uint2 w = __ldcg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.initial_state) + src));
      s = make_float4(bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y));
    }
  }
  grid_dependency_wait();
  // (eight runs' states and decays on their way at a time: one behind the other, a run takes 1.9 us)
  constexpr int kAhead = 8;
  for (int r0 = 0; r0 < runs; r0 += kAhead) {
    float4 local[kAhead];
    float d[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t slot = static_cast<int64_t>(first + r0 + i) * pairs + pair;
      if (r0 + i + 1 < runs) {
        local[i] = p.slots[slot * (32 * Ns) + at];
        d[i] = p.decays[2 * slot + h];
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (r0 + i >= runs) break;
      const int64_t slot = static_cast<int64_t>(first + r0 + i) * pairs + pair;
      p.slots[slot * (32 * Ns) + at] = s;
      if (r0 + i + 1 < runs) s = make_float4(fmaf(d[i], s.x, local[i].x), fmaf(d[i], s.y, local[i].y), fmaf(d[i], s.z, local[i].z), fmaf(d[i], s.w, local[i].w));
    }
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

template <int kNs, bool kWide, bool kFull, int kParts>
cudaError_t launch_walk(const SsmMaps& maps, const SsmScanParams& p, int64_t items, cudaStream_t stream) {
  if (items == 0) return cudaSuccess;
  static SmemOptIn opt_in;
  auto kernel = ssm_scan_kernel<kNs, kWide, kFull, kParts>;
  const cudaError_t e = opt_in.ensure(kernel, Smem<kNs>::kBytes);
  if (e != cudaSuccess) return e;
  const int64_t ctas = p.queue != nullptr && items > device_sm_count() ? device_sm_count() : items;
  return launch_after(kernel, dim3(static_cast<unsigned>(ctas)), kThreads, Smem<kNs>::kBytes, stream, maps, p);
}
template <bool kFull, int kParts>
cudaError_t launch_pass(const SsmMaps& maps, const SsmScanParams& p, int Ns, int64_t items, cudaStream_t stream) {
  if (Ns == 128) return p.P == 128 ? launch_walk<128, true, kFull, kParts>(maps, p, items, stream) : launch_walk<128, false, kFull, kParts>(maps, p, items, stream);
  return p.P == 128 ? launch_walk<64, true, kFull, kParts>(maps, p, items, stream) : launch_walk<64, false, kFull, kParts>(maps, p, items, stream);
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
    int64_t best = rounds(chains) * (blocks * 100 + kSsmStartCost);
    L.runs = 1;
    L.run_blocks = static_cast<int>(blocks);
    for (int64_t r = 2; r <= blocks && r <= 160 && chains < 4 * sms; ++r) {
      const int64_t len = (blocks + r - 1) / r;
      if ((r - 1) * len >= blocks) continue;                        // the last run would be empty
      const int64_t cost = rounds(chains * r) * (len * 100 + kSsmStartCost) + rounds(chains * (r - 1)) * (len * kSsmFirstCost + kSsmStartCost) + kSsmChainCost +
                           kSsmSlotCost * chains * r / 100;
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
  p.slots = reinterpret_cast<float4*>(ws + L.slot_off);
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
  p.wait_limit_us = aid.wait_limit_us;
  p.stop_loads_after = aid.stop_loads_after > 0 ? aid.stop_loads_after : 0x7fffffff;
  const bool exact = q.final_state != nullptr && q.state_fp32;        // (a state that is rounded to bf16 has no use for more than 16 bits of what is added to it)
  cudaError_t e = cudaSuccess;
  if (packed) {
    e = launch_after(ssm_scan::ssm_plan_kernel, dim3(1), ssm_scan::kPlanThreads, 0, stream, q.cu_seqlens, q.N, q.T, L.pairs, device_sm_count(), L.least, p.plan, p.status);
    // the sequences of a few tokens, decode steps among the prompts
    if (e == cudaSuccess) e = launch_ssm_step(q, kSsmStepT, nullptr, stream);
  } else if (clear_status) {
    e = cudaMemsetAsync(ws, 0, 4, stream);
  }
  if (e != cudaSuccess) return e;
  if (L.first_items > 0) {
    if (packed) p.queue = p.plan->next;
    e = exact ? ssm_scan::launch_pass<false, 3>(maps, p, q.Ns, L.first_items, stream) : ssm_scan::launch_pass<false, 2>(maps, p, q.Ns, L.first_items, stream);
    if (e != cudaSuccess) return e;
    const int64_t each = L.pairs * (128 * q.Ns / 1024), most = (8 * device_sm_count() + each - 1) / each;
    e = launch_after(ssm_scan::ssm_chain_kernel, dim3(static_cast<unsigned>(each * (L.chained < most ? L.chained : most))), 256, 0, stream, p, q.Ns, L.pairs);
    if (e != cudaSuccess) return e;
  }
  if (packed) p.queue = p.plan->next + 1;
  p.late = !packed && L.first_items > 0;
  return exact ? ssm_scan::launch_pass<true, 3>(maps, p, q.Ns, L.items, stream) : ssm_scan::launch_pass<true, 2>(maps, p, q.Ns, L.items, stream);
}

}  // namespace fkda
