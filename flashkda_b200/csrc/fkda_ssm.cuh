// What the block form of the selective scan (fkda_ssm_scan.cu) and the C ABI share: sizes, plan, workspace.
#pragma once
#include <cuda.h>

#include "fkda_layer.cuh"

namespace fkda {

constexpr int kSsmBlock = 128;       // tokens of a block
// Sequences of at most this many tokens go token by token (fkda_ssm_step.cu).  Both sides, us, with fp32 states in and out:
//     heads, P x Ns, batch      32, 64 x 128, 1    32, 64 x 128, 16    32, 64 x 128, 128    32, 128 x 128, 128    32, 64 x 64, 128
//     16 tokens one by one / in blocks   6.2 / 11.8          23 / 24            143 / 161             275 / 315              75 / 136
//     32 tokens                         10.4 / 11.9          42 / 25            257 / 163             500 / 317             133 / 137
// (One number for all: a single sequence, and states of 64 x 64, would gain up to 1.5 us in 12 and 4 in 137 from a later border; the others lose far more.)
constexpr int kSsmStepT = 16;
constexpr int kSsmPlanMost = 2048;   // packed batches of more sequences keep the given order and are not cut into runs
// What the planner of runs reckons with, in hundredths of a block's walk (some 3 us): a block of the first pass, what a walk takes beside its
// blocks, the launch that chains runs, and (in hundredths of that) what a run's state of a pair of heads takes on its way through memory.
constexpr int kSsmFirstCost = 48, kSsmStartCost = 170, kSsmChainCost = 150, kSsmSlotCost = 175;

// A packed batch as the plan kernel leaves it: sequences by rank (longest first), prefix sums over the ranks of their runs, and of the
// runs of those that are cut into more than one (`cut` of them, the first ranks).
struct SsmPlan {
  int run_blocks;
  int active;                // sequences that are walked in blocks
  int cut;
  unsigned next[2];          // walks handed out so far: first pass, second pass
  int walks[2];              // how many there are, of a pair of heads (the first pass's with the last run of each, which it leaves out)
  int pad;
  __host__ __device__ int* order() { return reinterpret_cast<int*>(this + 1); }
  __host__ __device__ int* prefix(int N) { return order() + N; }
  __host__ __device__ int* slot_prefix(int N) { return prefix(N) + N + 1; }
};

struct SsmMaps {
  CUtensorMap x, b, c, out;
};

struct SsmScanParams {
  const __nv_bfloat16* dt;
  __nv_bfloat16* out;
  const float* A_log;
  const float* dt_bias;
  const float* D;
  const void* initial_state;
  void* final_state;
  const int64_t* cu_seqlens;
  SsmPlan* plan;             // packed batches
  float4* slots;             // [slot][Ns / 4][128 rows] states of runs, slot = run * pairs + pair
  float* decays;             // [slot][2] decay over a run, per head
  int* status;
  unsigned* queue;           // packed batches: counter that hands the walks out, or nullptr: a CTA each
  Rows dts, os;
  int64_t T;
  int H, P, G, N;
  int pairs_per_group, pairs;
  int runs, run_blocks;      // equal lengths
  int packed;
  int late;                  // full pass behind a first one: waits for it where it wants the states, not before
  int state_fp32;
  int wait_limit_us;         // test aids, as in ScanParams
  int stop_loads_after;
};

// One CTA's walk (packed batches: called by whole warps).
struct SsmItem {
  bool there;                // false: no more walks
  int n, group, head0;
  bool two;                  // the second head is there
  bool last;                 // the sequence's last run
  int slot;                  // state to start from (first pass: to leave), or -1: the caller's
  int blocks;
  int64_t b, t0, tokens;
};
__device__ __forceinline__ SsmItem ssm_item(const SsmScanParams& p, unsigned index, bool full) {
  SsmItem it{};
  const int pair = static_cast<int>(index % static_cast<unsigned>(p.pairs));
  const int rs = static_cast<int>(index / static_cast<unsigned>(p.pairs));
  int run, runs, len;
  int64_t bos = 0, eos = p.T;
  it.slot = -1;
  it.there = !p.packed;
  if (p.packed) {
    SsmPlan* plan = p.plan;
    // (the runs of the first pass are those of the cut sequences, but each one's last: counted with the slots)
    const int* prefix = full ? plan->prefix(p.N) : plan->slot_prefix(p.N);
    const int ranks = full ? plan->active : plan->cut;
    if (rs >= plan->walks[full ? 1 : 0]) return it;
    it.there = true;
    // (by the whole warp, 32 entries at a time: what one load waits for behind the other is what a walk waits for to begin)
    int lo = 0, hi = ranks;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) >> 5, at = lo + (static_cast<int>(threadIdx.x & 31) + 1) * step;
      lo += __popc(__ballot_sync(0xffffffffu, at < hi && prefix[at] <= rs)) * step;
      if (lo + step < hi) hi = lo + step;
    }
    run = rs - prefix[lo];
    runs = prefix[lo + 1] - prefix[lo];
    if (!full && run + 1 >= runs) return it;
    len = plan->run_blocks;
    it.n = plan->order()[lo];
    if (runs > 1) it.slot = (plan->slot_prefix(p.N)[lo] + run) * p.pairs + pair;
    bos = p.cu_seqlens[it.n];
    eos = p.cu_seqlens[it.n + 1];
    bos = bos < 0 ? 0 : bos > p.T ? p.T : bos;
    eos = eos < bos ? bos : eos > p.T ? p.T : eos;
  } else {
    const int per = full ? p.runs : p.runs - 1;
    it.n = rs / per;
    run = rs - it.n * per;
    runs = p.runs;
    len = p.run_blocks;
    it.b = it.n;
    if (runs > 1) it.slot = (it.n * runs + run) * p.pairs + pair;
  }
  it.last = run == runs - 1;
  it.t0 = bos + (runs > 1 ? static_cast<int64_t>(run) * len * kSsmBlock : 0);
  it.tokens = it.last ? eos - it.t0 : static_cast<int64_t>(len) * kSsmBlock;
  it.blocks = static_cast<int>((it.tokens + kSsmBlock - 1) / kSsmBlock);
  const int per_pair = p.P == 128 ? 1 : 2, in_group = p.H / p.G;
  it.group = pair / p.pairs_per_group;
  const int first = (pair - it.group * p.pairs_per_group) * per_pair;
  it.head0 = it.group * in_group + first;
  it.two = per_pair == 2 && first + 1 < in_group;
  return it;
}

struct SsmLayout {
  int pairs_per_group, pairs;
  int runs, run_blocks;      // equal lengths
  int least;                 // packed: the shortest runs that may be chosen, 0: sequences stay whole
  int64_t items, first_items, chained, slots;
  int64_t plan_off, decay_off, slot_off, bytes;
};
SsmLayout ssm_layout(int64_t T, int64_t N, int H, int P, int G, int Ns, bool packed, int sms);

struct SsmAid {
  int wait_limit_us, stop_loads_after;
};
cudaError_t launch_ssm_scan(const SsmParams& p, const SsmLayout& L, const SsmAid& aid, void* workspace, bool clear_status, cudaStream_t stream);

}  // namespace fkda
