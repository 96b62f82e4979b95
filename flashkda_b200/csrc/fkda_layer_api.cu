// C ABI of the operators round the recurrence (include/fkda.h): argument checks and launches.
#include <cmath>
#include <initializer_list>

#include "../../include/fkda.h"
#include "../../include/fkda_testing.h"
#include "fkda_layer.cuh"
#include "fkda_ssm.cuh"

namespace {

using fkda::Rows;
using fkda::set_error;

int refuse(const char* what) { return set_error(FKDA_ERR_INVALID_ARGUMENT, "%s", what); }
int cuda_error(cudaError_t e, const char* what) { return set_error(FKDA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e)); }

// A [B][T][inner] tensor as the checks see it.
struct View {
  const char* name;
  const void* base;
  int64_t inner;            // elements of a token
  int64_t size;             // bytes of an element
  int64_t batch, token;     // strides in elements
};
struct Sizes {
  int64_t B, T;
};

// Strides as used: those of a dimension of one entry do not count, and a batch of single tokens is one row of tokens.
struct Normal {
  int64_t B, T, batch, token;
};
Normal normal(const View& v, const Sizes& s) {
  Normal r{s.B, s.T, v.batch, v.token};
  if (r.T <= 1) {
    r.T = r.B * (r.T > 0);
    r.token = r.batch;
    r.B = 1;
  }
  if (r.T <= 1) r.token = v.inner;
  if (r.B <= 1) r.batch = r.T * r.token;
  return r;
}

bool empty(const Sizes& s) { return s.B == 0 || s.T == 0; }

// Base, strides and extent of one tensor.  `wide`: read or written 16 bytes at a time.
int check_view(const View& v, const Sizes& s, bool wide = true) {
  if (empty(s)) return FKDA_OK;
  if (v.base == nullptr) return set_error(FKDA_ERR_INVALID_ARGUMENT, "%s must be non-NULL", v.name);
  const Normal r = normal(v, s);
  const int64_t limit = int64_t{1} << 46;
  if (r.token < 0 || r.batch < 0 || r.token > limit || r.batch > limit || r.token * (r.T - 1) > limit || (r.B > 1 && r.batch > limit / r.B))
    return set_error(FKDA_ERR_INVALID_ARGUMENT, "%s has strides out of range", v.name);
  const bool rows = r.token >= v.inner && (r.B == 1 || r.batch >= (r.T - 1) * r.token + v.inner);
  const bool woven = r.B > 1 && r.batch >= v.inner && r.token >= (r.B - 1) * r.batch + v.inner;
  if (!rows && !woven) return set_error(FKDA_ERR_INVALID_ARGUMENT, "the rows of %s overlap", v.name);
  if (wide) {
    if (reinterpret_cast<uintptr_t>(v.base) & 15u) return set_error(FKDA_ERR_INVALID_ARGUMENT, "%s must start on a 16-byte boundary", v.name);
    if ((r.T > 1 && r.token * v.size % 16) || (r.B > 1 && r.batch * v.size % 16))
      return set_error(FKDA_ERR_INVALID_ARGUMENT, "the strides of %s must be multiples of 16 bytes", v.name);
  }
  return FKDA_OK;
}

// Whether two tensors may share memory: their address ranges meet, and they are not columns of one tensor beside each other.
bool share(const View& a, const View& b, const Sizes& s) {
  if (empty(s) || a.base == nullptr || b.base == nullptr) return false;
  const Normal x = normal(a, s), y = normal(b, s);
  auto bytes = [](const View& v, const Normal& r) { return ((r.B - 1) * r.batch + (r.T - 1) * r.token + v.inner) * v.size; };
  const intptr_t pa = reinterpret_cast<intptr_t>(a.base), pb = reinterpret_cast<intptr_t>(b.base);
  if (pa + bytes(a, x) <= pb || pb + bytes(b, y) <= pa) return false;
  const int64_t pitch = x.token * a.size;
  if (pitch != y.token * b.size || (x.B > 1 && (x.batch * a.size != y.batch * b.size || x.batch % x.token != 0))) return true;
  const int64_t d = (((pb - pa) % pitch) + pitch) % pitch;          // where b's columns start within a row that starts with a's
  return !(d >= a.inner * a.size && d + b.inner * b.size <= pitch);
}
bool same(const View& a, const View& b, const Sizes& s) {
  const Normal x = normal(a, s), y = normal(b, s);
  return a.base == b.base && a.size == b.size && x.token == y.token && x.batch == y.batch;
}
bool ranges_meet(const void* a, int64_t na, const void* b, int64_t nb) {
  if (a == nullptr || b == nullptr || na <= 0 || nb <= 0) return false;
  const intptr_t x = reinterpret_cast<intptr_t>(a), y = reinterpret_cast<intptr_t>(b);
  return x < y + nb && y < x + na;
}
int64_t span(const View& v, const Sizes& s) {
  if (empty(s)) return 0;
  const Normal r = normal(v, s);
  return ((r.B - 1) * r.batch + (r.T - 1) * r.token + v.inner) * v.size;
}
Rows rows_of(const View& v, const Sizes& s) {
  // (strides of dimensions with one entry may be anything; the kernels multiply those by 0)
  return Rows{s.B > 1 ? v.batch : 0, s.T > 1 ? v.token : s.B > 1 && s.T == 1 ? v.batch : 0};
}
// Tokens of a batch row as the norms count them: all of them where every batch row follows the one before (no division then).
int64_t tokens_of(const Sizes& s, std::initializer_list<Rows> tensors) {
  for (const Rows& r : tensors)
    if (s.B > 1 && r.batch != s.T * r.token) return s.T;
  return INT64_MAX;
}
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool known(int32_t dtype) { return dtype == FKDA_STATE_BF16 || dtype == FKDA_STATE_FP32; }

int check_batch(int64_t B, int64_t T, int64_t N, const int64_t* cu) {
  if (B <= 0 || T < 0) return refuse("B must be positive and T non-negative");
  if (B > 0x7fffffffLL || T > (int64_t{1} << 40)) return refuse("B or T is too large");
  if (cu != nullptr) {
    if (B != 1) return refuse("B must be 1 when cu_seqlens is provided");
    if (N <= 0 || N > 0x7ffffffeLL) return refuse("cu_seqlens must have at least 2 elements");
  } else if (N != B) {
    return refuse("N must equal B when cu_seqlens is not provided");
  }
  return FKDA_OK;
}
// The state in and out: two tensors apart, or one and the same.
int check_states(const void* in, const void* out, int64_t bytes) {
  if (!aligned(in) || !aligned(out)) return refuse("initial_state and final_state must start on a 16-byte boundary");
  if (in != out && ranges_meet(in, bytes, out, bytes)) return refuse("final_state overlaps initial_state without being it");
  return FKDA_OK;
}

// A parameter (weight, bias) that an output would write over.
bool over(const View& out, const Sizes& s, const void* parameter, int64_t elements, int32_t dtype) {
  return ranges_meet(out.base, span(out, s), parameter, elements * (dtype == FKDA_STATE_FP32 ? 4 : 2));
}

#define FKDA_TRY(call)            \
  do {                            \
    const int rc_ = (call);       \
    if (rc_ != FKDA_OK) return rc_; \
  } while (0)

int check_ssm_sizes(const fkda_ssm_params* p) {
  FKDA_TRY(check_batch(p->B, p->T, p->N, p->cu_seqlens));
  if (p->H <= 0 || p->H > 65535 || p->G <= 0 || p->H % p->G != 0) return refuse("H must lie in [1, 65535] and be a multiple of G");
  if ((p->P != 64 && p->P != 128) || (p->Ns != 64 && p->Ns != 128)) return refuse("P and the columns of a state must be 64 or 128");
  if (p->N * p->H > 0x1fffffffLL) return refuse("N*H exceeds 2^29-1 chains");
  if (p->T > 0x7fff0000LL || (p->N + p->T / fkda::kSsmBlock * (p->cu_seqlens ? 1 : p->N)) * p->H > 0x3fffffffLL) return refuse("too many tokens for one call");
  return FKDA_OK;
}
// whether every sequence goes token by token
bool by_token(const fkda_ssm_params* p) { return p->T <= fkda::kSsmStepT; }
fkda::SsmLayout layout_of(const fkda_ssm_params* p) {
  return fkda::ssm_layout(p->T, p->N, static_cast<int>(p->H), static_cast<int>(p->P), static_cast<int>(p->G), static_cast<int>(p->Ns), p->cu_seqlens != nullptr,
                          fkda::device_sm_count());
}

int check_ssm(const fkda_ssm_params* p) {
  if (!p) return refuse("params is NULL");
  FKDA_TRY(check_ssm_sizes(p));
  if (!p->A_log || !p->dt_bias) return refuse("A_log and dt_bias must be non-NULL");
  if ((p->initial_state || p->final_state) && !known(p->state_dtype)) return refuse("state_dtype must be bf16 or fp32 when a state tensor is given");
  const Sizes s{p->B, p->T};
  const View x{"x", p->x, p->H * p->P, 2, p->x_batch_stride, p->x_token_stride}, dt{"dt", p->dt, p->H, 2, p->dt_batch_stride, p->dt_token_stride};
  const View b{"B", p->Bm, p->G * p->Ns, 2, p->B_batch_stride, p->B_token_stride}, c{"C", p->Cm, p->G * p->Ns, 2, p->C_batch_stride, p->C_token_stride};
  const View o{"out", p->out, p->H * p->P, 2, p->out_batch_stride, p->out_token_stride};
  FKDA_TRY(check_view(x, s));
  FKDA_TRY(check_view(dt, s, false));
  FKDA_TRY(check_view(b, s));
  FKDA_TRY(check_view(c, s));
  FKDA_TRY(check_view(o, s));
  for (const View* v : {&x, &dt, &b, &c})
    if (share(o, *v, s)) return set_error(FKDA_ERR_INVALID_ARGUMENT, "out shares memory with %s", v->name);
  const int64_t states = p->N * p->H * p->P * p->Ns * (p->state_dtype == FKDA_STATE_FP32 ? 4 : 2);
  FKDA_TRY(check_states(p->initial_state, p->final_state, states));
  for (const View* v : {&x, &dt, &b, &c, &o})
    if (ranges_meet(p->final_state, states, v->base, span(*v, s))) return set_error(FKDA_ERR_INVALID_ARGUMENT, "final_state shares memory with %s", v->name);
  if (ranges_meet(p->initial_state, states, p->out, span(o, s))) return refuse("out shares memory with initial_state");
  for (const float* parameter : {p->A_log, p->dt_bias, p->D})
    if (over(o, s, parameter, p->H, FKDA_STATE_FP32) || ranges_meet(p->final_state, states, parameter, p->H * 4)) return refuse("an output shares memory with A_log, dt_bias or D");
  return FKDA_OK;
}

int do_ssm(const fkda_ssm_params* p, const fkda::SsmAid& aid, void* cuda_stream) {
  FKDA_TRY(check_ssm(p));
  const Sizes s{p->B, p->T};
  fkda::SsmParams q{};
  q.x = static_cast<const __nv_bfloat16*>(p->x);
  q.dt = static_cast<const __nv_bfloat16*>(p->dt);
  q.Bm = static_cast<const __nv_bfloat16*>(p->Bm);
  q.Cm = static_cast<const __nv_bfloat16*>(p->Cm);
  q.out = static_cast<__nv_bfloat16*>(p->out);
  q.A_log = p->A_log;
  q.dt_bias = p->dt_bias;
  q.D = p->D;
  q.initial_state = p->initial_state;
  q.final_state = p->final_state;
  q.cu_seqlens = p->cu_seqlens;
  q.xs = rows_of(View{"x", p->x, 0, 2, p->x_batch_stride, p->x_token_stride}, s);
  q.dts = rows_of(View{"dt", p->dt, 0, 2, p->dt_batch_stride, p->dt_token_stride}, s);
  q.bs = rows_of(View{"B", p->Bm, 0, 2, p->B_batch_stride, p->B_token_stride}, s);
  q.cs = rows_of(View{"C", p->Cm, 0, 2, p->C_batch_stride, p->C_token_stride}, s);
  q.os = rows_of(View{"out", p->out, 0, 2, p->out_batch_stride, p->out_token_stride}, s);
  q.T = p->T;
  q.H = static_cast<int>(p->H);
  q.P = static_cast<int>(p->P);
  q.G = static_cast<int>(p->G);
  q.Ns = static_cast<int>(p->Ns);
  q.N = static_cast<int>(p->N);
  q.state_fp32 = p->state_dtype == FKDA_STATE_FP32;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  cudaError_t e;
  const bool word = p->workspace != nullptr && p->workspace_bytes >= static_cast<int64_t>(sizeof(int)), misplaced = (reinterpret_cast<uintptr_t>(p->workspace) & 255u) != 0;
  if (by_token(p)) {
    // (no scratch memory is needed; one that is given has the status word all the same)
    const bool told = word && !(p->flags & FKDA_FLAG_STATUS_UNREAD);
    if (told && misplaced) return refuse("workspace must be 256-byte aligned");
    e = fkda::launch_ssm_step(q, 0, told ? static_cast<int*>(p->workspace) : nullptr, stream);
    return e == cudaSuccess ? FKDA_OK : cuda_error(e, "selective scan launch");
  }
  const fkda::SsmLayout L = layout_of(p);
  if (!p->workspace || misplaced) return refuse("workspace must be non-NULL and 256-byte aligned");
  if (p->workspace_bytes < L.bytes)
    return set_error(FKDA_ERR_WORKSPACE_TOO_SMALL, "workspace has %lld bytes, %lld needed", (long long)p->workspace_bytes, (long long)L.bytes);
  e = fkda::launch_ssm_scan(q, L, aid, p->workspace, !(p->flags & FKDA_FLAG_STATUS_UNREAD), stream);
  if (e != cudaSuccess) return cuda_error(e, "selective scan launch");
  return FKDA_OK;
}

}  // namespace

extern "C" {

int fkda_short_conv(const fkda_conv_params* p, void* cuda_stream) {
  if (!p) return refuse("params is NULL");
  FKDA_TRY(check_batch(p->B, p->T, p->N, p->cu_seqlens));
  if (p->C <= 0 || p->C % 8 != 0 || p->C > (1 << 24)) return refuse("C must be a positive multiple of 8, at most 2^24");
  if (p->width < 2 || p->width > 4) return refuse("width must be 2, 3 or 4");
  if (!known(p->weight_dtype)) return refuse("weight_dtype must be bf16 or fp32");
  if (!p->weight) return refuse("weight must be non-NULL");
  if (!aligned(p->weight) || !aligned(p->bias)) return refuse("weight and bias must start on a 16-byte boundary");
  const Sizes s{p->B, p->T};
  const View x{"x", p->x, p->C, 2, p->x_batch_stride, p->x_token_stride}, o{"out", p->out, p->C, 2, p->out_batch_stride, p->out_token_stride};
  FKDA_TRY(check_view(x, s));
  FKDA_TRY(check_view(o, s));
  if (share(x, o, s)) return refuse("out shares memory with x");
  if (over(o, s, p->weight, p->C * p->width, p->weight_dtype) || over(o, s, p->bias, p->C, p->weight_dtype)) return refuse("out shares memory with weight or bias");
  const int64_t states = p->N * (p->width - 1) * p->C * 2;
  FKDA_TRY(check_states(p->initial_state, p->final_state, states));
  if (ranges_meet(p->final_state, states, p->x, span(x, s)) || ranges_meet(p->final_state, states, p->out, span(o, s)) ||
      ranges_meet(p->initial_state, states, p->out, span(o, s)))
    return refuse("a state shares memory with x or out");
  const int64_t size = p->weight_dtype == FKDA_STATE_FP32 ? 4 : 2;
  if (ranges_meet(p->final_state, states, p->weight, p->C * p->width * size) || ranges_meet(p->final_state, states, p->bias, p->C * size))
    return refuse("final_state shares memory with weight or bias");
  if ((p->B * p->T + p->N) * (p->C / 8) > (int64_t{1} << 37)) return refuse("too many elements for one call");
  fkda::ConvParams q{};
  q.x = static_cast<const __nv_bfloat16*>(p->x);
  q.weight = p->weight;
  q.bias = p->bias;
  q.out = static_cast<__nv_bfloat16*>(p->out);
  q.initial_state = static_cast<const __nv_bfloat16*>(p->initial_state);
  q.final_state = static_cast<__nv_bfloat16*>(p->final_state);
  q.cu_seqlens = p->cu_seqlens;
  q.xs = rows_of(x, s);
  q.os = rows_of(o, s);
  q.T = p->T;
  q.C = static_cast<int>(p->C);
  q.N = static_cast<int>(p->N);
  q.silu = p->silu != 0;
  const cudaError_t e = fkda::launch_short_conv(q, p->width, p->weight_dtype == FKDA_STATE_FP32, static_cast<cudaStream_t>(cuda_stream));
  return e == cudaSuccess ? FKDA_OK : cuda_error(e, "short convolution launch");
}

int fkda_ssm_scratch_bytes(const fkda_ssm_params* p, int64_t* bytes) {
  if (!p || !bytes) return refuse("NULL pointer");
  FKDA_TRY(check_ssm_sizes(p));
  *bytes = by_token(p) ? 0 : layout_of(p).bytes;
  return FKDA_OK;
}

int fkda_ssm_fwd(const fkda_ssm_params* p, void* cuda_stream) { return do_ssm(p, fkda::SsmAid{0, 0}, cuda_stream); }

int fkda_debug_ssm_giveup(const fkda_ssm_params* p, int stop_loads_after, int wait_limit_us, void* cuda_stream) {
  if (stop_loads_after < 1 || wait_limit_us < 1 || wait_limit_us > 1000000)
    return refuse("stop_loads_after >= 1 and 1 <= wait_limit_us <= 1000000 required");
  return do_ssm(p, fkda::SsmAid{wait_limit_us, stop_loads_after}, cuda_stream);
}

int fkda_gated_norm(const fkda_gated_norm_params* p, void* cuda_stream) {
  if (!p) return refuse("params is NULL");
  if (p->B <= 0 || p->T < 0 || p->H <= 0) return refuse("B and H must be positive and T non-negative");
  if (p->D <= 0 || p->D % 8 != 0 || p->D > 16384) return refuse("D must be a multiple of 8 from 8 to 16384");
  if (p->H > (1 << 24) || p->B > 0x7fffffffLL || p->T > (int64_t{1} << 40) || p->B * p->T > 0x7fffffffLL / p->H) return refuse("too many rows for one call");
  if (!known(p->weight_dtype)) return refuse("weight_dtype must be bf16 or fp32");
  if (!p->weight || !aligned(p->weight)) return refuse("weight must be non-NULL and start on a 16-byte boundary");
  if (!std::isfinite(p->eps) || p->eps < 0.f) return refuse("eps must be finite and not negative");
  const Sizes s{p->B, p->T};
  const View x{"x", p->x, p->H * p->D, 2, p->x_batch_stride, p->x_token_stride}, g{"gate", p->gate, p->H * p->D, 2, p->gate_batch_stride, p->gate_token_stride};
  const View o{"out", p->out, p->H * p->D, 2, p->out_batch_stride, p->out_token_stride};
  for (const View* v : {&x, &g, &o}) FKDA_TRY(check_view(*v, s));
  for (const View* v : {&x, &g})
    if (share(*v, o, s) && !same(*v, o, s)) return set_error(FKDA_ERR_INVALID_ARGUMENT, "out shares memory with %s without being it", v->name);
  if (over(o, s, p->weight, (p->weight_per_head ? p->H : 1) * p->D, p->weight_dtype)) return refuse("out shares memory with weight");
  const fkda::GatedNormParams q{static_cast<const __nv_bfloat16*>(p->x), static_cast<const __nv_bfloat16*>(p->gate), p->weight, static_cast<__nv_bfloat16*>(p->out),
                                rows_of(x, s), rows_of(g, s), rows_of(o, s), p->B * p->T * p->H, tokens_of(s, {rows_of(x, s), rows_of(g, s), rows_of(o, s)}), static_cast<int>(p->H), static_cast<int>(p->D), p->eps,
                                p->weight_per_head != 0};
  const cudaError_t e = fkda::launch_gated_norm(q, p->weight_dtype == FKDA_STATE_FP32, p->silu != 0, p->gate_first != 0, static_cast<cudaStream_t>(cuda_stream));
  return e == cudaSuccess ? FKDA_OK : cuda_error(e, "gated norm launch");
}

int fkda_add_norm(const fkda_add_norm_params* p, void* cuda_stream) {
  if (!p) return refuse("params is NULL");
  if (p->B <= 0 || p->T < 0) return refuse("B must be positive and T non-negative");
  if (p->D <= 0 || p->D % 8 != 0 || p->D > 16384) return refuse("D must be a multiple of 8 from 8 to 16384");
  if (p->B > 0x7fffffffLL || p->T > (int64_t{1} << 40) || p->B * p->T > 0x7fffffffLL) return refuse("too many rows for one call");
  if (!known(p->weight_dtype) || !known(p->residual_dtype)) return refuse("weight_dtype and residual_dtype must be bf16 or fp32");
  if (!p->weight || !aligned(p->weight)) return refuse("weight must be non-NULL and start on a 16-byte boundary");
  if (!std::isfinite(p->eps) || p->eps < 0.f || !std::isfinite(p->scale)) return refuse("eps and scale must be finite, eps not negative");
  const Sizes s{p->B, p->T};
  const int64_t size = p->residual_dtype == FKDA_STATE_FP32 ? 4 : 2;
  const View x{"x", p->x, p->D, 2, p->x_batch_stride, p->x_token_stride}, r{"residual", p->residual, p->D, size, p->residual_batch_stride, p->residual_token_stride};
  const View o{"out", p->out, p->D, 2, p->out_batch_stride, p->out_token_stride};
  const View ro{"residual_out", p->residual_out, p->D, size, p->residual_out_batch_stride, p->residual_out_token_stride};
  for (const View* v : {&x, &r, &o, &ro}) FKDA_TRY(check_view(*v, s));
  if (share(o, ro, s)) return refuse("out shares memory with residual_out");
  if (share(r, ro, s) && !same(r, ro, s)) return refuse("residual_out shares memory with residual without being it");
  if (share(x, o, s) && !same(x, o, s)) return refuse("out shares memory with x without being it");
  if (share(r, o, s)) return refuse("out shares memory with residual");
  if (share(x, ro, s)) return refuse("residual_out shares memory with x");
  if (over(o, s, p->weight, p->D, p->weight_dtype) || over(ro, s, p->weight, p->D, p->weight_dtype)) return refuse("an output shares memory with weight");
  const fkda::AddNormParams q{static_cast<const __nv_bfloat16*>(p->x), p->residual, p->weight, static_cast<__nv_bfloat16*>(p->out), p->residual_out,
                              rows_of(x, s), rows_of(r, s), rows_of(o, s), rows_of(ro, s), p->B * p->T, tokens_of(s, {rows_of(x, s), rows_of(r, s), rows_of(o, s), rows_of(ro, s)}), static_cast<int>(p->D), p->scale, p->eps};
  const cudaError_t e = fkda::launch_add_norm(q, p->weight_dtype == FKDA_STATE_FP32, p->residual_dtype == FKDA_STATE_FP32, static_cast<cudaStream_t>(cuda_stream));
  return e == cudaSuccess ? FKDA_OK : cuda_error(e, "residual norm launch");
}

}  // extern "C"
