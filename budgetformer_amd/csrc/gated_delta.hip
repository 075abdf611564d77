// The gated delta rule over packed sequences: checks, how a call is cut, workspaces (the kernels: gated_delta.h).
#include <cmath>

#include "gated_delta.h"

namespace bf {
namespace {

int check(const bf_gated_delta* p, const char* fn, bool step) {
  BF_CHECK_ARG(p != nullptr, "%s: no arguments", fn);
  BF_CHECK_ARG(p->dtype == BF_DTYPE_F32 || p->dtype == BF_DTYPE_BF16 || p->dtype == BF_DTYPE_F16, "%s: dtype %d", fn,
               p->dtype);
  for (int d : {p->dim_k, p->dim_v})
    if (d < 8 || d > 128 || d % 8) {
      set_error("%s: head dims (%d, %d) (multiples of 8 up to 128 are supported)", fn, p->dim_k, p->dim_v);
      return BF_ERR_UNSUPPORTED;
    }
  BF_CHECK_ARG(p->heads >= 1 && p->heads <= (1 << 16) && p->heads_k >= 1 && p->heads % p->heads_k == 0,
               "%s: %d value heads over %d key heads (a multiple expected, up to 2^16)", fn, p->heads, p->heads_k);
  BF_CHECK_ARG(p->n >= 0 && p->n < kMaxRows && p->n_seq >= 0 && p->n_seq < kMaxRows, "%s: bad sizes (%lld rows, %lld sequences)", fn,
               (long long)p->n, (long long)p->n_seq);
  BF_CHECK_ARG(p->scale == p->scale && p->scale <= 3e38f && p->scale >= -3e38f, "%s: scale %g", fn, double(p->scale));
  BF_CHECK_ARG(p->longest >= 0, "%s: longest sequence %d", fn, p->longest);
  BF_CHECK_ARG(p->n == 0 || (p->log_gate && p->beta), "%s: no gates or strengths", fn);
  BF_CHECK_ARG(aligned16({p->init, p->final_state}), "%s: states must be 16-byte aligned", fn);
  const int64_t per16 = step ? 1 : p->dtype == BF_DTYPE_F32 ? 4 : 8;
  for (const int64_t* s : {p->q_stride, p->k_stride, p->v_stride})
    BF_CHECK_ARG(s[0] >= 0 && s[1] >= 0 && s[0] % per16 == 0 && s[1] % per16 == 0,
                 "%s: strides (%lld, %lld) are not whole 16-byte steps", fn, (long long)s[0], (long long)s[1]);
  if (step) {
    BF_CHECK_ARG(p->n < (int64_t(1) << 24) / p->heads, "%s: %lld sequences of %d heads", fn, (long long)p->n, p->heads);
  } else {
    BF_CHECK_ARG(p->offsets != nullptr, "%s: no offsets", fn);
  }
  return BF_OK;
}

// Workgroups of a pass that a CU holds at once, by their registers and LDS.
int slots(int32_t dtype, int d, bool train) {
  if (dtype == BF_DTYPE_F32) return 128 / d;
  if (d == 32) return 8;
  if (d == 128) return train && dtype == BF_DTYPE_F16 ? 1 : 2;
  return train && dtype == BF_DTYPE_F16 ? 3 : 4;
}

// Chunks of a segment (2 to 64), by what a call with them takes. A pass (two with maps, six that train) takes the chunks of a workgroup
// one behind the other; a chunk takes longer the more workgroups a CU holds, but not in proportion while they mostly wait: with
// heads of 128 a chunk of the forward pass 3.5 us alone and 6 of two, of a pass of gradients 8.5 and 14; with heads of 64 4.7, 6, 7.6
// and 10.4 of one to four, of gradients 8.1, 8.8 and 9.7. So what fills the chip once is best, and some more workgroups cost a whole
// round; the carry takes 2 us (0.9, 0.7) a segment of the longest sequence. A call in us by segments of 2, 4, 8, 16 and 32 chunks: 8192 tokens,
// 16 heads of 128, bfloat16 467, 249, 184, 158, 227, training 1224, 794, 624, 591, 920; 1024 of 8 heads, training 153, 170, 247, 423,
// 614; 8192 of 8 heads of 64, training 346, 260, 246, 353, 619; 16 sequences of 21K tokens, 4 heads of 32, training 181, 154, 174, 258, 457.
// Sequences that fit a segment each need no maps and no carry.
int seg_chunks(const bf_gated_delta* p, bool train) {
  const int d = delta_pad(p->dim_k, p->dim_v), most = slots(p->dtype, d, train);
  const bool equal = p->longest > 0 && p->n == p->n_seq * int64_t(p->longest);
  const double chunks = double(p->n) / kDeltaChunk, longest = double(p->longest > 0 ? p->longest : p->n) / kDeltaChunk;
  const double seqs = double(p->n_seq), carry = d == 128 ? 2.0 : d == 64 ? 0.9 : 0.7;
  // of a chunk alone, of all passes and of those that a call without a carry has; of a pass's start
  const double all = train ? (d == 128 ? 22 : d == 64 ? 17 : 12) : (d == 128 ? 4.8 : d == 64 ? 3.7 : 2.9), few = all * (train ? 0.78 : 0.55);
  const double start = train ? 35 : 8;
  int best = 2;
  double least = 1e30;
  for (int len = 2; len <= 64; ++len) {
    const bool whole = longest <= len;
    // of sequences of unknown lengths the last segments are half full, more or less
    double segs = equal ? seqs * ceil(longest / len) : chunks / len + 0.5 * seqs;
    if (whole || segs < seqs) segs = seqs;
    const double groups = segs * p->heads, full = floor(groups / (256 * most));
    // a few more than fill it find room: last segments are short
    const double rest = full > 0 ? ceil((groups - full * 256 * most) / 256 - 0.1) : ceil(groups / 256 - (groups > 256 ? 0.1 : 0.0));
    const auto slower = [&](double at_once) {
      return d == 128 ? 0.32 + 0.68 * at_once : d == 32 ? 0.9 + 0.1 * at_once : at_once > 3 ? 1.9 : 0.8 + 0.2 * at_once;
    };
    const double rounds = full * slower(most) + (rest > 0 ? slower(rest) : 0);
    const double own = whole && longest < len ? (longest > 1 ? longest : 1) : len;
    const double cost = rounds * own * (whole ? few : all) + (full + (rest > 0)) * start + (whole ? 0 : longest / len * carry * (train ? 2 : 1));
    if (cost < least) least = cost, best = len;
    if (whole) break;
  }
  return best;
}

bool carries(const bf_gated_delta* p, bool train) {
  const int64_t seg = int64_t(seg_chunks(p, train)) * kDeltaChunk;
  return p->n > seg && p->n_seq > 0 && !(p->longest > 0 && p->longest <= seg);
}

// A call's workspaces, in floats: what the backward reads (kept), what only the forward needs, what only the backward does.
struct Sizes {
  int64_t chunks, segs;            // places
  int64_t rows, frags, map, state;
  int seg_len;                     // chunks
  bool carried;
  Sizes(const bf_gated_delta* p, bool train) : seg_len(seg_chunks(p, train)), carried(carries(p, train)) {
    const int64_t seg = int64_t(seg_len) * kDeltaChunk, d = delta_pad(p->dim_k, p->dim_v), parts = delta_mid_parts(p->dtype);
    chunks = p->n / kDeltaChunk + p->n_seq + 1;
    segs = p->n / seg + p->n_seq + 1;
    rows = ceil_div(p->n * p->heads, int64_t(4)) * 4;
    frags = chunks * p->heads * (2 * parts * 64 * 4);
    map = carried ? segs * p->heads * (parts * d * d / 2) : 0;
    state = carried ? segs * p->heads * int64_t(p->dim_k) * p->dim_v : 0;
  }
};

// A launch's threads are counted in 32 bits.
int check_grids(const bf_gated_delta* p, const Sizes& s, const char* fn) {
  const int64_t most = (int64_t(1) << 32) - 1, d = delta_pad(p->dim_k, p->dim_v);
  if (s.chunks * p->heads > most / 64 || s.segs * p->heads > most / (s.carried ? 4 * d : 2 * d) || p->n * p->heads_k * p->dim_k > 2 * (most - 1024)) {
    set_error("%s: %lld rows in %lld sequences of %d heads are more than a launch holds", fn, (long long)p->n, (long long)p->n_seq, p->heads);
    return BF_ERR_UNSUPPORTED;
  }
  return BF_OK;
}

int64_t kept_floats(const bf_gated_delta* p) {
  const Sizes s(p, true);
  return 3 * s.rows + 2 * s.frags + s.map + s.state + p->n * p->heads * p->dim_v;
}

int64_t fwd_floats(const bf_gated_delta* p, bool train) {
  const Sizes s(p, train);
  return 2 * s.frags + s.map + (train ? 0 : 3 * s.rows + s.state);
}

int64_t bwd_floats(const bf_gated_delta* p) {
  const Sizes s(p, true);
  const int64_t keys = p->n * p->heads * p->dim_k;
  return s.state + p->n * p->heads * p->dim_v + keys * (p->heads > p->heads_k ? 2 : 1);
}

DeltaArgs make_args(const bf_gated_delta* p, const Sizes& s, const void* q, const void* k, const void* v) {
  DeltaArgs a{};
  a.q = q, a.k = k, a.v = v;
  a.qs_t = p->q_stride[0], a.qs_h = p->q_stride[1];
  a.ks_t = p->k_stride[0], a.ks_h = p->k_stride[1];
  a.vs_t = p->v_stride[0], a.vs_h = p->v_stride[1];
  a.log_gate = p->log_gate, a.beta = p->beta, a.offsets = p->offsets;
  a.init = p->init, a.final_state = p->final_state;
  a.n = int32_t(p->n), a.n_seq = int32_t(p->n_seq), a.heads = p->heads, a.heads_k = p->heads_k, a.group = p->heads / p->heads_k;
  a.dim_k = p->dim_k, a.dim_v = p->dim_v;
  a.seg_chunks = s.seg_len, a.n_chunk = s.chunks, a.n_seg = s.segs;
  a.scale = p->scale;
  a.carried = s.carried;
  return a;
}

void take_kept(DeltaArgs& a, const Sizes& s, float* f) {
  a.inv_t = reinterpret_cast<uint4*>(f), f += s.frags;
  a.score_t = reinterpret_cast<uint4*>(f), f += s.frags;
  a.map_b = s.map ? reinterpret_cast<uint4*>(f) : nullptr, f += s.map;
  a.state = f, f += s.state;
  a.g2 = f, f += s.rows;
  a.gin = f, f += s.rows;
  a.gout = f, f += s.rows;
  a.e = f;
}

template <typename F> int with_launch(int32_t dtype, F&& f) {
  return with_type(dtype, [&](auto t) -> int { return f(DeltaLaunch<decltype(t)>()); });
}

}  // namespace
}  // namespace bf

using namespace bf;

extern "C" int64_t bf_gated_delta_kept_floats(const bf_gated_delta* p) {
  if (check(p, "gated_delta_kept_floats", false) != BF_OK) return -1;
  return check_grids(p, Sizes(p, true), "gated_delta_kept_floats") == BF_OK ? kept_floats(p) : -1;
}

extern "C" int64_t bf_gated_delta_fwd_floats(const bf_gated_delta* p, int32_t train) {
  if (check(p, "gated_delta_fwd_floats", false) != BF_OK) return -1;
  return check_grids(p, Sizes(p, train != 0), "gated_delta_fwd_floats") == BF_OK ? fwd_floats(p, train != 0) : -1;
}

extern "C" int bf_gated_delta_fwd(const bf_gated_delta* p, const void* q, const void* k, const void* v, void* out, float* kept,
                                  float* scratch, void* stream) {
  BF_CHECK_OK(check(p, "gated_delta_fwd", false));
  BF_CHECK_ARG(p->n == 0 || (q && k && v && out), "gated_delta_fwd: bad arguments");
  BF_CHECK_ARG(aligned16({q, k, v, out, kept, scratch}), "gated_delta_fwd: tensors and workspaces must be 16-byte aligned");
  if (p->n == 0 && !(p->final_state && p->n_seq > 0)) return BF_OK;
  BF_CHECK_ARG(scratch != nullptr, "gated_delta_fwd: no scratch (bf_gated_delta_fwd_floats)");
  const Sizes s(p, kept != nullptr);
  BF_CHECK_OK(check_grids(p, s, "gated_delta_fwd"));
  DeltaArgs a = make_args(p, s, q, k, v);
  a.out = out;
  float* f = scratch;
  a.inv = reinterpret_cast<uint4*>(f), f += s.frags;
  a.score = reinterpret_cast<uint4*>(f), f += s.frags;
  a.map_f = reinterpret_cast<uint4*>(f), f += s.map;
  if (kept) {
    take_kept(a, s, kept);
  } else {
    a.state = f, f += s.state;
    a.g2 = f, f += s.rows;
    a.gin = f, f += s.rows;
    a.gout = f;
  }
  const hipStream_t st = as_stream(stream);
  return with_launch(p->dtype, [&](auto l) -> int {
    if (a.n > 0) BF_CHECK_OK(l.prep(a, st));
    return l.forward(a, st);
  });
}

extern "C" int64_t bf_gated_delta_bwd_floats(const bf_gated_delta* p) {
  if (check(p, "gated_delta_bwd_floats", false) != BF_OK) return -1;
  return check_grids(p, Sizes(p, true), "gated_delta_bwd_floats") == BF_OK ? bwd_floats(p) : -1;
}

extern "C" int bf_gated_delta_bwd(const bf_gated_delta* p, const void* q, const void* k, const void* v, const void* dout,
                                  const float* kept, void* dq, void* dk, void* dv, float* dgate, float* dbeta, float* scratch,
                                  void* stream) {
  BF_CHECK_OK(check(p, "gated_delta_bwd", false));
  if (p->n == 0) return BF_OK;
  BF_CHECK_ARG(q && k && v && dout && kept && dq && dk && dv && dgate && dbeta && scratch, "gated_delta_bwd: bad arguments");
  BF_CHECK_ARG(aligned16({q, k, v, dout, kept, dq, dk, dv, scratch}), "gated_delta_bwd: tensors and workspaces must be 16-byte aligned");
  const Sizes s(p, true);
  BF_CHECK_OK(check_grids(p, s, "gated_delta_bwd"));
  DeltaArgs a = make_args(p, s, q, k, v);
  take_kept(a, s, const_cast<float*>(kept));
  a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv, a.dgate = dgate, a.dbeta = dbeta;
  float* f = scratch;
  a.dstate = f, f += s.state;
  a.z = f, f += p->n * p->heads * p->dim_v;
  a.dk32 = f, f += p->n * p->heads * p->dim_k;
  a.dq32 = a.group > 1 ? f : nullptr;
  return with_launch(p->dtype, [&](auto l) -> int { return l.backward(a, as_stream(stream)); });
}

extern "C" int bf_gated_delta_step(const bf_gated_delta* p, const void* q, const void* k, const void* v, void* out, void* stream) {
  BF_CHECK_OK(check(p, "gated_delta_step", true));
  if (p->n == 0) return BF_OK;
  BF_CHECK_ARG(q && k && v && out && p->init && p->final_state, "gated_delta_step: bad arguments");
  DeltaArgs a{};
  a.q = q, a.k = k, a.v = v;
  a.qs_t = p->q_stride[0], a.qs_h = p->q_stride[1];
  a.ks_t = p->k_stride[0], a.ks_h = p->k_stride[1];
  a.vs_t = p->v_stride[0], a.vs_h = p->v_stride[1];
  a.log_gate = p->log_gate, a.beta = p->beta, a.init = p->init, a.final_state = p->final_state;
  a.heads = p->heads, a.group = p->heads / p->heads_k, a.dim_k = p->dim_k, a.dim_v = p->dim_v;
  a.scale = p->scale, a.out = out;
  return with_launch(p->dtype, [&](auto l) -> int { return l.step(a, p->n, as_stream(stream)); });
}
