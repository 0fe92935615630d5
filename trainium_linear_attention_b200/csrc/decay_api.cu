// C entry points of the decayed linear attention: argument checks, the split
// into segments, and the launches (state of each segment, outputs).
#include <math.h>

#include "decay.cuh"
#include "decay_step.cuh"

namespace la {
namespace {

constexpr int64_t kMaxAutoSegments = 64;

int require_device(DeviceInfo *info) {
  const int st = current_device_info(info);
  if (st != LA_OK) return st;
  return info->cc_major == 10 ? LA_OK : LA_ERR_NO_DEVICE;
}

int check_sizes(int64_t batch, int64_t heads, int64_t n, int64_t d_qk, int64_t d_v, int dtype) {
  if (batch < 0 || heads < 0 || n < 0 || d_qk < 1 || d_v < 1) return LA_ERR_INVALID_ARGUMENT;
  if (dtype != LA_DTYPE_FLOAT32 && dtype != LA_DTYPE_BFLOAT16) return LA_ERR_INVALID_ARGUMENT;
  if (d_qk > kDecayMaxWidth || d_v > kDecayMaxWidth) return LA_ERR_UNSUPPORTED;
  if (batch > 65535 || heads > 65535 || batch * heads > 65535) return LA_ERR_UNSUPPORTED;
  if (n > INT32_MAX - 2 * kDecayTile) return LA_ERR_UNSUPPORTED;
  return LA_OK;
}

int64_t round_tile(int64_t n) { return (n + kDecayTile - 1) / kDecayTile * kDecayTile; }

// Segments actually used when `want` are asked for: none is empty.
int fit_segments(int64_t n, int64_t want, int64_t *len) {
  if (want <= 1 || n <= kDecayTile) {
    *len = n > 0 ? round_tile(n) : kDecayTile;
    return 1;
  }
  *len = round_tile((n + want - 1) / want);
  return (int)((n + *len - 1) / *len);
}

struct DecaySplit {
  int64_t whole = 0;  // heads walked unsplit
  int segments = 1;   // of the others
  int64_t len = 0;    // tokens per segment
  int lead = 0;       // tiles of the first of two parts without a state pass
};

// How the heads are split: the choice with the lowest estimated time.  A split
// head's segments but the last are walked twice (the state pass, then the
// output) and the later ones start by joining the states before them; unsplit
// heads leave SMs idle where there are few, or in a last, partial wave of CTAs.
// So all heads are walked whole, or all in g segments, or as many whole as fill
// k waves and the rest in g segments that share the SMs of one more, or all in two
// parts without a state pass.
DecaySplit estimate_split(int64_t bh, int64_t n, int64_t d_qk, int64_t d_v, int dtype,
                          bool backward, int sm_count) {
  DecaySplit best;
  const int64_t sq = (d_qk + kDecaySlice - 1) / kDecaySlice;
  const int64_t sv = (d_v + kDecaySlice - 1) / kDecaySlice;
  const int64_t per_head = backward ? 2 * sq + sv : sv;    // CTAs that walk a head
  const int64_t state_per_head = backward ? 2 * sv : sv;   // and in a state pass
  const bool wide = backward ? (d_qk > 64 || d_v > 64) : d_qk > 64;
  // microseconds per 128 tokens of a CTA's walk (output, state) and per wave
  // of CTAs (start-up, first loads, drain), measured on a B200.  (bf16, d = 64:
  // 64 heads of 2048 / 4096 / 8192 tokens unsplit 24 / 45 / 82 us, in two
  // segments 28 / 45 / 76; the gradients of 64 heads of 4096 tokens, 192 CTAs,
  // unsplit 89 us, in two segments 94.  fp32: 64 heads of 4096 tokens unsplit
  // 468 us, in 2 / 4 / 8 segments 324 / 321 / 337.)
  const bool simt = dtype == LA_DTYPE_FLOAT32 || d_qk % 8 || d_v % 8;  // (TMA addresses the rest)
  const double t_out = simt ? (wide ? 25.0 : 14.3) : (wide ? 2.1 : 1.3);
  const double t_state = simt ? (wide ? 9.0 : 5.1) : (wide ? 1.2 : 0.8);
  const double t_pre = wide ? 1.4 : 0.9;  // tiles the output kernel walks for the state
  constexpr double kWaveOut = 4.0, kWaveState = 3.0, kSplit = 5.0, kJoin = 0.4;
  const int64_t slots = sm_count;  // one CTA per SM
  const int64_t tiles = (n + kDecayTile - 1) / kDecayTile;
  const int64_t most = tiles < 1 ? 1 : tiles < kMaxAutoSegments ? tiles : kMaxAutoSegments;
  const int64_t full_waves = simt ? 0 : bh * per_head / slots;
  best.segments = fit_segments(n, 1, &best.len);
  double best_t = (double)((bh * per_head + slots - 1) / slots) * (kWaveOut + tiles * t_out);
  for (int64_t waves = 0; waves <= full_waves; ++waves) {
    const int64_t whole = waves * slots / per_head;
    if (whole >= bh) break;
    if (waves > 0 && waves + 2 < full_waves) continue;  // only the last few waves matter
    const int64_t rest = bh - whole;
    for (int64_t want = 2; want <= most; ++want) {
      int64_t l = 0;
      const int g = fit_segments(n, want, &l);
      if (g != want) continue;  // the same split as a smaller count
      const double per_seg = (double)(l / kDecayTile);
      const double t =
          waves * (kWaveOut + tiles * t_out) +
          (double)((rest * per_head * g + slots - 1) / slots) * (kWaveOut + per_seg * t_out) +
          kSplit + kJoin * (g - 1) +
          (double)((rest * state_per_head * (g - 1) + slots - 1) / slots) *
              (kWaveState + per_seg * t_state);
      if (t < best_t) {
        best_t = t;
        best.whole = whole;
        best.segments = g;
        best.len = l;
      }
    }
  }
  // Two parts in one launch, the second of which walks the first one's tiles for the
  // state before its own: no state pass to wait for, and parts of unequal length.  For
  // walks that fit the SMs twice: 64 heads of 2048 x 64 in 22.2 us (whole 24.4, in two
  // segments 27.3), 15 heads of 1000 x 64 / 128 in 12.9 (14.6), 30 heads of 4096 x 128
  // in 52.5 (60.6).
  if (!simt && tiles > 1 && bh * per_head * 2 <= slots) {
    int64_t x = (int64_t)(tiles * t_out / (2 * t_out - t_pre) + 0.5);
    x = x < 1 ? 1 : x > tiles - 1 ? tiles - 1 : x;
    const double first = x * t_out, second = x * t_pre + (tiles - x) * t_out;
    const double t = kWaveOut + (first > second ? first : second);
    if (t < best_t) {
      best = DecaySplit{};
      best.segments = 2;
      best.len = round_tile(n);
      best.lead = (int)x;
    }
  }
  return best;
}

DecaySplit plan_split(int64_t bh, int64_t n, int64_t d_qk, int64_t d_v, int dtype, bool backward,
                      int requested, int sm_count) {
  if (requested != 0) {
    DecaySplit s;
    s.segments = fit_segments(n, requested, &s.len);
    return s;
  }
  // the estimate takes some microseconds for a long sequence: the last one of
  // each kind is kept per thread
  struct Kept {
    int64_t sizes[6] = {-1, -1, -1, -1, -1, -1};
    DecaySplit split;
  };
  static thread_local Kept kept[2];
  Kept &k = kept[backward ? 1 : 0];
  const int64_t sizes[6] = {bh, n, d_qk, d_v, dtype, sm_count};
  bool same = true;
  for (int i = 0; i < 6; ++i) same = same && k.sizes[i] == sizes[i];
  if (!same) {
    k.split = estimate_split(bh, n, d_qk, d_v, dtype, backward, sm_count);
    for (int i = 0; i < 6; ++i) k.sizes[i] = sizes[i];
  }
  return k.split;
}

// States of the split heads: of the walk ahead, and of the one back.
size_t state_bytes(int64_t bh, const DecaySplit &s, int64_t d_qk, int64_t d_v, bool backward) {
  if (s.segments <= 1 || s.lead > 0) return 0;
  return (size_t)(backward ? 2 : 1) * (size_t)(bh - s.whole) * s.segments * (size_t)d_qk *
         (size_t)d_v * 4;
}

DecayView view(const void *p, const int64_t *strides) {
  DecayView v;
  v.p = p;
  v.sb = strides[0];
  v.sh = strides[1];
  v.st = strides[2];
  return v;
}

// bf16 whose rows TMA can address runs on tensor cores.
bool use_tensor_cores(const DecayCall &c) {
  if (c.dtype != LA_DTYPE_BFLOAT16 || c.n == 0) return false;
  for (int r = 0; r < c.roles; ++r) {
    const DecayRole &f = c.role[r];
    if (!decay_tc_view(f.a, f.da, c) || !decay_tc_view(f.b, f.da, c) ||
        !decay_tc_view(f.v, f.dvo, c) || !decay_tc_view(f.out, f.dvo, c))
      return false;
  }
  return true;
}

int run_decay(const DecayCall &call, const DecayRole *state_roles, int n_state_roles,
              cudaStream_t s) {
  const bool tc = use_tensor_cores(call);
  // (bf16 that TMA cannot address: the plan for tensor cores may leave heads
  // whole or have no workspace, the CUDA-core kernels walk every head alike)
  if (!tc && (call.whole > 0 || call.lead > 0)) {
    DecayCall same = call;
    same.whole = same.lead = 0;
    same.segments = fit_segments(call.n, 1, &same.seg_len);
    return launch_decay_output_simt(same, s);
  }
  if (call.segments > 1 && call.lead == 0) {
    DecayCall pass = call;
    pass.roles = n_state_roles;
    for (int r = 0; r < n_state_roles; ++r) pass.role[r] = state_roles[r];
    const int st = tc ? launch_decay_state_tc(pass, s) : launch_decay_state_simt(pass, s);
    if (st != LA_OK) return st;
  }
  return tc ? launch_decay_output_tc(call, s) : launch_decay_output_simt(call, s);
}

bool null_strides(const int64_t *const *s, int n) {
  for (int i = 0; i < n; ++i)
    if (!s[i]) return true;
  return false;
}

}  // namespace
}  // namespace la

using namespace la;

extern "C" {

int la_decay_plan(int64_t batch, int64_t heads, int64_t seq_len, int64_t d_qk, int64_t d_v,
                  int dtype, int backward, int segments_requested, int *segments_out,
                  size_t *workspace_bytes_out) {
  if (!segments_out || !workspace_bytes_out || segments_requested < 0)
    return LA_ERR_INVALID_ARGUMENT;
  int st = check_sizes(batch, heads, seq_len, d_qk, d_v, dtype);
  if (st != LA_OK) return st;
  DeviceInfo info;
  info.sm_count = 1;
  if (segments_requested == 0 && (st = require_device(&info)) != LA_OK) return st;
  const DecaySplit split = plan_split(batch * heads, seq_len, d_qk, d_v, dtype, backward != 0,
                                      segments_requested, info.sm_count);
  *segments_out = split.segments;
  *workspace_bytes_out = state_bytes(batch * heads, split, d_qk, d_v, backward != 0);
  return LA_OK;
}

int la_decay_chunked_fwd(const void *q, const int64_t *q_strides, const void *k,
                         const int64_t *k_strides, const void *v, const int64_t *v_strides,
                         void *out, const int64_t *out_strides, const float *log_decay,
                         int64_t batch, int64_t heads, int64_t seq_len, int64_t d_qk, int64_t d_v,
                         int dtype, float scale, const float *init_state, float *final_state,
                         void *workspace, size_t workspace_bytes, int segments, void *stream) {
  int st = check_sizes(batch, heads, seq_len, d_qk, d_v, dtype);
  if (st != LA_OK) return st;
  if (segments < 0) return LA_ERR_INVALID_ARGUMENT;
  const int64_t bh = batch * heads;
  if (bh == 0) return LA_OK;
  const int64_t *strides[] = {q_strides, k_strides, v_strides, out_strides};
  if (!log_decay || null_strides(strides, 4)) return LA_ERR_INVALID_ARGUMENT;
  if (seq_len > 0 && (!q || !k || !v || !out)) return LA_ERR_INVALID_ARGUMENT;
  if (seq_len == 0 && !final_state) return LA_OK;
  DeviceInfo info;
  if ((st = require_device(&info)) != LA_OK) return st;
  DecayCall c;
  const DecaySplit split =
      plan_split(bh, seq_len, d_qk, d_v, dtype, false, segments, info.sm_count);
  c.whole = split.whole, c.segments = split.segments, c.seg_len = split.len;
  c.lead = split.lead;
  const size_t need = state_bytes(bh, split, d_qk, d_v, false);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255)))
    return LA_ERR_WORKSPACE;
  c.roles = 1;
  c.log_decay = log_decay;
  c.batch = batch;
  c.heads = heads;
  c.n = seq_len;
  c.dtype = dtype;
  DecayRole &f = c.role[0];
  f.a = view(q, q_strides);
  f.b = view(k, k_strides);
  f.v = view(v, v_strides);
  f.out = view(out, out_strides);
  f.da = (int)d_qk;
  f.dvo = (int)d_v;
  f.init = init_state;
  f.states = (float *)workspace;
  f.final_state = final_state;
  f.intra = f.inter = scale;
  return run_decay(c, &f, 1, (cudaStream_t)stream);
}

int la_decay_chunked_bwd(const void *q, const int64_t *q_strides, const void *k,
                         const int64_t *k_strides, const void *v, const int64_t *v_strides,
                         const void *d_out, const int64_t *d_out_strides, void *dq,
                         const int64_t *dq_strides, void *dk, const int64_t *dk_strides, void *dv,
                         const int64_t *dv_strides, const float *log_decay, int64_t batch,
                         int64_t heads, int64_t seq_len, int64_t d_qk, int64_t d_v, int dtype,
                         float scale, const float *init_state, const float *d_final_state,
                         float *d_init_state, void *workspace, size_t workspace_bytes,
                         int segments, void *stream) {
  int st = check_sizes(batch, heads, seq_len, d_qk, d_v, dtype);
  if (st != LA_OK) return st;
  if (segments < 0) return LA_ERR_INVALID_ARGUMENT;
  const int64_t bh = batch * heads;
  if (bh == 0) return LA_OK;
  const int64_t *strides[] = {q_strides,  k_strides,  v_strides, d_out_strides,
                              dq_strides, dk_strides, dv_strides};
  if (!log_decay || null_strides(strides, 7)) return LA_ERR_INVALID_ARGUMENT;
  if (seq_len > 0 && (!q || !k || !v || !d_out || !dq || !dk || !dv))
    return LA_ERR_INVALID_ARGUMENT;
  if (seq_len == 0 && !d_init_state) return LA_OK;
  DeviceInfo info;
  if ((st = require_device(&info)) != LA_OK) return st;
  DecayCall c;
  const DecaySplit split =
      plan_split(bh, seq_len, d_qk, d_v, dtype, true, segments, info.sm_count);
  c.whole = split.whole, c.segments = split.segments, c.seg_len = split.len;
  c.lead = split.lead;
  const size_t need = state_bytes(bh, split, d_qk, d_v, true);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255)))
    return LA_ERR_WORKSPACE;
  float *ahead = (float *)workspace;  // the segments' states, first token first
  float *back = ahead + need / (2 * sizeof(float));  // last token first
  c.roles = 3;
  c.log_decay = log_decay;
  c.batch = batch;
  c.heads = heads;
  c.n = seq_len;
  c.dtype = dtype;
  const DecayView Q = view(q, q_strides), K = view(k, k_strides), V = view(v, v_strides),
                  G = view(d_out, d_out_strides);
  DecayRole &a = c.role[0], &b = c.role[1], &d = c.role[2];
  a.a = G, a.b = V, a.v = K, a.out = view(dq, dq_strides);
  a.da = (int)d_v, a.dvo = (int)d_qk;
  a.init = init_state, a.states = ahead;
  a.transposed = 1;
  a.intra = a.inter = scale;
  b.a = K, b.b = Q, b.v = G, b.out = view(dv, dv_strides);
  b.da = (int)d_qk, b.dvo = (int)d_v;
  b.init = d_final_state, b.states = back;
  b.final_state = d_init_state;
  b.reverse = 1;
  b.intra = b.inc = scale;
  d.a = V, d.b = G, d.v = Q, d.out = view(dk, dk_strides);
  d.da = (int)d_v, d.dvo = (int)d_qk;
  d.init = d_final_state, d.states = back;
  d.transposed = 1;
  d.reverse = 1;
  d.intra = d.inc = scale;
  DecayRole pass[2];
  pass[0].b = K, pass[0].v = V, pass[0].da = (int)d_qk, pass[0].dvo = (int)d_v;
  pass[0].states = ahead;
  pass[1] = b;
  return run_decay(c, pass, 2, (cudaStream_t)stream);
}

int la_decay_step(const void *q, const int64_t *q_strides, const void *k, const int64_t *k_strides,
                  const void *v, const int64_t *v_strides, void *out, float *state,
                  const int64_t *state_strides, const float *log_decay, int64_t batch,
                  int64_t heads, int64_t d_qk, int64_t d_v, int dtype, float scale, void *stream) {
  int st = check_sizes(0, 0, 1, d_qk, d_v, dtype);
  if (st != LA_OK) return st;
  if (batch < 0 || heads < 0) return LA_ERR_INVALID_ARGUMENT;
  if (batch == 0 || heads == 0) return LA_OK;
  if (batch > INT32_MAX / heads) return LA_ERR_UNSUPPORTED;
  const int64_t *strides[] = {q_strides, k_strides, v_strides, state_strides};
  if (!q || !k || !v || !out || !state || !log_decay || null_strides(strides, 4))
    return LA_ERR_INVALID_ARGUMENT;
  DeviceInfo info;
  if ((st = require_device(&info)) != LA_OK) return st;
  DecayStep p;
  p.q = q, p.k = k, p.v = v, p.out = out, p.state = state, p.log_decay = log_decay;
  p.q_sb = q_strides[0], p.q_sh = q_strides[1];
  p.k_sb = k_strides[0], p.k_sh = k_strides[1];
  p.v_sb = v_strides[0], p.v_sh = v_strides[1];
  p.state_sb = state_strides[0], p.state_sh = state_strides[1];
  p.heads = heads;
  p.dk = (int)d_qk, p.dv = (int)d_v;
  p.scale = scale;
  return launch_decay_step(p, batch, dtype, (cudaStream_t)stream);
}

}  // extern "C"
