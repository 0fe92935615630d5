// C entry points of the decayed linear attention: argument checks, the split
// into segments, and the launches (state of each segment, running states,
// outputs).
#include <math.h>

#include "decay.cuh"
#include "decay_step.cuh"

namespace la {
namespace {

// A segment is worth its share of the state pass from this many tokens on.
constexpr int64_t kMinDecaySegment = 4 * kDecayTile;

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

// Segments of each walk: as many as fill the SMs with one wave of CTAs.
int plan_segments(int64_t bh, int64_t n, int64_t d_qk, int64_t d_v, bool backward, int requested,
                  int sm_count, int64_t *len) {
  int64_t want = requested;
  if (want == 0) {
    const int64_t sq = (d_qk + kDecaySlice - 1) / kDecaySlice;
    const int64_t sv = (d_v + kDecaySlice - 1) / kDecaySlice;
    const int64_t ctas = bh * (backward ? 2 * sq + sv : sv);
    want = ctas > 0 ? sm_count / ctas : 1;
    const int64_t most = n / kMinDecaySegment;
    if (want > most) want = most;
  }
  return fit_segments(n, want, len);
}

size_t state_bytes(int64_t bh, int segments, int64_t d_qk, int64_t d_v, bool backward) {
  if (segments <= 1) return 0;
  return (size_t)(backward ? 2 : 1) * (size_t)bh * segments * (size_t)d_qk * (size_t)d_v * 4;
}

DecayView view(const void *p, const int64_t *strides) {
  DecayView v;
  v.p = p;
  v.sb = strides[0];
  v.sh = strides[1];
  v.st = strides[2];
  return v;
}

// In place: the state of each segment becomes the state before it,
//   seed_0 = init,  seed_{o+1} = lambda^len_o seed_o + state_o.
struct RunningArgs {
  float *states[2];
  const float *init[2];
  int64_t len0[2];  // tokens of the walk's first segment (the ragged one of a reversed walk)
};

__global__ void decay_running_kernel(const RunningArgs a, const float *log_decay, int64_t heads,
                                     int segments, int64_t per_head, int64_t seg_len) {
  const int64_t bh = blockIdx.y;
  float *s = a.states[blockIdx.z] + bh * segments * per_head;
  const float *init = a.init[blockIdx.z];
  const float g = log_decay[bh % heads];
  const float keep0 = decay_pow(g, (int)a.len0[blockIdx.z]), keep = decay_pow(g, (int)seg_len);
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < per_head;
       i += (int64_t)gridDim.x * blockDim.x) {
    float run = init ? init[bh * per_head + i] : 0.f;
    for (int o = 0; o < segments; ++o) {
      const float x = s[o * per_head + i];
      s[o * per_head + i] = run;
      run = fmaf(o == 0 ? keep0 : keep, run, x);
    }
  }
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

int run_decay(DecayCall &call, const DecayRole *state_roles, int n_state_roles,
              const float *const *inits, int64_t d_qk, int64_t d_v, cudaStream_t s) {
  const bool tc = use_tensor_cores(call);
  if (call.segments > 1) {
    DecayCall pass = call;
    pass.roles = n_state_roles;
    RunningArgs run{};
    for (int r = 0; r < n_state_roles; ++r) {
      pass.role[r] = state_roles[r];
      run.states[r] = state_roles[r].states;
      run.init[r] = inits[r];
      run.len0[r] = state_roles[r].reverse ? call.n - (call.segments - 1) * call.seg_len
                                           : call.seg_len;
    }
    int st = tc ? launch_decay_state_tc(pass, s) : launch_decay_state_simt(pass, s);
    if (st != LA_OK) return st;
    const int64_t per_head = d_qk * d_v;
    const dim3 grid((unsigned)((per_head + 255) / 256), (unsigned)(call.batch * call.heads),
                    (unsigned)n_state_roles);
    decay_running_kernel<<<grid, 256, 0, s>>>(run, call.log_decay, call.heads, call.segments,
                                              per_head, call.seg_len);
    st = check_launch();
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
  int64_t len = 0;
  *segments_out = plan_segments(batch * heads, seq_len, d_qk, d_v, backward != 0,
                                segments_requested, info.sm_count, &len);
  *workspace_bytes_out = state_bytes(batch * heads, *segments_out, d_qk, d_v, backward != 0);
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
  c.segments = plan_segments(bh, seq_len, d_qk, d_v, false, segments, info.sm_count, &c.seg_len);
  const size_t need = state_bytes(bh, c.segments, d_qk, d_v, false);
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
  f.seeds = c.segments > 1 ? (const float *)workspace : init_state;
  f.final_state = final_state;
  f.intra = f.inter = scale;
  DecayRole pass = f;
  pass.states = (float *)workspace;
  return run_decay(c, &pass, 1, &init_state, d_qk, d_v, (cudaStream_t)stream);
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
  c.segments = plan_segments(bh, seq_len, d_qk, d_v, true, segments, info.sm_count, &c.seg_len);
  const size_t need = state_bytes(bh, c.segments, d_qk, d_v, true);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255)))
    return LA_ERR_WORKSPACE;
  float *before = (float *)workspace;  // states before each segment, first token first
  float *after = before + bh * c.segments * d_qk * d_v;  // and of the reversed walk
  const bool split = c.segments > 1;
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
  a.seeds = split ? before : init_state;
  a.seed_transposed = 1;
  a.intra = a.inter = scale;
  b.a = K, b.b = Q, b.v = G, b.out = view(dv, dv_strides);
  b.da = (int)d_qk, b.dvo = (int)d_v;
  b.seeds = split ? after : d_final_state;
  b.final_state = d_init_state;
  b.reverse = 1;
  b.intra = b.inc = scale;
  d.a = V, d.b = G, d.v = Q, d.out = view(dk, dk_strides);
  d.da = (int)d_v, d.dvo = (int)d_qk;
  d.seeds = split ? after : d_final_state;
  d.seed_transposed = 1;
  d.reverse = 1;
  d.intra = d.inc = scale;
  DecayRole pass[2];
  pass[0].b = K, pass[0].v = V, pass[0].da = (int)d_qk, pass[0].dvo = (int)d_v;
  pass[0].states = before;
  pass[1] = b;
  pass[1].states = after;
  const float *inits[2] = {init_state, d_final_state};
  return run_decay(c, pass, 2, inits, d_qk, d_v, (cudaStream_t)stream);
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
