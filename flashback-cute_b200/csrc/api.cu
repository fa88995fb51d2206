// C-ABI entry points (include/flashback_b200.h): argument validation, parameter-block
// construction and dispatch to the tensor-core (tcgen05) or CUDA-core kernels.
// There is no CPU path: on a machine without an sm_100 device every compute entry point
// returns FB_ERR_ARCH / FB_ERR_CUDA.
#include "../../include/flashback_b200.h"
#include "fb_params.h"

#include <atomic>
#include <initializer_list>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>

namespace fb {

__device__ int g_device_status = 0;

namespace {

thread_local int tl_launches = 0;
thread_local char tl_cuda_error[256] = "";

constexpr int kMaxDevices = 64;
// Per-device facts, looked up once. The entry points may be called from several host threads at
// once (autograd runs backward passes on worker threads), so the look-up takes a mutex and the
// "known" flag is published last, with release ordering, after the pointer it guards.
// (cudaDeviceReset invalidates these cached device addresses; the library does not support it.)
std::atomic<int> g_arch_major[kMaxDevices];  // 0 = not looked up yet
int* g_status_ptr[kMaxDevices];              // device address of g_device_status per device
std::mutex g_setup_mutex;

}  // namespace

int record_cuda(cudaError_t e) {
  snprintf(tl_cuda_error, sizeof(tl_cuda_error), "%s: %s", cudaGetErrorName(e), cudaGetErrorString(e));
  return FB_ERR_CUDA;
}

void set_launch_count(int n) { tl_launches = n; }

// Per-device lazy set-up: architecture check and the address of the status word.
int device_setup(int** status_ptr) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return record_cuda(e);
  if (dev < 0 || dev >= kMaxDevices) return FB_ERR_ARCH;
  int major = g_arch_major[dev].load(std::memory_order_acquire);
  if (major == 0) {
    std::lock_guard<std::mutex> lock(g_setup_mutex);
    major = g_arch_major[dev].load(std::memory_order_relaxed);
    if (major == 0) {
      e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
      if (e != cudaSuccess) return record_cuda(e);
      int* sp = nullptr;
      if (major == 10) {
        e = cudaGetSymbolAddress(reinterpret_cast<void**>(&sp), g_device_status);
        if (e != cudaSuccess) return record_cuda(e);
      }
      g_status_ptr[dev] = sp;
      g_arch_major[dev].store(major, std::memory_order_release);
    }
  }
  if (major != 10) return FB_ERR_ARCH;
  *status_ptr = g_status_ptr[dev];
  return FB_OK;
}

namespace {

// Environment switches are read once, before any thread can race on them.
struct EnvSwitches {
  bool force_simt;
  int debug;
  EnvSwitches() {
    const char* s = getenv("FLASHBACK_FORCE_SIMT");
    force_simt = s && s[0] == '1';
    const char* d = getenv("FLASHBACK_DEBUG");
    debug = d ? atoi(d) : 0;
  }
};
const EnvSwitches g_env;

bool env_force_simt() { return g_env.force_simt; }

}  // namespace

int check_problem(const fb_problem& pr) {
  if (pr.dtype != FB_BF16 && pr.dtype != FB_F16 && pr.dtype != FB_F32) return FB_ERR_DTYPE;
  if (pr.head_dim != 64 && pr.head_dim != 128) return FB_ERR_HEAD_DIM;
  if (pr.heads_q <= 0 || pr.heads_kv <= 0 || pr.heads_q % pr.heads_kv != 0) return FB_ERR_HEADS;
  if (pr.batch <= 0 || pr.seqlen_q < 0 || pr.seqlen_k < 0 || pr.total_q < 0 || pr.total_k < 0) return FB_ERR_SHAPE;
  if ((pr.cu_seqlens_q == nullptr) != (pr.cu_seqlens_k == nullptr)) return FB_ERR_MODE;
  if (!pr.cu_seqlens_q) {
    if (pr.total_q != (int64_t)pr.batch * pr.seqlen_q || pr.total_k != (int64_t)pr.batch * pr.seqlen_k) return FB_ERR_SHAPE;
  }
  if (pr.total_q >= (1ll << 31) || pr.total_k >= (1ll << 31)) return FB_ERR_TOO_LARGE;
  if (pr.batch > 65535 || pr.heads_q > 65535) return FB_ERR_TOO_LARGE;
  const int split = (pr.flags >> 8) & 15;
  if (split != 0 && split != 1 && split != 2 && split != 4 && split != 8) return FB_ERR_MODE;
  int prev_row = 0, prev_shift = INT32_MAX;
  bool ended = false;
  const int seg_len = (pr.flags & FB_FLAG_SEG_KEYS) ? pr.seqlen_k : pr.seqlen_q;
  for (int t = 0; t < 4; ++t) {  // row segments: dense causal, breaks on owner-tile boundaries, positions growing with the row
    if (pr.seg_rows[t] == 0 && pr.seg_shift[t] == 0) { ended = true; continue; }
    if (!pr.causal || pr.cu_seqlens_q) return FB_ERR_MODE;
    if (ended || pr.seg_rows[t] <= prev_row || pr.seg_rows[t] > seg_len || pr.seg_rows[t] % 128 != 0) return FB_ERR_SHAPE;
    if (pr.seg_shift[t] < 0 || pr.seg_shift[t] > prev_shift) return FB_ERR_SHAPE;
    prev_row = pr.seg_rows[t];
    prev_shift = pr.seg_shift[t];
  }
  return FB_OK;
}

namespace {

// Required tensor: non-NULL, 16-byte aligned, strides multiples of 8 elements (16 bytes for
// 16-bit types; what TMA and the vector accesses need).
int check_tensor(const fb_tensor& t, bool required) {
  if (!t.ptr) return required ? FB_ERR_NULL_ARG : FB_OK;
  if (reinterpret_cast<uintptr_t>(t.ptr) % 16 != 0) return FB_ERR_ALIGNMENT;
  if (t.row_stride % 8 != 0 || t.head_stride % 8 != 0 || t.row_stride <= 0 || t.head_stride <= 0) return FB_ERR_ALIGNMENT;
  return FB_OK;
}

SeqT cvt(const fb_tensor& t) { return SeqT{t.ptr, t.row_stride, t.head_stride}; }

void fill_problem(Params& p, const fb_problem& pr) {
  memset(&p, 0, sizeof(p));
  p.dtype = pr.dtype;
  p.B = pr.batch; p.Hq = pr.heads_q; p.Hkv = pr.heads_kv; p.D = pr.head_dim;
  p.Sq = pr.seqlen_q; p.Sk = pr.seqlen_k; p.causal = pr.causal ? 1 : 0;
  p.Tq = pr.total_q; p.Tk = pr.total_k;
  for (int t = 0; t < 4 && pr.seg_rows[t] > 0; ++t) { p.seg_rows[t] = pr.seg_rows[t]; p.seg_shift[t] = pr.seg_shift[t]; p.seg_n = t + 1; }
  p.seg_keys = (p.seg_n > 0 && (pr.flags & FB_FLAG_SEG_KEYS)) ? 1 : 0;
  p.cu_q = pr.cu_seqlens_q; p.cu_k = pr.cu_seqlens_k;
  p.scale = pr.softmax_scale;
  p.debug = g_env.debug;
  p.group = (pr.flags & FB_FLAG_TILE_MAJOR) ? 1 : ((pr.flags >> 12) & 0xfff);  // 0 = chosen by the launcher
  p.split = (pr.flags >> 8) & 15;  // 0 = chosen by the launcher
  p.kv_f32 = (pr.flags & FB_FLAG_KV_OUT_F32) ? 1 : 0;
  p.kv_accum = (pr.flags & FB_FLAG_KV_ACCUMULATE) ? 1 : 0;
  p.kv_accum_rows = INT64_MAX;
  p.wait_budget = 0;
}

bool use_tensor_cores(const fb_problem& pr) {
  return pr.dtype != FB_F32 && !(pr.flags & FB_FLAG_FORCE_SIMT) && !env_force_simt();
}

// key segments: only the kernels that own key rows (dK/dV side) take them
bool has_key_segments(const fb_problem& pr) { return (pr.flags & FB_FLAG_SEG_KEYS) && pr.seg_rows[0] > 0; }

#define FB_TRY(expr) do { int _s = (expr); if (_s != FB_OK) return _s; } while (0)

}  // namespace
}  // namespace fb

using namespace fb;

extern "C" int fb_jvp_fwd(const fb_jvp_args* a, fb_stream_t stream) {
  tl_launches = 0;
  if (!a) return FB_ERR_NULL_ARG;
  FB_TRY(check_problem(a->prob));
  const bool tangent = a->q_dot.ptr || a->k_dot.ptr || a->v_dot.ptr;
  if (tangent && !(a->q_dot.ptr && a->k_dot.ptr && a->v_dot.ptr)) return FB_ERR_MODE;
  FB_TRY(check_tensor(a->q, true)); FB_TRY(check_tensor(a->k, true)); FB_TRY(check_tensor(a->v, true));
  FB_TRY(check_tensor(a->q_dot, tangent)); FB_TRY(check_tensor(a->k_dot, tangent)); FB_TRY(check_tensor(a->v_dot, tangent));
  FB_TRY(check_tensor(a->out, true));
  FB_TRY(check_tensor(a->out_dot, tangent));
  if (!a->lse) return FB_ERR_NULL_ARG;
  if (tangent && !a->z1) return FB_ERR_NULL_ARG;
  if (a->lse_known && !tangent) return FB_ERR_MODE;
  if (has_key_segments(a->prob)) return FB_ERR_MODE;
  FB_TRY(check_tensor(a->dout, false)); FB_TRY(check_tensor(a->dout_dot, false));
  if (a->dout_dot.ptr && !(a->dout.ptr && tangent)) return FB_ERR_MODE;
  if (a->dout.ptr && (!a->dpsum || (tangent && !a->ddot))) return FB_ERR_NULL_ARG;
  if (a->prob.total_q == 0) return FB_OK;

  Params p;
  fill_problem(p, a->prob);
  FB_TRY(device_setup(&p.status));
  p.q = cvt(a->q); p.k = cvt(a->k); p.v = cvt(a->v);
  p.qd = cvt(a->q_dot); p.kd = cvt(a->k_dot); p.vd = cvt(a->v_dot);
  p.o = cvt(a->out); p.od = cvt(a->out_dot);
  p.lse = a->lse; p.z1 = a->z1;
  p.dout = cvt(a->dout); p.doutd = cvt(a->dout_dot);
  p.dpsum = a->dpsum; p.ddot = a->ddot;
  p.lse_known = a->lse_known ? 1 : 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int n = use_tensor_cores(a->prob) ? launch_tc_fwd(p, s) : launch_simt_fwd(p, s);
  if (n < 0) { if (n == FB_ERR_CUDA) record_cuda(cudaGetLastError()); return n; }
  tl_launches = n;
  return FB_OK;
}

extern "C" int fb_bwd_row_stats(const fb_stats_args* a, fb_stream_t stream) {
  tl_launches = 0;
  if (!a) return FB_ERR_NULL_ARG;
  FB_TRY(check_problem(a->prob));
  FB_TRY(check_tensor(a->out, true)); FB_TRY(check_tensor(a->dout, true));
  FB_TRY(check_tensor(a->out_dot, false)); FB_TRY(check_tensor(a->dout_dot, false));
  if (!a->dpsum) return FB_ERR_NULL_ARG;
  if (a->out_dot.ptr && !a->ddot) return FB_ERR_NULL_ARG;
  if (a->dout_dot.ptr && !a->out_dot.ptr) return FB_ERR_MODE;
  if (a->prob.total_q == 0) return FB_OK;
  Params p;
  fill_problem(p, a->prob);
  FB_TRY(device_setup(&p.status));
  p.o = cvt(a->out); p.dout = cvt(a->dout); p.od = cvt(a->out_dot); p.doutd = cvt(a->dout_dot);
  p.dpsum = a->dpsum; p.ddot = a->out_dot.ptr ? a->ddot : nullptr;
  int n = launch_row_stats(p, reinterpret_cast<cudaStream_t>(stream));
  if (n < 0) { if (n == FB_ERR_CUDA) record_cuda(cudaGetLastError()); return n; }
  tl_launches = n;
  return FB_OK;
}

static int hvp_bwd_impl(const fb_hvp_args* a, const fb_kv_scatter* sc, fb_stream_t stream) {
  tl_launches = 0;
  if (!a) return FB_ERR_NULL_ARG;
  FB_TRY(check_problem(a->prob));
  const bool tangent = a->q_dot.ptr || a->k_dot.ptr || a->v_dot.ptr;
  if (tangent && !(a->q_dot.ptr && a->k_dot.ptr && a->v_dot.ptr)) return FB_ERR_MODE;
  const bool want_dot = a->dq_dot.ptr || a->dk_dot.ptr || a->dv_dot.ptr;
  if (want_dot && !tangent) return FB_ERR_MODE;
  if (a->dout_dot.ptr && !tangent) return FB_ERR_MODE;
  FB_TRY(check_tensor(a->q, true)); FB_TRY(check_tensor(a->k, true)); FB_TRY(check_tensor(a->v, true));
  FB_TRY(check_tensor(a->dout, true));
  FB_TRY(check_tensor(a->q_dot, tangent)); FB_TRY(check_tensor(a->k_dot, tangent)); FB_TRY(check_tensor(a->v_dot, tangent));
  FB_TRY(check_tensor(a->dout_dot, false));
  FB_TRY(check_tensor(a->dq, false)); FB_TRY(check_tensor(a->dk, false)); FB_TRY(check_tensor(a->dv, false));
  FB_TRY(check_tensor(a->dq_dot, false)); FB_TRY(check_tensor(a->dk_dot, false)); FB_TRY(check_tensor(a->dv_dot, false));
  if (!a->lse || !a->dpsum) return FB_ERR_NULL_ARG;
  if (tangent && (!a->z1 || !a->ddot)) return FB_ERR_NULL_ARG;
  if (has_key_segments(a->prob) && (a->dq.ptr || a->dq_dot.ptr)) return FB_ERR_MODE;
  if (a->prob.flags & (FB_FLAG_KV_OUT_F32 | FB_FLAG_KV_ACCUMULATE)) {
    // float32 / accumulating dK,dV-side outputs: tensor-core kernels only, and accumulation needs float32
    if (!use_tensor_cores(a->prob)) return FB_ERR_MODE;
    if ((a->prob.flags & FB_FLAG_KV_ACCUMULATE) && !(a->prob.flags & FB_FLAG_KV_OUT_F32)) return FB_ERR_MODE;
  }
  if (a->prob.total_q == 0 || a->prob.total_k == 0) return FB_OK;

  Params p;
  fill_problem(p, a->prob);
  FB_TRY(device_setup(&p.status));
  p.q = cvt(a->q); p.k = cvt(a->k); p.v = cvt(a->v); p.dout = cvt(a->dout);
  // Tangent inputs only matter if a directional derivative is requested.
  if (want_dot) { p.qd = cvt(a->q_dot); p.kd = cvt(a->k_dot); p.vd = cvt(a->v_dot); p.doutd = cvt(a->dout_dot); }
  p.lse = const_cast<float*>(a->lse); p.dpsum = const_cast<float*>(a->dpsum);
  p.z1 = const_cast<float*>(a->z1); p.ddot = const_cast<float*>(a->ddot);
  p.dq = cvt(a->dq); p.dk = cvt(a->dk); p.dv = cvt(a->dv);
  p.dqd = cvt(a->dq_dot); p.dkd = cvt(a->dk_dot); p.dvd = cvt(a->dv_dot);
  if (sc) {
    // scatter mode: float32 results of the dK/dV kernels go to the owners of the key rows
    if (!p.kv_f32 || a->prob.batch != 1 || a->prob.cu_seqlens_q) return FB_ERR_MODE;
    if (sc->n_peers < 1 || sc->n_peers > 8 || sc->rows_per_peer <= 0 || sc->rows_per_peer % 128 != 0) return FB_ERR_SHAPE;
    if ((int64_t)sc->n_peers * sc->rows_per_peer < a->prob.seqlen_k) return FB_ERR_SHAPE;
    if (sc->row_stride <= 0 || sc->head_stride <= 0 || sc->row_stride % 4 != 0 || sc->head_stride % 4 != 0) return FB_ERR_ALIGNMENT;
    void* const* lists[4] = {sc->dk, sc->dv, sc->dk_dot, sc->dv_dot};
    const void* wanted[4] = {a->dk.ptr, a->dv.ptr, a->dk_dot.ptr, a->dv_dot.ptr};
    for (int o = 0; o < 4; ++o)
      for (int i = 0; i < sc->n_peers; ++i) {
        if (wanted[o] && !lists[o][i]) return FB_ERR_NULL_ARG;
        if (reinterpret_cast<uintptr_t>(lists[o][i]) % 16 != 0) return FB_ERR_ALIGNMENT;
        p.scat[o][i] = lists[o][i];
      }
    if (sc->accumulate_rows < 0 || sc->accumulate_rows % 128 != 0) return FB_ERR_SHAPE;
    if (sc->accumulate_rows > 0) p.kv_accum_rows = sc->accumulate_rows;
    p.scat_n = sc->n_peers; p.scat_rows = sc->rows_per_peer;
    p.scat_row_stride = sc->row_stride; p.scat_head_stride = sc->head_stride;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int n = use_tensor_cores(a->prob) ? launch_tc_bwd(p, s) : launch_simt_bwd(p, s);
  if (n < 0) { if (n == FB_ERR_CUDA) record_cuda(cudaGetLastError()); return n; }
  tl_launches = n;
  return FB_OK;
}

extern "C" int fb_hvp_bwd(const fb_hvp_args* a, fb_stream_t stream) { return hvp_bwd_impl(a, nullptr, stream); }

extern "C" int fb_hvp_bwd_scatter(const fb_hvp_args* a, const fb_kv_scatter* sc, fb_stream_t stream) {
  if (!sc) { tl_launches = 0; return FB_ERR_NULL_ARG; }
  return hvp_bwd_impl(a, sc, stream);
}

extern "C" int fb_sum_slots(const float* slots, int32_t n_slots, int64_t slot_stride, int64_t count, int64_t period, const int64_t* valid,
                            float* out, fb_stream_t stream) {
  tl_launches = 0;
  if (!slots || !out) return FB_ERR_NULL_ARG;
  if (n_slots < 1 || n_slots > 8 || count < 0 || slot_stride < count || period < 0) return FB_ERR_SHAPE;
  if (period % 4 != 0 || (period > 0 && count % period != 0)) return FB_ERR_SHAPE;
  if (valid)
    for (int s = 0; s < n_slots; ++s)
      if (valid[s] < 0 || valid[s] % 4 != 0) return FB_ERR_SHAPE;
  if (count % 4 != 0 || slot_stride % 4 != 0 || reinterpret_cast<uintptr_t>(slots) % 16 != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0)
    return FB_ERR_ALIGNMENT;
  if (count == 0) return FB_OK;
  int* status_word = nullptr;
  FB_TRY(device_setup(&status_word));
  int n = launch_sum_slots(slots, n_slots, slot_stride, count, period, valid, out, reinterpret_cast<cudaStream_t>(stream));
  if (n < 0) { if (n == FB_ERR_CUDA) record_cuda(cudaGetLastError()); return n; }
  tl_launches = n;
  return FB_OK;
}

// ---- relative position bias ----
namespace {

// Checks the bias and fills the kernels' copy of it. need_table: the table itself is read.
int convert_relpos(RelPos& r, const fb_relpos& b, bool need_table) {
  if (!b.starts || (need_table && !b.table)) return FB_ERR_NULL_ARG;
  if (b.num_buckets < 2 || b.num_buckets > FB_RELPOS_MAX_BUCKETS) return FB_ERR_RELPOS;
  if (b.bidirectional != 0 && b.bidirectional != 1) return FB_ERR_RELPOS;
  if (b.bidirectional && (b.num_buckets < 4 || b.num_buckets % 2 != 0)) return FB_ERR_RELPOS;
  memset(&r, 0, sizeof(r));
  r.table = b.table;
  r.bucket_stride = b.bucket_stride;
  r.head_stride = b.head_stride;
  r.nb = b.num_buckets;
  r.two = b.bidirectional;
  r.side = r.two ? r.nb / 2 : r.nb;
  for (int t = 0; t < r.side - 1; ++t) {
    if (b.starts[t] < 0 || (t > 0 && b.starts[t] < b.starts[t - 1])) return FB_ERR_RELPOS;
    r.starts[t] = b.starts[t];
  }
  r.far = r.starts[r.side - 2];
  for (int t = 0; t < r.nb; ++t) {  // r > 0 starts at distance 1
    const int side = t >= r.side, x = t - side * r.side, first = x > 0 ? r.starts[x - 1] : 0, end = x < r.side - 1 ? r.starts[x] : INT32_MAX;
    if (end > (side && first < 1 ? 1 : first)) r.used[t / 32] |= 1u << (t % 32);
  }
  uint8_t* bytes = reinterpret_cast<uint8_t*>(r.near_words);
  for (int t = 0, n = 0; t < r.side; ++t) {
    const int end = t < r.side - 1 && r.starts[t] < kRelNear ? r.starts[t] : kRelNear;
    if (end > n) { memset(bytes + n, t, (size_t)(end - n)); n = end; }
  }
  return FB_OK;
}

// The problems the biased attention takes: any of fb_jvp_fwd without row segments and float32 key-side outputs.
int check_relpos_problem(const fb_problem& pr) {
  FB_TRY(check_problem(pr));
  if (pr.seg_rows[0] != 0 || pr.seg_shift[0] != 0) return FB_ERR_MODE;
  if (pr.flags & (FB_FLAG_KV_OUT_F32 | FB_FLAG_KV_ACCUMULATE | FB_FLAG_SEG_KEYS)) return FB_ERR_MODE;
  if (pr.seqlen_q > (1 << 30) || pr.seqlen_k > (1 << 30)) return FB_ERR_TOO_LARGE;
  return FB_OK;
}

int relpos_tiles(const fb_problem& pr) {
  const int rows = use_tensor_cores(pr) ? kTcOwnerRows : kSimtOwnerRows;
  return (pr.seqlen_q + rows - 1) / rows;
}

// D in the workspace of the backward, rounded up so that what follows is 16-byte aligned
size_t relpos_dot_floats(const fb_problem& pr) { return ((size_t)pr.heads_q * (size_t)pr.total_q + 3) / 4 * 4; }

int check_bias_sizes(int dtype, int heads, int sq, int sk) {
  if (dtype != FB_BF16 && dtype != FB_F16 && dtype != FB_F32) return FB_ERR_DTYPE;
  if (heads <= 0 || sq < 0 || sk < 0) return FB_ERR_SHAPE;
  if (heads > 65535 || sq > (1 << 20) || sk > (1 << 30)) return FB_ERR_TOO_LARGE;
  return FB_OK;
}

}  // namespace

extern "C" int fb_relpos_fwd(const fb_relpos_fwd_args* a, fb_stream_t stream) {
  tl_launches = 0;
  if (!a) return FB_ERR_NULL_ARG;
  FB_TRY(check_relpos_problem(a->prob));
  RelPos rel;
  FB_TRY(convert_relpos(rel, a->bias, true));
  FB_TRY(check_tensor(a->q, true)); FB_TRY(check_tensor(a->k, true)); FB_TRY(check_tensor(a->v, true));
  FB_TRY(check_tensor(a->out, true)); FB_TRY(check_tensor(a->out_low, false));
  if (a->prob.total_q == 0) return FB_OK;
  if (a->prob.total_k == 0) return FB_ERR_SHAPE;
  Params p;
  fill_problem(p, a->prob);
  rel.zero_rest = (a->prob.flags & FB_FLAG_ZERO_REST) && a->prob.cu_seqlens_q ? 1 : 0;
  FB_TRY(device_setup(&p.status));
  p.q = cvt(a->q); p.k = cvt(a->k); p.v = cvt(a->v); p.o = cvt(a->out); p.od = cvt(a->out_low);
  p.lse = a->lse;
  rel.shift = a->shift;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int n = use_tensor_cores(a->prob) ? launch_tc_fwd_rel(p, rel, s) : launch_simt_fwd_rel(p, rel, s);
  if (n < 0) { if (n == FB_ERR_CUDA) record_cuda(cudaGetLastError()); return n; }
  tl_launches = n;
  return FB_OK;
}

extern "C" int fb_relpos_bwd(const fb_relpos_bwd_args* a, fb_stream_t stream) {
  tl_launches = 0;
  if (!a) return FB_ERR_NULL_ARG;
  FB_TRY(check_relpos_problem(a->prob));
  RelPos rel;
  FB_TRY(convert_relpos(rel, a->bias, true));
  FB_TRY(check_tensor(a->q, true)); FB_TRY(check_tensor(a->k, true)); FB_TRY(check_tensor(a->v, true));
  FB_TRY(check_tensor(a->out, true)); FB_TRY(check_tensor(a->dout, true)); FB_TRY(check_tensor(a->out_low, false));
  FB_TRY(check_tensor(a->dq, false)); FB_TRY(check_tensor(a->dk, false)); FB_TRY(check_tensor(a->dv, false));
  if (!a->lse || !a->workspace) return FB_ERR_NULL_ARG;
  if (reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0) return FB_ERR_ALIGNMENT;
  if (a->prob.total_q == 0 || a->prob.total_k == 0) return FB_ERR_SHAPE;
  if (!a->shift) return FB_ERR_NULL_ARG;
  rel.shift = const_cast<float*>(a->shift);
  Params p;
  fill_problem(p, a->prob);
  rel.zero_rest = (a->prob.flags & FB_FLAG_ZERO_REST) && a->prob.cu_seqlens_q ? 1 : 0;
  FB_TRY(device_setup(&p.status));
  p.q = cvt(a->q); p.k = cvt(a->k); p.v = cvt(a->v); p.dout = cvt(a->dout);
  p.o = cvt(a->out); p.od = cvt(a->out_low);
  p.lse = const_cast<float*>(a->lse); p.dpsum = a->workspace;
  p.dq = cvt(a->dq); p.dk = cvt(a->dk); p.dv = cvt(a->dv);
  if (!a->dtable && !p.dq.ptr && !p.dk.ptr && !p.dv.ptr) return FB_OK;
  rel.dpart = a->dtable ? a->workspace + relpos_dot_floats(a->prob) : nullptr;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int n = use_tensor_cores(a->prob) ? launch_tc_bwd_rel(p, rel, s) : launch_simt_bwd_rel(p, rel, s);
  if (n >= 0 && a->dtable) {
    const int r = launch_rel_reduce(p.dtype, rel.dpart, p.B, p.Hq, relpos_tiles(a->prob), rel.nb, a->dtable, a->dtable_bucket_stride,
                                    a->dtable_head_stride, s);
    n = r < 0 ? r : n + r;
  }
  if (n < 0) { if (n == FB_ERR_CUDA) record_cuda(cudaGetLastError()); return n; }
  tl_launches = n;
  return FB_OK;
}

extern "C" size_t fb_relpos_workspace_bytes(const fb_problem* pr, int num_buckets) {
  if (!pr || check_relpos_problem(*pr) != FB_OK || num_buckets < 2 || num_buckets > FB_RELPOS_MAX_BUCKETS) return 0;
  return sizeof(float) * (relpos_dot_floats(*pr) + (size_t)pr->batch * (size_t)pr->heads_q * (size_t)relpos_tiles(*pr) * (size_t)num_buckets);
}

extern "C" int fb_relpos_bias(const fb_relpos_bias_args* a, fb_stream_t stream) {
  tl_launches = 0;
  if (!a) return FB_ERR_NULL_ARG;
  FB_TRY(check_bias_sizes(a->dtype, a->heads, a->seqlen_q, a->seqlen_k));
  RelPos rel;
  FB_TRY(convert_relpos(rel, a->bias, true));
  if (!a->out) return FB_ERR_NULL_ARG;
  if (reinterpret_cast<uintptr_t>(a->out) % 16 != 0) return FB_ERR_ALIGNMENT;
  if (a->seqlen_q == 0 || a->seqlen_k == 0) return FB_OK;
  int* status_word = nullptr;
  FB_TRY(device_setup(&status_word));
  int n = launch_relpos_fill(a->dtype, rel, a->heads, a->seqlen_q, a->seqlen_k, a->out, reinterpret_cast<cudaStream_t>(stream));
  if (n < 0) { if (n == FB_ERR_CUDA) record_cuda(cudaGetLastError()); return n; }
  tl_launches = n;
  return FB_OK;
}

extern "C" int fb_relpos_bias_grad(const fb_relpos_bias_grad_args* a, fb_stream_t stream) {
  tl_launches = 0;
  if (!a) return FB_ERR_NULL_ARG;
  FB_TRY(check_bias_sizes(a->dtype, a->heads, a->seqlen_q, a->seqlen_k));
  RelPos rel;
  FB_TRY(convert_relpos(rel, a->bias, false));
  if (!a->grad || !a->dtable || !a->workspace) return FB_ERR_NULL_ARG;
  if (reinterpret_cast<uintptr_t>(a->grad) % 16 != 0) return FB_ERR_ALIGNMENT;
  if (a->seqlen_q == 0 || a->seqlen_k == 0) return FB_ERR_SHAPE;
  int* status_word = nullptr;
  FB_TRY(device_setup(&status_word));
  rel.dpart = a->workspace;
  int n = launch_relpos_grad(a->dtype, rel, a->heads, a->seqlen_q, a->seqlen_k, a->grad, a->dtable, a->dtable_bucket_stride,
                             a->dtable_head_stride, reinterpret_cast<cudaStream_t>(stream));
  if (n < 0) { if (n == FB_ERR_CUDA) record_cuda(cudaGetLastError()); return n; }
  tl_launches = n;
  return FB_OK;
}

extern "C" size_t fb_relpos_bias_workspace_bytes(int dtype, int heads, int sq, int sk, int num_buckets) {
  if (check_bias_sizes(dtype, heads, sq, sk) != FB_OK || sq == 0 || sk == 0 || num_buckets < 2 || num_buckets > FB_RELPOS_MAX_BUCKETS) return 0;
  return sizeof(float) * (size_t)heads * (size_t)relpos_bias_parts(dtype, heads, sq, sk) * (size_t)num_buckets;
}

namespace {

int check_cache(const fb_cache& t) {
  if (!t.ptr) return FB_ERR_NULL_ARG;
  if (reinterpret_cast<uintptr_t>(t.ptr) % 16 != 0) return FB_ERR_ALIGNMENT;
  for (int64_t s : {t.batch_stride, t.row_stride, t.head_stride})
    if (s < 0 || s % 8 != 0) return FB_ERR_ALIGNMENT;
  return FB_OK;
}

int check_decode(const fb_relpos_decode_args& a) {
  if (a.dtype != FB_BF16 && a.dtype != FB_F16) return FB_ERR_DTYPE;
  if (a.head_dim != 64 && a.head_dim != 128) return FB_ERR_HEAD_DIM;
  if (a.heads_q <= 0 || a.heads_kv <= 0 || a.heads_q % a.heads_kv != 0) return FB_ERR_HEADS;
  if (a.batch < 0 || a.seqlen_q < 0 || a.seqlen_k < 0) return FB_ERR_SHAPE;
  if (a.batch > 65535 || a.seqlen_k > (1 << 30) || a.heads_q > 65535 || (int64_t)a.seqlen_q * a.heads_q > (1 << 20)) return FB_ERR_TOO_LARGE;
  if ((int64_t)a.heads_kv * (((int64_t)(a.heads_q / a.heads_kv) * a.seqlen_q + 15) / 16) > 65535) return FB_ERR_TOO_LARGE;  // grid
  if ((int64_t)(a.heads_q / a.heads_kv) * a.bias.num_buckets > kDecodeMaxTable) return FB_ERR_TOO_LARGE;
  return FB_OK;
}

DecodeShape shape_of(const fb_relpos_decode_args& a) {
  return decode_shape(a.batch, a.heads_kv, a.heads_q / a.heads_kv * a.seqlen_q, a.seqlen_k);
}

}  // namespace

extern "C" size_t fb_relpos_decode_workspace_bytes(const fb_relpos_decode_args* a) {
  if (!a || check_decode(*a) != FB_OK || a->batch == 0 || a->seqlen_q == 0) return 0;
  const DecodeShape shape = shape_of(*a);
  return shape.splits == 1 || shape.cluster ? 0 : (size_t)a->batch * a->seqlen_q * a->heads_q * (size_t)shape.splits * (a->head_dim + 2) * sizeof(float);
}

extern "C" int fb_relpos_decode(const fb_relpos_decode_args* a, fb_stream_t stream) {
  tl_launches = 0;
  if (!a) return FB_ERR_NULL_ARG;
  FB_TRY(check_decode(*a));
  RelPos rel;
  FB_TRY(convert_relpos(rel, a->bias, true));
  FB_TRY(check_cache(a->q)); FB_TRY(check_cache(a->k)); FB_TRY(check_cache(a->v));
  if (!a->out) return FB_ERR_NULL_ARG;
  if (reinterpret_cast<uintptr_t>(a->out) % 16 != 0 || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0) return FB_ERR_ALIGNMENT;
  if (a->batch == 0 || a->seqlen_q == 0) return FB_OK;
  DecodeParams p;
  memset(&p, 0, sizeof(p));
  p.B = a->batch; p.Hq = a->heads_q; p.Hkv = a->heads_kv; p.G = a->heads_q / a->heads_kv;
  p.Sq = a->seqlen_q; p.Sk = a->seqlen_k; p.D = a->head_dim;
  p.scale = a->softmax_scale;
  p.q = CacheT{a->q.ptr, a->q.batch_stride, a->q.row_stride, a->q.head_stride};
  p.k = CacheT{a->k.ptr, a->k.batch_stride, a->k.row_stride, a->k.head_stride};
  p.v = CacheT{a->v.ptr, a->v.batch_stride, a->v.row_stride, a->v.head_stride};
  p.lens = a->lens;
  p.out = a->out;
  const DecodeShape shape = shape_of(*a);
  p.splits = shape.splits;
  p.cluster = shape.cluster ? 1 : 0;
  if (p.splits > 1 && !p.cluster) {
    if (!a->workspace) return FB_ERR_NULL_ARG;
    p.part = a->workspace;  // row length head_dim floats: the (maximum, sum) pairs behind them stay 8-byte aligned
    p.part_ml = reinterpret_cast<float2*>(a->workspace + (size_t)p.B * p.Sq * p.Hq * p.splits * p.D);
  }
  int* status_word = nullptr;
  FB_TRY(device_setup(&status_word));
  int n = launch_decode(a->dtype, p, rel, reinterpret_cast<cudaStream_t>(stream));
  if (n < 0) { if (n == FB_ERR_CUDA) record_cuda(cudaGetLastError()); return n; }
  tl_launches = n;
  return FB_OK;
}

extern "C" int fb_last_launch_count(void) { return tl_launches; }

extern "C" int fb_check_device_status(void) {
  int* sp = nullptr;
  FB_TRY(device_setup(&sp));
  cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess) return record_cuda(e);
  int v = 0;
  e = cudaMemcpy(&v, sp, sizeof(int), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return record_cuda(e);
  if (v != 0) {
    int zero = 0;
    cudaMemcpy(sp, &zero, sizeof(int), cudaMemcpyHostToDevice);
    snprintf(tl_cuda_error, sizeof(tl_cuda_error), "device status word = 0x%x (bits 0-2: a bounded wait gave up in the FWD/DQ/DKV kernel; bit 8: shared memory misaligned)", v);
    return FB_ERR_DEVICE_TIMEOUT;
  }
  return FB_OK;
}

extern "C" const char* fb_status_string(int status) {
  switch (status) {
    case FB_OK: return "ok";
    case FB_ERR_NULL_ARG: return "a required pointer is NULL";
    case FB_ERR_DTYPE: return "q, k, v must share a dtype in {float16, bfloat16, float32}";
    case FB_ERR_HEAD_DIM: return "head_dim must equal head_dim_v and be 64 or 128";
    case FB_ERR_HEADS: return "number of q heads must be divisible by number of kv heads";
    case FB_ERR_SHAPE: return "inconsistent problem sizes";
    case FB_ERR_ALIGNMENT: return "pointers must be 16-byte aligned and strides multiples of 8 elements";
    case FB_ERR_ARCH: return "flashback_b200 supports only sm_100 (Blackwell B200) GPUs";
    case FB_ERR_CUDA: return "CUDA call failed";
    case FB_ERR_MODE: return "inconsistent combination of optional tensors";
    case FB_ERR_TOO_LARGE: return "size exceeds a documented maximum";
    case FB_ERR_RELPOS: return "the bias table needs 2 to 128 buckets (even and at least 4 when bidirectional) and ascending bucket starts >= 0";
    case FB_ERR_DEVICE_TIMEOUT: return "a bounded device-side wait gave up";
  }
  return "unknown status";
}

extern "C" const char* fb_last_cuda_error(void) { return tl_cuda_error; }

extern "C" int fb_version(void) { return 200; }

extern "C" int fb_debug_profile(long long* out16) { return out16 ? read_profile(out16) : FB_ERR_NULL_ARG; }

extern "C" int fb_debug_wait_timeout(const fb_jvp_args* a, long long budget_cycles, fb_stream_t stream) {
  tl_launches = 0;
  if (!a) return FB_ERR_NULL_ARG;
  FB_TRY(check_problem(a->prob));
  if (a->prob.dtype != FB_BF16 || a->prob.head_dim != 64) return FB_ERR_MODE;
  if (budget_cycles < 1000 || budget_cycles > 2000000000ll) return FB_ERR_MODE;
  FB_TRY(check_tensor(a->q, true)); FB_TRY(check_tensor(a->k, true)); FB_TRY(check_tensor(a->v, true));
  FB_TRY(check_tensor(a->out, true));
  if (!a->lse) return FB_ERR_NULL_ARG;
  if (a->prob.total_q == 0) return FB_OK;
  Params p;
  fill_problem(p, a->prob);
  FB_TRY(device_setup(&p.status));
  p.q = cvt(a->q); p.k = cvt(a->k); p.v = cvt(a->v); p.o = cvt(a->out);
  p.lse = a->lse;
  p.wait_budget = budget_cycles;
  int n = launch_tc_fwd_wait_hook(p, reinterpret_cast<cudaStream_t>(stream));
  if (n < 0) { if (n == FB_ERR_CUDA) record_cuda(cudaGetLastError()); return n; }
  tl_launches = n;
  return FB_OK;
}

extern "C" size_t fb_workspace_bytes(const fb_problem* pr, int which) {
  if (!pr || which != 0 || pr->heads_q <= 0 || pr->total_q < 0) return 0;
  return (size_t)pr->heads_q * (size_t)pr->total_q * sizeof(float);
}

extern "C" size_t fb_abi_sizeof(int which) {
  switch (which) {
    case 0: return sizeof(fb_tensor);
    case 1: return sizeof(fb_problem);
    case 2: return sizeof(fb_jvp_args);
    case 3: return sizeof(fb_stats_args);
    case 4: return sizeof(fb_hvp_args);
    case 5: return sizeof(fb_bwd_noalloc_args);
    case 6: return sizeof(fb_kv_scatter);
    case 8: return sizeof(fb_relpos);
    case 9: return sizeof(fb_relpos_fwd_args);
    case 10: return sizeof(fb_relpos_bwd_args);
    case 11: return sizeof(fb_relpos_bias_args);
    case 12: return sizeof(fb_relpos_bias_grad_args);
    case 13: return sizeof(fb_cache);
    case 14: return sizeof(fb_relpos_decode_args);
  }
  return 0;
}
