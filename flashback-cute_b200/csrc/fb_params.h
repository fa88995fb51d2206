// Internal kernel parameter block shared by the CUDA-core (SIMT) and tensor-core (tcgen05)
// kernels. Built by api.cu from the public C structs in include/flashback_b200.h.
#pragma once
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/flashback_b200.h"

namespace fb {

struct SeqT {
  void* ptr;
  int64_t row_stride;
  int64_t head_stride;
};

struct Params {
  int dtype;
  int B, Hq, Hkv, D;
  int Sq, Sk;  // dense: per-sequence rows; varlen: max lengths
  int causal;
  // row segments (dense causal only; seg_n = 0: off) of the query rows, or with seg_keys of the key rows:
  // seg_n break rows, ascending; the rows below break s (and not below an earlier one) sit seg_shift[s]
  // positions earlier than bottom-right alignment puts them, the rows from the last break on do not
  int seg_n, seg_keys, seg_rows[4], seg_shift[4];
  int64_t Tq, Tk;
  const int32_t* cu_q;
  const int32_t* cu_k;
  float scale;
  int lse_known;
  // inputs
  SeqT q, k, v, qd, kd, vd, dout, doutd;
  // forward outputs (inputs of the backward / of lse_known mode)
  SeqT o, od;
  float *lse, *z1, *dpsum, *ddot;
  // backward outputs
  SeqT dq, dk, dv, dqd, dkd, dvd;
  // device status word (bounded-wait timeouts)
  int* status;
  int debug;  // FLASHBACK_DEBUG bits (kernel bring-up switches; 0 in normal use)
  // dK/dV-side outputs (dk, dv, dkd, dvd) as float32 tensors, optionally added to what they already hold
  int kv_f32, kv_accum;
  // dK/dV-side results scattered to the owners of the key rows (fb_hvp_bwd_scatter): key row r of output o
  // goes to scat[o][r / scat_rows] at row r % scat_rows; o = 0 dk, 1 dv, 2 dk_dot, 3 dv_dot. The
  // destinations may be another GPU's memory (plain stores over NVLink). scat_n = 0: off.
  void* scat[4][8];
  int scat_n, scat_rows;
  int64_t scat_row_stride, scat_head_stride;
  int64_t kv_accum_rows;  // kv_accum applies to key rows below this only
  // launch geometry of the tensor-core kernels (filled in by their launcher)
  int tma_out;            // 1: full owner tiles leave (and the forward's dO rows enter) through shared memory + TMA
  int ntiles;             // owner tiles per sequence
  int split;              // dK/dV kernels: CTAs (one cluster) sharing an owner tile, each a slice of its streamed blocks
  int group;              // (head, batch) pairs per scheduling group, see TcCta::setup (0 on entry = chosen by the launcher)
  long long wait_budget;  // clock budget of one bounded wait (test hook instantiation only)
};

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }

template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// Learned relative position bias (fb_relpos), passed to the kernels that add it as a parameter of its own, so that the
// others keep theirs as they are.
struct RelPos {
  const void* table;  // (bucket, head), the problem's dtype
  int64_t bucket_stride, head_stride;
  int nb, side, two;  // buckets in all / per side, 1 = both sides have buckets of their own
  float* dpart;       // backward: partial table gradients [(batch, query head)][query tile][nb], or nullptr
  float* shift;       // the rows' shifts (forward: out, may be nullptr; backward: in)
  int zero_rest;      // packed problems: rows of no sequence are zeroed (FB_FLAG_ZERO_REST); tensor-core kernels: by that many CTAs at the grid's end
  uint32_t used[FB_RELPOS_MAX_BUCKETS / 32];  // bit t: some distance falls in bucket t
  int far;            // distances from here on lie in the last bucket of their side
  int starts[FB_RELPOS_MAX_BUCKETS - 1];  // side - 1 entries
  uint32_t near_words[256];  // the buckets of distances 0 .. 1023, a byte each
};
// The bucket function in shared memory: a byte per near distance (the usual case: one load), a search beyond them.
constexpr int kRelNear = 1024;
struct RelBuckets {
  uint32_t near_words[kRelNear / 4];
  int starts[FB_RELPOS_MAX_BUCKETS];
};
struct NoRel {};

// Bucket of relative position r (key - query): the number of bucket starts at or below its distance. Each bucket is one
// interval of r (r falls monotonically through the buckets of a side), so a range of positions whose ends share a
// bucket lies in it altogether.
// (its parameters by value: read once, not again behind every barrier)
struct RelFn {
  const RelBuckets* b;
  int two, far, side;
  RelFn() = default;
  __device__ __forceinline__ RelFn(const RelPos& rel, const RelBuckets& buckets) : b(&buckets), two(rel.two), far(rel.far), side(rel.side) {}
  // Without a branch, so that several look-ups overlap; only where `byte_table()`.
  __device__ __forceinline__ bool byte_table() const { return far < kRelNear; }
  __device__ __forceinline__ int near(int r) const {
    const int n = min(two ? abs(r) : max(-r, 0), far);
    return reinterpret_cast<const uint8_t*>(b->near_words)[n] + ((two && r > 0) ? side : 0);
  }
  __device__ __forceinline__ int operator()(int r) const {
    const int n = min(two ? abs(r) : max(-r, 0), far);
    int lo;
    if (n < kRelNear) {
      lo = reinterpret_cast<const uint8_t*>(b->near_words)[n];
    } else {
      lo = 0;
      int hi = side - 1;  // answer in [lo, hi]
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (b->starts[mid] <= n) lo = mid + 1;
        else hi = mid;
      }
    }
    return lo + ((two && r > 0) ? side : 0);
  }
};
// A table entry as the attention kernels use it. Entries at or below -2^100 (the lowest bfloat16 and float32 values among them) hide their
// pairs like -inf: kept as numbers they would swallow the scores of a row that sees nothing else and make its log-sum-exp
// useless for the backward.
constexpr float kRelHidden = -1.2676506002282294e30f;  // -2^100
template <typename T>
__device__ __forceinline__ float relpos_entry(const RelPos& rel, int bucket, int head) {
  const float x = to_f<T>(reinterpret_cast<const T*>(rel.table)[bucket * rel.bucket_stride + head * rel.head_stride]);
  return x <= kRelHidden ? -INFINITY : x;
}
// An entry in log2 units, as the tensor-core kernels add it: finite stays finite (3e38 log2(e) is beyond float32).
__device__ __forceinline__ float relpos_log2(float x) {
  const float y = x * 1.4426950408889634f;
  return y == INFINITY && x != INFINITY ? 3.402823466e38f : y;
}
// The shift of a row: the largest entry that its keys have. Scores are formed as c q.k + (entry - shift): the difference is exact where it
// matters, while beside an entry of 1e6 the sum would have no room for c q.k, and neither would a log-sum-exp for what the backward needs.
//
// Where no entry of the head is larger than kRelLarge the shifts are 0: there the sum is good to 2^-18, and the look-ups (they cost 4 % of a
// packed prompt's time, and 15 % of the drafted tokens') are left out.
constexpr float kRelLarge = 64.f;
__device__ __forceinline__ bool relpos_large(float x) { return fabsf(x) > kRelLarge && fabsf(x) != INFINITY; }
// Prefix maxima of a head's entries over the buckets of each side that some distance falls in, by one warp.
template <typename T>
__device__ __forceinline__ void relpos_prefix(float* pre, const RelPos& rel, int head, int lane) {
  for (int first = 0; first < rel.nb; first += rel.side) {
    float carry = -INFINITY;
    for (int t0 = 0; t0 < rel.side; t0 += 32) {
      const int t = t0 + lane, b = first + t;
      float x = -INFINITY;
      if (t < rel.side && (rel.used[b >> 5] >> (b & 31) & 1u)) x = relpos_entry<T>(rel, b, head);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x = fmaxf(x, y);
      }
      x = fmaxf(x, carry);
      if (t < rel.side) pre[b] = x;
      carry = __shfl_sync(0xffffffffu, x, 31);
    }
  }
}
// The shift of a row whose keys lie at positions lo .. hi, hi >= 0.
template <typename T>
__device__ __forceinline__ float relpos_shift(const float* pre, const RelPos& rel, const RelFn& bucket_of, int head, int lo, int hi) {
  float x = -INFINITY;
  if (!rel.two || lo <= 0) x = pre[bucket_of(min(lo, 0))];  // distances 0 .. -lo (r > 0 counts as 0 when one side has buckets)
  if (rel.two && hi > 0) {
    const int last = bucket_of(hi);
    if (lo <= 1) {
      x = fmaxf(x, pre[last]);
    } else {  // a row ahead of the first key
      for (int b = bucket_of(lo); b <= last; ++b)
        if (rel.used[b >> 5] >> (b & 31) & 1u) x = fmaxf(x, relpos_entry<T>(rel, b, head));
    }
  }
  return x == -INFINITY ? 0.f : x;
}
// Fills `b`, thread `i` of `n`. Only what the search will look at: bytes up to the first far distance.
__device__ __forceinline__ void relpos_load_buckets(RelBuckets& b, const RelPos& rel, int i, int n) {
  const int words = min(rel.far, kRelNear - 1) / 4 + 1;
  // Through generic addresses: as constant-bank reads with a different index per lane these would be served one lane at a time.
  const uint32_t* near_words = rel.near_words;
  const int* starts = rel.starts;
  asm("" : "+l"(near_words));
  asm("" : "+l"(starts));
  for (int t = i; t < words; t += n) b.near_words[t] = near_words[t];
  if (rel.far >= kRelNear)
    for (int t = i; t < rel.side - 1; t += n) b.starts[t] = starts[t];
}
// Sum of `v` over the lanes that hold the same key, for keys that form one run of neighbouring lanes each. Returns whether this lane
// is the first of its run; `v` is the run's sum there. Fixed order.
__device__ __forceinline__ bool run_sum(float& v, int key, int lane) {
  const int prev = __shfl_up_sync(0xffffffffu, key, 1);
  const bool head = lane == 0 || prev != key;
  const uint32_t behind = __ballot_sync(0xffffffffu, head) & ~((2u << lane) - 1u);  // first lanes of later runs
  const int left = (behind ? __ffs((int)behind) - 2 : 31) - lane;                   // lanes of this run behind this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float ov = __shfl_down_sync(0xffffffffu, v, o);
    if (o <= left) v += ov;
  }
  return head;
}

// Decoding against a cache (decode.cu).
struct CacheT {
  const void* ptr;
  int64_t batch_stride, row_stride, head_stride;
};
struct DecodeParams {
  int B, Hq, Hkv, G, Sq, Sk, D;
  float scale;
  CacheT q, k, v;
  const int32_t* lens;  // nullptr: Sk each
  void* out;            // contiguous (B, Sq, Hq, D)
  int splits, row_tiles;
  int cluster;          // the slices of a sequence are one thread-block cluster
  float* part;          // splits > 1: [(b, token, query head)][split][D] and their (maximum, sum)
  float2* part_ml;
};

struct SeqInfo {
  int q0, k0;    // first global row of this sequence
  int sq, sk;    // its lengths
};

__device__ __forceinline__ SeqInfo seq_info(const Params& p, int b) {
  SeqInfo s;
  if (p.cu_q) { s.q0 = p.cu_q[b]; s.sq = p.cu_q[b + 1] - s.q0; } else { s.q0 = b * p.Sq; s.sq = p.Sq; }
  if (p.cu_k) { s.k0 = p.cu_k[b]; s.sk = p.cu_k[b + 1] - s.k0; } else { s.k0 = b * p.Sk; s.sk = p.Sk; }
  return s;
}

// CTAs of a tensor-core launch that zero the rows of no sequence, behind those of the tiles.
constexpr int kRestCtas = 16;
// Zeroes the rows of `t` that belong to no sequence (before cu[0], from cu[B] on); this CTA as part `part` of `parts`.
template <typename T>
__device__ __forceinline__ void rel_zero_rest(const Params& p, const SeqT& t, const int32_t* cu, int64_t total, int heads, int part, int parts) {
  if (!t.ptr) return;
  constexpr int VEC = 16 / sizeof(T);
  const int units = p.D / VEC;
  const int64_t lead = cu[0], end = cu[p.B], rows = lead + (total - end);
  for (int64_t x = (int64_t)part * blockDim.x + threadIdx.x; x < rows * heads * units; x += (int64_t)parts * blockDim.x) {
    const int u = (int)(x % units), h = (int)(x / units % heads);
    const int64_t r = x / units / heads, row = r < lead ? r : end + r - lead;
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(t.ptr) + row * t.row_stride + (int64_t)h * t.head_stride + u * VEC) = make_uint4(0, 0, 0, 0);
  }
}
// The same as a call, for the tensor-core kernels: inlined at their entry it cost every launch 2 us (12 packed prompts of up to 2048: 197.0 us, 195.0 as a
// call, 194.8 without). The CUDA-core kernels inline it: a call costs them registers (training step B2 S200, 4 heads of 64: 163 us, 142 inlined).
template <typename T>
__device__ __noinline__ void rel_zero_rest_call(const Params& p, const SeqT& t, const int32_t* cu, int64_t total, int heads, int part, int parts) {
  rel_zero_rest<T>(p, t, cu, total, heads, part, parts);
}

// Shift of sequence-local row `row` of the segmented side (fb_problem.seg_rows / seg_shift).
__device__ __forceinline__ int seg_shift_of(const Params& p, int row) {
  int shift = 0;
  for (int t = p.seg_n - 1; t >= 0; --t)
    if (row < p.seg_rows[t]) shift = p.seg_shift[t];
  return shift;
}
// Causal masking: key j is visible to query row i (both sequence-local) iff j <= i + pair_off(p, s, i, j):
// bottom-right aligned, corrected by the shift of the segment the query (or, with key segments, the key) lies in.
__device__ __forceinline__ int pair_off(const Params& p, const SeqInfo& s, int i, int j) {
  return s.sk - s.sq + (p.seg_keys ? seg_shift_of(p, j) : -seg_shift_of(p, i));
}
// The same for a whole query row (query segments or none; kernels that own query rows do not take key segments).
__device__ __forceinline__ int causal_off(const Params& p, const SeqInfo& s, int i) {
  return s.sk - s.sq - (p.seg_keys ? 0 : seg_shift_of(p, i));
}
// First query row that sees key row j (positions grow with the row index, across the segment breaks too).
__device__ __forceinline__ int first_query_of_key(const Params& p, const SeqInfo& s, int j) {
  const int off = s.sk - s.sq;
  if (p.seg_keys) return max(0, j - (off + seg_shift_of(p, j)));
  int lo = 0;
  for (int t = 0; t < p.seg_n; ++t) {
    const int i = max(lo, j - (off - p.seg_shift[t]));
    if (i < p.seg_rows[t]) return i;
    lo = p.seg_rows[t];
  }
  return max(lo, j - off);
}

// host-side launchers (each returns the number of kernels enqueued, or a negative fb_status)
int launch_simt_fwd(const Params& p, cudaStream_t stream);
int launch_simt_bwd(const Params& p, cudaStream_t stream);
int launch_row_stats(const Params& p, cudaStream_t stream);
int launch_tc_fwd(const Params& p, cudaStream_t stream);
int launch_tc_bwd(const Params& p, cudaStream_t stream);
// the same with a relative position bias (first order only); launch_rel_reduce adds up the partial table gradients of
// `ntiles` query tiles per (batch, head)
int launch_simt_fwd_rel(const Params& p, const RelPos& rel, cudaStream_t stream);
int launch_simt_bwd_rel(const Params& p, const RelPos& rel, cudaStream_t stream);
int launch_tc_fwd_rel(const Params& p, const RelPos& rel, cudaStream_t stream);
int launch_tc_bwd_rel(const Params& p, const RelPos& rel, cudaStream_t stream);
int launch_rel_reduce(int dtype, const float* part, int batch, int heads, int ntiles, int nb, void* dtable, int64_t bucket_stride,
                      int64_t head_stride, cudaStream_t stream);
int launch_relpos_fill(int dtype, const RelPos& rel, int heads, int sq, int sk, void* out, cudaStream_t stream);
int launch_relpos_grad(int dtype, const RelPos& rel, int heads, int sq, int sk, const void* grad, void* dtable, int64_t bucket_stride,
                       int64_t head_stride, cudaStream_t stream);
int64_t relpos_bias_parts(int dtype, int heads, int sq, int sk);  // partial table gradients per head of launch_relpos_grad
struct DecodeShape {
  int splits;    // slices of a sequence's keys
  bool cluster;  // they are one cluster (and need no workspace)
};
DecodeShape decode_shape(int batch, int heads_kv, int rows, int seqlen_k);
constexpr int kDecodeMaxTable = 4096;  // query heads per kv head x buckets
int launch_decode(int dtype, DecodeParams& p, RelPos& rel, cudaStream_t stream);
constexpr int kTcOwnerRows = 128, kSimtOwnerRows = 16;  // query rows per partial table gradient
int launch_tc_fwd_wait_hook(const Params& p, cudaStream_t stream);  // test instantiation, see fb_debug_wait_timeout
int launch_sum_slots(const float* slots, int n_slots, int64_t slot_stride, int64_t count, int64_t period, const int64_t* valid, float* out,
                     cudaStream_t stream);
int read_profile(long long* out16);

// shared host helpers (api.cu)
int check_problem(const fb_problem& pr);
int record_cuda(cudaError_t e);        // remembers the error text for fb_last_cuda_error(); returns FB_ERR_CUDA
int device_setup(int** status_ptr);    // architecture check + device address of the status word (cached per device)
void set_launch_count(int n);          // what fb_last_launch_count() reports for this thread

}  // namespace fb
