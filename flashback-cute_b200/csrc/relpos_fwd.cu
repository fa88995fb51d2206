// Forward of attention with a learned relative position bias on the tensor cores (16-bit types).
//
// Online softmax, in log2 units: V_ij = c log2(e) (Q K^T)_ij + log2(e) (T[bucket] - shift_i), P = 2^(V - m), O = P V / l (the shift: fb_params.h).
//
// What bounds it: per 128 x 64 scores, S = Q K^T and O += P V keep the tensor pipe busy for 384 + 256 clk (head_dim 128; 192 +
// 128 at 64), the 8192 exponentials the special-function units for 512 clk, and the softmax warps need about 1100 clk from
// a tile's scores to its P, plus several hundred clk for every hand-over. So a CTA owns TWO tiles of 128 query rows with
// two buffers of scores each: while the warpgroup of a tile works on one block of 64 keys, the tensor pipe computes its next one and
// the other tile's. One thread owns one query row (TMEM lane) and has 64 scores at a time in registers: row maximum and sum need no
// exchange between threads. K and V blocks are shared by the two tiles.
//
//   warp 0 (one lane)   TMA: Q tiles once, K and V blocks through three stages
//   warp 1 (one lane)   every tcgen05.mma: PV(t, j) and, right behind it, S(t, j + 2) into the buffer it read, for the tiles t in turn
//   warps 2, 3          biases of the coming blocks' positions into shared memory; zeros behind a sequence's last key
//   warps 4-7, 8-11     softmax, rescaling and epilogue of tile 0 and tile 1
//
// TMEM (512 columns): per tile 2 x 64 columns of scores, overwritten by P (16 bit) as it is computed, and head_dim of output.
//
// The bias. Blocks whose 128 x 64 positions share a bucket (all but a few around the diagonal) take one number, folded into the
// exponent's FMA. In the others every pair reads its own: entry (key column - row) of 319 staged values. A warp's lanes
// read neighbouring entries; four copies, each shifted by one entry, let every thread fetch four columns with one
// 16-byte load whatever its row.
//
// Measured: non-causal B2 Hq16 Hkv4 S4096 bf16, 281 us at head_dim 128 (978 TFLOP/s, 0.59 of the measured cuBLAS burst rate) and 253 at 64;
// causal at 128, 146 us (300, 264 and 160 within a training step, with the outputs that the backward wants). Per block the softmax warps wait 400 of 1900 clk for scores, spend 350 on the maximum and 800 on exponentials.
// Tried (non-causal B2 Hq16 Hkv4 S4096 D128, at a clock where this version takes 317): blocks of 128 keys with one buffer of scores per tile 340 us (a tile waits 1550 of 3800 clk
// for its scores); the same with the exponentials started on the maximum known so far, 348 us; two CTAs per SM with one
// tile each and two warps per row, 372 us.
#include "fb_params.h"
#include "ptx_sm100.cuh"
#include "tc_host.h"

#include <cuda.h>
#include <mutex>
#include <type_traits>

namespace fb {
namespace {

using namespace ptx;

constexpr int BM = 128;  // query rows per tile = TMEM lanes
constexpr int BN = 64;   // keys per block
constexpr int kRoleThreads = 128, kSoftThreads = 256, kThreads = kRoleThreads + kSoftThreads;
// The role warps give registers back, the softmax warpgroups take them: no more than the launch left (see tc_kernels.cu).
constexpr int kLaunchRegs = 168, kRoleRegs = 104, kSoftRegs = 200;
static_assert(kRoleThreads * (kLaunchRegs - kRoleRegs) >= kSoftThreads * (kSoftRegs - kLaunchRegs), "registers that nobody releases");
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRescaleThreshold = 8.f;  // log2 units: rescale O only when the row maximum grew by more than 2^8
constexpr int kSpan = 2 * BM + BN;        // positions of a block seen from both tiles (one more than there are)
constexpr int kCopyStride = kSpan + 8;    // floats between the shifted copies: 8 banks apart

constexpr int KS = 3;                     // stages of K and of V
enum {
  BAR_Q = 0,            // + tile
  BAR_K_FULL = 2,       // + stage
  BAR_K_EMPTY = 5,
  BAR_V_FULL = 8,
  BAR_V_EMPTY = 11,
  BAR_S_FULL = 14,      // + 2 * tile + slot: scores complete and biases staged
  BAR_P_FULL = 18,      // + 2 * tile + slot
  BAR_ST_EMPTY = 22,    // + 2 * tile + slot: biases read
  BAR_PV_DONE = 26,     // + tile
  BAR_O_DONE = 28,      // + tile
  BAR_TAIL = 30,        // keys behind the sequence zeroed in the last V block
  BAR_COUNT = 31
};
// Bytes behind the tiles
enum {
  M_SLOT = 256,                       // TMEM address, abort flag
  M_UNI = M_SLOT + 16,                // [2 buffers][2 tiles] kinds of blocks, then the same of biases
  M_LARGE = M_UNI + 32,               // 1: the rows have shifts
  M_TAB = M_UNI + 32 + 208,           // 512: table column in log2 units
  M_PRE = M_TAB + FB_RELPOS_MAX_BUCKETS * 4,      // prefix maxima of the entries (relpos_prefix)
  M_BUCKETS = M_PRE + FB_RELPOS_MAX_BUCKETS * 4,  // RelBuckets
  M_BIAS = M_BUCKETS + (int)sizeof(RelBuckets),   // [2][4][kCopyStride]
  M_SHIFT = M_BIAS + 2 * 4 * kCopyStride * 4,     // [2 tiles][BM] the rows' shifts, negated, in log2 units (each read by the thread that wrote it)
  M_BYTES = M_SHIFT + 2 * BM * 4
};
static_assert(M_TAB == 512 && M_BIAS % 16 == 0, "layout");

template <int D>
struct FwdCfg {
  static constexpr int qTile = BM * D * 2, kvTile = BN * D * 2;
  static constexpr int kOff = 2 * qTile, vOff = kOff + KS * kvTile;
  static constexpr int tileBytes = vOff + KS * kvTile;
  // at least half of shared memory: TMEM takes one CTA per SM
  static constexpr int smemBytes = tileBytes + M_BYTES < 120 * 1024 ? 120 * 1024 : tileBytes + M_BYTES;
  static_assert(smemBytes <= 232448, "shared memory");
  static constexpr int tmemCols = 512;  // 2 x (2 x 64 scores + D): 384 at head_dim 64, and allocations are powers of two
};

// Kinds of blocks: one bias for all pairs; the rows have shifts
enum { BLK_SHIFTED = 1, BLK_ONE = 2 };

struct FwdMaps {
  CUtensorMap q, k, v, o, lo;
};

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t u);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u)); }
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }

// The two parts of the shifts as calls: heads without large entries jump over them, and code in their place cost every CTA's set-up and epilogue.
template <typename T>
__device__ __noinline__ void prefix_call(float* pre, const RelPos& rel, int head, int lane) { relpos_prefix<T>(pre, rel, head, lane); }
template <typename T>
__device__ __noinline__ float shift_call(const float* pre, const RelBuckets& buckets, const RelPos& rel, int head, int lo, int hi) {
  return relpos_shift<T>(pre, rel, RelFn(rel, buckets), head, lo, hi);
}

template <typename T, int D>
struct RelFwd {
  using C = FwdCfg<D>;
  static constexpr int fmt = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  static constexpr uint32_t idesc_s = make_idesc(fmt, BM, BN, 0, 0);
  static constexpr uint32_t idesc_o = make_idesc(fmt, BM, D, 0, 1);

  const FwdMaps& maps;
  const Params& p;
  const RelPos& rel;
  uint8_t* const smem;
  uint8_t* misc;
  uint32_t sbase, bar0, tmem_base;
  volatile int* abort_flag;
  int warp, lane, head, hk, off, r0, n_it;
  int n_of[2];  // blocks of the two tiles (0: the tile lies behind its sequence)
  SeqInfo si;

  __device__ __forceinline__ RelFwd(const FwdMaps& m, const Params& p_, const RelPos& r, uint8_t* s) : maps(m), p(p_), rel(r), smem(s) {}

  __device__ __forceinline__ uint32_t bar(int i) const { return bar0 + 8 * i; }
  __device__ __forceinline__ bool wait1(int b, int parity) const { return mbar_wait(bar(b), parity, abort_flag); }
  __device__ __forceinline__ void warp_wait(int b, int parity) const {
    if (lane == 0) wait1(b, parity);
    __syncwarp();
  }
  __device__ __forceinline__ bool aborted() const { return *abort_flag != 0; }
  __device__ __forceinline__ uint32_t q_addr(int t) const { return sbase + t * C::qTile; }
  __device__ __forceinline__ uint32_t k_addr(int s) const { return sbase + C::kOff + s * C::kvTile; }
  __device__ __forceinline__ uint32_t v_addr(int s) const { return sbase + C::vOff + s * C::kvTile; }
  __device__ __forceinline__ uint32_t s_cols(int t, int slot) const { return tmem_base + (2 * t + slot) * BN; }
  __device__ __forceinline__ uint32_t o_cols(int t) const { return tmem_base + 4 * BN + t * D; }

  // False: nothing to do (the whole CTA leaves together).
  __device__ __forceinline__ bool setup() {
    sbase = smem_u32(smem);
    if (sbase & 1023u) {
      if (threadIdx.x == 0) atomicOr(p.status, 0x100);
      return false;
    }
    if (*reinterpret_cast<volatile int*>(p.status) != 0) return false;  // see tc_kernels.cu
    misc = smem + C::tileBytes;
    bar0 = sbase + C::tileBytes;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + M_SLOT);
    abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    warp = threadIdx.x >> 5;
    lane = threadIdx.x & 31;
    // (head, batch) pairs in groups, heaviest tiles of a group first: see tc_kernels.cu
    const uint32_t lin = blockIdx.x, pairs = (uint32_t)p.Hq * (uint32_t)p.B, gsz = (uint32_t)p.group;
    const uint32_t grp = lin / (gsz * (uint32_t)p.ntiles), rem = lin - grp * gsz * (uint32_t)p.ntiles;
    const uint32_t in_grp = min(gsz, pairs - grp * gsz);
    const int tidx = (int)(rem / in_grp);
    const uint32_t pair = grp * gsz + rem % in_grp;
    head = (int)(pair % (uint32_t)p.Hq);
    hk = head / (p.Hq / p.Hkv);
    if (p.cu_q) grid_dependency_wait();
    si = seq_info(p, (int)(pair / (uint32_t)p.Hq));
    r0 = (p.causal ? p.ntiles - 1 - tidx : tidx) * (2 * BM);
    if (r0 >= si.sq) return false;
    off = si.sk - si.sq;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      int kmax = si.sk;
      if (p.causal) kmax = max(0, min(si.sk, r0 + (t + 1) * BM + off));
      n_of[t] = r0 + t * BM < si.sq ? (kmax + BN - 1) / BN : 0;
    }
    n_it = max(n_of[0], n_of[1]);

    if (threadIdx.x == 0) {
      for (int i = 0; i < BAR_COUNT; ++i) {
        uint32_t count = 1;
        if (i >= BAR_S_FULL && i < BAR_S_FULL + 4) count = 3;    // the MMAs and both bias warps
        if (i >= BAR_P_FULL && i < BAR_ST_EMPTY + 4) count = 4;  // a tile's softmax warps
        mbar_init(bar(i), count);
      }
      *abort_flag = 0;
      fence_barrier_init();
      if (n_it > 0) {
        grid_dependency_wait();
        prefetch_tmap(&maps.q); prefetch_tmap(&maps.k); prefetch_tmap(&maps.v);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (n_of[t] == 0) continue;
          mbar_expect_tx(bar(BAR_Q + t), C::qTile);
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_3d(q_addr(t) + c * (BM * 128), &maps.q, bar(BAR_Q + t), c * 64, si.q0 + r0 + t * BM, head);
        }
      }
    }
    if (warp == 1) {
      tmem_alloc(smem_u32(tmem_slot), C::tmemCols);
      tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    tmem_base = *tmem_slot;
    grid_launch_dependents();
    grid_dependency_wait();
    return true;
  }

  __device__ __forceinline__ void producer() {
    for (int it = 0; it < n_it; ++it) {
      const int s = it % KS, ph = ((it / KS) & 1) ^ 1, row = si.k0 + it * BN;
      if (!wait1(BAR_K_EMPTY + s, ph)) return;
      mbar_expect_tx(bar(BAR_K_FULL + s), C::kvTile);
#pragma unroll
      for (int c = 0; c < D / 64; ++c) tma_load_3d(k_addr(s) + c * (BN * 128), &maps.k, bar(BAR_K_FULL + s), c * 64, row, hk);
      if (!wait1(BAR_V_EMPTY + s, ph)) return;
      mbar_expect_tx(bar(BAR_V_FULL + s), C::kvTile);
#pragma unroll
      for (int c = 0; c < D / 64; ++c) tma_load_3d(v_addr(s) + c * (BN * 128), &maps.v, bar(BAR_V_FULL + s), c * 64, row, hk);
    }
  }

  // The last block reaches past the sequence's keys. Their P is 0, but 0 x Inf or 0 x NaN is NaN: whatever lies there (the next
  // sequence, rows nobody filled) is zeroed in shared memory before the second product reads it.
  __device__ __forceinline__ bool has_tail() const { return n_it * BN > si.sk; }

  __device__ __forceinline__ void issuer() {
    bool live = true;
    const uint32_t kd = smem_desc_lo(k_addr(0), 16), vd = smem_desc_lo(v_addr(0), BN * 128);
    uint32_t qd[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) qd[t] = smem_desc_lo(q_addr(t), 16);
    auto issue_s = [&](int t, int it) {
      const uint32_t o = (uint32_t)(((it % KS) * C::kvTile) >> 4);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        mma_ss(s_cols(t, it & 1), qd[t] + (uint32_t)(((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4),
               kd + o + (uint32_t)(((kk >> 2) * (BN * 128) + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
      mma_commit(bar(BAR_S_FULL + 2 * t + (it & 1)));
    };
    auto issue_o = [&](int t, int it) {
      const uint32_t o = (uint32_t)(((it % KS) * C::kvTile) >> 4);
#pragma unroll
      for (int kk = 0; kk < BN / 16; ++kk)
        mma_ts(o_cols(t), s_cols(t, it & 1) + kk * 16, vd + o + (uint32_t)((kk * 16 * 128) >> 4), idesc_o, (it > 0 || kk > 0) ? 1u : 0u);
      mma_commit(bar((it == n_of[t] - 1 ? BAR_O_DONE : BAR_PV_DONE) + t));
    };
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      if (it >= n_it) break;
      live = wait1(BAR_K_FULL + it, 0) && live;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (it >= n_of[t]) continue;
        if (it == 0) live = wait1(BAR_Q + t, 0) && live;
        if (!live) return;
        tc_fence_after();
        issue_s(t, it);
      }
      mma_commit(bar(BAR_K_EMPTY + it));
    }
    for (int it = 0; it < n_it; ++it) {
      const int s = it % KS, s2 = (it + 2) % KS;
      live = wait1(BAR_V_FULL + s, (it / KS) & 1) && live;
      if (it == n_it - 1 && has_tail()) live = wait1(BAR_TAIL, 0) && live;
      if (it + 2 < n_it) live = wait1(BAR_K_FULL + s2, ((it + 2) / KS) & 1) && live;
      if (!live) return;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (it >= n_of[t]) continue;
        if (!wait1(BAR_P_FULL + 2 * t + (it & 1), (it >> 1) & 1)) return;
        tc_fence_after();
        issue_o(t, it);
        if (it + 2 < n_of[t]) issue_s(t, it + 2);  // behind PV in the pipe: it overwrites the P that PV reads
      }
      mma_commit(bar(BAR_V_EMPTY + s));
      if (it + 2 < n_it) mma_commit(bar(BAR_K_EMPTY + s2));
    }
  }

  // Warps 2 and 3 (w = 0, 1): biases of block `it` into buffer it % 2. Entry u: key column - row = u - (2 BM - 1).
  __device__ __forceinline__ void bias_warp(int w) {
    float* tab = reinterpret_cast<float*>(misc + M_TAB);
    RelBuckets& buckets = *reinterpret_cast<RelBuckets*>(misc + M_BUCKETS);
    bool large = false;
    for (int t = w * 32 + lane; t < rel.nb; t += 64) {
      const float x = relpos_entry<T>(rel, t, head);
      large = large || relpos_large(x);
      tab[t] = relpos_log2(x);
    }
    relpos_load_buckets(buckets, rel, w * 32 + lane, 64);
    large = named_barrier_or(1, 64, large);
    if (w == 1) {
      if (large) prefix_call<T>(reinterpret_cast<float*>(misc + M_PRE), rel, head, lane);
      if (lane == 0) *reinterpret_cast<int*>(misc + M_LARGE) = large;
    }
    const int shifted = large ? BLK_SHIFTED : 0;
    const RelFn bucket_of(rel, buckets);
    for (int it = 0; it < n_it; ++it) {
      const int buf = it & 1;
      // looked up into registers before the wait for the buffer (see rel_look_up in tc_kernels.cu)
      const int base = it * BN - r0 - off - (2 * BM - 1);
      auto bucket_at = [&](int u) { return bucket_of(base + u); };
      // first and last positions of tile 1 (u = 0 and BM + BN - 2), tile 0 (BM and 2 BM + BN - 2)
      const int mine = bucket_at((lane & 1 ? BM + BN - 2 : 0) + (lane & 2 ? 0 : BM));
      const int f0 = __shfl_sync(0xffffffffu, mine, 0), l0 = __shfl_sync(0xffffffffu, mine, 1);
      const int f1 = __shfl_sync(0xffffffffu, mine, 2), l1 = __shfl_sync(0xffffffffu, mine, 3);
      // (with a negative or zero scale the row maximum does not follow the scores': such calls take the general path)
      const bool uni0 = f0 == l0 && p.scale > 0.f, uni1 = f1 == l1 && p.scale > 0.f;
      const float v0 = tab[f0], v1 = tab[f1];
      float bias[kSpan / 64];
      if (!(uni0 && uni1)) {
        const int r = base + w * (kSpan / 2) + lane;
        if (bucket_of.byte_table()) {
#pragma unroll
          for (int i = 0; i < kSpan / 64; ++i) bias[i] = tab[bucket_of.near(r + i * 32)];
        } else {
#pragma unroll
          for (int i = 0; i < kSpan / 64; ++i) bias[i] = tab[bucket_of(r + i * 32)];
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (it >= 2 && it - 2 < n_of[t]) warp_wait(BAR_ST_EMPTY + 2 * t + buf, ((it >> 1) & 1) ^ 1);  // (then their barrier's phase is over too)
      if (aborted()) return;
      if (w == 0 && lane == 0) {
        int* flag = reinterpret_cast<int*>(misc + M_UNI) + 2 * buf;
        float* val = reinterpret_cast<float*>(misc + M_UNI + 16) + 2 * buf;
        flag[0] = (uni0 ? BLK_ONE : 0) | shifted; flag[1] = (uni1 ? BLK_ONE : 0) | shifted;
        val[0] = v0; val[1] = v1;
      }
      if (!(uni0 && uni1)) {
        float* arr = reinterpret_cast<float*>(misc + M_BIAS) + buf * 4 * kCopyStride;
#pragma unroll
        for (int i = 0; i < kSpan / 64; ++i) {
          const int u = w * (kSpan / 2) + i * 32 + lane;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (u >= k) arr[k * kCopyStride + u - k] = bias[i];
        }
      }
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (it < n_of[t]) mbar_arrive(bar(BAR_S_FULL + 2 * t + buf));
        }
      }
      __syncwarp();
    }
  }
  // Warp 3 as well: zeros behind the last key (see has_tail).
  __device__ __forceinline__ void zero_tail() {
    const int it = n_it - 1, s = it % KS;
    // Parities repeat: the stage's previous phase (block it - KS) has to be over. It is once S(it - 1), which was issued behind
    // PV(it - 3), is complete; that barrier has no phase behind the one waited for, and block it - 3 of its slot has been read.
    static_assert(KS == 3, "the parity of the last V stage");
    if (it >= KS) warp_wait(BAR_S_FULL + 2 * (n_of[1] == n_it ? 1 : 0) + ((it - 1) & 1), ((it - 1) >> 1) & 1);
    warp_wait(BAR_V_FULL + s, (it / KS) & 1);
    if (aborted()) return;
    const int first = si.sk - it * BN;  // rows first .. BN - 1 of the block
    uint8_t* v = smem + C::vOff + s * C::kvTile;
    for (int x = lane; x < (BN - first) * (D / 8); x += 32) {
      const int r = first + x / (D / 8), u = x % (D / 8);  // whole rows: the swizzle only permutes units inside a row's 128 bytes
      *reinterpret_cast<uint4*>(v + (u >> 3) * (BN * 128) + r * 128 + (u & 7) * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(BAR_TAIL));
  }

  // ---- softmax and epilogue of tile t: one thread per row ----
  __device__ __forceinline__ void softmax(int t) {
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const int orow = r0 + t * BM + row;
    const bool row_ok = orow < si.sq;
    const float scale2 = p.scale * kLog2e;
    const float2 sc2 = make_float2(scale2, scale2);
    const int n = t ? n_of[1] : n_of[0];  // (a dynamic index would put the array into local memory)
    float m = -INFINITY, l = 0.f;
    float* const nshift2 = reinterpret_cast<float*>(misc + M_SHIFT) + t * BM + row;
    // this row's staged biases: entry a + column, read 4 at a time from the copy that is aligned for it
    const int a = 2 * BM - 1 - (t * BM + row);
    const float* bias_row = reinterpret_cast<const float*>(misc + M_BIAS) + (a & 3) * kCopyStride + (a & ~3);

    for (int it = 0; it < n; ++it) {
      const int buf = it & 1, c0 = it * BN;
      int cmax = si.sk - 1 - c0;
      bool need_mask = c0 + BN > si.sk;
      if (p.causal) {
        need_mask = need_mask || c0 + BN - 1 > r0 + t * BM + off;
        cmax = min(cmax, orow + off - c0);
      }
      warp_wait(BAR_S_FULL + 2 * t + buf, (it >> 1) & 1);
      tc_fence_after();
      uint32_t raw[BN / 32][32];
#pragma unroll
      for (int q = 0; q < BN / 32; ++q) tmem_ld32(s_cols(t, buf) + lane_off + q * 32, raw[q]);
      const int kind = reinterpret_cast<const int*>(misc + M_UNI)[2 * buf + t];
      const bool uni = (kind & BLK_ONE) != 0;
      float ub = reinterpret_cast<const float*>(misc + M_UNI + 16)[2 * buf + t];
      if (kind & BLK_SHIFTED) {
        if (it == 0) *nshift2 = -relpos_log2(row_shift(orow));  // (both bias warps' tables are complete when they hand over block 0)
        ub += *nshift2;
      }
      tmem_ld_wait();
      float v[BN], mx;
#pragma unroll
      for (int c = 0; c < BN; ++c) v[c] = __uint_as_float(raw[c / 32][c % 32]);
      const bool fold = uni && !need_mask;  // scale and bias folded into the exponent
      if (fold) {
        mx = fmaf(row_max(v), scale2, ub);
      } else if (uni) {
#pragma unroll
        for (int c = 0; c < BN; ++c) v[c] = c > cmax ? -INFINITY : fmaf(v[c], scale2, ub);
        mx = row_max(v);
      } else {
        const float4* b4 = reinterpret_cast<const float4*>(bias_row + buf * 4 * kCopyStride);
        auto add_bias = [&](auto shifted) {
          const float2 ns2 = decltype(shifted)::value ? make_float2(*nshift2, *nshift2) : make_float2(0.f, 0.f);
#pragma unroll
          for (int c = 0; c < BN / 4; ++c) {
            const float4 b = b4[c];
            float2 lo = make_float2(b.x, b.y), hi = make_float2(b.z, b.w);
            if (decltype(shifted)::value) { lo = __fadd2_rn(lo, ns2); hi = __fadd2_rn(hi, ns2); }
            const float2 x = __ffma2_rn(make_float2(v[4 * c], v[4 * c + 1]), sc2, lo);
            const float2 y = __ffma2_rn(make_float2(v[4 * c + 2], v[4 * c + 3]), sc2, hi);
            v[4 * c] = x.x; v[4 * c + 1] = x.y; v[4 * c + 2] = y.x; v[4 * c + 3] = y.y;
          }
        };
        if (kind & BLK_SHIFTED) add_bias(std::true_type{});
        else add_bias(std::false_type{});
        if (need_mask) {
#pragma unroll
          for (int c = 0; c < BN; ++c) if (c > cmax) v[c] = -INFINITY;
        }
        mx = row_max(v);
      }
      const float m_new = fmaxf(m, mx);
      const bool grow = m_new - m > kRescaleThreshold;  // false when both are -inf (NaN)
      if (__any_sync(0xffffffffu, grow)) {
        const float alpha = grow ? (m == -INFINITY ? 0.f : ex2(m - m_new)) : 1.f;
        if (grow) { m = m_new; l *= alpha; }
        if (it > 0) {
          warp_wait(BAR_PV_DONE + t, (it - 1) & 1);  // (PV(it - 2) is complete: S(it) was issued behind it)
          tc_fence_after();
#pragma unroll 1
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            tmem_ld32(o_cols(t) + lane_off + q * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
            tmem_st32(o_cols(t) + lane_off + q * 32, o);
          }
        }
      }
      const float moff = m == -INFINITY ? 0.f : m;
      const float2 mul = fold ? sc2 : make_float2(1.f, 1.f);
      const float2 add = fold ? make_float2(ub - moff, ub - moff) : make_float2(-moff, -moff);
      // The two tiles' exponentials alternate: the warps of a TMEM lane quadrant share a scheduler and its special-function unit.
      const int pairs = min(n_of[0], n_of[1]);
      if (it < pairs && (t == 1 || it > 0)) named_barrier_sync(4 + 4 * t + (warp & 3), 64);
      float2 ls[4] = {};
      // 16 keys = one k-step of PV: their 8 packed columns go back over the first 8 of the 16 score columns they came from
#pragma unroll
      for (int h = 0; h < BN / 16; ++h) {
        uint32_t pk[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float2 e = __ffma2_rn(make_float2(v[h * 16 + 2 * c], v[h * 16 + 2 * c + 1]), mul, add);
          const float2 x = make_float2(ex2(e.x), ex2(e.y));
          ls[c & 3] = __fadd2_rn(ls[c & 3], x);
          pk[c] = pack2<T>(x.x, x.y);
        }
        tmem_st8(s_cols(t, buf) + lane_off + h * 16, pk);
      }
      if (it < pairs && (t == 0 || it + 1 < pairs)) named_barrier_arrive(8 - 4 * t + (warp & 3), 64);
      const float2 sum = __fadd2_rn(__fadd2_rn(ls[0], ls[1]), __fadd2_rn(ls[2], ls[3]));
      l += sum.x + sum.y;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(BAR_P_FULL + 2 * t + buf));
        mbar_arrive(bar(BAR_ST_EMPTY + 2 * t + buf));
      }
    }
    if (r0 + t * BM >= si.sq) return;  // a tile behind its sequence
    if (n > 0) {
      warp_wait(BAR_O_DONE + t, 0);
      tc_fence_after();
    }
    // ---- epilogue: O / l; the tile's Q buffer is free (every product that read it is complete) ----
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const bool staged = r0 + (t + 1) * BM <= si.sq;
    const int64_t grow_ = si.q0 + orow;
    if (p.lse && row_ok) {
      const float lse = l > 0.f ? m * kLn2 + logf(l) : -INFINITY, shift = n > 0 ? row_shift(orow) : 0.f;  // less the shift
      p.lse[(int64_t)head * p.Tq + grow_] = rel.shift ? lse : lse + shift;
      if (rel.shift) rel.shift[(int64_t)head * p.Tq + grow_] = shift;
    }
    write_out(t, row, lane_off, inv, staged, row_ok, grow_, n > 0, false);
    if (p.od.ptr) write_out(t, row, lane_off, inv, staged, row_ok, grow_, n > 0, true);
    tc_fence_before();
  }
  // The shift of query row `i` of the sequence (0 for a row behind it).
  __device__ __forceinline__ float row_shift(int i) const {
    if (*reinterpret_cast<const int*>(misc + M_LARGE) == 0 || i >= si.sq || (p.causal && i + off < 0)) return 0.f;
    return shift_call<T>(reinterpret_cast<const float*>(misc + M_PRE), *reinterpret_cast<const RelBuckets*>(misc + M_BUCKETS), rel, head,
                         -(i + off), p.causal ? 0 : si.sk - 1 - (i + off));
  }
  __device__ __forceinline__ static float row_max(const float (&v)[BN]) {
    float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int c = 4; c < BN; ++c) mx[c & 3] = fmaxf(mx[c & 3], v[c]);
    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
  }
  // low: what rounding O to 16 bits left out, rounded to 16 bits itself (the backward forms rowsum(dO O) from both)
  __device__ __forceinline__ void write_out(int t, int row, uint32_t lane_off, float inv, bool staged, bool row_ok, int64_t grow_, bool any, bool low) {
    const SeqT& dst = low ? p.od : p.o;
    uint8_t* tile = smem + t * C::qTile;
    T* rowp = reinterpret_cast<T*>(dst.ptr) + (int64_t)head * dst.head_stride + grow_ * dst.row_stride;
    if (low && staged) {  // the bulk store of O still reads the buffer
      if ((threadIdx.x & 127) == 0) bulk_wait_group_read0();
      named_barrier_sync(2 + t, 128);
    }
#pragma unroll 1
    for (int q = 0; q < D / 32; ++q) {
      uint32_t o[32];
      if (any) {
        tmem_ld32(o_cols(t) + lane_off + q * 32, o);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] = 0u;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __uint_as_float(o[8 * i + 2 * e]) * inv, y = __uint_as_float(o[8 * i + 2 * e + 1]) * inv;
          w[e] = pack2<T>(x, y);
          if (low) {
            const float2 r = unpack2<T>(w[e]);
            w[e] = pack2<T>(x - r.x, y - r.y);
          }
        }
        const uint4 u = make_uint4(w[0], w[1], w[2], w[3]);
        if (staged) *reinterpret_cast<uint4*>(tile + (q >> 1) * (BM * 128) + row * 128 + ((((q & 1) * 4 + i) ^ (row & 7)) << 4)) = u;
        else if (row_ok) *reinterpret_cast<uint4*>(rowp + q * 32 + i * 8) = u;
      }
    }
    if (staged) {
      fence_proxy_async_smem();
      named_barrier_sync(2 + t, 128);
      if ((threadIdx.x & 127) == 0) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) tma_store_3d(low ? &maps.lo : &maps.o, q_addr(t) + c * (BM * 128), c * 64, si.q0 + r0 + t * BM, head);
        bulk_commit_group();
        bulk_wait_group_read0();  // shared memory must outlive the reads
      }
    }
  }

  __device__ __forceinline__ void run_role() {
    if (warp < 4) {
      reg_dealloc<kRoleRegs>();
      if (n_it == 0) return;
      if (warp == 0) {
        if (elect_one()) producer();
      } else if (warp == 1) {
        if (elect_one()) issuer();
      } else {
        bias_warp(warp - 2);
        if (warp == 3 && has_tail() && !aborted()) zero_tail();
      }
    } else {
      reg_alloc<kSoftRegs>();
      softmax((warp >> 2) - 1);
    }
  }

  __device__ __forceinline__ void teardown() {
    __syncwarp();
    __syncthreads();
    if (*abort_flag) {
      if (threadIdx.x == 0) atomicOr(p.status, 1);
      for (int i = 0; i < 64; ++i) __nanosleep(20000);  // copies and products in flight land before anything is released
      __syncthreads();
    }
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem_base, C::tmemCols);
    }
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
relpos_fwd_kernel(const __grid_constant__ FwdMaps maps, const __grid_constant__ Params p, const __grid_constant__ RelPos rel) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if (rel.zero_rest > 0 && blockIdx.x >= gridDim.x - (unsigned)rel.zero_rest) {
    grid_dependency_wait();
    rel_zero_rest_call<T>(p, p.o, p.cu_q, p.Tq, p.Hq, (int)(gridDim.x - 1 - blockIdx.x), rel.zero_rest);
    return;
  }
  RelFwd<T, D> cta(maps, p, rel, smem);
  if (!cta.setup()) return;
  cta.run_role();
  cta.teardown();
}

template <typename T, int D>
int launch_typed(const Params& p_in, const RelPos& rel, cudaStream_t s) {
  using C = FwdCfg<D>;
  Params p = p_in;
  FwdMaps maps;
  int r;
  if ((r = tc_tensor_map(&maps.q, p.q, p.dtype, D, p.Tq, p.Hq, BM))) return r;
  if ((r = tc_tensor_map(&maps.k, p.k, p.dtype, D, p.Tk, p.Hkv, BN))) return r;
  if ((r = tc_tensor_map(&maps.v, p.v, p.dtype, D, p.Tk, p.Hkv, BN))) return r;
  if ((r = tc_tensor_map(&maps.o, p.o, p.dtype, D, p.Tq, p.Hq, BM))) return r;
  if ((r = tc_tensor_map(&maps.lo, p.od, p.dtype, D, p.Tq, p.Hq, BM))) return r;
  auto kern = relpos_fwd_kernel<T, D>;
  int sms = 0;
  if ((r = tc_prepare_launch(reinterpret_cast<const void*>(kern), C::smemBytes, &sms))) return r;
  p.ntiles = (p.Sq + 2 * BM - 1) / (2 * BM);
  p.group = tc_choose_group(p, false, p.ntiles, sms);
  const long long ctas = (long long)p.ntiles * p.Hq * p.B;
  RelPos bias = rel;
  bias.zero_rest = rel.zero_rest ? kRestCtas : 0;
  if (ctas <= 0 || ctas + bias.zero_rest > 0x7fffffffll) return FB_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctas + bias.zero_rest), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = C::smemBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, maps, p, bias) == cudaSuccess ? 1 : FB_ERR_CUDA;
}

}  // namespace

int launch_tc_fwd_rel(const Params& p, const RelPos& rel, cudaStream_t s) {
  if (p.dtype == FB_BF16) return p.D == 64 ? launch_typed<__nv_bfloat16, 64>(p, rel, s) : launch_typed<__nv_bfloat16, 128>(p, rel, s);
  return p.D == 64 ? launch_typed<__half, 64>(p, rel, s) : launch_typed<__half, 128>(p, rel, s);
}

}  // namespace fb
