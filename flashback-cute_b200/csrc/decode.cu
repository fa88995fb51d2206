// Attention of a few new tokens per sequence against a cache of keys and values, with a learned relative position bias.
//
// Bound by HBM: every key and value row up to the sequence's length is read once, 4 D bytes for the 4 rows D flops that the
// rows = (new tokens) x (query heads per kv head) sharing them need. So the rows of a kv head form ONE 16-row operand (two for
// more rows) of warp-level MMAs, and the kernel is built around keeping loads in flight:
//
//   * a CTA of 4 warps (8 in a cluster) takes a slice of one (sequence, kv head)'s keys; every warp is a flash-attention of its own over every
//     4th (8th) group of 16 keys (own running maximum, sum and accumulator; own shared-memory stages filled by cp.async), so nothing in
//     the main loop waits for another warp;
//   * the slices divide the sequence's OWN length, so ragged batches stay balanced. For small batches over short caches (decode_shape) they are one
//     thread-block cluster: its CTAs leave their partial results (float32, unnormalised, with maximum and sum) in shared memory and join them
//     through distributed shared memory, each a part of the rows. Otherwise they go through a workspace and a second kernel. Fixed
//     order either way.
//
// Measured: 48 sequences of up to 8192 keys, 32 / 8 heads of 128, bf16 (897 MB): 139 + 5 us, 150 us a call, 6.0 TB/s, 91 % of the measured copy bandwidth.
//
// Far from the newest token all keys of a group share the last bucket and the bias is one number per row.
#include "fb_params.h"
#include "ptx_sm100.cuh"

#include <type_traits>

namespace fb {
namespace {

using namespace ptx;

constexpr int kWarps = 4, kThreads = kWarps * 32;  // of the join kernel; the decode kernel has 4 or 8 warps
constexpr int KG = 16;      // keys per group = MMA k of the second product
constexpr int kStages = 3;  // groups in flight per warp
constexpr float kRescaleThreshold = 8.f;  // log2 units
constexpr int kMaxTable = kDecodeMaxTable;  // entries of the table's columns that a CTA keeps
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {  // invalid: zero fill, nothing read
  const int n = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// 16-byte unit u of row r of a [rows][D] 16-bit tile, swizzled so that ldmatrix (8 rows, one unit each) meets 8 different banks
template <int D>
__device__ __forceinline__ uint32_t unit_off(int r, int u) { return (uint32_t)(r * D * 2 + ((u ^ (r & 7)) << 4)); }

template <typename T, int D>
__device__ __forceinline__ void store_out(const DecodeParams& p, int b, int t, int h, int d4, float4 v, float l) {
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T* dst = reinterpret_cast<T*>(p.out) + ((int64_t)(b * p.Sq + t) * p.Hq + h) * D + d4 * 4;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack16<T>(v.x * inv, v.y * inv), pack16<T>(v.z * inv, v.w * inv));
}

template <typename T, int D, int MT, int NW>
__global__ void __launch_bounds__(NW * 32) decode_kernel(const __grid_constant__ DecodeParams p, const __grid_constant__ RelPos rel) {
  constexpr int NT = NW * 32;
  constexpr int R = 16 * MT;           // rows per CTA
  constexpr int U = D / 8;             // 16-byte units per row
  constexpr int kTile = KG * D * 2;    // bytes of one K or V group
  constexpr int kWarpBytes = kStages * 2 * kTile;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* const qs = smem;                       // [R][D]
  uint8_t* const stages = smem + R * D * 2;       // per warp [kStages][K, V]
  __shared__ RelBuckets buckets;
  __shared__ float s_m[NW][R], s_l[NW][R], s_shift[R];
  __shared__ float2 joint_ml[R];
  float* const tab = reinterpret_cast<float*>(smem + R * D * 2 + NW * kWarpBytes);  // [heads of the CTA's rows][nb], log2 units

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x;
  const int hk = blockIdx.y / p.row_tiles, rt = blockIdx.y - hk * p.row_tiles;
  const int b = blockIdx.z;
  const int rows = p.G * p.Sq;
  relpos_load_buckets(buckets, rel, threadIdx.x, NT);
  grid_dependency_wait();
  grid_launch_dependents();
  const int len = p.lens ? min(max(p.lens[b], 0), p.Sk) : p.Sk;
  // this slice of the sequence's keys: [k0, k1), whole rounds of the CTA's warps
  const int per = ((len + p.splits - 1) / p.splits + NW * KG - 1) / (NW * KG) * (NW * KG);
  const int k0 = min(len, split * per), k1 = min(len, k0 + per);
  const int ngroups = (k1 - k0 + KG - 1) / KG;
  const int mine = ngroups > warp ? (ngroups - warp + NW - 1) / NW : 0;

  const T* kb = reinterpret_cast<const T*>(p.k.ptr) + b * p.k.batch_stride + hk * p.k.head_stride;
  const T* vb = reinterpret_cast<const T*>(p.v.ptr) + b * p.v.batch_stride + hk * p.v.head_stride;
  const uint32_t my = smem_u32(stages) + warp * kWarpBytes;
  auto load = [&](int i) {  // group i of this warp into its stage
    if (i < mine) {
      const int j0 = k0 + (warp + i * NW) * KG;
      const uint32_t dst = my + (i % kStages) * 2 * kTile;
#pragma unroll
      for (int x = 0; x < KG * U / 32; ++x) {
        const int at = x * 32 + lane, r = at / U, u = at % U;
        const bool ok = j0 + r < k1;
        const int64_t j = ok ? j0 + r : k0;
        cp_async16(dst + unit_off<D>(r, u), kb + j * p.k.row_stride + u * 8, ok);
        cp_async16(dst + kTile + unit_off<D>(r, u), vb + j * p.v.row_stride + u * 8, ok);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load(i);

  // the table's columns of this kv head's query heads
  bool large = false;
  for (int at = threadIdx.x; at < p.G * rel.nb; at += NT) {
    const int g = at / rel.nb, t = at - g * rel.nb;
    const float x = relpos_entry<T>(rel, t, hk * p.G + g);
    large = large || relpos_large(x);
    tab[at] = relpos_log2(x);
  }
  // the queries: row x of the CTA is new token (rt * R + x) / G, query head hk * G + (rt * R + x) % G
  for (int at = threadIdx.x; at < R * U; at += NT) {
    const int x = at / U, u = at % U, row = rt * R + x;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows) {
      const int t = row / p.G, g = row - t * p.G;
      v = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q.ptr) + b * p.q.batch_stride + t * p.q.row_stride + (int64_t)(hk * p.G + g) * p.q.head_stride + u * 8);
    }
    *reinterpret_cast<uint4*>(qs + unit_off<D>(x, u)) = v;
  }
  large = __syncthreads_or(large) != 0;

  const RelFn bucket_of(rel, buckets);
  if (large) {  // the rows' shifts (fb_params.h): the largest entry of the buckets up to the first key's, a warp per row
#pragma unroll 1
    for (int x = warp; x < R; x += NW) {
      const int row = min(rt * R + x, rows - 1), t = row / p.G, at = len - p.Sq + t;
      float top = -INFINITY;
      if (at >= 0) {
        const int last = bucket_of(-at);
        for (int u = lane; u <= last; u += 32)
          if (rel.used[u >> 5] >> (u & 31) & 1u) top = fmaxf(top, tab[(row - t * p.G) * rel.nb + u]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) s_shift[x] = top == -INFINITY ? 0.f : top;
    }
    __syncthreads();
  }

  // this thread's rows of the MMA fragments: lane / 4 and lane / 4 + 8 of every 16
  const float scale2 = p.scale * kLog2e;
  int pos[MT][2];
  const float* row_tab[MT][2];
  float far_bias[MT][2], shift[MT][2], m[MT][2], l[MT][2];
  float o[MT][D / 8][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = min(rt * R + mt * 16 + lane / 4 + 8 * x, rows - 1);
      const int t = row / p.G;
      row_tab[mt][x] = tab + (row - t * p.G) * rel.nb;
      pos[mt][x] = len - p.Sq + t;  // the new token's place in its sequence
      shift[mt][x] = large ? s_shift[mt * 16 + lane / 4 + 8 * x] : 0.f;
      far_bias[mt][x] = row_tab[mt][x][rel.side - 1] - shift[mt][x];
      m[mt][x] = -INFINITY;
      l[mt][x] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
  }
  const int pos_min = len - p.Sq + (rt * R) / p.G;  // the earliest row of the CTA

  // the query fragments stay in registers unless the accumulators need them
  constexpr bool kQRegs = MT * D <= 128;
  uint32_t q_regs[kQRegs ? MT : 1][kQRegs ? D / 16 : 1][4];
  if constexpr (kQRegs) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) ldsm4(smem_u32(qs) + unit_off<D>(mt * 16 + (lane & 15), kk * 2 + (lane >> 4)), q_regs[mt][kk]);
  }

  for (int i = 0; i < mine; ++i) {
    load(i + kStages - 1);
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const uint32_t ks = my + (i % kStages) * 2 * kTile, vs = ks + kTile;
    const int j0 = k0 + (warp + i * NW) * KG;
    float s[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][n][e] = 0.f;
    // S = Q K^T: matrices of one x4 load: keys 0-7 | k 0-7, keys 0-7 | k 8-15, keys 8-15 | k 0-7, keys 8-15 | k 8-15
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t kf[4];
      ldsm4(ks + unit_off<D>((lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)), kf);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t qf[4];
        if constexpr (kQRegs) {
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[e] = q_regs[mt][kk][e];
        } else {
          ldsm4(smem_u32(qs) + unit_off<D>(mt * 16 + (lane & 15), kk * 2 + (lane >> 4)), qf);
        }
        mma16816<T>(s[mt][0], qf, kf[0], kf[1]);
        mma16816<T>(s[mt][1], qf, kf[2], kf[3]);
      }
    }
    // bias and mask; element e of tile n: row lane / 4 + 8 (e / 2), key j0 + 8 n + 2 (lane % 4) + e % 2
    const bool all_far = pos_min - (j0 + KG - 1) >= bucket_of.far && j0 + KG <= k1;
    float mx[MT][2];
    auto add_bias = [&](auto which) {
      constexpr int mode = decltype(which)::value;  // 0: one bucket per row, 1: by the byte table, 2: with a search
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mx[mt][0] = mx[mt][1] = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int x = e >> 1, j = j0 + 8 * n + 2 * (lane & 3) + (e & 1);
            if (mode == 0) {
              s[mt][n][e] = fmaf(s[mt][n][e], scale2, far_bias[mt][x]);
            } else {
              const int r = j - pos[mt][x];
              const float bias = row_tab[mt][x][mode == 1 ? bucket_of.near(min(r, 0)) : bucket_of(min(r, 0))] - shift[mt][x];
              // selected, not added: the key of a later token may hold infinities or NaN
              s[mt][n][e] = r > 0 || j >= k1 ? -INFINITY : fmaf(s[mt][n][e], scale2, bias);
            }
            mx[mt][x] = fmaxf(mx[mt][x], s[mt][n][e]);
          }
      }
    };
    if (all_far) add_bias(std::integral_constant<int, 0>{});
    else if (bucket_of.byte_table()) add_bias(std::integral_constant<int, 1>{});
    else add_bias(std::integral_constant<int, 2>{});
    // running maximum, every row's steps side by side; it moves (and the accumulators are rescaled) only when it grew by more than 2^8
    bool grow = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        mx[mt][x] = fmaxf(mx[mt][x], __shfl_xor_sync(0xffffffffu, mx[mt][x], 1));
        mx[mt][x] = fmaxf(mx[mt][x], __shfl_xor_sync(0xffffffffu, mx[mt][x], 2));
        grow = grow || mx[mt][x] - m[mt][x] > kRescaleThreshold;  // (false when both are -inf: NaN)
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (!(mx[mt][x] - m[mt][x] > kRescaleThreshold)) continue;
          const float alpha = ex2(m[mt][x] - mx[mt][x]);  // m = -inf: 0
          m[mt][x] = mx[mt][x];
          l[mt][x] *= alpha;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) { o[mt][n][2 * x] *= alpha; o[mt][n][2 * x + 1] *= alpha; }
        }
    }
    uint32_t pf[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float off = m[mt][x] == -INFINITY ? 0.f : m[mt][x];  // nothing visible so far: every exponential is 0
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 2 * x; e < 2 * x + 2; ++e) s[mt][n][e] = ex2(s[mt][n][e] - off);
        // this lane's keys only; the four lanes of a row are added up at the end
        l[mt][x] += (s[mt][0][2 * x] + s[mt][0][2 * x + 1]) + (s[mt][1][2 * x] + s[mt][1][2 * x + 1]);
      }
      // the score fragments of two 8-key tiles are the 16-key operand of the second product
      pf[mt][0] = pack16<T>(s[mt][0][0], s[mt][0][1]);
      pf[mt][1] = pack16<T>(s[mt][0][2], s[mt][0][3]);
      pf[mt][2] = pack16<T>(s[mt][1][0], s[mt][1][1]);
      pf[mt][3] = pack16<T>(s[mt][1][2], s[mt][1][3]);
    }
#pragma unroll
    for (int n2 = 0; n2 < D / 16; ++n2) {
      uint32_t vf[4];
      ldsm4t(vs + unit_off<D>(lane & 15, n2 * 2 + (lane >> 4)), vf);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mma16816<T>(o[mt][2 * n2], pf[mt], vf[0], vf[1]);
        mma16816<T>(o[mt][2 * n2 + 1], pf[mt], vf[2], vf[3]);
      }
    }
    __syncwarp();  // every lane has read the stage before it is filled again
  }

  // ---- join the warps ----
  cp_async_wait<0>();
  __syncthreads();  // the stages are free: [warp][R][D] float32 accumulators
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[mt][x] += __shfl_xor_sync(0xffffffffu, l[mt][x], 1);
      l[mt][x] += __shfl_xor_sync(0xffffffffu, l[mt][x], 2);
      if ((lane & 3) == 0) {
        s_m[warp][mt * 16 + lane / 4 + 8 * x] = m[mt][x];
        s_l[warp][mt * 16 + lane / 4 + 8 * x] = l[mt][x];
      }
    }
  float* const acc = reinterpret_cast<float*>(stages);
  float* const joint = acc + NW * R * D;  // [R][D], cluster: this slice's sum
  static_assert((NW + 1) * R * D * 4 <= NW * kWarpBytes, "the accumulators fit the stages");
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        *reinterpret_cast<float2*>(acc + (warp * R + mt * 16 + lane / 4 + 8 * x) * D + n * 8 + 2 * (lane & 3)) = make_float2(o[mt][n][2 * x], o[mt][n][2 * x + 1]);
  __syncthreads();
  for (int at = threadIdx.x; at < R * D / 4; at += NT) {
    const int x = at / (D / 4), d4 = at - x * (D / 4), row = rt * R + x;
    if (row >= rows) break;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mm = fmaxf(mm, s_m[w][x]);
    const float off = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = ex2(s_m[w][x] - off);
      const float4 a = *reinterpret_cast<const float4*>(acc + (w * R + x) * D + d4 * 4);
      ll += s_l[w][x] * f;
      v.x += a.x * f; v.y += a.y * f; v.z += a.z * f; v.w += a.w * f;
    }
    const int t = row / p.G, h = hk * p.G + row - t * p.G;
    if (p.splits == 1) {
      store_out<T, D>(p, b, t, h, d4, v, ll);
    } else if (p.cluster) {
      *reinterpret_cast<float4*>(joint + x * D + d4 * 4) = v;
      if (d4 == 0) joint_ml[x] = make_float2(mm, ll);
    } else {
      const int64_t at_row = ((int64_t)(b * p.Sq + t) * p.Hq + h) * p.splits + split;
      *reinterpret_cast<float4*>(p.part + at_row * D + d4 * 4) = v;
      if (d4 == 0) p.part_ml[at_row] = make_float2(mm, ll);
    }
  }
  if (p.cluster) {
    cluster_sync_all();  // every slice's result is in its CTA's shared memory
    const uint32_t my_joint = smem_u32(joint), my_ml = smem_u32(joint_ml);
    for (int at = split * NT + threadIdx.x; at < R * D / 4; at += p.splits * NT) {
      const int x = at / (D / 4), d4 = at - x * (D / 4), row = rt * R + x;
      if (row >= rows) break;
      float mm = -INFINITY;
      float2 ml[kMaxCluster];
      float4 a[kMaxCluster];
#pragma unroll
      for (int s = 0; s < kMaxCluster; ++s) {
        ml[s] = make_float2(-INFINITY, 0.f);
        if (s < p.splits) {
          ml[s] = ld_cluster_f2(map_to_cta(my_ml + x * 8, (uint32_t)s));
          a[s] = ld_cluster_f4(map_to_cta(my_joint + (x * D + d4 * 4) * 4, (uint32_t)s));
          mm = fmaxf(mm, ml[s].x);
        }
      }
      const float off = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int s = 0; s < kMaxCluster; ++s) {
        if (s < p.splits) {
          const float f = ex2(ml[s].x - off);
          ll += ml[s].y * f;
          v.x += a[s].x * f; v.y += a[s].y * f; v.z += a[s].z * f; v.w += a[s].w * f;
        }
      }
      const int t = row / p.G, h = hk * p.G + row - t * p.G;
      store_out<T, D>(p, b, t, h, d4, v, ll);
    }
    cluster_sync_all();  // nobody reads this CTA's shared memory any more
  }
}

// One warp per (sequence, new token, query head): joins the slices in order.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) decode_join_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int E = D / 32;  // elements per lane
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  grid_dependency_wait();
  if (row >= (int64_t)p.B * p.Sq * p.Hq) return;
  const float2* ml = p.part_ml + row * p.splits;
  const float* part = p.part + row * p.splits * D + lane * E;
  float mm = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) mm = fmaxf(mm, ml[s].x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, x));
  const float off = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f, v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float2 x = ml[s];
    const float f = ex2(x.x - off);
    ll += x.y * f;
    if constexpr (E == 4) {
      const float4 a = *reinterpret_cast<const float4*>(part + (int64_t)s * D);
      v[0] += a.x * f; v[1] += a.y * f; v[2] += a.z * f; v[3] += a.w * f;
    } else {
      const float2 a = *reinterpret_cast<const float2*>(part + (int64_t)s * D);
      v[0] += a.x * f; v[1] += a.y * f;
    }
  }
  const float inv = ll > 0.f ? 1.f / ll : 0.f;
  T* dst = reinterpret_cast<T*>(p.out) + row * D + lane * E;
  if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pack16<T>(v[0] * inv, v[1] * inv), pack16<T>(v[2] * inv, v[3] * inv));
  else *reinterpret_cast<uint32_t*>(dst) = pack16<T>(v[0] * inv, v[1] * inv);
}

template <typename K>
cudaError_t launch(K kern, dim3 grid, int threads, size_t smem, int cluster, cudaStream_t s, void** args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];  // programmatic dependent launch: both kernels wait for the one before at their start
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kern), args);
}

template <typename T, int D, int MT, int NW>
int decode_typed(DecodeParams& p, RelPos& rel, cudaStream_t s) {
  constexpr int R = 16 * MT;
  constexpr size_t tiles = R * D * 2 + NW * kStages * 2 * KG * D * 2;
  const size_t smem = tiles + (size_t)p.G * rel.nb * sizeof(float);
  auto kern = decode_kernel<T, D, MT, NW>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(tiles + kMaxTable * sizeof(float))) != cudaSuccess) return FB_ERR_CUDA;
  p.row_tiles = (p.G * p.Sq + R - 1) / R;
  void* args[2] = {&p, &rel};
  if (launch(kern, dim3((unsigned)p.splits, (unsigned)(p.Hkv * p.row_tiles), (unsigned)p.B), NW * 32, smem, p.cluster ? p.splits : 1, s, args) != cudaSuccess)
    return FB_ERR_CUDA;
  if (p.splits == 1 || p.cluster) return 1;
  const int64_t rows = (int64_t)p.B * p.Sq * p.Hq;
  if (launch(decode_join_kernel<T, D>, dim3((unsigned)((rows + kWarps - 1) / kWarps)), kThreads, 0, 1, s, args) != cudaSuccess) return FB_ERR_CUDA;
  return 2;
}

template <typename T>
int decode_dispatch(DecodeParams& p, RelPos& rel, cudaStream_t s) {
  // A cluster's problem is small: one CTA per SM, whose 8 warps have the schedulers to themselves.
  if (p.cluster) {
    if (p.G * p.Sq <= 16) return p.D == 64 ? decode_typed<T, 64, 1, 8>(p, rel, s) : decode_typed<T, 128, 1, 8>(p, rel, s);
    return p.D == 64 ? decode_typed<T, 64, 2, 8>(p, rel, s) : decode_typed<T, 128, 2, 8>(p, rel, s);
  }
  if (p.G * p.Sq <= 16) return p.D == 64 ? decode_typed<T, 64, 1, 4>(p, rel, s) : decode_typed<T, 128, 1, 4>(p, rel, s);
  return p.D == 64 ? decode_typed<T, 64, 2, 4>(p, rel, s) : decode_typed<T, 128, 2, 4>(p, rel, s);
}

}  // namespace

// Slices of a sequence's keys and how they are joined: enough CTAs for a few waves on the whole GPU, slices of at least one round of the CTA's warps. A
// power of two up to 8 (a cluster: one launch) for small batches whose slices then have at most 8 rounds; otherwise a workspace and a
// second launch, since a cluster holds its SMs until its last CTA is done: 48 sequences of up to 8192 keys, 8 kv heads of 128
// in 4 slices each: 171 us as clusters, 152 + 5 us through the workspace; 24 sequences of 9000 keys, 8 kv heads of 128 in 7 slices: 222 and 141 us.
DecodeShape decode_shape(int batch, int heads_kv, int rows, int seqlen_k) {
  const int per = rows <= 16 ? 16 : 32;
  const int64_t base = (int64_t)batch * heads_kv * ((rows + per - 1) / per);
  const int64_t want = (148 * 2 * 4 + base - 1) / base;
  const int64_t rounds = (seqlen_k + kWarps * KG - 1) / (kWarps * KG);
  const int64_t rounds8 = (rounds + 1) / 2;  // of 8 warps
  if (base < 2 * 148 && rounds8 <= 8 * kMaxCluster) {
    int n = 1;
    while (n < kMaxCluster && n < want && 2 * n <= rounds8) n *= 2;
    return {n, n > 1};
  }
  const int64_t n = want < rounds ? want : rounds;
  return {(int)(n < 1 ? 1 : n > 128 ? 128 : n), false};
}

int launch_decode(int dtype, DecodeParams& p, RelPos& rel, cudaStream_t s) {
  return dtype == FB_BF16 ? decode_dispatch<__nv_bfloat16>(p, rel, s) : decode_dispatch<__half>(p, rel, s);
}

}  // namespace fb
