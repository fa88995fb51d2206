// The learned relative position bias as a tensor, out[h][i][j] = T[bucket(j - i - (sk - sq)), h], and the gradient of the
// table for a given gradient of it; and the last step of the table's gradient in the attention backward.
//
// Both directions are bound by HBM: the forward writes, the gradient reads heads * sq * sk elements once.
#include "fb_params.h"

namespace fb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// ---------------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------------
// One CTA = kRows rows x kCols columns of one head. The values depend on j - i alone: the kRows + kCols - 1 of them that
// the tile needs are looked up once, into shared memory, and a warp per row copies its stretch out in 16-byte stores
// (aligned in the flat tensor, since rows of odd length start anywhere; the ends of a row go out one by one). The stretch of a row
// starts at any element: one copy of the values per element of a 16-byte unit, each shifted by one more, gives every
// row 16-byte loads too. (One copy and an element at a time was bound by shared memory: 168 us for 16 x 4095 x 4099 bf16.)
// The columns are split evenly into stretches of at most kCols.
constexpr int kRows = 128, kCols = 2304;

template <typename T>
__global__ void __launch_bounds__(kThreads) relpos_fill_kernel(const __grid_constant__ RelPos rel, int sq, int sk, int rows_per_cta, int cols_per_cta, T* __restrict__ out) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int LEN = kRows + kCols + VEC;  // entries per copy, whole units
  extern __shared__ __align__(16) uint8_t smem[];
  T* const val = reinterpret_cast<T*>(smem);  // [VEC][LEN]: copy k, entry u = value u + k
  __shared__ T tab[FB_RELPOS_MAX_BUCKETS];
  __shared__ RelBuckets buckets;
  const int h = blockIdx.z, i0 = blockIdx.y * rows_per_cta, j0 = blockIdx.x * cols_per_cta;
  const int rows = min(rows_per_cta, sq - i0), cols = min(cols_per_cta, sk - j0);
  for (int t = threadIdx.x; t < rel.nb; t += kThreads) tab[t] = reinterpret_cast<const T*>(rel.table)[t * rel.bucket_stride + h * rel.head_stride];
  relpos_load_buckets(buckets, rel, threadIdx.x, kThreads);
  __syncthreads();
  const RelFn bucket_of(rel, buckets);
  const int base = j0 - (i0 + rows - 1) - (sk - sq);  // position of value 0: the tile's last row, first column
  for (int x = threadIdx.x; x < (rows + cols - 1 + VEC - 1) / VEC; x += kThreads) {
    T v[2 * VEC];  // values VEC x .. VEC x + 2 VEC - 1
    if (bucket_of.byte_table()) {
#pragma unroll
      for (int e = 0; e < 2 * VEC; ++e) v[e] = tab[bucket_of.near(base + x * VEC + e)];
    } else {
#pragma unroll
      for (int e = 0; e < 2 * VEC; ++e) v[e] = tab[bucket_of(base + x * VEC + e)];
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      alignas(16) T w[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = v[k + e];
      *reinterpret_cast<uint4*>(val + k * LEN + x * VEC) = *reinterpret_cast<const uint4*>(w);
    }
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = warp; r < rows; r += kWarps) {
    const int64_t flat = ((int64_t)h * sq + i0 + r) * sk + j0;
    const int first = rows - 1 - r;  // value of the row's first column
    T* dst = out + flat;
    const int head = min(cols, (int)((VEC - flat % VEC) % VEC));
    if (lane < head) dst[lane] = val[first + lane];
    const int nvec = (cols - head) / VEC, start = first + head;
    const uint4* src = reinterpret_cast<const uint4*>(val + (start % VEC) * LEN + start / VEC * VEC);
    uint4* to = reinterpret_cast<uint4*>(dst + head);
#pragma unroll 4
    for (int k = lane; k < nvec; k += 32) to[k] = src[k];
    const int j = head + nvec * VEC + lane;
    if (j < cols) dst[j] = val[first + j];
  }
}

// ---------------------------------------------------------------------------------------------------
// gradient
// ---------------------------------------------------------------------------------------------------
// The sum over a bucket is a sum over diagonals. Diagonal c = j - i + (sq - 1) of row i sits at flat offset
// i * (sk + 1) + c - (sq - 1): rows that are VEC = 16 bytes / element apart keep their place relative to a 16-byte
// boundary. So a CTA takes kSpan of the diagonals that meet a stretch of rows, each of VEC residues of the row index gets an equal share of
// the warps, and a thread adds up VEC neighbouring diagonals in registers over its rows with 16-byte loads: no
// atomics, no reordering, every element read once. At the end the CTA adds up its warps' diagonals, then those of
// each bucket (neighbours), and leaves one number per bucket in the workspace.
// A warp reads one 16-byte vector per lane and row, 512 bytes of it; 4 rows in flight, 256 rows per CTA. Measured on 16 x 4095 x 4099 bf16
// (537 MB): 141 us; 8 rows in flight 153; 512 / 1024 rows per CTA 178 / 196; 1 KB of a row per warp 158, 2 KB 222. Many small
// CTAs that read one region of the tensor at a time beat fewer, longer ones. Interior rows without predicates and packed
// additions were worth 8 %.

template <typename T> struct Vec;
template <> struct Vec<__nv_bfloat16> { static constexpr int n = 8; };
template <> struct Vec<__half> { static constexpr int n = 8; };
template <> struct Vec<float> { static constexpr int n = 4; };

template <typename T>
__global__ void __launch_bounds__(kThreads) relpos_grad_kernel(const __grid_constant__ RelPos rel, int sq, int sk, int rows_per_cta, const T* __restrict__ grad) {
  constexpr int VEC = Vec<T>::n;
  constexpr int kSpan = 32 * VEC;  // diagonals per CTA
  constexpr int kBatch = 4;        // rows of a warp in flight
  __shared__ float part[kWarps][kSpan + VEC];
  __shared__ float acc[FB_RELPOS_MAX_BUCKETS];
  __shared__ RelBuckets buckets;
  const int h = blockIdx.z;
  int i_lo = blockIdx.y * rows_per_cta, i_hi = min(sq, i_lo + rows_per_cta);
  const int c0 = sq - i_hi + blockIdx.x * kSpan;  // first diagonal; the stretch's first is that of its last row's first column
  const int ndiag = sq + sk - 1;
  float* out = rel.dpart + (((int64_t)h * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * rel.nb;
  // rows whose columns j = c - (sq - 1) + i meet [0, sk) for some diagonal of the CTA
  i_lo = max(i_lo, sq - 1 - (c0 + kSpan - 1));
  i_hi = min(i_hi, sk + sq - 1 - c0);
  if (i_lo >= i_hi) {
    if ((int)threadIdx.x < rel.nb) out[threadIdx.x] = 0.f;
    return;
  }
  relpos_load_buckets(buckets, rel, threadIdx.x, kThreads);
  if (threadIdx.x < FB_RELPOS_MAX_BUCKETS) acc[threadIdx.x] = 0.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* g = grad + (int64_t)h * sq * sk;
  const int64_t g_at = (int64_t)h * sq * sk;  // flat offset of the head (its own place relative to a boundary)

  // this warp's rows: i = first + step * k
  const int first = i_lo + warp;
  // vectors start where (g_at + i * (sk + 1) + c - (sq - 1)) is a multiple of VEC: diagonal c0 - shift + VEC * k
  const int shift = (int)(((g_at + (int64_t)first * (sk + 1) + c0 - (sq - 1)) % VEC + VEC) % VEC);
  float sum[VEC], tail[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[e] = tail[e] = 0.f;
  // One residue needs kSpan + VEC diagonals when shift > 0: the first `shift` of its first vector belong to the CTA before
  // and are masked, the last vector's are masked by the next; so the span of a warp is [c0 - shift, c0 - shift + kSpan)
  // plus one more vector, which lane 0 takes.

  // a vector in row i whose first column is j and that an end of the row cuts; where both do, the first call takes it
  auto cut = [&](float (&s)[VEC], int i, int j, int end) {
    if (end == 1 && j < 0) return;
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (j + e >= 0 && j + e < sk) s[e] += to_f<T>(g[(int64_t)i * sk + j + e]);
  };
  // Vectors that lie inside [0, sk) altogether, kBatch rows' in flight together (predicated, no branches between the loads)
  const int lo = c0 - shift - (sq - 1) + lane * VEC;  // this lane's first column, in row 0
  const int warp_lo = lo - lane * VEC;
  const int64_t step = (int64_t)kWarps * (sk + 1);  // elements from a row's vector to that of the warp's next row
  const T* at = g + (int64_t)first * sk + first + lo;
  float2 sum2[VEC / 2];
#pragma unroll
  for (int e = 0; e < VEC / 2; ++e) sum2[e] = make_float2(0.f, 0.f);
  for (int i = first; i < i_hi; i += kBatch * kWarps, at += kBatch * step) {
    const int last = i + (kBatch - 1) * kWarps;
    uint4 u[kBatch];
    if (last < i_hi && warp_lo + i >= 0 && warp_lo + kSpan + last <= sk) {  // every lane's vectors of these rows
#pragma unroll
      for (int b = 0; b < kBatch; ++b) u[b] = *reinterpret_cast<const uint4*>(at + b * step);
    } else {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int row = i + b * kWarps, j = lo + row;
        u[b] = make_uint4(0, 0, 0, 0);
        if (row < i_hi && j >= 0 && j + VEC <= sk) u[b] = *reinterpret_cast<const uint4*>(at + b * step);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const T* v = reinterpret_cast<const T*>(&u[b]);
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) sum2[e] = __fadd2_rn(sum2[e], make_float2(to_f<T>(v[2 * e]), to_f<T>(v[2 * e + 1])));
    }
  }
#pragma unroll
  for (int e = 0; e < VEC / 2; ++e) { sum[2 * e] = sum2[e].x; sum[2 * e + 1] = sum2[e].y; }
  // ... and those that an end of their row cuts: the column moves by kWarps per row of this warp, so that happens at most once per end
  static_assert(kWarps >= VEC, "a vector is cut in one row per end at most");
#pragma unroll
  for (int end = 0; end < 2; ++end) {
    // the row whose column lies in (edge - VEC, edge)
    const int edge = end ? sk : 0, ahead = edge - 1 - (lo + first), k = ahead / kWarps;
    const int row = first + k * kWarps, col = lo + row;
    if (ahead >= 0 && row < i_hi && col > edge - VEC && (col < 0 || col + VEC > sk)) cut(sum, row, col, end);
  }
  if (shift > 0 && lane == 0)
    for (int i = first; i < i_hi; i += kWarps) {
      const int j = lo + kSpan + i;
      for (int e = 0; e < VEC; ++e)
        if (j + e >= 0 && j + e < sk && e < shift) tail[e] += to_f<T>(g[(int64_t)i * sk + j + e]);
    }
#pragma unroll
  for (int e = 0; e < VEC; ++e) part[warp][lane * VEC + e] = sum[e];
  if (lane == 0) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[warp][kSpan + e] = tail[e];
  }
  __shared__ int shifts[kWarps];
  if (lane == 0) shifts[warp] = shift;
  __syncthreads();
  // diagonal c0 + t, the warps' sums in a fixed order; then the diagonals of a bucket, warp by warp
  const int t = threadIdx.x, c = c0 + t;
  float s = 0.f;
  int bucket = -1;
  if (t < kSpan) {
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += part[w][shifts[w] + t];
    if (c < ndiag) bucket = RelFn(rel, buckets)(c - (sq - 1) - (sk - sq));
  }
  static_assert(kSpan <= kThreads, "a thread per diagonal");
  const bool run = run_sum(s, bucket, lane);
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp && run && bucket >= 0) acc[bucket] += s;
    __syncthreads();
  }
  if ((int)threadIdx.x < rel.nb) out[threadIdx.x] = acc[threadIdx.x];
}

// ---------------------------------------------------------------------------------------------------
// dtable[t][h] = sum over the rows of `part` that belong to head h: rows ((b * heads + h) * ntiles + tile), nb numbers each
// ---------------------------------------------------------------------------------------------------
// Latency-bound (a few hundred KB at most): one CTA per head, as many slices of the rows as fit, each thread one bucket of
// a slice; slices are added up in order. Sums in double: the summands cancel (every row of dS sums to zero).
constexpr int kReduceThreads = 1024;
template <typename T>
__global__ void __launch_bounds__(kReduceThreads) relpos_reduce_kernel(const float* __restrict__ part, int batch, int heads, int ntiles, int nb,
                                                                       T* __restrict__ dtable, int64_t bucket_stride, int64_t head_stride) {
  __shared__ double sums[kReduceThreads];
  const int h = blockIdx.x;
  const int slices = kReduceThreads / nb, slice = threadIdx.x / nb, t = threadIdx.x - slice * nb;
  double s = 0.0;
  if (slice < slices) {
    const int rows = batch * ntiles;
#pragma unroll 8
    for (int r = slice; r < rows; r += slices) {
      const int b = r / ntiles, tile = r - b * ntiles;
      s += (double)part[((int64_t)(b * heads + h) * ntiles + tile) * nb + t];
    }
  }
  sums[threadIdx.x] = s;
  __syncthreads();
  if ((int)threadIdx.x < nb) {
    for (int q = 1; q < slices; ++q) s += sums[q * nb + threadIdx.x];
    dtable[threadIdx.x * bucket_stride + h * head_stride] = from_f<T>((float)s);
  }
}

template <typename T>
int fill_typed(const RelPos& rel, int heads, int sq, int sk, void* out, cudaStream_t s) {
  const int n = (sk + kCols - 1) / kCols, cols = ((sk + n - 1) / n + 7) / 8 * 8;
  int rows = kRows;
  while (rows > 16 && (int64_t)n * heads * ((sq + rows - 1) / rows) < 148 * 4) rows /= 2;  // small: more CTAs
  const dim3 grid((sk + cols - 1) / cols, (sq + rows - 1) / rows, heads);
  if (grid.y > 65535 || grid.z > 65535) return FB_ERR_TOO_LARGE;
  constexpr int VEC = 16 / sizeof(T), smem = VEC * (kRows + kCols + VEC) * (int)sizeof(T);
  static_assert(smem <= 48 * 1024, "without an opt-in");
  relpos_fill_kernel<T><<<grid, kThreads, smem, s>>>(rel, sq, sk, rows, cols, reinterpret_cast<T*>(out));
  return cudaGetLastError() == cudaSuccess ? 1 : FB_ERR_CUDA;
}

template <typename T>
int reduce_typed(const float* part, int batch, int heads, int ntiles, int nb, void* dtable, int64_t bs, int64_t hs, cudaStream_t s) {
  relpos_reduce_kernel<T><<<heads, kReduceThreads, 0, s>>>(part, batch, heads, ntiles, nb, reinterpret_cast<T*>(dtable), bs, hs);
  return cudaGetLastError() == cudaSuccess ? 1 : FB_ERR_CUDA;
}

// Shape of the gradient's CTAs: 256 rows, fewer where the problem would not fill the GPU. The same rule sizes the workspace.
struct GradShape {
  int rows, spans, row_blocks;
};
GradShape grad_shape(int dtype, int heads, int sq, int sk) {
  GradShape g;
  const int span = 32 * (dtype == FB_F32 ? 4 : 8);
  for (g.rows = 256;; g.rows /= 2) {
    g.spans = (g.rows + sk - 1 + span - 1) / span;  // of a stretch of rows
    g.row_blocks = (sq + g.rows - 1) / g.rows;
    if (g.rows <= 32 || (int64_t)g.spans * heads * g.row_blocks >= 148 * 8) return g;
  }
}

template <typename T>
int grad_typed(const RelPos& rel, const GradShape& g, int heads, int sq, int sk, const void* grad, cudaStream_t s) {
  const dim3 grid(g.spans, g.row_blocks, heads);
  if (grid.y > 65535 || grid.z > 65535) return FB_ERR_TOO_LARGE;
  const T* in = reinterpret_cast<const T*>(grad);
  relpos_grad_kernel<T><<<grid, kThreads, 0, s>>>(rel, sq, sk, g.rows, in);
  return cudaGetLastError() == cudaSuccess ? 1 : FB_ERR_CUDA;
}

}  // namespace

int launch_rel_reduce(int dtype, const float* part, int batch, int heads, int ntiles, int nb, void* dtable, int64_t bs, int64_t hs, cudaStream_t s) {
  switch (dtype) {
    case FB_BF16: return reduce_typed<__nv_bfloat16>(part, batch, heads, ntiles, nb, dtable, bs, hs, s);
    case FB_F16: return reduce_typed<__half>(part, batch, heads, ntiles, nb, dtable, bs, hs, s);
    case FB_F32: return reduce_typed<float>(part, batch, heads, ntiles, nb, dtable, bs, hs, s);
  }
  return FB_ERR_DTYPE;
}

int64_t relpos_bias_parts(int dtype, int heads, int sq, int sk) {
  const GradShape g = grad_shape(dtype, heads, sq, sk);
  return (int64_t)g.spans * g.row_blocks;
}

int launch_relpos_fill(int dtype, const RelPos& rel, int heads, int sq, int sk, void* out, cudaStream_t s) {
  switch (dtype) {
    case FB_BF16: return fill_typed<__nv_bfloat16>(rel, heads, sq, sk, out, s);
    case FB_F16: return fill_typed<__half>(rel, heads, sq, sk, out, s);
    case FB_F32: return fill_typed<float>(rel, heads, sq, sk, out, s);
  }
  return FB_ERR_DTYPE;
}

int launch_relpos_grad(int dtype, const RelPos& rel, int heads, int sq, int sk, const void* grad, void* dtable, int64_t bs, int64_t hs, cudaStream_t s) {
  const GradShape g = grad_shape(dtype, heads, sq, sk);
  int r;
  switch (dtype) {
    case FB_BF16: r = grad_typed<__nv_bfloat16>(rel, g, heads, sq, sk, grad, s); break;
    case FB_F16: r = grad_typed<__half>(rel, g, heads, sq, sk, grad, s); break;
    case FB_F32: r = grad_typed<float>(rel, g, heads, sq, sk, grad, s); break;
    default: return FB_ERR_DTYPE;
  }
  if (r < 0) return r;
  const int r2 = launch_rel_reduce(dtype, rel.dpart, 1, heads, g.spans * g.row_blocks, rel.nb, dtable, bs, hs, s);
  return r2 < 0 ? r2 : r + r2;
}

}  // namespace fb
