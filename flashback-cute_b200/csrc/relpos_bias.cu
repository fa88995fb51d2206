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
// (aligned in the flat tensor, since rows of odd length start anywhere; the ends of a row go out one by one).
constexpr int kRows = 32, kCols = 2048;

template <typename T>
__global__ void __launch_bounds__(kThreads) relpos_fill_kernel(const __grid_constant__ RelPos rel, int sq, int sk, T* __restrict__ out) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ T val[kRows + kCols];
  __shared__ T tab[FB_RELPOS_MAX_BUCKETS];
  __shared__ RelBuckets buckets;
  const int h = blockIdx.z, i0 = blockIdx.y * kRows, j0 = blockIdx.x * kCols;
  const int rows = min(kRows, sq - i0), cols = min(kCols, sk - j0);
  for (int t = threadIdx.x; t < rel.nb; t += kThreads) tab[t] = reinterpret_cast<const T*>(rel.table)[t * rel.bucket_stride + h * rel.head_stride];
  relpos_load_buckets(buckets, rel, threadIdx.x, kThreads);
  __syncthreads();
  const RelFn bucket_of(rel, buckets);
  const int base = j0 - (i0 + rows - 1) - (sk - sq);  // position of entry 0: the tile's last row, first column
  for (int u = threadIdx.x; u < rows + cols - 1; u += kThreads) val[u] = tab[bucket_of(base + u)];
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = warp; r < rows; r += kWarps) {
    const int64_t flat = ((int64_t)h * sq + i0 + r) * sk + j0;
    const T* src = val + (rows - 1 - r);
    T* dst = out + flat;
    const int head = min(cols, (int)((VEC - flat % VEC) % VEC));
    if (lane < head) dst[lane] = src[lane];
    const int nvec = (cols - head) / VEC;
    for (int k = lane; k < nvec; k += 32) {
      const int j = head + k * VEC;
      alignas(16) T v[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = src[j + e];
      *reinterpret_cast<uint4*>(dst + j) = *reinterpret_cast<const uint4*>(v);
    }
    const int j = head + nvec * VEC + lane;
    if (j < cols) dst[j] = src[j];
  }
}

// ---------------------------------------------------------------------------------------------------
// gradient
// ---------------------------------------------------------------------------------------------------
// The sum over a bucket is a sum over diagonals. Diagonal c = j - i + (sq - 1) of row i sits at flat offset
// i * (sk + 1) + c - (sq - 1): rows that are VEC = 16 bytes / element apart keep their place relative to a 16-byte
// boundary. So a CTA takes kDiag diagonals x a stretch of rows, each of VEC residues of the row index gets an equal share of
// the warps, and a thread adds up VEC neighbouring diagonals in registers over its rows with 16-byte loads: no
// atomics, no reordering, every element read once. At the end the CTA adds up its warps' diagonals, then those of
// each bucket (neighbours), and leaves one number per bucket in the workspace.
constexpr int kSpan = 256;  // diagonals per warp: 32 lanes x 8 elements (16 bit); 32 x 4 x 2 (float32)

template <typename T> struct Vec;
template <> struct Vec<__nv_bfloat16> { static constexpr int n = 8; };
template <> struct Vec<__half> { static constexpr int n = 8; };
template <> struct Vec<float> { static constexpr int n = 4; };

template <typename T>
__global__ void __launch_bounds__(kThreads) relpos_grad_kernel(const __grid_constant__ RelPos rel, int sq, int sk, int rows_per_cta, const T* __restrict__ grad) {
  constexpr int VEC = Vec<T>::n;
  constexpr int PER = kSpan / 32 / VEC;  // vectors per lane and row
  __shared__ float part[kWarps][kSpan + VEC];
  __shared__ float acc[FB_RELPOS_MAX_BUCKETS];
  __shared__ RelBuckets buckets;
  const int h = blockIdx.z;
  const int c0 = blockIdx.x * kSpan;  // first diagonal
  const int ndiag = sq + sk - 1;
  int i_lo = blockIdx.y * rows_per_cta, i_hi = min(sq, i_lo + rows_per_cta);
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
  float sum[PER][VEC];
#pragma unroll
  for (int q = 0; q < PER; ++q)
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[q][e] = 0.f;
  // One residue needs kSpan + VEC diagonals when shift > 0: the first `shift` of its first vector belong to the CTA before
  // and are masked, the last vector's are masked by the next; so the span of a warp is [c0 - shift, c0 - shift + kSpan)
  // plus one more vector, which lane 0 takes.
  float tail[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) tail[e] = 0.f;

  auto add = [&](float (&s)[VEC], int i, int c) {  // the vector that starts at diagonal c of row i
    const int j = c - (sq - 1) + i;
    if (j >= 0 && j + VEC <= sk) {
      const uint4 u = *reinterpret_cast<const uint4*>(g + (int64_t)i * sk + j);
      const T* v = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[e] += to_f<T>(v[e]);
    } else if (j + VEC > 0 && j < sk) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (j + e >= 0 && j + e < sk) s[e] += to_f<T>(g[(int64_t)i * sk + j + e]);
    }
  };
#pragma unroll 4
  for (int i = first; i < i_hi; i += kWarps) {
#pragma unroll
    for (int q = 0; q < PER; ++q) add(sum[q], i, c0 - shift + (q * 32 + lane) * VEC);
    if (shift > 0 && lane == 0) add(tail, i, c0 - shift + kSpan);
  }
#pragma unroll
  for (int q = 0; q < PER; ++q)
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[warp][(q * 32 + lane) * VEC + e] = sum[q][e];
  if (lane == 0) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[warp][kSpan + e] = tail[e];
  }
  __shared__ int shifts[kWarps];
  if (lane == 0) shifts[warp] = shift;
  __syncthreads();
  // thread t: diagonal c0 + t, the warps' sums in a fixed order; then the diagonals of a bucket, warp by warp
  float s = 0.f;
  const int c = c0 + threadIdx.x;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) s += part[w][shifts[w] + threadIdx.x];
  const int bucket = c < ndiag ? RelFn(rel, buckets)(c - (sq - 1) - (sk - sq)) : -1;
  const bool run = run_head(bucket, lane);
  s = run_sum(s, bucket, lane);
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
#pragma unroll 4
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
  const dim3 grid((sk + kCols - 1) / kCols, (sq + kRows - 1) / kRows, heads);
  if (grid.y > 65535 || grid.z > 65535) return FB_ERR_TOO_LARGE;
  relpos_fill_kernel<T><<<grid, kThreads, 0, s>>>(rel, sq, sk, reinterpret_cast<T*>(out));
  return cudaGetLastError() == cudaSuccess ? 1 : FB_ERR_CUDA;
}

template <typename T>
int reduce_typed(const float* part, int batch, int heads, int ntiles, int nb, void* dtable, int64_t bs, int64_t hs, cudaStream_t s) {
  relpos_reduce_kernel<T><<<heads, kReduceThreads, 0, s>>>(part, batch, heads, ntiles, nb, reinterpret_cast<T*>(dtable), bs, hs);
  return cudaGetLastError() == cudaSuccess ? 1 : FB_ERR_CUDA;
}

// Rows per CTA of the gradient: long stretches spread the end of a CTA (its sums by bucket) over more reads, short ones
// fill the GPU. The same rule sizes the workspace.
int grad_rows(int heads, int sq, int sk) {
  const long long spans = (sq + sk - 1 + kSpan - 1) / kSpan;
  int rows = 512;
  while (rows > 32 && spans * heads * ((sq + rows - 1) / rows) < 148 * 8) rows /= 2;
  return rows;
}

template <typename T>
int grad_typed(const RelPos& rel, int heads, int sq, int sk, const void* grad, cudaStream_t s) {
  const int rows = grad_rows(heads, sq, sk);
  const dim3 grid((sq + sk - 1 + kSpan - 1) / kSpan, (sq + rows - 1) / rows, heads);
  if (grid.y > 65535 || grid.z > 65535) return FB_ERR_TOO_LARGE;
  relpos_grad_kernel<T><<<grid, kThreads, 0, s>>>(rel, sq, sk, rows, reinterpret_cast<const T*>(grad));
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

int64_t relpos_bias_parts(int heads, int sq, int sk) {
  const int rows = grad_rows(heads, sq, sk);
  return (int64_t)((sq + sk - 1 + kSpan - 1) / kSpan) * ((sq + rows - 1) / rows);
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
  int r;
  switch (dtype) {
    case FB_BF16: r = grad_typed<__nv_bfloat16>(rel, heads, sq, sk, grad, s); break;
    case FB_F16: r = grad_typed<__half>(rel, heads, sq, sk, grad, s); break;
    case FB_F32: r = grad_typed<float>(rel, heads, sq, sk, grad, s); break;
    default: return FB_ERR_DTYPE;
  }
  if (r < 0) return r;
  const int r2 = launch_rel_reduce(dtype, rel.dpart, 1, heads, (int)relpos_bias_parts(heads, sq, sk), rel.nb, dtable, bs, hs, s);
  return r2 < 0 ? r2 : r + r2;
}

}  // namespace fb
