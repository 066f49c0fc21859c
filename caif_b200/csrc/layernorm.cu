// Layer norm in front of the frozen projections, the other norm beside norm.cu's RMSNorm:
//   mean = sum x / n, rstd = 1 / sqrt(sum (x - mean)^2 / n + epsilon), y = (x - mean) * rstd * gamma + beta
//   xh = (x - mean) * rstd, g = dy * gamma
//   dx = rstd * (g - sum(g) / n - xh * sum(g * xh) / n),  dgamma = sum_rows dy * xh,  dbeta = sum_rows dy
// All sums are fp32 and run in a fixed order: a row's variance is taken around its mean (a second pass over the row, not the
// difference of two large sums), and the gradients of gamma and beta are partial sums per slice of rows, added slice by
// slice by a second launch, so that two calls give the same bits.  y and dx are rounded once.
#include <atomic>

#include "umma.cuh"

namespace caifq
{

namespace
{

constexpr int kLnThreads = 256;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16(v); }

// sum of one value a thread over WARPS warps; every thread gets it.  slots: [WARPS] floats that nobody else uses before the
// next barrier of these threads
template <int WARPS>
__device__ __forceinline__ float sum_of(float v, float *slots)
{
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
  {
    v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  }
  if constexpr (WARPS > 1)
  {
    __syncthreads();   // the slots may still be read from the sum before
    if ((threadIdx.x & 31) == 0)
    {
      slots[(threadIdx.x >> 5) % WARPS] = v;
    }
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
    {
      v += slots[w];
    }
  }
  return v;
}

// ---- any width, any alignment (tensors off a 16-byte boundary, rows wider than the forms below hold): a block a row, read in every
// pass ----

template <typename T>
__global__ void __launch_bounds__(kLnThreads)
layernorm_fwd_kernel(const T *x, const float *__restrict__ gamma, const float *__restrict__ beta, T *y,
                     float *__restrict__ mean_out, float *__restrict__ rstd_out, float epsilon, int rows, int64_t dim)
{
  __shared__ float slots[kLnThreads / 32];
  asm volatile("griddepcontrol.wait;" : "+l"(gamma), "+l"(beta)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
  {
    const T *src = x + r * dim;
    T *dst = y + r * dim;
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < dim; c += kLnThreads)
    {
      s += to_f<T>(src[c]);
    }
    const float mean = sum_of<kLnThreads / 32>(s, slots) / static_cast<float>(dim);
    s = 0.0f;
    for (int64_t c = threadIdx.x; c < dim; c += kLnThreads)
    {
      const float d = to_f<T>(src[c]) - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = 1.0f / sqrtf(sum_of<kLnThreads / 32>(s, slots) / static_cast<float>(dim) + epsilon);
    for (int64_t c = threadIdx.x; c < dim; c += kLnThreads)
    {
      const float v = (to_f<T>(src[c]) - mean) * rstd;
      dst[c] = from_f<T>(fmaf(v, gamma != nullptr ? gamma[c] : 1.0f, beta != nullptr ? beta[c] : 0.0f));
    }
    if (threadIdx.x == 0)
    {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kLnThreads)
layernorm_dx_kernel(const T *dy, const T *x, const float *__restrict__ gamma, const float *__restrict__ mean_in,
                    const float *__restrict__ rstd_in, T *dx, int rows, int64_t dim)
{
  __shared__ float slots[kLnThreads / 32];
  asm volatile("griddepcontrol.wait;" : "+l"(gamma), "+l"(mean_in), "+l"(rstd_in)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
  {
    const int64_t at = r * dim;
    const float mean = mean_in[r];
    const float rstd = rstd_in[r];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t c = threadIdx.x; c < dim; c += kLnThreads)
    {
      const float g = to_f<T>(dy[at + c]) * (gamma != nullptr ? gamma[c] : 1.0f);
      s1 += g;
      s2 = fmaf(g, (to_f<T>(x[at + c]) - mean) * rstd, s2);
    }
    s1 = sum_of<kLnThreads / 32>(s1, slots) / static_cast<float>(dim);
    s2 = sum_of<kLnThreads / 32>(s2, slots) / static_cast<float>(dim);
    for (int64_t c = threadIdx.x; c < dim; c += kLnThreads)
    {
      const float g = to_f<T>(dy[at + c]) * (gamma != nullptr ? gamma[c] : 1.0f);
      const float xh = (to_f<T>(x[at + c]) - mean) * rstd;
      dx[at + c] = from_f<T>(rstd * (g - s1 - xh * s2));
    }
  }
}

// the slices' sums, in a fixed order: 32 threads a column take every 32nd slice each (with eight, 296 slices of 4096 columns
// took 10 us)
__global__ void __launch_bounds__(1024)
layernorm_finish_kernel(const float *part, float *grad_gamma, float *grad_beta, int slices, int64_t dim, int accumulate)
{
  __shared__ float tile[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int group = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float *grad = blockIdx.y == 0 ? grad_gamma : grad_beta;
  if (grad == nullptr)
  {
    return;
  }
  float s = 0.0f;
  if (c < dim)
  {
    const float *src = part + static_cast<int64_t>(blockIdx.y) * dim + c;
#pragma unroll 10
    for (int i = group; i < slices; i += 32)
    {
      s += src[static_cast<int64_t>(i) * 2 * dim];
    }
  }
  tile[group][lane] = s;
  __syncthreads();
  s = tile[lane][group];   // a warp a column
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
  {
    s += __shfl_xor_sync(0xFFFFFFFFu, s, off);
  }
  const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 + group;
  if (lane == 0 && column < dim)
  {
    grad[column] = accumulate != 0 ? grad[column] + s : s;
  }
}

// ---- rows in registers ----
// WARPS warps own a row; a thread holds P pieces of V columns, 16 bytes each.  The row comes in once and all its loads are in flight
// together.  A row that does not begin with a piece begins
// `shift` columns into one, and its first and last piece are read and written element by element.

template <typename T, int V>
struct alignas(sizeof(T) * V) LnPiece
{
  T e[V];
};

// threads of a block: several short rows, or one long one
template <int WARPS>
constexpr int kLnSlots = WARPS < 8 ? 8 / WARPS : 1;
template <int WARPS>
constexpr int kLnBlock = WARPS * 32 * kLnSlots<WARPS>;

// a piece of a row from column c on, and back; its elements that are not the row's are zeros, or left alone
template <typename T, int V, bool SHIFT>
__device__ __forceinline__ LnPiece<T, V> load_piece(const T *row, int c, int dim)
{
  LnPiece<T, V> p;
  if (!SHIFT || (c >= 0 && c + V <= dim))
  {
    p = *reinterpret_cast<const LnPiece<T, V> *>(row + c);
  }
  else
  {
#pragma unroll
    for (int i = 0; i < V; ++i)
    {
      p.e[i] = c + i >= 0 && c + i < dim ? row[c + i] : from_f<T>(0.0f);
    }
  }
  return p;
}

template <typename T, int V, bool SHIFT>
__device__ __forceinline__ void store_piece(T *row, int c, int dim, const LnPiece<T, V> &p)
{
  if (!SHIFT || (c >= 0 && c + V <= dim))
  {
    *reinterpret_cast<LnPiece<T, V> *>(row + c) = p;
  }
  else
  {
#pragma unroll
    for (int i = 0; i < V; ++i)
    {
      if (c + i >= 0 && c + i < dim)
      {
        row[c + i] = p.e[i];
      }
    }
  }
}

// fp32 values of a piece's columns; `other` without a vector.  `vector`: p on a 16-byte boundary.  Columns that do not begin on one
// are taken out of the 16-byte pieces around them.
template <int V, bool SHIFT>
__device__ __forceinline__ void load_columns(float (&out)[V], const float *p, int c, int dim, bool vector, float other)
{
  if (p == nullptr)
  {
#pragma unroll
    for (int i = 0; i < V; ++i)
    {
      out[i] = other;
    }
    return;
  }
  const int skip = SHIFT ? c & 3 : 0;
  if (vector && c >= 0 && c - skip + V + (SHIFT ? 4 : 0) <= dim)
  {
    float f[V + 4];
#pragma unroll
    for (int i = 0; i < V + (SHIFT ? 4 : 0); i += 4)
    {
      const float4 v = __ldg(reinterpret_cast<const float4 *>(p + c - skip + i));
      f[i] = v.x;
      f[i + 1] = v.y;
      f[i + 2] = v.z;
      f[i + 3] = v.w;
    }
    if constexpr (SHIFT)
    {
#pragma unroll
      for (int i = 0; i < V + 2; ++i)
      {
        f[i] = (skip & 2) != 0 ? f[i + 2] : f[i];
      }
#pragma unroll
      for (int i = 0; i < V; ++i)
      {
        f[i] = (skip & 1) != 0 ? f[i + 1] : f[i];
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
    {
      out[i] = f[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
  {
    out[i] = c + i >= 0 && c + i < dim ? __ldg(p + c + i) : 0.0f;
  }
}

__device__ __forceinline__ bool on_16_dev(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// columns of the first piece that belong to the row before
template <int V>
__device__ __forceinline__ int shift_of(int64_t row, int dim)
{
  return static_cast<int>(row * dim % V);
}

// rows too wide for the form below, which keeps gamma and beta: one row a block
template <typename T, int V, int P, int WARPS, bool SHIFT>
__global__ void __launch_bounds__(WARPS * 32)
layernorm_fwd_rows_kernel(const T *x, const float *__restrict__ gamma, const float *__restrict__ beta, T *y,
                          float *__restrict__ mean_out, float *__restrict__ rstd_out, float epsilon, int dim)
{
  constexpr int THREADS = WARPS * 32;
  __shared__ float sums[WARPS];
  asm volatile("griddepcontrol.wait;" : "+l"(gamma), "+l"(beta)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t r = blockIdx.x;
  const bool vector = on_16_dev(gamma) && on_16_dev(beta);
  const int c0 = static_cast<int>(threadIdx.x) * V - (SHIFT ? shift_of<V>(r, dim) : 0);
  using Piece = LnPiece<T, V>;
  Piece v[P];
  const T *src = x + r * dim;
#pragma unroll
  for (int j = 0; j < P; ++j)
  {
    const int c = c0 + j * THREADS * V;
    if (c < dim)
    {
      v[j] = load_piece<T, V, SHIFT>(src, c, dim);
    }
  }
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < P; ++j)
  {
    if (c0 + j * THREADS * V < dim)
    {
#pragma unroll
      for (int i = 0; i < V; ++i)
      {
        s += to_f<T>(v[j].e[i]);
      }
    }
  }
  const float mean = sum_of<WARPS>(s, sums) / static_cast<float>(dim);
  s = 0.0f;
#pragma unroll
  for (int j = 0; j < P; ++j)
  {
    const int c = c0 + j * THREADS * V;
    if (c < dim)
    {
#pragma unroll
      for (int i = 0; i < V; ++i)
      {
        const float d = !SHIFT || (c + i >= 0 && c + i < dim) ? to_f<T>(v[j].e[i]) - mean : 0.0f;
        s = fmaf(d, d, s);
      }
    }
  }
  const float rstd = 1.0f / sqrtf(sum_of<WARPS>(s, sums) / static_cast<float>(dim) + epsilon);
  T *dst = y + r * dim;
#pragma unroll
  for (int j = 0; j < P; ++j)
  {
    const int c = c0 + j * THREADS * V;
    if (c < dim)
    {
      float g[V], b[V];
      load_columns<V, SHIFT>(g, gamma, c, dim, vector, 1.0f);
      load_columns<V, SHIFT>(b, beta, c, dim, vector, 0.0f);
      Piece o;
#pragma unroll
      for (int i = 0; i < V; ++i)
      {
        o.e[i] = from_f<T>(fmaf((to_f<T>(v[j].e[i]) - mean) * rstd, g[i], b[i]));
      }
      store_piece<T, V, SHIFT>(dst, c, dim, o);
    }
  }
  if (threadIdx.x == 0)
  {
    mean_out[r] = mean;
    rstd_out[r] = rstd;
  }
}

// part[slice][0][c] = sum of dy * xh, part[slice][1][c] = sum of dy over slice blockIdx.y of the rows: a warp every eighth row of it, a
// lane V neighbouring columns (V = 1, rows that are not whole pieces: eight columns, 32 apart); the eight warps' sums meet in shared
// memory.  HBM-bound: dy and x once.
template <typename T, int V>
__global__ void __launch_bounds__(kLnThreads)
layernorm_columns_kernel(const T *dy, const T *x, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                         float *__restrict__ part, int rows, int64_t dim)
{
  constexpr int N = V == 1 ? 8 : V;   // columns of a thread
  __shared__ float2 tile[kLnThreads / 32][32 * N + 1];
  asm volatile("griddepcontrol.wait;" : "+l"(mean_in), "+l"(rstd_in)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int64_t begin = static_cast<int64_t>(rows) * blockIdx.y / gridDim.y;
  const int64_t end = static_cast<int64_t>(rows) * (blockIdx.y + 1) / gridDim.y;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 32 * N;
  float sg[N], sb[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
  {
    sg[i] = sb[i] = 0.0f;
  }
#pragma unroll 2
  for (int64_t r = begin + warp; r < end; r += kLnThreads / 32)
  {
    const float mean = mean_in[r], rstd = rstd_in[r];
    T d[N], v[N];
    if constexpr (V > 1)
    {
      const int64_t c = first + lane * V;
      if (c < dim)
      {
        *reinterpret_cast<LnPiece<T, V> *>(d) = *reinterpret_cast<const LnPiece<T, V> *>(dy + r * dim + c);
        *reinterpret_cast<LnPiece<T, V> *>(v) = *reinterpret_cast<const LnPiece<T, V> *>(x + r * dim + c);
      }
    }
    else
    {
#pragma unroll
      for (int i = 0; i < N; ++i)
      {
        const int64_t c = first + lane + 32 * i;
        if (c < dim)
        {
          d[i] = dy[r * dim + c];
          v[i] = x[r * dim + c];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)   // (sums of columns that are not there are not stored)
    {
      const float g = to_f<T>(d[i]);
      sg[i] = fmaf(g, (to_f<T>(v[i]) - mean) * rstd, sg[i]);
      sb[i] += g;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
  {
    tile[warp][V > 1 ? lane * V + i : lane + 32 * i] = make_float2(sg[i], sb[i]);
  }
  __syncthreads();
  float *dst = part + static_cast<int64_t>(blockIdx.y) * 2 * dim;
  for (int i = threadIdx.x; i < 32 * N; i += kLnThreads)
  {
    if (first + i < dim)
    {
      float2 s = tile[0][i];
#pragma unroll
      for (int w = 1; w < kLnThreads / 32; ++w)
      {
        s.x += tile[w][i].x;
        s.y += tile[w][i].y;
      }
      dst[first + i] = s.x;
      dst[dim + first + i] = s.y;
    }
  }
}

// ---- many rows: a block takes rows one after the other ----
// gamma and beta (or the columns' sums of the backward pass) stay in registers from row to row, and the next rows are on their
// way: 16-byte pieces come by asynchronous copies through a ring of RING rows in shared memory, of which every thread reads
// back exactly what it copied, so that no barrier belongs to the copies.  A sum's slots alternate from row to row: one barrier a
// sum.
// Rows that are not whole pieces begin anywhere in one.  A block's rows are a multiple of V apart then, so that all of them begin
// `shift` columns into a piece and a thread's columns stay the same from row to row; the pieces that reach into a neighbouring row
// are masked, and stored element by element.

// blocks an SM
template <int WARPS, bool SHIFT>
constexpr int kFwdBlocks = WARPS <= 8 ? (SHIFT ? 2 : 3) : (WARPS <= 12 ? 2 : 1);
template <int WARPS>
constexpr int kBwdBlocks = WARPS <= 8 ? 2 : 1;

template <typename T>
constexpr int kLnRing = sizeof(T) == 4 ? 3 : 4;

// 16 bytes, of which the first `bytes` are read and the others zero
__device__ __forceinline__ void copy_16(void *to, const void *from, int bytes)
{
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from),
               "r"(bytes)
               : "memory");
}

// pairs of floats: Blackwell adds and multiplies two at a time, and these kernels would be bound by their instructions
// (forward, 16384 x 4096 bf16: 20 an element one by one, 0.75 of the issue slots, 54 us)
using Two = uint64_t;

__device__ __forceinline__ Two two(float a, float b)
{
  return static_cast<Two>(__float_as_uint(a)) | (static_cast<Two>(__float_as_uint(b)) << 32);
}
__device__ __forceinline__ float first_of(Two v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float second_of(Two v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ Two add2(Two a, Two b)
{
  Two d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b)
{
  Two d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c)
{
  Two d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// sums of N values a thread over WARPS warps of CL blocks of a cluster, every thread gets them; `slots` [N][CL * WARPS] must not be
// in use by an earlier sum that a barrier of these threads has not closed
template <int WARPS, int CL, int N>
__device__ __forceinline__ void sums_of(float (&v)[N], float (*slots)[CL * WARPS])
{
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
  {
#pragma unroll
    for (int n = 0; n < N; ++n)
    {
      v[n] += __shfl_xor_sync(0xFFFFFFFFu, v[n], off);
    }
  }
  const int lane = threadIdx.x & 31;
  if constexpr (CL > 1)
  {
    // a warp's sums go to every block's slots, a lane a block; one barrier of the cluster then serves block and cluster
    const int at = static_cast<int>(cluster_ctarank()) * WARPS + static_cast<int>(threadIdx.x >> 5);
    if (lane < CL)
    {
#pragma unroll
      for (int n = 0; n < N; ++n)
      {
        st_shared_cluster(map_to_cta(smem_u32(&slots[n][at]), static_cast<uint32_t>(lane)), v[n]);
      }
    }
    cluster_sync_all();
#pragma unroll
    for (int n = 0; n < N; ++n)
    {
      v[n] = 0.0f;
#pragma unroll
      for (int w = 0; w < CL * WARPS; w += 32)
      {
        v[n] += (CL * WARPS) % 32 == 0 || w + lane < CL * WARPS ? slots[n][w + lane] : 0.0f;
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
    {
#pragma unroll
      for (int n = 0; n < N; ++n)
      {
        v[n] += __shfl_xor_sync(0xFFFFFFFFu, v[n], off);
      }
    }
  }
  else if constexpr (WARPS > 1)
  {
    if (lane == 0)
    {
#pragma unroll
      for (int n = 0; n < N; ++n)
      {
        slots[n][(threadIdx.x >> 5) % WARPS] = v[n];
      }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n)
    {
      if constexpr (WARPS % 4 == 0)
      {
        const float4 *p = reinterpret_cast<const float4 *>(slots[n]);
        float4 s = p[0];
#pragma unroll
        for (int w = 1; w < WARPS / 4; ++w)
        {
          const float4 o = p[w];
          s.x += o.x;
          s.y += o.y;
          s.z += o.z;
          s.w += o.w;
        }
        v[n] = (s.x + s.y) + (s.z + s.w);
      }
      else
      {
        v[n] = slots[n][0];
#pragma unroll
        for (int w = 1; w < WARPS; ++w)
        {
          v[n] += slots[n][w];
        }
      }
    }
  }
}

// 1 / sqrt(v): the approximation and one step of Newton's method, except where the step would meet 0 * infinity
__device__ __forceinline__ float inverse_root(float v)
{
  const float r = rsqrtf(v);
  const float better = fmaf(0.5f * r, fmaf(-v * r, r, 1.0f), r);
  return v > 0.0f && v < __int_as_float(0x7F800000) ? better : r;
}

// the rows of N tensors that a block walks over: start() once, then next() for each row in turn gives this thread's pieces
template <typename T, int V, int P, int THREADS, int BLOCK, int N, bool SHIFT>
struct RowsAhead
{
  using Piece = LnPiece<T, V>;
  static constexpr int RING = kLnRing<T>;
  static constexpr size_t kBytes = static_cast<size_t>(RING) * N * P * BLOCK * 16;
  const T *src[N];
  int64_t row;     // the next row to fetch
  int64_t step;
  int rows, dim, t;
  int shift;       // columns of the first piece that belong to the row before
  uint4 *ring;
  int at;          // ring row that next() reads

  // first column of piece j; below 0 or past the row where the piece reaches into a neighbouring one
  __device__ __forceinline__ int column(int j) const { return (t + j * THREADS) * V - (SHIFT ? shift : 0); }

  // whether all of piece j, or nothing of it, is the row's
  __device__ __forceinline__ bool whole(int j) const { return !SHIFT || (column(j) >= 0 && column(j) + V <= dim) || column(j) >= dim; }

  __device__ __forceinline__ void fetch(int stage)
  {
    if (row < rows)
    {
      const int64_t left = (rows - row) * dim;   // elements from the row's first on
#pragma unroll
      for (int n = 0; n < N; ++n)
      {
#pragma unroll
        for (int j = 0; j < P; ++j)
        {
          const int c = column(j);
          if (c < dim)
          {
            // (of the tensor's last piece only what belongs to it)
            const int bytes = SHIFT && left - c < V ? static_cast<int>(left - c) * static_cast<int>(sizeof(T)) : 16;
            copy_16(ring + ((stage * N + n) * P + j) * BLOCK + threadIdx.x, src[n] + row * dim + c, bytes);
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    row += step;
  }

  __device__ __forceinline__ void start()
  {
    at = 0;
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
    {
      fetch(i);
    }
  }

  // the row's values of this thread in pairs; zeros where the thread has no column, or the block no row
  __device__ __forceinline__ void next(Two (&out)[N][P * V / 2], bool live)
  {
    // (the ring row before this one, which this thread has read, is filled again)
    fetch(at == 0 ? RING - 1 : at - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
#pragma unroll
    for (int n = 0; n < N; ++n)
    {
#pragma unroll
      for (int j = 0; j < P; ++j)
      {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        const int c = column(j);
        if (live && c < dim)
        {
          v = ring[((at * N + n) * P + j) * BLOCK + threadIdx.x];
          if (!whole(j))
          {
            mask(v, c);
          }
        }
        pairs_of(out[n] + j * (V / 2), v);
      }
    }
    at = at == RING - 1 ? 0 : at + 1;
  }

  // zeros for the elements of a piece that are not the row's
  __device__ __forceinline__ void mask(uint4 &v, int c) const
  {
    Piece p = *reinterpret_cast<const Piece *>(&v);
#pragma unroll
    for (int i = 0; i < V; ++i)
    {
      if (c + i < 0 || c + i >= dim)
      {
        p.e[i] = from_f<T>(0.0f);
      }
    }
    v = *reinterpret_cast<const uint4 *>(&p);
  }

  static __device__ __forceinline__ void pairs_of(Two *out, const uint4 &v)
  {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (sizeof(T) == 4)
    {
      out[0] = static_cast<Two>(w[0]) | (static_cast<Two>(w[1]) << 32);
      out[1] = static_cast<Two>(w[2]) | (static_cast<Two>(w[3]) << 32);
    }
    else
    {
#pragma unroll
      for (int i = 0; i < 4; ++i)
      {
        const LnPiece<T, 2> p = *reinterpret_cast<const LnPiece<T, 2> *>(&w[i]);
        out[i] = two(to_f<T>(p.e[0]), to_f<T>(p.e[1]));
      }
    }
  }

  // the row's results
  __device__ __forceinline__ void store(T *row_out, const Two (&v)[P * V / 2]) const
  {
#pragma unroll
    for (int j = 0; j < P; ++j)
    {
      const int c = column(j);
      if (c < dim)
      {
        Piece o;
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
          const int e = j * V + i;
          o.e[i] = from_f<T>((e & 1) != 0 ? second_of(v[e / 2]) : first_of(v[e / 2]));
        }
        if (whole(j))
        {
          *reinterpret_cast<Piece *>(row_out + c) = o;
        }
        else
        {
#pragma unroll
          for (int i = 0; i < V; ++i)
          {
            if (c + i >= 0 && c + i < dim)
            {
              row_out[c + i] = o.e[i];
            }
          }
        }
      }
    }
  }

  // column of element e of the thread, and whether the row has it
  __device__ __forceinline__ int column_of(int e) const { return column(e / V) + e % V; }
  __device__ __forceinline__ bool has(int e) const { return column_of(e) >= 0 && column_of(e) < dim; }

  // fp32 values of this thread's columns; `other` without a vector, zeros where the thread has no column
  __device__ __forceinline__ void columns(Two (&out)[P * V / 2], const float *p, float other) const
  {
    float f[P * V];
#pragma unroll
    for (int j = 0; j < P; ++j)
    {
      if (!SHIFT && column(j) < dim && p != nullptr && on_16_dev(p))
      {
#pragma unroll
        for (int i = 0; i < V; i += 4)
        {
          const float4 v = __ldg(reinterpret_cast<const float4 *>(p + column(j) + i));
          f[j * V + i] = v.x;
          f[(j * V + i + 1) % (P * V)] = v.y;
          f[(j * V + i + 2) % (P * V)] = v.z;
          f[(j * V + i + 3) % (P * V)] = v.w;
        }
      }
      else
      {
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
          const int e = j * V + i;
          f[e] = !has(e) ? 0.0f : (p != nullptr ? __ldg(p + column_of(e)) : other);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < P * V; e += 2)
    {
      out[e / 2] = two(f[e], f[e + 1]);
    }
  }
};

template <typename T, int V, int P, int WARPS, bool SHIFT>
__global__ void __launch_bounds__(kLnBlock<WARPS>, kFwdBlocks<WARPS, SHIFT>)
layernorm_fwd_many_kernel(const T *x, const float *__restrict__ gamma, const float *__restrict__ beta, T *y,
                          float *__restrict__ mean_out, float *__restrict__ rstd_out, float epsilon, int rows, int dim)
{
  constexpr int BLOCK = kLnBlock<WARPS>;
  constexpr int SLOTS = kLnSlots<WARPS>;
  constexpr int THREADS = WARPS * 32;
  constexpr int PAIRS = P * V / 2;
  extern __shared__ uint4 ln_ring[];
  __shared__ __align__(16) float sums[2][2][SLOTS][1][WARPS];
  asm volatile("griddepcontrol.wait;" : "+l"(gamma), "+l"(beta)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int slot = threadIdx.x / THREADS;
  const int t = threadIdx.x % THREADS;
  const int first = static_cast<int>(blockIdx.x) * SLOTS;
  const int step = static_cast<int>(gridDim.x) * SLOTS;
  RowsAhead<T, V, P, THREADS, BLOCK, 1, SHIFT> in;
  in.src[0] = x;
  in.row = first + slot;
  in.step = step;
  in.rows = rows;
  in.dim = dim;
  in.t = t;
  in.shift = SHIFT ? static_cast<int>(static_cast<int64_t>(first + slot) * dim % V) : 0;
  in.ring = ln_ring;
  in.start();
  Two g[PAIRS], b[PAIRS];
  in.columns(g, gamma, 1.0f);
  in.columns(b, beta, 0.0f);
  const float inverse = 1.0f / static_cast<float>(dim);
  int turn = 0;
  for (int64_t base = first; base < rows; base += step, turn ^= 1)   // (every slot takes part in the sums' barriers)
  {
    const int64_t r = base + slot;
    const bool live = r < rows;
    Two v[1][PAIRS];
    in.next(v, live);
    Two a = v[0][0];
#pragma unroll
    for (int i = 1; i < PAIRS; ++i)
    {
      a = add2(a, v[0][i]);
    }
    float s[1] = {first_of(a) + second_of(a)};
    sums_of<WARPS, 1>(s, sums[turn][0][slot]);
    const float mean = s[0] * inverse;
    a = two(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
    {
      v[0][i] = add2(v[0][i], two(-mean, -mean));
      if (i % (V / 2) == V / 2 - 1)   // the piece's last pair
      {
        constexpr int H = V / 2;
        const int j = i / H;
        if (in.column(j) >= dim)
        {
#pragma unroll
          for (int k = 0; k < H; ++k)
          {
            v[0][j * H + k] = two(0.0f, 0.0f);
          }
        }
        else if (!in.whole(j))
        {
#pragma unroll
          for (int k = 0; k < H; ++k)
          {
            const int e = 2 * (j * H + k);
            v[0][j * H + k] = two(in.has(e) ? first_of(v[0][j * H + k]) : 0.0f, in.has(e + 1) ? second_of(v[0][j * H + k]) : 0.0f);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
    {
      a = fma2(v[0][i], v[0][i], a);
    }
    s[0] = first_of(a) + second_of(a);
    sums_of<WARPS, 1>(s, sums[turn][1][slot]);
    const float rstd = inverse_root(fmaf(s[0], inverse, epsilon));
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
    {
      v[0][i] = fma2(mul2(v[0][i], two(rstd, rstd)), g[i], b[i]);
    }
    if (live)
    {
      in.store(y + r * dim, v[0]);
      if (t == 0)
      {
        mean_out[r] = mean;
        rstd_out[r] = rstd;
      }
    }
  }
}

// dx and this block's share of dgamma and dbeta in one pass: a thread keeps its columns' sums over all rows of the block, a fp32 chain of
// rows / 296 up to 8192 columns and of rows / 74, 32 or 16 in clusters of 2, 4 or 8 blocks.
// part[block][0][c], part[block][1][c] as in layernorm_columns_kernel.  A row of more than 8192 columns takes a cluster of CL blocks,
// which share its sums; the cluster's barrier costs 0.7 us a row, and still 16384 columns run at 0.48 (bf16) and 0.67 (fp32) of the copy
// rate where two launches, the columns' sums and dx, reach 0.31 and 0.42.  (Waiting for a row's sums only after the next row's are taken
// hides the barrier but reads and converts the ring twice: 0.44, 0.65.  Clusters of four smaller blocks, two an SM: 0.47, 0.69, but 0.55
// instead of 0.70 where one block does.)
template <typename T, int V, int P, int WARPS, int CL, bool SHIFT>
__global__ void __launch_bounds__(kLnBlock<WARPS>, kBwdBlocks<WARPS>)
layernorm_bwd_rows_kernel(const T *dy, const T *x, const float *__restrict__ gamma, const float *__restrict__ mean_in,
                          const float *__restrict__ rstd_in, T *dx, float *__restrict__ part, int rows, int dim)
{
  constexpr int BLOCK = kLnBlock<WARPS>;
  constexpr int SLOTS = kLnSlots<WARPS>;
  constexpr int THREADS = CL * WARPS * 32;   // of a row
  constexpr int PAIRS = P * V / 2;
  extern __shared__ uint4 ln_ring[];   // the ring; then, where SLOTS > 1, the columns' sums [2][dim]
  __shared__ __align__(16) float sums[2][SLOTS][2][CL * WARPS];
  asm volatile("griddepcontrol.wait;" : "+l"(gamma), "+l"(mean_in), "+l"(rstd_in)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  using Rows = RowsAhead<T, V, P, THREADS, BLOCK, 2, SHIFT>;
  const int slot = threadIdx.x / (WARPS * 32);
  const int t = (CL > 1 ? static_cast<int>(cluster_ctarank()) * WARPS * 32 : 0) + threadIdx.x % (WARPS * 32);
  const int first = static_cast<int>(blockIdx.x) / CL * SLOTS;
  const int step = static_cast<int>(gridDim.x) / CL * SLOTS;
  Rows in;
  in.src[0] = x;
  in.src[1] = dy;
  in.row = first + slot;
  in.step = step;
  in.rows = rows;
  in.dim = dim;
  in.t = t;
  in.shift = SHIFT ? static_cast<int>(static_cast<int64_t>(first + slot) * dim % V) : 0;
  in.ring = ln_ring;
  in.start();
  if constexpr (CL > 1)
  {
    cluster_sync_all();   // every block's slots are there before another writes to them
  }
  Two g[PAIRS], sg[PAIRS], sb[PAIRS];
  in.columns(g, gamma, 1.0f);
#pragma unroll
  for (int i = 0; i < PAIRS; ++i)
  {
    sg[i] = sb[i] = two(0.0f, 0.0f);
  }
  const float inverse = 1.0f / static_cast<float>(dim);
  // the statistics of this row and the two after it
  float means[3], rstds[3];
  auto statistics = [&](int64_t r, float &m, float &s) {
    m = r < rows ? mean_in[r] : 0.0f;
    s = r < rows ? rstd_in[r] : 0.0f;
  };
  for (int i = 0; i < 3; ++i)
  {
    statistics(first + slot + i * static_cast<int64_t>(step), means[i], rstds[i]);
  }
  int turn = 0;
  for (int64_t base = first; base < rows; base += step, turn ^= 1)   // (every slot takes part in the sums' barriers)
  {
    const int64_t r = base + slot;
    const bool live = r < rows;
    Two v[2][PAIRS];   // x, then x_hat; dy, then dy * gamma
    in.next(v, live);
    const float mean = means[0];
    const float rstd = rstds[0];
    means[0] = means[1];
    rstds[0] = rstds[1];
    means[1] = means[2];
    rstds[1] = rstds[2];
    statistics(r + 3 * static_cast<int64_t>(step), means[2], rstds[2]);
    Two a = two(0.0f, 0.0f), b = two(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
    {
      v[0][i] = mul2(add2(v[0][i], two(-mean, -mean)), two(rstd, rstd));
      sg[i] = fma2(v[1][i], v[0][i], sg[i]);
      sb[i] = add2(sb[i], v[1][i]);
      v[1][i] = mul2(v[1][i], g[i]);
      a = add2(a, v[1][i]);
      b = fma2(v[1][i], v[0][i], b);
    }
    float s[2] = {first_of(a) + second_of(a), first_of(b) + second_of(b)};
    sums_of<WARPS, CL>(s, sums[turn][slot]);
    const float s1 = -s[0] * inverse;
    const float s2 = -s[1] * inverse;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
    {
      v[1][i] = mul2(fma2(v[0][i], two(s2, s2), add2(v[1][i], two(s1, s1))), two(rstd, rstd));
    }
    if (live)
    {
      in.store(dx + r * dim, v[1]);
    }
  }
  if (part == nullptr)
  {
    return;
  }
  float *columns = reinterpret_cast<float *>(reinterpret_cast<char *>(ln_ring) + Rows::kBytes);
  float *mine = part + static_cast<int64_t>(blockIdx.x / CL) * 2 * dim;
  float *to = SLOTS > 1 ? columns : mine;
#pragma unroll 1
  for (int turns = 0; turns < SLOTS; ++turns)   // slot by slot, in order
  {
    if (slot == turns)
    {
#pragma unroll
      for (int e = 0; e < P * V; ++e)
      {
        const int c = in.column_of(e);
        if (c >= 0 && c < dim)
        {
          const float vg = (e & 1) != 0 ? second_of(sg[e / 2]) : first_of(sg[e / 2]);
          const float vb = (e & 1) != 0 ? second_of(sb[e / 2]) : first_of(sb[e / 2]);
          to[c] = turns > 0 ? to[c] + vg : vg;
          to[dim + c] = turns > 0 ? to[dim + c] + vb : vb;
        }
      }
    }
    if (SLOTS > 1)
    {
      __syncthreads();
    }
  }
  if (SLOTS > 1)
  {
    for (int c = threadIdx.x; c < 2 * dim; c += BLOCK)
    {
      mine[c] = columns[c];
    }
  }
}

// slices of rows with partial sums of their own, at most
int ln_slices(int rows) { return rows < 148 * 2 ? rows : 148 * 2; }

unsigned ln_grid(int rows) { return static_cast<unsigned>(rows < 148 * 8 ? rows : 148 * 8); }

constexpr size_t kLnPlainSmem = 40 * 1024;   // dynamic, beside the static slots, without asking

bool on_16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// columns that the threads of a row must reach: its own, and those of its first piece that are not
template <int V>
int64_t reach_of(int dim)
{
  return static_cast<int64_t>(dim) + (dim % V != 0 ? V - 1 : 0);
}

// clusters of CL blocks that the SMs hold at a time, one block an SM: those of four and eight do not fill every group of SMs
template <int CL>
constexpr int kLnClusters = CL == 1 ? 148 : (CL == 2 ? 74 : (CL == 4 ? 32 : 16));

// blocks (or clusters) of a launch that walks over the rows: one wave.  Where rows are not whole pieces a block's rows lie a multiple
// of V apart.
template <int V>
int walk_blocks(int rows, int slots, int dim, int most)
{
  const int blocks = (rows - 1) / slots + 1;
  return blocks <= most ? blocks : (dim % V != 0 ? most / 8 * 8 : most);
}

template <typename T, int V, int P, int WARPS>
int ln_fwd_rows(const T *x, const float *gamma, const float *beta, T *y, float *mean, float *rstd, float epsilon, int rows,
                int dim, cudaStream_t s)
{
  auto kernel = dim % V == 0 ? layernorm_fwd_rows_kernel<T, V, P, WARPS, false> : layernorm_fwd_rows_kernel<T, V, P, WARPS, true>;
  CAIFQ_CHECK_CUDA(launch_dependent(kernel, dim3(static_cast<unsigned>(rows)), dim3(WARPS * 32), 0, s, x, gamma, beta, y, mean, rstd, epsilon, dim));
  return CAIFQ_OK;
}

// dynamic shared memory beyond 48 KB is asked for once per kernel and device
template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes, std::atomic<uint64_t> &done)
{
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev < 0 || dev >= kMaxDevices || (done.load(std::memory_order_relaxed) >> dev & 1u) != 0)
  {
    return e;
  }
  const cudaError_t set =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (set == cudaSuccess)
  {
    done.fetch_or(static_cast<uint64_t>(1) << dev, std::memory_order_relaxed);
  }
  return set;
}

template <typename T, int V, int P, int WARPS, bool SHIFT>
int ln_fwd_many(const T *x, const float *gamma, const float *beta, T *y, float *mean, float *rstd, float epsilon, int rows,
                int dim, cudaStream_t s)
{
  constexpr int BLOCK = kLnBlock<WARPS>;
  constexpr size_t kBytes = RowsAhead<T, V, P, WARPS * 32, BLOCK, 1, SHIFT>::kBytes;
  static std::atomic<uint64_t> done{0};
  auto kernel = layernorm_fwd_many_kernel<T, V, P, WARPS, SHIFT>;
  if (kBytes > kLnPlainSmem)
  {
    CAIFQ_CHECK_CUDA(allow_smem(kernel, kBytes, done));
  }
  const int blocks = walk_blocks<V>(rows, kLnSlots<WARPS>, dim, 148 * kFwdBlocks<WARPS, SHIFT>);
  CAIFQ_CHECK_CUDA(launch_dependent(kernel, dim3(static_cast<unsigned>(blocks)), dim3(BLOCK), kBytes, s, x, gamma, beta, y, mean, rstd, epsilon, rows, dim));
  return CAIFQ_OK;
}

// the fewest warps whose registers hold `reach` columns, ELEMENTS of them a thread
#define CAIFQ_LN_CASE(CALL, W, ELEMENTS) \
  if (reach <= 32 * (W) * (ELEMENTS))    \
  {                                      \
    return CALL(W);                      \
  }
#define CAIFQ_LN_WARPS(CALL, ELEMENTS) \
  CAIFQ_LN_CASE(CALL, 1, ELEMENTS)     \
  CAIFQ_LN_CASE(CALL, 2, ELEMENTS)     \
  CAIFQ_LN_CASE(CALL, 3, ELEMENTS)     \
  CAIFQ_LN_CASE(CALL, 4, ELEMENTS)     \
  CAIFQ_LN_CASE(CALL, 6, ELEMENTS)     \
  CAIFQ_LN_CASE(CALL, 8, ELEMENTS)     \
  CAIFQ_LN_CASE(CALL, 10, ELEMENTS)    \
  CAIFQ_LN_CASE(CALL, 12, ELEMENTS)    \
  CAIFQ_LN_CASE(CALL, 16, ELEMENTS)

// the fewest blocks of a cluster, and then the fewest warps, that hold them
#define CAIFQ_LN_CLUSTER_CASE(CALL, W, CL, ELEMENTS)               \
  if (reach <= static_cast<int64_t>(32) * (W) * (CL) * (ELEMENTS)) \
  {                                                                \
    return CALL(W, CL);                                            \
  }
#define CAIFQ_LN_CLUSTERS(CALL, ELEMENTS)     \
  CAIFQ_LN_CLUSTER_CASE(CALL, 10, 2, ELEMENTS) \
  CAIFQ_LN_CLUSTER_CASE(CALL, 12, 2, ELEMENTS) \
  CAIFQ_LN_CLUSTER_CASE(CALL, 16, 2, ELEMENTS) \
  CAIFQ_LN_CLUSTER_CASE(CALL, 12, 4, ELEMENTS) \
  CAIFQ_LN_CLUSTER_CASE(CALL, 16, 4, ELEMENTS) \
  CAIFQ_LN_CLUSTER_CASE(CALL, 16, 8, ELEMENTS)

template <typename T>
int ln_fwd(const void *xv, const float *gamma, const float *beta, void *yv, float *mean, float *rstd, float epsilon, int rows,
           int dim, cudaStream_t s)
{
  const T *x = static_cast<const T *>(xv);
  T *y = static_cast<T *>(yv);
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  if (on_16(x) && on_16(y))
  {
    const int64_t reach = reach_of<V>(dim);
    // (gamma and beta of 16 columns a thread fit the registers)
    if (dim % V == 0)
    {
      if (dim <= 32 * V)
      {
        return ln_fwd_many<T, V, 1, 1, false>(x, gamma, beta, y, mean, rstd, epsilon, rows, dim, s);
      }
#define CAIFQ_LN_CALL(W) ln_fwd_many<T, V, 16 / V, W, false>(x, gamma, beta, y, mean, rstd, epsilon, rows, dim, s)
      CAIFQ_LN_WARPS(CAIFQ_LN_CALL, 16)
#undef CAIFQ_LN_CALL
    }
    else
    {
#define CAIFQ_LN_CALL(W) ln_fwd_many<T, V, 16 / V, W, true>(x, gamma, beta, y, mean, rstd, epsilon, rows, dim, s)
      CAIFQ_LN_WARPS(CAIFQ_LN_CALL, 16)
#undef CAIFQ_LN_CALL
    }
    if (sizeof(T) == 2 && reach <= 512 * 4 * V)
    {
      return ln_fwd_rows<T, V, 4, 16>(x, gamma, beta, y, mean, rstd, epsilon, rows, dim, s);
    }
    if (reach <= 1024 * 4 * V)
    {
      return ln_fwd_rows<T, V, 4, 32>(x, gamma, beta, y, mean, rstd, epsilon, rows, dim, s);
    }
  }
  CAIFQ_CHECK_CUDA(launch_dependent(layernorm_fwd_kernel<T>, dim3(ln_grid(rows)), dim3(kLnThreads), 0, s, x, gamma, beta, y,
                                    mean, rstd, epsilon, rows, static_cast<int64_t>(dim)));
  return CAIFQ_OK;
}

template <typename T, int V, int P, int WARPS, int CL, bool SHIFT>
int ln_bwd_rows(const T *dy, const T *x, const float *gamma, const float *mean, const float *rstd, T *dx, float *part,
                int *slices, int rows, int dim, cudaStream_t s)
{
  constexpr int BLOCK = kLnBlock<WARPS>;
  constexpr int SLOTS = kLnSlots<WARPS>;
  constexpr size_t kBytes = RowsAhead<T, V, P, CL * WARPS * 32, BLOCK, 2, SHIFT>::kBytes;
  constexpr size_t kColumns = SLOTS > 1 ? sizeof(float) * 2 * P * V * WARPS * 32 : 0;   // of the widest row
  static std::atomic<uint64_t> done{0};
  auto kernel = layernorm_bwd_rows_kernel<T, V, P, WARPS, CL, SHIFT>;
  if (kBytes + kColumns > kLnPlainSmem)
  {
    CAIFQ_CHECK_CUDA(allow_smem(kernel, kBytes + kColumns, done));
  }
  *slices = walk_blocks<V>(rows, SLOTS, dim, kLnClusters<CL> * kBwdBlocks<WARPS>);
  const dim3 grid(static_cast<unsigned>(*slices * CL));
  const size_t smem = kBytes + (SLOTS > 1 ? sizeof(float) * 2 * static_cast<size_t>(dim) : 0);
  if constexpr (CL == 1)
  {
    CAIFQ_CHECK_CUDA(launch_dependent(kernel, grid, dim3(BLOCK), smem, s, dy, x, gamma, mean, rstd, dx, part, rows, dim));
  }
  else
  {
    CAIFQ_CHECK_CUDA(launch_dependent_clusters(kernel, grid, dim3(BLOCK), smem, s, CL, dy, x, gamma, mean, rstd, dx, part, rows, dim));
  }
  return CAIFQ_OK;
}

// part: null where the columns' sums are not wanted; *slices: how many of them the launches leave
template <typename T>
int ln_bwd(const void *dyv, const void *xv, const float *gamma, const float *mean, const float *rstd, void *dxv, float *part,
           int *slices, int rows, int dim, cudaStream_t s)
{
  const T *dy = static_cast<const T *>(dyv);
  const T *x = static_cast<const T *>(xv);
  T *dx = static_cast<T *>(dxv);
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  const bool pieces = on_16(dy) && on_16(x) && on_16(dx);
  const int64_t reach = reach_of<V>(dim);
  if (pieces && dim % V == 0)
  {
    if (dim <= 32 * V)
    {
      return ln_bwd_rows<T, V, 1, 1, 1, false>(dy, x, gamma, mean, rstd, dx, part, slices, rows, dim, s);
    }
#define CAIFQ_LN_CLUSTER_CALL(W, CL) ln_bwd_rows<T, V, 16 / V, W, CL, false>(dy, x, gamma, mean, rstd, dx, part, slices, rows, dim, s)
#define CAIFQ_LN_CALL(W) CAIFQ_LN_CLUSTER_CALL(W, 1)
    CAIFQ_LN_WARPS(CAIFQ_LN_CALL, 16)
    CAIFQ_LN_CLUSTERS(CAIFQ_LN_CLUSTER_CALL, 16)
#undef CAIFQ_LN_CALL
#undef CAIFQ_LN_CLUSTER_CALL
  }
  else if (pieces)
  {
    constexpr int P = V == 4 ? 3 : 2;   // (four shifted pieces of two tensors in fp32 do not fit the registers)
#define CAIFQ_LN_CLUSTER_CALL(W, CL) ln_bwd_rows<T, V, P, W, CL, true>(dy, x, gamma, mean, rstd, dx, part, slices, rows, dim, s)
#define CAIFQ_LN_CALL(W) CAIFQ_LN_CLUSTER_CALL(W, 1)
    CAIFQ_LN_WARPS(CAIFQ_LN_CALL, P * V)
    CAIFQ_LN_CLUSTERS(CAIFQ_LN_CLUSTER_CALL, P * V)
#undef CAIFQ_LN_CALL
#undef CAIFQ_LN_CLUSTER_CALL
  }
  // slices of at least 64 rows: a warp takes every eighth.  (Of 8 rows, when this launch served rows of 8192 columns and more: 512 x 10000
  // bf16 34.7 us instead of 25.7, 2000 x 12000 140 instead of 90, 100 x 12000 13.0 instead of 13.7)
  const int most = rows / 64 < 1 ? 1 : rows / 64;
  *slices = most < ln_slices(rows) ? most : ln_slices(rows);
  if (part != nullptr)
  {
    // (before dx, which may be written over dy)
    const bool whole = pieces && dim % V == 0;
    const int wide = 32 * (whole ? V : 8);
    CAIFQ_CHECK_CUDA(launch_dependent(whole ? layernorm_columns_kernel<T, V> : layernorm_columns_kernel<T, 1>,
                                      dim3(static_cast<unsigned>((static_cast<int64_t>(dim) + wide - 1) / wide), static_cast<unsigned>(*slices)),
                                      dim3(kLnThreads), 0, s, dy, x, mean, rstd, part, rows, static_cast<int64_t>(dim)));
  }
  CAIFQ_CHECK_CUDA(launch_dependent(layernorm_dx_kernel<T>, dim3(ln_grid(rows)), dim3(kLnThreads), 0, s, dy, x, gamma, mean,
                                    rstd, dx, rows, static_cast<int64_t>(dim)));
  return CAIFQ_OK;
}

}  // namespace

size_t layernorm_bwd_workspace_bytes(int rows, int dim)
{
  return static_cast<size_t>(ln_slices(rows)) * 2 * static_cast<size_t>(dim) * sizeof(float);
}

int launch_layernorm_fwd(const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd,
                         float epsilon, int dtype, int rows, int dim, cudaStream_t s)
{
  if (rows <= 0)
  {
    return CAIFQ_OK;
  }
  switch (dtype)
  {
    case CAIFQ_F32:
      return ln_fwd<float>(x, gamma, beta, y, mean, rstd, epsilon, rows, dim, s);
    case CAIFQ_F16:
      return ln_fwd<__half>(x, gamma, beta, y, mean, rstd, epsilon, rows, dim, s);
    default:
      return ln_fwd<__nv_bfloat16>(x, gamma, beta, y, mean, rstd, epsilon, rows, dim, s);
  }
}

int launch_layernorm_bwd(const void *dy, const void *x, const float *gamma, const float *mean, const float *rstd, void *dx,
                         float *grad_gamma, float *grad_beta, int accumulate, float *workspace, int dtype, int rows, int dim,
                         cudaStream_t s)
{
  const bool columns = grad_gamma != nullptr || grad_beta != nullptr;
  int slices = 0;
  if (rows > 0)
  {
    float *part = columns ? workspace : nullptr;
    int rc = CAIFQ_OK;
    switch (dtype)
    {
      case CAIFQ_F32:
        rc = ln_bwd<float>(dy, x, gamma, mean, rstd, dx, part, &slices, rows, dim, s);
        break;
      case CAIFQ_F16:
        rc = ln_bwd<__half>(dy, x, gamma, mean, rstd, dx, part, &slices, rows, dim, s);
        break;
      default:
        rc = ln_bwd<__nv_bfloat16>(dy, x, gamma, mean, rstd, dx, part, &slices, rows, dim, s);
        break;
    }
    if (rc != CAIFQ_OK)
    {
      return rc;
    }
  }
  if (columns)
  {
    CAIFQ_CHECK_CUDA(launch_dependent(layernorm_finish_kernel, dim3(static_cast<unsigned>((static_cast<int64_t>(dim) + 31) / 32), 2), dim3(1024), 0, s,
                                      static_cast<const float *>(workspace), grad_gamma, grad_beta, slices,
                                      static_cast<int64_t>(dim), accumulate));
  }
  return CAIFQ_OK;
}

}  // namespace caifq
