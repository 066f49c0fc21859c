// Layer norm in front of the frozen projections, the other norm beside norm.cu's RMSNorm:
//   mean = sum x / n, rstd = 1 / sqrt(sum (x - mean)^2 / n + epsilon), y = (x - mean) * rstd * gamma + beta
//   xh = (x - mean) * rstd, g = dy * gamma
//   dx = rstd * (g - sum(g) / n - xh * sum(g * xh) / n),  dgamma = sum_rows dy * xh,  dbeta = sum_rows dy
// All sums are fp32 and run in a fixed order: a row's variance is taken around its mean (a second pass over the row, not the
// difference of two large sums), and the gradients of gamma and beta are partial sums per slice of rows, added slice by
// slice by a second launch, so that two calls give the same bits.  y and dx are rounded once.
#include <atomic>

#include "common.cuh"

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

// ---- any width, any alignment: a CTA a row, the row read from memory (the cache) in every pass ----

template <typename T>
__global__ void __launch_bounds__(kLnThreads)
layernorm_fwd_kernel(const T *x, const float *__restrict__ gamma, const float *__restrict__ beta, T *y,
                     float *__restrict__ mean_out, float *__restrict__ rstd_out, float epsilon, int rows, int64_t dim)
{
  __shared__ float slots[kLnThreads / 32];
  asm volatile("griddepcontrol.wait;" : "+l"(gamma), "+l"(beta)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int r = blockIdx.x; r < rows; r += gridDim.x)
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
  for (int r = blockIdx.x; r < rows; r += gridDim.x)
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

// partial sums over slice blockIdx.y of the rows: part[slice][0][c] = sum dy * xh, part[slice][1][c] = sum dy
template <typename T>
__global__ void __launch_bounds__(kLnThreads)
layernorm_columns_kernel(const T *dy, const T *x, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                         float *__restrict__ part, int rows, int64_t dim)
{
  __shared__ float2 tile[8][33];
  asm volatile("griddepcontrol.wait;" : "+l"(mean_in), "+l"(rstd_in)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int group = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const int64_t begin = static_cast<int64_t>(rows) * blockIdx.y / gridDim.y;
  const int64_t end = static_cast<int64_t>(rows) * (blockIdx.y + 1) / gridDim.y;
  float2 s = make_float2(0.0f, 0.0f);
  if (c < dim)
  {
    for (int64_t r = begin + group; r < end; r += 8)
    {
      const float g = to_f<T>(dy[r * dim + c]);
      s.x = fmaf(g, (to_f<T>(x[r * dim + c]) - mean_in[r]) * rstd_in[r], s.x);
      s.y += g;
    }
  }
  tile[group][lane] = s;
  __syncthreads();
  if (group == 0 && c < dim)
  {
    for (int i = 1; i < 8; ++i)
    {
      s.x += tile[i][lane].x;
      s.y += tile[i][lane].y;
    }
    float *dst = part + static_cast<int64_t>(blockIdx.y) * 2 * dim + c;
    dst[0] = s.x;
    dst[dim] = s.y;
  }
}

// the slices' sums, in a fixed order: eight threads a column take every eighth slice each
__global__ void __launch_bounds__(kLnThreads)
layernorm_finish_kernel(const float *part, float *grad_gamma, float *grad_beta, int slices, int64_t dim, int accumulate)
{
  __shared__ float tile[8][33];
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
#pragma unroll 8
    for (int i = group; i < slices; i += 8)
    {
      s += src[static_cast<int64_t>(i) * 2 * dim];
    }
  }
  tile[group][lane] = s;
  __syncthreads();
  if (group == 0 && c < dim)
  {
    for (int i = 1; i < 8; ++i)
    {
      s += tile[i][lane];
    }
    grad[c] = accumulate != 0 ? grad[c] + s : s;
  }
}

// ---- rows in registers ----
// WARPS warps own a row; a thread holds P pieces of V columns, 16 bytes each where the rows allow it (V = 1: rows off a
// 16-byte boundary or of odd length, element by element).  The row comes in once and all its loads are in flight together.

template <typename T, int V>
struct alignas(sizeof(T) * V) LnPiece
{
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_floats(float (&out)[V], const float *p, float other)
{
  if (p == nullptr)
  {
#pragma unroll
    for (int i = 0; i < V; ++i)
    {
      out[i] = other;
    }
  }
  else if constexpr (V >= 4)
  {
#pragma unroll
    for (int i = 0; i < V; i += 4)
    {
      const float4 v = __ldg(reinterpret_cast<const float4 *>(p + i));
      out[i] = v.x;
      out[i + 1] = v.y;
      out[i + 2] = v.z;
      out[i + 3] = v.w;
    }
  }
  else
  {
#pragma unroll
    for (int i = 0; i < V; ++i)
    {
      out[i] = __ldg(p + i);
    }
  }
}

// threads of a block: several short rows, or one long one
template <int WARPS, int LEAST>
constexpr int kLnBlock = WARPS * 32 > LEAST ? WARPS * 32 : LEAST;

template <typename T, int V, int P, int WARPS>
__global__ void __launch_bounds__(kLnBlock<WARPS, 128>)
layernorm_fwd_rows_kernel(const T *x, const float *__restrict__ gamma, const float *__restrict__ beta, T *y,
                          float *__restrict__ mean_out, float *__restrict__ rstd_out, float epsilon, int rows, int dim)
{
  constexpr int SLOTS = kLnBlock<WARPS, 128> / (WARPS * 32);
  constexpr int THREADS = WARPS * 32;   // of a row
  __shared__ float sums[SLOTS][WARPS];
  asm volatile("griddepcontrol.wait;" : "+l"(gamma), "+l"(beta)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int slot = threadIdx.x / THREADS;
  const int t = threadIdx.x % THREADS;
  const int r = blockIdx.x * SLOTS + slot;
  const bool live = r < rows;
  using Piece = LnPiece<T, V>;
  Piece v[P];
  const T *src = x + static_cast<int64_t>(live ? r : 0) * dim;
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < P; ++j)
  {
    const int c = (t + j * THREADS) * V;
    if (live && c < dim)
    {
      v[j] = *reinterpret_cast<const Piece *>(src + c);
    }
  }
#pragma unroll
  for (int j = 0; j < P; ++j)
  {
    if (live && (t + j * THREADS) * V < dim)
    {
#pragma unroll
      for (int i = 0; i < V; ++i)
      {
        s += to_f<T>(v[j].e[i]);
      }
    }
  }
  const float mean = sum_of<WARPS>(s, sums[slot]) / static_cast<float>(dim);
  s = 0.0f;
#pragma unroll
  for (int j = 0; j < P; ++j)
  {
    if (live && (t + j * THREADS) * V < dim)
    {
#pragma unroll
      for (int i = 0; i < V; ++i)
      {
        const float d = to_f<T>(v[j].e[i]) - mean;
        s = fmaf(d, d, s);
      }
    }
  }
  const float rstd = 1.0f / sqrtf(sum_of<WARPS>(s, sums[slot]) / static_cast<float>(dim) + epsilon);
  if (!live)
  {
    return;
  }
  T *dst = y + static_cast<int64_t>(r) * dim;
#pragma unroll
  for (int j = 0; j < P; ++j)
  {
    const int c = (t + j * THREADS) * V;
    if (c < dim)
    {
      float g[V], b[V];
      load_floats<T, V>(g, gamma != nullptr ? gamma + c : nullptr, 1.0f);
      load_floats<T, V>(b, beta != nullptr ? beta + c : nullptr, 0.0f);
      Piece o;
#pragma unroll
      for (int i = 0; i < V; ++i)
      {
        o.e[i] = from_f<T>(fmaf((to_f<T>(v[j].e[i]) - mean) * rstd, g[i], b[i]));
      }
      *reinterpret_cast<Piece *>(dst + c) = o;
    }
  }
  if (t == 0)
  {
    mean_out[r] = mean;
    rstd_out[r] = rstd;
  }
}

// ---- many rows: a block takes rows one after the other ----
// gamma and beta (or the columns' sums of the backward pass) stay in registers from row to row, and the next rows are on their
// way: 16-byte pieces come by asynchronous copies through a ring of RING rows in shared memory, of which every thread reads
// back exactly what it copied, so that no barrier belongs to the copies.  Rows that no 16-byte piece fits are fetched one row
// ahead into registers.  A sum's slots alternate from row to row: one barrier a sum.

template <typename T>
constexpr int kLnRing = sizeof(T) == 4 ? 3 : 4;

__device__ __forceinline__ void copy_16(void *to, const void *from)
{
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from)
               : "memory");
}

template <int WARPS>
__device__ __forceinline__ float2 sums_of(float2 v, float2 *slots)
{
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
  {
    v.x += __shfl_xor_sync(0xFFFFFFFFu, v.x, off);
    v.y += __shfl_xor_sync(0xFFFFFFFFu, v.y, off);
  }
  if constexpr (WARPS > 1)
  {
    if ((threadIdx.x & 31) == 0)
    {
      slots[(threadIdx.x >> 5) % WARPS] = v;
    }
    __syncthreads();
    v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
    {
      v.x += slots[w].x;
      v.y += slots[w].y;
    }
  }
  return v;
}

template <int WARPS>
__device__ __forceinline__ float one_sum_of(float v, float *slots)
{
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
  {
    v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  }
  if constexpr (WARPS > 1)
  {
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

// the rows of N tensors that a block walks over: start() once, then next() for each row in turn gives this thread's pieces
template <typename T, int V, int P, int THREADS, int BLOCK, int N>
struct RowsAhead
{
  using Piece = LnPiece<T, V>;
  static constexpr int RING = kLnRing<T>;
  static constexpr size_t kBytes = V > 1 ? static_cast<size_t>(RING) * N * P * BLOCK * 16 : 0;
  const T *src[N];
  int64_t row;     // the next row to fetch
  int64_t step;
  int rows, dim, t;
  uint4 *ring;
  int at;          // ring row that next() reads
  Piece ahead[V > 1 ? 1 : N][V > 1 ? 1 : P];

  __device__ __forceinline__ void fetch(int stage)
  {
    if constexpr (V > 1)
    {
      if (row < rows)
      {
#pragma unroll
        for (int n = 0; n < N; ++n)
        {
#pragma unroll
          for (int j = 0; j < P; ++j)
          {
            const int c = (t + j * THREADS) * V;
            if (c < dim)
            {
              copy_16(ring + ((stage * N + n) * P + j) * BLOCK + threadIdx.x, src[n] + row * dim + c);
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    else
    {
      if (row < rows)
      {
#pragma unroll
        for (int n = 0; n < N; ++n)
        {
#pragma unroll
          for (int j = 0; j < P; ++j)
          {
            const int c = (t + j * THREADS) * V;
            if (c < dim)
            {
              ahead[n][j] = *reinterpret_cast<const Piece *>(src[n] + row * dim + c);
            }
          }
        }
      }
    }
    row += step;
  }

  __device__ __forceinline__ void start()
  {
    at = 0;
#pragma unroll
    for (int i = 0; i < (V > 1 ? RING - 1 : 1); ++i)
    {
      fetch(i);
    }
  }

  __device__ __forceinline__ void next(Piece (&out)[N][P])
  {
    if constexpr (V > 1)
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
          const uint4 v = ring[((at * N + n) * P + j) * BLOCK + threadIdx.x];
          out[n][j] = *reinterpret_cast<const Piece *>(&v);
        }
      }
      at = at == RING - 1 ? 0 : at + 1;
    }
    else
    {
#pragma unroll
      for (int n = 0; n < N; ++n)
      {
#pragma unroll
        for (int j = 0; j < P; ++j)
        {
          out[n][j] = ahead[n][j];
        }
      }
      fetch(0);
    }
  }
};

template <typename T, int V, int P, int WARPS>
__global__ void __launch_bounds__(kLnBlock<WARPS, 256>, WARPS <= 8 ? 3 : 1)
layernorm_fwd_many_kernel(const T *x, const float *__restrict__ gamma, const float *__restrict__ beta, T *y,
                          float *__restrict__ mean_out, float *__restrict__ rstd_out, float epsilon, int rows, int dim)
{
  constexpr int BLOCK = kLnBlock<WARPS, 256>;
  constexpr int SLOTS = BLOCK / (WARPS * 32);
  constexpr int THREADS = WARPS * 32;
  extern __shared__ uint4 ln_ring[];
  __shared__ float sums[2][2][SLOTS][WARPS];
  asm volatile("griddepcontrol.wait;" : "+l"(gamma), "+l"(beta)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  using Rows = RowsAhead<T, V, P, THREADS, BLOCK, 1>;
  const int slot = threadIdx.x / THREADS;
  const int t = threadIdx.x % THREADS;
  const int first = static_cast<int>(blockIdx.x) * SLOTS;
  const int step = static_cast<int>(gridDim.x) * SLOTS;
  Rows in;
  in.src[0] = x;
  in.row = first + slot;
  in.step = step;
  in.rows = rows;
  in.dim = dim;
  in.t = t;
  in.ring = ln_ring;
  in.start();
  float g[P][V], b[P][V];
#pragma unroll
  for (int j = 0; j < P; ++j)
  {
    const int c = (t + j * THREADS) * V;
    if (c < dim)
    {
      load_floats<T, V>(g[j], gamma != nullptr ? gamma + c : nullptr, 1.0f);
      load_floats<T, V>(b[j], beta != nullptr ? beta + c : nullptr, 0.0f);
    }
  }
  int turn = 0;
  for (int64_t base = first; base < rows; base += step, turn ^= 1)   // (every slot takes part in the sums' barriers)
  {
    const int64_t r = base + slot;
    const bool live = r < rows;
    LnPiece<T, V> v[1][P];
    in.next(v);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j)
    {
      if (live && (t + j * THREADS) * V < dim)
      {
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
          s += to_f<T>(v[0][j].e[i]);
        }
      }
    }
    const float mean = one_sum_of<WARPS>(s, sums[turn][0][slot]) / static_cast<float>(dim);
    s = 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j)
    {
      if (live && (t + j * THREADS) * V < dim)
      {
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
          const float d = to_f<T>(v[0][j].e[i]) - mean;
          s = fmaf(d, d, s);
        }
      }
    }
    const float rstd = 1.0f / sqrtf(one_sum_of<WARPS>(s, sums[turn][1][slot]) / static_cast<float>(dim) + epsilon);
#pragma unroll
    for (int j = 0; j < P; ++j)
    {
      const int c = (t + j * THREADS) * V;
      if (live && c < dim)
      {
        LnPiece<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
          o.e[i] = from_f<T>(fmaf((to_f<T>(v[0][j].e[i]) - mean) * rstd, g[j][i], b[j][i]));
        }
        *reinterpret_cast<LnPiece<T, V> *>(y + r * dim + c) = o;
      }
    }
    if (live && t == 0)
    {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
  }
}

// dx and this block's share of dgamma and dbeta in one pass: a thread keeps its columns' sums over all rows of the block.
// part[block][0][c], part[block][1][c] as in layernorm_columns_kernel.
template <typename T, int V, int P, int WARPS>
__global__ void __launch_bounds__(kLnBlock<WARPS, 256>)
layernorm_bwd_rows_kernel(const T *dy, const T *x, const float *__restrict__ gamma, const float *__restrict__ mean_in,
                          const float *__restrict__ rstd_in, T *dx, float *__restrict__ part, int rows, int dim)
{
  constexpr int BLOCK = kLnBlock<WARPS, 256>;
  constexpr int SLOTS = BLOCK / (WARPS * 32);
  constexpr int THREADS = WARPS * 32;
  extern __shared__ uint4 ln_ring[];   // the ring; then, where SLOTS > 1, the columns' sums [2][dim]
  __shared__ float2 sums[2][SLOTS][WARPS];
  asm volatile("griddepcontrol.wait;" : "+l"(gamma), "+l"(mean_in), "+l"(rstd_in)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  using Rows = RowsAhead<T, V, P, THREADS, BLOCK, 2>;
  const int slot = threadIdx.x / THREADS;
  const int t = threadIdx.x % THREADS;
  const int first = static_cast<int>(blockIdx.x) * SLOTS;
  const int step = static_cast<int>(gridDim.x) * SLOTS;
  Rows in;
  in.src[0] = x;
  in.src[1] = dy;
  in.row = first + slot;
  in.step = step;
  in.rows = rows;
  in.dim = dim;
  in.t = t;
  in.ring = ln_ring;
  in.start();
  float g[P][V], sg[P][V], sb[P][V];
#pragma unroll
  for (int j = 0; j < P; ++j)
  {
    const int c = (t + j * THREADS) * V;
    if (c < dim)
    {
      load_floats<T, V>(g[j], gamma != nullptr ? gamma + c : nullptr, 1.0f);
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
    {
      sg[j][i] = sb[j][i] = 0.0f;
    }
  }
  float next_mean = 0.0f, next_rstd = 0.0f;
  if (first + slot < rows)
  {
    next_mean = mean_in[first + slot];
    next_rstd = rstd_in[first + slot];
  }
  int turn = 0;
  for (int64_t base = first; base < rows; base += step, turn ^= 1)   // (every slot takes part in the sums' barriers)
  {
    const int64_t r = base + slot;
    const bool live = r < rows;
    LnPiece<T, V> v[2][P];
    in.next(v);
    const float mean = next_mean, rstd = next_rstd;
    if (r + step < rows)
    {
      next_mean = mean_in[r + step];
      next_rstd = rstd_in[r + step];
    }
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < P; ++j)
    {
      if (live && (t + j * THREADS) * V < dim)
      {
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
          const float d = to_f<T>(v[1][j].e[i]);
          const float xh = (to_f<T>(v[0][j].e[i]) - mean) * rstd;
          const float w = d * g[j][i];
          s.x += w;
          s.y = fmaf(w, xh, s.y);
          sg[j][i] = fmaf(d, xh, sg[j][i]);
          sb[j][i] += d;
        }
      }
    }
    s = sums_of<WARPS>(s, sums[turn][slot]);
    const float s1 = s.x / static_cast<float>(dim);
    const float s2 = s.y / static_cast<float>(dim);
#pragma unroll
    for (int j = 0; j < P; ++j)
    {
      const int c = (t + j * THREADS) * V;
      if (live && c < dim)
      {
        LnPiece<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
          const float xh = (to_f<T>(v[0][j].e[i]) - mean) * rstd;
          o.e[i] = from_f<T>(rstd * (to_f<T>(v[1][j].e[i]) * g[j][i] - s1 - xh * s2));
        }
        *reinterpret_cast<LnPiece<T, V> *>(dx + r * dim + c) = o;
      }
    }
  }
  if (part == nullptr)
  {
    return;
  }
  float *columns = reinterpret_cast<float *>(reinterpret_cast<char *>(ln_ring) + Rows::kBytes);
  float *mine = part + static_cast<int64_t>(blockIdx.x) * 2 * dim;
  float *to = SLOTS > 1 ? columns : mine;
#pragma unroll 1
  for (int i = 0; i < SLOTS; ++i)   // slot by slot, in order
  {
    if (slot == i)
    {
#pragma unroll
      for (int j = 0; j < P; ++j)
      {
        const int c = (t + j * THREADS) * V;
        if (c < dim)
        {
#pragma unroll
          for (int e = 0; e < V; ++e)
          {
            to[c + e] = i > 0 ? to[c + e] + sg[j][e] : sg[j][e];
            to[dim + c + e] = i > 0 ? to[dim + c + e] + sb[j][e] : sb[j][e];
          }
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

// slices of rows with partial sums of their own
int ln_slices(int rows) { return rows < 148 * 2 ? rows : 148 * 2; }

unsigned ln_grid(int rows) { return static_cast<unsigned>(rows < 148 * 8 ? rows : 148 * 8); }

constexpr size_t kLnPlainSmem = 40 * 1024;   // dynamic, beside the static slots, without asking

bool on_16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, int V, int P, int WARPS>
int ln_fwd_rows(const T *x, const float *gamma, const float *beta, T *y, float *mean, float *rstd, float epsilon, int rows,
                int dim, cudaStream_t s)
{
  constexpr int BLOCK = kLnBlock<WARPS, 128>;
  constexpr int SLOTS = BLOCK / (WARPS * 32);
  CAIFQ_CHECK_CUDA(launch_dependent(layernorm_fwd_rows_kernel<T, V, P, WARPS>,
                                    dim3(static_cast<unsigned>((static_cast<int64_t>(rows) + SLOTS - 1) / SLOTS)), dim3(BLOCK), 0, s, x,
                                    gamma, beta, y, mean, rstd, epsilon, rows, dim));
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

template <typename T, int V, int P, int WARPS>
int ln_fwd_many(const T *x, const float *gamma, const float *beta, T *y, float *mean, float *rstd, float epsilon, int rows,
                int dim, cudaStream_t s)
{
  constexpr int BLOCK = kLnBlock<WARPS, 256>;
  constexpr int SLOTS = BLOCK / (WARPS * 32);
  constexpr size_t kBytes = RowsAhead<T, V, P, WARPS * 32, BLOCK, 1>::kBytes;
  static std::atomic<uint64_t> done{0};
  if (kBytes > kLnPlainSmem)
  {
    CAIFQ_CHECK_CUDA(allow_smem(layernorm_fwd_many_kernel<T, V, P, WARPS>, kBytes, done));
  }
  const int blocks = (rows - 1) / SLOTS + 1;
  const int most = 148 * (WARPS <= 8 ? 3 : 1);
  CAIFQ_CHECK_CUDA(launch_dependent(layernorm_fwd_many_kernel<T, V, P, WARPS>,
                                    dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(BLOCK), kBytes, s, x,
                                    gamma, beta, y, mean, rstd, epsilon, rows, dim));
  return CAIFQ_OK;
}

// the fewest warps (a power of two) whose registers hold the row
#define CAIFQ_LN_WARPS(CALL, ELEMENTS)  \
  if (dim <= 32 * (ELEMENTS))           \
  {                                     \
    return CALL(1);                     \
  }                                     \
  if (dim <= 64 * (ELEMENTS))           \
  {                                     \
    return CALL(2);                     \
  }                                     \
  if (dim <= 128 * (ELEMENTS))          \
  {                                     \
    return CALL(4);                     \
  }                                     \
  if (dim <= 256 * (ELEMENTS))          \
  {                                     \
    return CALL(8);                     \
  }                                     \
  if (dim <= 512 * (ELEMENTS))          \
  {                                     \
    return CALL(16);                    \
  }

template <typename T>
int ln_fwd(const void *xv, const float *gamma, const float *beta, void *yv, float *mean, float *rstd, float epsilon, int rows,
           int dim, cudaStream_t s)
{
  const T *x = static_cast<const T *>(xv);
  T *y = static_cast<T *>(yv);
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  if ((dim % V) == 0 && on_16(x) && on_16(y) && on_16(gamma) && on_16(beta))
  {
#define CAIFQ_LN_CALL(W) ln_fwd_many<T, V, 16 / V, W>(x, gamma, beta, y, mean, rstd, epsilon, rows, dim, s)
    if (rows > 148)
    {
      CAIFQ_LN_WARPS(CAIFQ_LN_CALL, 16)
    }
#undef CAIFQ_LN_CALL
#define CAIFQ_LN_CALL(W) ln_fwd_rows<T, V, 4, W>(x, gamma, beta, y, mean, rstd, epsilon, rows, dim, s)
    CAIFQ_LN_WARPS(CAIFQ_LN_CALL, 4 * V)
    if (dim <= 1024 * 4 * V)
    {
      return CAIFQ_LN_CALL(32);
    }
#undef CAIFQ_LN_CALL
  }
  else
  {
#define CAIFQ_LN_CALL(W) ln_fwd_rows<T, 1, 16, W>(x, gamma, beta, y, mean, rstd, epsilon, rows, dim, s)
    CAIFQ_LN_WARPS(CAIFQ_LN_CALL, 16)
    if (dim <= 1024 * 16)
    {
      return CAIFQ_LN_CALL(32);
    }
#undef CAIFQ_LN_CALL
  }
  CAIFQ_CHECK_CUDA(launch_dependent(layernorm_fwd_kernel<T>, dim3(ln_grid(rows)), dim3(kLnThreads), 0, s, x, gamma, beta, y,
                                    mean, rstd, epsilon, rows, static_cast<int64_t>(dim)));
  return CAIFQ_OK;
}

template <typename T, int V, int P, int WARPS>
int ln_bwd_rows(const T *dy, const T *x, const float *gamma, const float *mean, const float *rstd, T *dx, float *part,
                int *slices, int rows, int dim, cudaStream_t s)
{
  constexpr int BLOCK = kLnBlock<WARPS, 256>;
  constexpr int SLOTS = BLOCK / (WARPS * 32);
  constexpr size_t kBytes = RowsAhead<T, V, P, WARPS * 32, BLOCK, 2>::kBytes;
  constexpr size_t kColumns = SLOTS > 1 ? sizeof(float) * 2 * 16 * WARPS * 32 : 0;   // of the widest row
  static std::atomic<uint64_t> done{0};
  if (kBytes + kColumns > kLnPlainSmem)
  {
    CAIFQ_CHECK_CUDA(allow_smem(layernorm_bwd_rows_kernel<T, V, P, WARPS>, kBytes + kColumns, done));
  }
  const int blocks = (rows - 1) / SLOTS + 1;
  const int most = WARPS <= 8 ? 148 * 2 : 148;
  *slices = blocks < most ? blocks : most;
  CAIFQ_CHECK_CUDA(launch_dependent(layernorm_bwd_rows_kernel<T, V, P, WARPS>, dim3(static_cast<unsigned>(*slices)), dim3(BLOCK),
                                    kBytes + (SLOTS > 1 ? sizeof(float) * 2 * static_cast<size_t>(dim) : 0), s, dy, x, gamma,
                                    mean, rstd, dx, part, rows, dim));
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
  if ((dim % V) == 0 && on_16(dy) && on_16(x) && on_16(dx) && on_16(gamma))
  {
#define CAIFQ_LN_CALL(W) ln_bwd_rows<T, V, 16 / V, W>(dy, x, gamma, mean, rstd, dx, part, slices, rows, dim, s)
    CAIFQ_LN_WARPS(CAIFQ_LN_CALL, 16)
#undef CAIFQ_LN_CALL
  }
  else
  {
#define CAIFQ_LN_CALL(W) ln_bwd_rows<T, 1, 16, W>(dy, x, gamma, mean, rstd, dx, part, slices, rows, dim, s)
    CAIFQ_LN_WARPS(CAIFQ_LN_CALL, 16)
#undef CAIFQ_LN_CALL
  }
  *slices = ln_slices(rows);
  if (part != nullptr)
  {
    // (before dx, which may be written over dy)
    CAIFQ_CHECK_CUDA(launch_dependent(layernorm_columns_kernel<T>, dim3((dim + 31) / 32, static_cast<unsigned>(*slices)),
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
    CAIFQ_CHECK_CUDA(launch_dependent(layernorm_finish_kernel, dim3((dim + 31) / 32, 2), dim3(kLnThreads), 0, s,
                                      static_cast<const float *>(workspace), grad_gamma, grad_beta, slices,
                                      static_cast<int64_t>(dim), accumulate));
  }
  return CAIFQ_OK;
}

}  // namespace caifq
