// Layer norm in front of the frozen projections, the other norm beside norm.cu's RMSNorm:
//   mean = sum x / n, rstd = 1 / sqrt(sum (x - mean)^2 / n + epsilon), y = (x - mean) * rstd * gamma + beta
//   xh = (x - mean) * rstd, g = dy * gamma
//   dx = rstd * (g - sum(g) / n - xh * sum(g * xh) / n),  dgamma = sum_rows dy * xh,  dbeta = sum_rows dy
// All sums are fp32 and run in a fixed order: a row's variance is taken around its mean (a second pass over the row, not the
// difference of two large sums), and the gradients of gamma and beta are partial sums per slice of rows, added slice by
// slice by a second launch, so that two calls give the same bits.  y and dx are rounded once.
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

// slices of rows with partial sums of their own
int ln_slices(int rows) { return rows < 148 * 2 ? rows : 148 * 2; }

unsigned ln_grid(int rows) { return static_cast<unsigned>(rows < 148 * 8 ? rows : 148 * 8); }

template <typename T>
int ln_fwd(const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd, float epsilon, int rows,
           int dim, cudaStream_t s)
{
  CAIFQ_CHECK_CUDA(launch_dependent(layernorm_fwd_kernel<T>, dim3(ln_grid(rows)), dim3(kLnThreads), 0, s,
                                    static_cast<const T *>(x), gamma, beta, static_cast<T *>(y), mean, rstd, epsilon, rows,
                                    static_cast<int64_t>(dim)));
  return CAIFQ_OK;
}

template <typename T>
int ln_bwd(const void *dy, const void *x, const float *gamma, const float *mean, const float *rstd, void *dx, float *part,
           int slices, int rows, int dim, cudaStream_t s)
{
  if (part != nullptr)
  {
    // (before dx, which may be written over dy)
    CAIFQ_CHECK_CUDA(launch_dependent(layernorm_columns_kernel<T>, dim3((dim + 31) / 32, static_cast<unsigned>(slices)),
                                      dim3(kLnThreads), 0, s, static_cast<const T *>(dy), static_cast<const T *>(x), mean,
                                      rstd, part, rows, static_cast<int64_t>(dim)));
  }
  CAIFQ_CHECK_CUDA(launch_dependent(layernorm_dx_kernel<T>, dim3(ln_grid(rows)), dim3(kLnThreads), 0, s,
                                    static_cast<const T *>(dy), static_cast<const T *>(x), gamma, mean, rstd,
                                    static_cast<T *>(dx), rows, static_cast<int64_t>(dim)));
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
  const int slices = ln_slices(rows);
  if (rows > 0)
  {
    float *part = columns ? workspace : nullptr;
    int rc = CAIFQ_OK;
    switch (dtype)
    {
      case CAIFQ_F32:
        rc = ln_bwd<float>(dy, x, gamma, mean, rstd, dx, part, slices, rows, dim, s);
        break;
      case CAIFQ_F16:
        rc = ln_bwd<__half>(dy, x, gamma, mean, rstd, dx, part, slices, rows, dim, s);
        break;
      default:
        rc = ln_bwd<__nv_bfloat16>(dy, x, gamma, mean, rstd, dx, part, slices, rows, dim, s);
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
