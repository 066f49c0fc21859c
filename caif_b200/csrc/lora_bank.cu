// Low-rank adapters of many requests beside one frozen projection: row t of the batch takes adapter a = adapter_of_row[t],
//   y[t] = x[t] . W^T + scale_a (x[t] . A_a^T) . B_a^T
// Two kernels write the adapters' part into y, and the frozen product then adds itself to it in its own epilogue:
//   down: h[t, :] = x[t] . A_a^T, fp32        up: y[t, :] = scale_a h[t, :] . B_a^T, rounded once
// Rows need no order.  The adapters lie in a table in device memory that the kernels read, so a batch is described by the
// rows' indices alone and a captured call follows them.  A row whose index is outside the table gets zeros here; what its
// x or another adapter's factors hold (infinities, NaN) never reaches it, since rows are selected, not multiplied by zero.
#include "common.cuh"

namespace caifq
{

namespace
{

constexpr int kBankThreads = 256;

template <typename T>
__device__ __forceinline__ float bank_f(T v);
template <>
__device__ __forceinline__ float bank_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float bank_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float bank_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T bank_t(float v);
template <>
__device__ __forceinline__ float bank_t<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half bank_t<__half>(float v) { return __float2half(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 bank_t<__nv_bfloat16>(float v) { return __float2bfloat16(v); }

// ---- any type, rank and width: fp32 multiply-adds ----

// a CTA a row, a warp a column of h at a time
template <typename T>
__global__ void __launch_bounds__(kBankThreads)
bank_down_kernel(const T *x, const int32_t *__restrict__ adapter_of_row, const caifq_lora_entry *__restrict__ entries, int count,
                 float *h, int ld, int in_dim)
{
  asm volatile("griddepcontrol.wait;" : "+l"(adapter_of_row), "+l"(entries)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t row = blockIdx.x;
  const int id = adapter_of_row[row];
  if (id < 0 || id >= count)
  {
    return;
  }
  const int lane = threadIdx.x & 31;
  const int rank = entries[id].rank;
  const T *a = static_cast<const T *>(entries[id].a);
  const T *src = x + row * in_dim;
  const int step = static_cast<int>(gridDim.y) * (kBankThreads / 32);
  for (int j = blockIdx.y * (kBankThreads / 32) + static_cast<int>(threadIdx.x >> 5); j < rank; j += step)
  {
    const T *w = a + static_cast<int64_t>(j) * in_dim;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int c = lane;
    for (; c + 96 < in_dim; c += 128)
    {
#pragma unroll
      for (int i = 0; i < 4; ++i)
      {
        s[i] = fmaf(bank_f<T>(src[c + 32 * i]), bank_f<T>(w[c + 32 * i]), s[i]);
      }
    }
    for (; c < in_dim; c += 32)
    {
      s[0] = fmaf(bank_f<T>(src[c]), bank_f<T>(w[c]), s[0]);
    }
    float v = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
    {
      v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
    }
    if (lane == 0)
    {
      h[row * ld + j] = v;
    }
  }
}

// a thread a column of y
template <typename T>
__global__ void __launch_bounds__(kBankThreads)
bank_up_kernel(const float *h, const int32_t *__restrict__ adapter_of_row, const caifq_lora_entry *__restrict__ entries,
               int count, T *y, int ld, int out_dim)
{
  __shared__ float sh[kBankMaxRank];
  asm volatile("griddepcontrol.wait;" : "+l"(adapter_of_row), "+l"(entries)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t row = blockIdx.x;
  const int id = adapter_of_row[row];
  const bool mine = id >= 0 && id < count;
  const int rank = mine ? entries[id].rank : 0;
  for (int j = threadIdx.x; j < rank; j += kBankThreads)
  {
    sh[j] = h[row * ld + j];
  }
  __syncthreads();
  const int col = blockIdx.y * kBankThreads + static_cast<int>(threadIdx.x);
  if (col >= out_dim)
  {
    return;
  }
  float v = 0.0f;
  if (mine)
  {
    const T *b = static_cast<const T *>(entries[id].b) + static_cast<int64_t>(col) * rank;
    for (int j = 0; j < rank; ++j)
    {
      v = fmaf(sh[j], bank_f<T>(b[j]), v);
    }
    v *= entries[id].scale;
  }
  y[row * out_dim + col] = bank_t<T>(v);
}

template <typename T>
int bank_general(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const void *x, int64_t m, void *y, float *h,
                 cudaStream_t s)
{
  const unsigned parts = static_cast<unsigned>((bank.max_rank + 7) / 8);
  CAIFQ_CHECK_CUDA(launch_dependent(bank_down_kernel<T>, dim3(static_cast<unsigned>(m), parts), dim3(kBankThreads), 0, s,
                                    static_cast<const T *>(x), adapter_of_row, bank.entries, bank.count, h, bank.max_rank,
                                    bank.in_dim));
  CAIFQ_CHECK_CUDA(launch_dependent(bank_up_kernel<T>, dim3(static_cast<unsigned>(m), static_cast<unsigned>((bank.out_dim + kBankThreads - 1) / kBankThreads)),
                                    dim3(kBankThreads), 0, s, static_cast<const float *>(h), adapter_of_row, bank.entries,
                                    bank.count, static_cast<T *>(y), bank.max_rank, bank.out_dim));
  return CAIFQ_OK;
}

}  // namespace

// y[m, out] = the adapters' part alone, zeros for rows without one; h: fp32 [m, max_rank].  m >= 1
int launch_lora_bank(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const void *x, int64_t m, void *y, float *h,
                     cudaStream_t s)
{
  switch (bank.dtype)
  {
    case CAIFQ_F32:
      return bank_general<float>(bank, adapter_of_row, x, m, y, h, s);
    case CAIFQ_F16:
      return bank_general<__half>(bank, adapter_of_row, x, m, y, h, s);
    default:
      return bank_general<__nv_bfloat16>(bank, adapter_of_row, x, m, y, h, s);
  }
}

}  // namespace caifq
