// Low-rank adapters of many requests beside one frozen projection: row t of the batch takes adapter a = adapter_of_row[t],
//   y[t] = x[t] . W^T + scale_a (x[t] . A_a^T) . B_a^T
//   down: h[t, :] = x[t] . A_a^T, fp32
//   the frozen product, fp32
//   up: y[t, :] = frozen[t, :] + scale_a h[t, :] . B_a^T, rounded once
// Why the frozen product first and in fp32, not the adapters' part first and the product added to it in the epilogues that add
// a residual: those read y where their other operands leave no time for it (4096 -> 14336 int4, 768 rows: 78 us without, 145
// with; 4096 -> 4096 bf16, 8192 rows: 176 and 209), and y would be rounded twice.
// Rows need no order.  The adapters lie in a table in device memory that the kernels read, so a batch is described by the
// rows' indices alone and a captured call follows them.  A row whose index is outside the table is the frozen product alone;
// what another row or another row's adapter holds (infinities, NaN) never reaches it, since rows are selected, not
// multiplied by zero.
#include "umma.cuh"

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
bank_up_kernel(const float *frozen, const float *h, const int32_t *__restrict__ adapter_of_row,
               const caifq_lora_entry *__restrict__ entries, int count, T *y, int ld, int out_dim)
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
  const float f = frozen[row * out_dim + col];
  y[row * out_dim + col] = bank_t<T>(mine ? f + v : f);
}

// ---- bf16 factors of rank 8, 16, ... 64 on 16-byte boundaries: the tensor core on 16 rows of the batch as they lie ----
// A block takes 16 neighbouring rows and goes through the adapters that they name, one after the other (gridDim blocks share
// them).  The rows of a prompt share one adapter, 16 decoding sequences may name 16: their factors are read once a tile in
// either case, and no sorting of rows, and no launch for it, comes before.  Each adapter's product has accumulators of its
// own and is stored for its own rows alone.

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1)
{
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the adapters of 16 rows: ids[i] of row i (-1: none); returns the rows at which one appears for the first time
__device__ __forceinline__ uint32_t first_rows(const int (&ids)[16])
{
  const int lane = threadIdx.x & 31;
  const int id = lane < 16 ? ids[lane] : -1;
  const uint32_t same = __match_any_sync(0xFFFFFFFFu, id);
  return __ballot_sync(0xFFFFFFFFu, id >= 0 && (same & ((1u << lane) - 1u)) == 0u);
}

// ids and table entries of a tile's rows, once for all turns
__device__ __forceinline__ void load_ids(int (&ids)[16], caifq_lora_entry (&mine)[16], const int32_t *adapter_of_row,
                                         const caifq_lora_entry *entries, int64_t row0, int64_t m, int count)
{
  if (threadIdx.x < 16)
  {
    const int64_t row = row0 + threadIdx.x;
    int id = row < m ? adapter_of_row[row] : -1;
    id = id < count ? (id < 0 ? -1 : id) : -1;
    ids[threadIdx.x] = id;
    if (id >= 0)
    {
      mine[threadIdx.x] = entries[id];
    }
  }
  __syncthreads();
}

// h of 16 rows.  As in the adapter's own thin product, a lane streams 16 bytes of two rows of x and of a row of A per 32
// columns straight into fragments (the order of the columns inside a fragment is the same for both); the eight warps split
// the columns, and so do the blocks of a cluster where there are few rows.
template <int NT>   // eights of the largest rank
__global__ void __launch_bounds__(256)
bank_down_mma_kernel(const __nv_bfloat16 *x, const int32_t *__restrict__ adapter_of_row,
                     const caifq_lora_entry *__restrict__ entries, int count, float *h, int ld, int64_t m, int in_dim,
                     int cluster)
{
  __shared__ float part[8][16][NT * 8 + 1];
  __shared__ int ids[16];
  __shared__ caifq_lora_entry entry[16];
  // (what invariant loads read is addressed out of the wait, so that they stay behind it)
  asm volatile("griddepcontrol.wait;" : "+l"(adapter_of_row), "+l"(entries), "+l"(x)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2;
  const int t = lane & 3;
  const int rank_in_cluster = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / cluster) * 16;
  load_ids(ids, entry, adapter_of_row, entries, row0, m, count);
  uint32_t firsts = first_rows(ids);
  const int steps = in_dim / 32;
  const int begin = static_cast<int>(static_cast<int64_t>(steps) * (rank_in_cluster * 8 + warp) / (8 * cluster));
  const int end = static_cast<int>(static_cast<int64_t>(steps) * (rank_in_cluster * 8 + warp + 1) / (8 * cluster));
  const uint4 zero4 = make_uint4(0u, 0u, 0u, 0u);
  // (ids has the same content in all blocks of a cluster, so they run the same turns)
  for (int turn = 0; firsts != 0u; ++turn, firsts &= firsts - 1u)
  {
    if (turn % static_cast<int>(gridDim.y) != static_cast<int>(blockIdx.y))
    {
      continue;
    }
    const int at = __ffs(static_cast<int>(firsts)) - 1;
    const int id = ids[at];
    const int eights = entry[at].rank / 8;
    const __nv_bfloat16 *a = static_cast<const __nv_bfloat16 *>(entry[at].a);
    const bool lo = ids[g] == id;
    const bool hi = ids[g + 8] == id;
    const uint4 *x_lo = reinterpret_cast<const uint4 *>(x + (lo ? row0 + g : 0) * in_dim) + t;
    const uint4 *x_hi = reinterpret_cast<const uint4 *>(x + (hi ? row0 + g + 8 : 0) * in_dim) + t;
    const uint4 *a_row = reinterpret_cast<const uint4 *>(a + static_cast<int64_t>(g) * in_dim) + t;
    float c[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
    {
      c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.0f;
    }
#pragma unroll 4
    for (int st = begin; st < end; ++st)
    {
      const uint4 xa = lo ? __ldg(x_lo + st * 4) : zero4;
      const uint4 xb = hi ? __ldg(x_hi + st * 4) : zero4;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
      {
        if (nt < eights)
        {
          const uint4 w = __ldg(a_row + static_cast<int64_t>(nt) * in_dim + st * 4);
          mma_16816(c[nt], xa.x, xb.x, xa.y, xb.y, w.x, w.y);
          mma_16816(c[nt], xa.z, xb.z, xa.w, xb.w, w.z, w.w);
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
    {
      part[warp][g][nt * 8 + 2 * t] = c[nt][0];
      part[warp][g][nt * 8 + 2 * t + 1] = c[nt][1];
      part[warp][g + 8][nt * 8 + 2 * t] = c[nt][2];
      part[warp][g + 8][nt * 8 + 2 * t + 1] = c[nt][3];
    }
    __syncthreads();
    // the block's eight partial tiles become one, in the first of them (an element is one thread's)
    for (int e = threadIdx.x; e < 16 * NT * 8; e += 256)
    {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w)
      {
        v += part[w][e / (NT * 8)][e % (NT * 8)];
      }
      part[0][e / (NT * 8)][e % (NT * 8)] = v;
    }
    if (cluster > 1)
    {
      cluster_sync_all();
    }
    else
    {
      __syncthreads();
    }
    const int share = 16 / cluster;
    for (int e = threadIdx.x; e < share * NT * 8; e += 256)
    {
      const int rr = rank_in_cluster * share + e / (NT * 8);
      const int col = e % (NT * 8);
      if (ids[rr] == id && col < eights * 8)
      {
        float v = part[0][rr][col];
        if (cluster > 1)
        {
          v = 0.0f;
          const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(&part[0][rr][col]));
          for (int b = 0; b < cluster; ++b)
          {
            v += __uint_as_float(ld_shared_cluster(map_to_cta(mine, static_cast<uint32_t>(b))));
          }
        }
        h[(row0 + rr) * ld + col] = v;
      }
    }
    // nobody's partial tile is written again, or left, while it is read
    if (cluster > 1)
    {
      cluster_sync_all();
    }
    else
    {
      __syncthreads();
    }
  }
}

// y of 16 rows and 128 columns: a warp 32 columns.  h enters as two bf16 terms (2^-16 relative).  The columns of a warp's four
// 8-wide tiles are dealt out so that a lane ends with eight neighbouring ones of a row: 16-byte accesses of y.
struct UpOperands
{
  uint2 w[4];                // rows of B, four columns of it each
  uint32_t top[2][2];        // h of rows g and g + 8: the first terms
  uint32_t rest[2][2];       // and the second
};

__global__ void __launch_bounds__(128)
bank_up_mma_kernel(const float *frozen, const float *h, const int32_t *__restrict__ adapter_of_row,
                   const caifq_lora_entry *__restrict__ entries, int count, __nv_bfloat16 *y, int ld, int64_t m, int out_dim)
{
  __shared__ int ids[16];
  __shared__ caifq_lora_entry entry[16];
  asm volatile("griddepcontrol.wait;" : "+l"(adapter_of_row), "+l"(entries)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2;
  const int t = lane & 3;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int col0 = static_cast<int>(blockIdx.y) * 128 + static_cast<int>(threadIdx.x >> 5) * 32;
  const bool stores = col0 + 8 * t < out_dim;
  // the frozen product's part of this lane's sixteen results is on its way meanwhile
  float4 f[2][2];
#pragma unroll
  for (int half = 0; half < 2; ++half)
  {
    const int64_t row = row0 + g + 8 * half;
    if (stores && row < m)
    {
      const float4 *src = reinterpret_cast<const float4 *>(frozen + row * out_dim + col0 + 8 * t);
      f[half][0] = src[0];
      f[half][1] = src[1];
    }
  }
  load_ids(ids, entry, adapter_of_row, entries, row0, m, count);
  uint32_t firsts = first_rows(ids);
  const int n0 = col0 + 8 * (g >> 1) + (g & 1);   // the column whose row of B this lane feeds, plus 2 * tile
  const int id_of[2] = {ids[g], ids[g + 8]};
  auto operands = [&](int at, int k) {
    UpOperands o;
    const int rank = entry[at].rank;
    const __nv_bfloat16 *b = static_cast<const __nv_bfloat16 *>(entry[at].b);
    const int kk = k + 4 * t;
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
    {
      o.w[nt] = make_uint2(0u, 0u);
      if (kk < rank && n0 + 2 * nt < out_dim)
      {
        o.w[nt] = __ldg(reinterpret_cast<const uint2 *>(b + static_cast<int64_t>(n0 + 2 * nt) * rank + kk));
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half)
    {
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (id_of[half] == ids[at] && kk < rank)
      {
        v = *reinterpret_cast<const float4 *>(h + (row0 + g + 8 * half) * ld + kk);
      }
      const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 2; ++i)
      {
        const uint32_t top = pack_bf16x2(e[2 * i], e[2 * i + 1]);
        // (an infinity has no second term)
        const float r0 = isfinite(e[2 * i]) ? e[2 * i] - __uint_as_float(top << 16) : 0.0f;
        const float r1 = isfinite(e[2 * i + 1]) ? e[2 * i + 1] - __uint_as_float(top & 0xFFFF0000u) : 0.0f;
        o.top[half][i] = top;
        o.rest[half][i] = pack_bf16x2(r0, r1);
      }
    }
    return o;
  };
  auto multiply = [](float(&c)[4][4], const UpOperands &o) {
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
    {
      mma_16816(c[nt], o.top[0][0], o.top[1][0], o.top[0][1], o.top[1][1], o.w[nt].x, o.w[nt].y);
      mma_16816(c[nt], o.rest[0][0], o.rest[1][0], o.rest[0][1], o.rest[1][1], o.w[nt].x, o.w[nt].y);
    }
  };
  auto add = [&](const float(&c)[4][4], int at) {
    const float scale = entry[at].scale;
#pragma unroll
    for (int half = 0; half < 2; ++half)
    {
      if (id_of[half] == ids[at] && stores)
      {
        uint4 o;
        o.x = pack_bf16x2(fmaf(c[0][2 * half], scale, f[half][0].x), fmaf(c[0][2 * half + 1], scale, f[half][0].y));
        o.y = pack_bf16x2(fmaf(c[1][2 * half], scale, f[half][0].z), fmaf(c[1][2 * half + 1], scale, f[half][0].w));
        o.z = pack_bf16x2(fmaf(c[2][2 * half], scale, f[half][1].x), fmaf(c[2][2 * half + 1], scale, f[half][1].y));
        o.w = pack_bf16x2(fmaf(c[3][2 * half], scale, f[half][1].z), fmaf(c[3][2 * half + 1], scale, f[half][1].w));
        *reinterpret_cast<uint4 *>(y + (row0 + g + 8 * half) * out_dim + col0 + 8 * t) = o;
      }
    }
  };
  // this block's share of the tile's adapters, two at a time so that the loads of one hide behind the other's
  int turn = 0;
  auto next = [&]() {
    while (firsts != 0u)
    {
      const int at = __ffs(static_cast<int>(firsts)) - 1;
      firsts &= firsts - 1u;
      if (turn++ % static_cast<int>(gridDim.z) == static_cast<int>(blockIdx.z))
      {
        return at;
      }
    }
    return -1;
  };
  for (int a = next(); a >= 0; a = next())
  {
    const int b = next();
    UpOperands oa = operands(a, 0);
    UpOperands ob = oa;
    if (b >= 0)
    {
      ob = operands(b, 0);
    }
    float ca[4][4] = {}, cb[4][4] = {};
    multiply(ca, oa);
#pragma unroll 1
    for (int k = 16; k < entry[a].rank; k += 16)
    {
      multiply(ca, operands(a, k));
    }
    add(ca, a);
    if (b >= 0)
    {
      multiply(cb, ob);
#pragma unroll 1
      for (int k = 16; k < entry[b].rank; k += 16)
      {
        multiply(cb, operands(b, k));
      }
      add(cb, b);
    }
  }
  if (blockIdx.z == 0 && stores)
  {
#pragma unroll
    for (int half = 0; half < 2; ++half)
    {
      const int64_t row = row0 + g + 8 * half;
      if (row < m && id_of[half] < 0)
      {
        *reinterpret_cast<uint4 *>(y + row * out_dim + col0 + 8 * t) =
            make_uint4(pack_bf16x2(f[half][0].x, f[half][0].y), pack_bf16x2(f[half][0].z, f[half][0].w),
                       pack_bf16x2(f[half][1].x, f[half][1].y), pack_bf16x2(f[half][1].z, f[half][1].w));
      }
    }
  }
}

// blocks that share a tile's adapters, no more than there can be: as many as keep the launch near `most` blocks.  (Most of
// them find nothing to do where a tile's rows are one prompt's, and leave at once.)
int bank_shares(int64_t blocks, int64_t most, int64_t m, int count)
{
  int64_t n = most / blocks;
  n = n > 16 ? 16 : n;
  n = n > m ? m : n;
  n = n > count ? count : n;
  return static_cast<int>(n < 1 ? 1 : n);
}

int down_mma(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const void *x, int64_t m, float *h, cudaStream_t s)
{
  const int64_t tiles = (m + 15) / 16;
  // blocks of a cluster: as in the adapter's own thin product, with at least two steps of 32 columns for every warp
  int cluster = 1;
  while (cluster < 8 && tiles * cluster < 4 * 148 && bank.in_dim / 32 >= 2 * cluster * 8 * 2)
  {
    cluster *= 2;
  }
  const int shares = bank_shares(tiles * cluster, 32 * 148, m, bank.count);
  void (*down)(const __nv_bfloat16 *, const int32_t *, const caifq_lora_entry *, int, float *, int, int64_t, int, int) =
      bank.max_rank <= 8 ? bank_down_mma_kernel<1>
                         : (bank.max_rank <= 16 ? bank_down_mma_kernel<2>
                                                : (bank.max_rank <= 32 ? bank_down_mma_kernel<4> : bank_down_mma_kernel<8>));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * cluster), static_cast<unsigned>(shares));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent_launches() ? 2 : 1;
  CAIFQ_CHECK_CUDA(cudaLaunchKernelEx(&cfg, down, static_cast<const __nv_bfloat16 *>(x), adapter_of_row, bank.entries,
                                      bank.count, h, bank.max_rank, m, bank.in_dim, cluster));
  return CAIFQ_OK;
}

int up_mma(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const float *frozen, const float *h, int64_t m, void *y,
           cudaStream_t s)
{
  const int64_t tiles = (m + 15) / 16;
  const int64_t columns = (bank.out_dim + 127) / 128;
  CAIFQ_CHECK_CUDA(launch_dependent(bank_up_mma_kernel,
                                    dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(columns),
                                         static_cast<unsigned>(bank_shares(tiles * columns, 16 * 148, m, bank.count))),
                                    dim3(128), 0, s, frozen, h, adapter_of_row, bank.entries, bank.count,
                                    static_cast<__nv_bfloat16 *>(y), bank.max_rank, m, bank.out_dim));
  return CAIFQ_OK;
}

template <typename T>
int down_general(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const void *x, int64_t m, float *h, cudaStream_t s)
{
  CAIFQ_CHECK_CUDA(launch_dependent(bank_down_kernel<T>, dim3(static_cast<unsigned>(m), static_cast<unsigned>((bank.max_rank + 7) / 8)),
                                    dim3(kBankThreads), 0, s, static_cast<const T *>(x), adapter_of_row, bank.entries, bank.count,
                                    h, bank.max_rank, bank.in_dim));
  return CAIFQ_OK;
}

template <typename T>
int up_general(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const float *frozen, const float *h, int64_t m, void *y,
               cudaStream_t s)
{
  CAIFQ_CHECK_CUDA(launch_dependent(bank_up_kernel<T>,
                                    dim3(static_cast<unsigned>(m), static_cast<unsigned>((bank.out_dim + kBankThreads - 1) / kBankThreads)),
                                    dim3(kBankThreads), 0, s, frozen, h, adapter_of_row, bank.entries, bank.count,
                                    static_cast<T *>(y), bank.max_rank, bank.out_dim));
  return CAIFQ_OK;
}

bool on_16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

// h[m, max_rank] (fp32, 16-byte aligned) = x . A^T of each row's adapter; rows without one are left as they are.  m >= 1
int launch_lora_bank_down(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const void *x, int64_t m, float *h,
                          cudaStream_t s)
{
  if (bank.vectors != 0 && (bank.in_dim % 32) == 0 && on_16(x))
  {
    return down_mma(bank, adapter_of_row, x, m, h, s);
  }
  switch (bank.dtype)
  {
    case CAIFQ_F32:
      return down_general<float>(bank, adapter_of_row, x, m, h, s);
    case CAIFQ_F16:
      return down_general<__half>(bank, adapter_of_row, x, m, h, s);
    default:
      return down_general<__nv_bfloat16>(bank, adapter_of_row, x, m, h, s);
  }
}

// y[m, out] = frozen[m, out] + the adapters' part; frozen (fp32) may be y itself.  m >= 1
int launch_lora_bank_up(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const float *frozen, const float *h,
                        int64_t m, void *y, cudaStream_t s)
{
  if (bank.vectors != 0 && (bank.out_dim % 8) == 0 && bank.out_dim <= 65535 * 128 && on_16(y) && on_16(frozen))
  {
    return up_mma(bank, adapter_of_row, frozen, h, m, y, s);
  }
  switch (bank.dtype)
  {
    case CAIFQ_F32:
      return up_general<float>(bank, adapter_of_row, frozen, h, m, y, s);
    case CAIFQ_F16:
      return up_general<__half>(bank, adapter_of_row, frozen, h, m, y, s);
    default:
      return up_general<__nv_bfloat16>(bank, adapter_of_row, frozen, h, m, y, s);
  }
}

}  // namespace caifq
