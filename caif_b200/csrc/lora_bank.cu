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

// A block a row; `split` of its eight warps share a column of h at a time, a part of the row each.  Bound by latency: sixteen loads of
// each operand on their way, and short parts where there are few rows (one row of 2048, rank 16: 13 us by whole rows).
template <typename T>
__global__ void __launch_bounds__(kBankThreads)
bank_down_kernel(const T *x, const int32_t *__restrict__ adapter_of_row, const caifq_lora_entry *__restrict__ entries, int count,
                 float *h, int ld, int in_dim, int split)
{
  __shared__ float sums[kBankThreads / 32];
  asm volatile("griddepcontrol.wait;" : "+l"(adapter_of_row), "+l"(entries)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t row = blockIdx.x;
  const int id = adapter_of_row[row];
  if (id < 0 || id >= count)
  {
    return;
  }
  const int lane = threadIdx.x & 31;
  const int warp = static_cast<int>(threadIdx.x >> 5);
  const int rank = entries[id].rank;
  const T *a = static_cast<const T *>(entries[id].a);
  const T *src = x + row * in_dim;
  const int part = warp % split;
  const int begin = static_cast<int>(static_cast<int64_t>(in_dim) * part / split);
  const int end = static_cast<int>(static_cast<int64_t>(in_dim) * (part + 1) / split);
  const int per = kBankThreads / 32 / split;   // columns of h at a time
  for (int j0 = blockIdx.y * per; j0 < rank; j0 += static_cast<int>(gridDim.y) * per)
  {
    const int j = j0 + warp / split;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (j < rank)
    {
      const T *w = a + static_cast<int64_t>(j) * in_dim;
      int c = begin + lane;
      for (; c + 480 < end; c += 512)
      {
        T u[16], v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
          u[i] = src[c + 32 * i];
          v[i] = w[c + 32 * i];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
          s[i & 3] = fmaf(bank_f<T>(u[i]), bank_f<T>(v[i]), s[i & 3]);
        }
      }
#pragma unroll 8
      for (; c < end; c += 32)
      {
        s[0] = fmaf(bank_f<T>(src[c]), bank_f<T>(w[c]), s[0]);
      }
    }
    float v = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
    {
      v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
    }
    if (split > 1)
    {
      __syncthreads();   // the sums before have been read
      if (lane == 0)
      {
        sums[warp] = v;
      }
      __syncthreads();
      v = 0.0f;
      for (int k = 0; k < split; ++k)
      {
        v += sums[warp - part + k];
      }
    }
    if (lane == 0 && part == 0 && j < rank)
    {
      h[row * ld + j] = v;
    }
  }
}

// A block 64 columns of a row of y, four threads a column: B's rows lie one behind the other and come through shared memory, 64 ranks at a
// time, whose products are added up by themselves and then to those before.  (A thread a column straight from memory: 64 rows of 2048
// columns, rank 64, 35 us)
constexpr int kBankColumns = 64;

template <typename T>
__global__ void __launch_bounds__(kBankThreads)
bank_up_kernel(const float *frozen, const float *h, const int32_t *__restrict__ adapter_of_row,
               const caifq_lora_entry *__restrict__ entries, int count, T *y, int ld, int out_dim)
{
  __shared__ float sh[64];
  __shared__ float sb[kBankColumns][64 + 1];
  asm volatile("griddepcontrol.wait;" : "+l"(adapter_of_row), "+l"(entries)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t row = blockIdx.x;
  const int id = adapter_of_row[row];
  const bool mine = id >= 0 && id < count;
  const int rank = mine ? entries[id].rank : 0;
  const T *b = mine ? static_cast<const T *>(entries[id].b) : nullptr;
  const int col0 = static_cast<int>(blockIdx.y) * kBankColumns;
  const int columns = out_dim - col0 < kBankColumns ? out_dim - col0 : kBankColumns;
  const int col = static_cast<int>(threadIdx.x) / 4;
  const int quarter = static_cast<int>(threadIdx.x) % 4;
  float v = 0.0f;
  for (int j0 = 0; j0 < rank; j0 += 64)
  {
    const int n = rank - j0 < 64 ? rank - j0 : 64;
    __syncthreads();   // the ranks before have been read
    if (static_cast<int>(threadIdx.x) < n)
    {
      sh[threadIdx.x] = h[row * ld + j0 + threadIdx.x];
    }
#pragma unroll 8
    for (int e = threadIdx.x; e < columns * n; e += kBankThreads)
    {
      sb[e / n][e % n] = bank_f<T>(b[static_cast<int64_t>(col0 + e / n) * rank + j0 + e % n]);
    }
    __syncthreads();
    if (col < columns)
    {
      float some = 0.0f;
      for (int k = quarter; k < n; k += 4)
      {
        some = fmaf(sh[k], sb[col][k], some);
      }
      v += some;
    }
  }
  v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
  v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
  if (quarter == 0 && col < columns)
  {
    const float f = frozen[row * out_dim + col0 + col];
    y[row * out_dim + col0 + col] = bank_t<T>(mine ? fmaf(v, entries[id].scale, f) : f);
  }
}

// The frozen product of few rows and a weight whose width no other kernel takes (they want whole 128s): a warp a row of codes for eight
// rows of x, fp32 multiply-adds, code times scale in fp32 (int8: the scale at the end).  Bound by the loads of x from L1 where there are
// many rows and by latency where there are few (1408 -> 1776 int4, 2 rows of fp32: the kernel for any cell takes 187 us).
constexpr int kFrozenRows = 8;

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) BankPiece
{
  T e[N];
};

template <typename T, bool I4>
__global__ void __launch_bounds__(kBankThreads)
bank_frozen_kernel(const T *x, const uint8_t *__restrict__ codes, const void *__restrict__ scales, float *frozen, int64_t m, int in_dim,
                   int out_dim, int group_size)
{
  constexpr int N = I4 ? 8 : 4;   // codes of a lane at a time: four bytes
  asm volatile("griddepcontrol.wait;" : "+l"(codes), "+l"(scales)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t o = static_cast<int64_t>(blockIdx.x) * (kBankThreads / 32) + static_cast<int>(threadIdx.x >> 5);
  if (o >= out_dim)
  {
    return;
  }
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * kFrozenRows;
  const int64_t flat = o * in_dim;
  const bool whole = I4 && in_dim % group_size == 0;   // (no group in two rows)
  const int64_t first_group = whole ? o * (in_dim / group_size) : 0;
  float s[kFrozenRows] = {};
#pragma unroll 2
  for (int c = lane * N; c < in_dim; c += 32 * N)
  {
    const uint32_t word = *reinterpret_cast<const uint32_t *>(codes + (I4 ? (flat + c) / 2 : flat + c));
    float scale = 1.0f;
    if constexpr (I4)
    {
      const int64_t group = whole ? first_group + c / group_size : (flat + c) / group_size;
      scale = __half2float(static_cast<const __half *>(scales)[group]);
    }
    float w[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
    {
      w[i] = I4 ? static_cast<float>(static_cast<int>((word >> (4 * i)) & 15u ^ 8u) - 8) * scale
                : static_cast<float>(static_cast<int8_t>(word >> (8 * (i & 3))));
    }
#pragma unroll
    for (int k = 0; k < kFrozenRows; ++k)
    {
      if (row0 + k < m)
      {
        const BankPiece<T, N> v = *reinterpret_cast<const BankPiece<T, N> *>(x + (row0 + k) * in_dim + c);
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
          s[k] = fmaf(bank_f<T>(v.e[i]), w[i], s[k]);
        }
      }
    }
  }
  const float last = !I4 && scales != nullptr ? *static_cast<const float *>(scales) : 1.0f;
#pragma unroll
  for (int k = 0; k < kFrozenRows; ++k)
  {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
    {
      s[k] += __shfl_xor_sync(0xFFFFFFFFu, s[k], off);
    }
    if (lane == k && row0 + k < m)
    {
      frozen[(row0 + k) * out_dim + o] = s[k] * last;
    }
  }
}

// ---- bf16 factors of rank 8, 16, ... 64 on 16-byte boundaries: the tensor core on tiles of up to 16 rows of one adapter ----
// Rows are dealt to tiles by adapter first, wherever they stand in the batch (those without one make tiles of their own, which
// `up` copies).  In a call of up to 128 rows every block does that by itself, longer ones have a launch for it.  Tiles
// of neighbouring rows as they lie, with a turn for every adapter that they name, need neither; but 200 decoding sequences of
// 24 adapters are then 13 tiles of 14 turns, which held up `up` for 28 us beside 131 tiles of prompts, and here they are 24.
// Which tile and slot a row gets does not change its arithmetic, so results do not depend on the rows' order.

constexpr int kTileRows = 16;
// rows that a block sorts by itself.  4096 -> 4096 int4, 48 rows of 16 adapters: 19.1 us so, 24.3 with the launch ahead; 1024 -> 1024, 128
// rows of 16: 15.7 and 19.2; 4096 -> 14336, 128 rows of 48: 43.1 and 43.5
constexpr int kSmallCall = 128;
constexpr int kTableMost = 4096;    // adapters that the launch ahead counts in shared memory

// what `down` leaves for `up`, in the workspace
struct BankPlan
{
  caifq_lora_entry *entry;   // [tiles] of the tile's adapter; rank 0: rows without one; rank -1: no tile
  int32_t *rows;             // [tiles][16], -1: no row
  float *h;                  // [tiles][16][ld]
};

int64_t most_tiles(int64_t m, int count)
{
  const int64_t groups = m < count + 1 ? m : count + 1;
  return (m + 15 * groups) / 16;
}

__device__ __forceinline__ int group_of(const int32_t *adapter_of_row, int64_t row, int count)
{
  const int id = adapter_of_row[row];
  return id >= 0 && id < count ? id : count;
}

// tiles of a longer call: count, number the tiles, deal the rows.  (The slots inside an adapter follow the order in which
// atomics are served; nothing but the rows' places depends on it.)
__global__ void __launch_bounds__(1024)
bank_plan_kernel(const int32_t *__restrict__ adapter_of_row, const caifq_lora_entry *__restrict__ entries, int count,
                 const BankPlan plan, int64_t m, int most)
{
  extern __shared__ int table[];   // [count + 1] rows so far, [count + 1] first tile
  __shared__ int warp_sums[32];
  asm volatile("griddepcontrol.wait;" : "+l"(adapter_of_row), "+l"(entries)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  int *rows_of = table;
  int *first = table + count + 1;
  for (int i = threadIdx.x; i <= count; i += 1024)
  {
    rows_of[i] = 0;
  }
  __syncthreads();
  // one addition for the lanes of a warp that have one adapter; the row's place in it
  auto place = [&](int id) {
    const bool live = id >= 0;
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, id);
    const int leader = __ffs(static_cast<int>(same)) - 1;
    int at = 0;
    if (live && lane == leader)
    {
      at = atomicAdd(&rows_of[id], __popc(same));
    }
    return __shfl_sync(0xFFFFFFFFu, at, leader) + __popc(same & ((1u << lane) - 1u));
  };
  // four rows a thread a trip, so that their indices come together
  auto groups = [&](int (&id)[4], int64_t base) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
      const int64_t row = base + i * 1024 + threadIdx.x;
      id[i] = row < m ? group_of(adapter_of_row, row, count) : -1;
    }
  };
  // (a call of one trip keeps its rows' places)
  int kept[4], kept_at[4];
  for (int64_t base = 0; base < m; base += 4096)
  {
    groups(kept, base);
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
      kept_at[i] = place(kept[i]);
    }
  }
  __syncthreads();
  // first tiles: an exclusive sum over the adapters, a run of them for each thread
  const int run = (count + 1024) / 1024;
  const int begin = static_cast<int>(threadIdx.x) * run;
  int sum = 0;
  for (int i = begin; i < begin + run && i <= count; ++i)
  {
    sum += (rows_of[i] + kTileRows - 1) / kTileRows;
  }
  int inclusive = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1)
  {
    const int other = __shfl_up_sync(0xFFFFFFFFu, inclusive, off);
    inclusive += lane >= off ? other : 0;
  }
  if (lane == 31)
  {
    warp_sums[warp] = inclusive;
  }
  __syncthreads();
  int before = 0, tiles = 0;
  for (int w = 0; w < 32; ++w)
  {
    before += w < warp ? warp_sums[w] : 0;
    tiles += warp_sums[w];
  }
  int tile = before + inclusive - sum;
  for (int i = begin; i < begin + run && i <= count; ++i)
  {
    first[i] = tile;
    const int rows = rows_of[i];
    const int mine = (rows + kTileRows - 1) / kTileRows;
    caifq_lora_entry e{};
    if (i < count && rows > 0)
    {
      e = entries[i];
    }
    for (int k = 0; k < mine; ++k)
    {
      plan.entry[tile + k] = e;
    }
    for (int r = rows; r < mine * kTileRows; ++r)
    {
      plan.rows[static_cast<int64_t>(tile) * kTileRows + r] = -1;
    }
    tile += mine;
  }
  for (int i = tiles + static_cast<int>(threadIdx.x); i < most; i += 1024)
  {
    plan.entry[i].rank = -1;
  }
  __syncthreads();
  auto deal = [&](const int (&id)[4], const int (&at)[4], int64_t base) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
      if (id[i] >= 0)
      {
        plan.rows[static_cast<int64_t>(first[id[i]]) * kTileRows + at[i]] = static_cast<int32_t>(base + i * 1024 + threadIdx.x);
      }
    }
  };
  if (m <= 4096)
  {
    deal(kept, kept_at, 0);
    return;
  }
  for (int i = threadIdx.x; i <= count; i += 1024)
  {
    rows_of[i] = 0;
  }
  __syncthreads();
  for (int64_t base = 0; base < m; base += 4096)
  {
    groups(kept, base);
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
      kept_at[i] = place(kept[i]);
    }
    deal(kept, kept_at, base);
  }
}

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1)
{
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the rows and adapter of tile `tile` of a call of m <= kSmallCall rows; false: there is no such tile.  All threads of the block
// (kSmallCall or more).
__device__ __forceinline__ bool small_tile(const int32_t *adapter_of_row, const caifq_lora_entry *entries, int count, int m, int tile,
                                           int (&rows)[kTileRows], caifq_lora_entry &entry)
{
  __shared__ __align__(16) int id_of[kSmallCall];
  __shared__ int warp_tiles[kSmallCall / 32];
  __shared__ int lead[2];   // the row that begins the tile, and how many of its adapter come before it
  const int i = threadIdx.x;
  const int id = i < m ? group_of(adapter_of_row, i, count) : -1;
  if (i < kSmallCall)
  {
    id_of[i] = id;
  }
  if (i < kTileRows)
  {
    rows[i] = -1;
  }
  __syncthreads();
  int before = __popc(__match_any_sync(0xFFFFFFFFu, id) & ((1u << (i & 31)) - 1u));
  for (int k = 0; k < (i < m ? (i & ~31) : 0); k += 4)
  {
    const int4 o = *reinterpret_cast<const int4 *>(id_of + k);
    before += (o.x == id ? 1 : 0) + (o.y == id ? 1 : 0) + (o.z == id ? 1 : 0) + (o.w == id ? 1 : 0);
  }
  const bool begins = i < m && before % kTileRows == 0;
  const uint32_t mask = __ballot_sync(0xFFFFFFFFu, begins);
  if ((i & 31) == 0 && i < kSmallCall)
  {
    warp_tiles[i >> 5] = __popc(mask);
  }
  __syncthreads();
  int tiles = 0, earlier = 0;
#pragma unroll
  for (int w = 0; w < kSmallCall / 32; ++w)
  {
    earlier += w < (i >> 5) ? warp_tiles[w] : 0;
    tiles += warp_tiles[w];
  }
  if (begins && earlier + __popc(mask & ((1u << (i & 31)) - 1u)) == tile)
  {
    lead[0] = i;
    lead[1] = before;
    entry = caifq_lora_entry{};
    if (id < count)
    {
      entry = entries[id];
    }
  }
  __syncthreads();
  if (tile >= tiles)
  {
    return false;
  }
  if (i < m && id == id_of[lead[0]] && before >= lead[1] && before < lead[1] + kTileRows)
  {
    rows[before - lead[1]] = i;
  }
  __syncthreads();
  return true;
}

// h of a tile.  As in the adapter's own thin product, a lane streams 16 bytes of two rows of x and of a row of A per 32 columns
// straight into fragments (the order of the columns inside a fragment is the same for both); the eight warps split the columns,
// and so do the blocks of a cluster where there are few tiles.
//
// h_part: the sums of this block's share of the columns, for the rows of a tile, in `part[0]`
template <int NT>   // eights of the largest rank
__device__ __forceinline__ void h_part(const __nv_bfloat16 *x, const int (&rows)[kTileRows], const caifq_lora_entry &entry, int in_dim,
                                       int cluster, int rank_in_cluster, float (&part)[8][kTileRows][NT * 8 + 1])
{
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2;
  const int t = lane & 3;
  const int eights = entry.rank / 8;
  const int steps = in_dim / 32;
  const int begin = static_cast<int>(static_cast<int64_t>(steps) * (rank_in_cluster * 8 + warp) / (8 * cluster));
  const int end = static_cast<int>(static_cast<int64_t>(steps) * (rank_in_cluster * 8 + warp + 1) / (8 * cluster));
  const uint4 zero4 = make_uint4(0u, 0u, 0u, 0u);
  const bool lo = rows[g] >= 0;
  const bool hi = rows[g + 8] >= 0;
  const uint4 *x_lo = reinterpret_cast<const uint4 *>(x + static_cast<int64_t>(lo ? rows[g] : 0) * in_dim) + t;
  const uint4 *x_hi = reinterpret_cast<const uint4 *>(x + static_cast<int64_t>(hi ? rows[g + 8] : 0) * in_dim) + t;
  const uint4 *a_row = reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(entry.a) + static_cast<int64_t>(g) * in_dim) + t;
  float c[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
  {
    c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.0f;
  }
  if constexpr (NT <= 4)
  {
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
  }
  else
  {
    // (all loads of two steps before the first product: 7000 rows, 50 adapters up to rank 64, 336 -> 317 us, 64 rows 38 -> 36; with
    // fewer rows of A a step the products on zeros cost more than the branches)
#pragma unroll 2
    for (int st = begin; st < end; ++st)
    {
      const uint4 xa = lo ? __ldg(x_lo + st * 4) : zero4;
      const uint4 xb = hi ? __ldg(x_hi + st * 4) : zero4;
      uint4 w[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
      {
        w[nt] = nt < eights ? __ldg(a_row + static_cast<int64_t>(nt) * in_dim + st * 4) : zero4;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
      {
        mma_16816(c[nt], xa.x, xb.x, xa.y, xb.y, w[nt].x, w[nt].y);
        mma_16816(c[nt], xa.z, xb.z, xa.w, xb.w, w[nt].z, w[nt].w);
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
  for (int e = threadIdx.x; e < kTileRows * NT * 8; e += 256)
  {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w)
    {
      v += part[w][e / (NT * 8)][e % (NT * 8)];
    }
    part[0][e / (NT * 8)][e % (NT * 8)] = v;
  }
}

template <int NT, bool SMALL>
__global__ void __launch_bounds__(256)
bank_down_mma_kernel(const __nv_bfloat16 *x, const int32_t *__restrict__ adapter_of_row,
                     const caifq_lora_entry *__restrict__ entries, int count, const BankPlan plan, int ld, int64_t m, int in_dim,
                     int cluster)
{
  __shared__ float part[8][kTileRows][NT * 8 + 1];
  __shared__ int rows[kTileRows];
  __shared__ caifq_lora_entry entry;
  // (what invariant loads read is addressed out of the wait, so that they stay behind it.  The wait comes before the next launch is
  // let in: `up` relies on it)
  asm volatile("griddepcontrol.wait;" : "+l"(adapter_of_row), "+l"(entries), "+l"(x)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int rank_in_cluster = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int64_t tile = blockIdx.x / cluster;
  if constexpr (SMALL)
  {
    // (every block of a cluster finds the same)
    if (!small_tile(adapter_of_row, entries, count, static_cast<int>(m), static_cast<int>(tile), rows, entry))
    {
      return;
    }
  }
  else
  {
    if (threadIdx.x < kTileRows)
    {
      rows[threadIdx.x] = plan.rows[tile * kTileRows + threadIdx.x];
    }
    if (threadIdx.x == 0)
    {
      entry = plan.entry[tile];
    }
    __syncthreads();
  }
  const int eights = entry.rank / 8;
  if (eights <= 0)
  {
    return;
  }
  h_part<NT>(x, rows, entry, in_dim, cluster, rank_in_cluster, part);
  if (cluster > 1)
  {
    cluster_sync_all();
  }
  else
  {
    __syncthreads();
  }
  const int share = kTileRows / cluster;
  for (int e = threadIdx.x; e < share * NT * 8; e += 256)
  {
    const int rr = rank_in_cluster * share + e / (NT * 8);
    const int col = e % (NT * 8);
    if (rows[rr] >= 0 && col < eights * 8)
    {
      float v = part[0][rr][col];
      if (cluster > 1)
      {
        const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(&part[0][rr][col]));
        float from[8];
#pragma unroll
        for (int b = 0; b < 8; ++b)   // (all on their way before the first is added)
        {
          from[b] = b < cluster ? __uint_as_float(ld_shared_cluster(map_to_cta(mine, static_cast<uint32_t>(b)))) : 0.0f;
        }
        v = ((from[0] + from[1]) + (from[2] + from[3])) + ((from[4] + from[5]) + (from[6] + from[7]));
      }
      plan.h[(tile * kTileRows + rr) * ld + col] = v;
    }
  }
  if (cluster > 1)
  {
    cluster_sync_all();   // nobody's partial tile is left while it is read
  }
}

// ---- y of 32 columns of a tile: a warp's work ----
// h enters as two bf16 terms (2^-16 relative).  The columns are dealt out to the four 8-wide tiles so that a lane ends with eight
// neighbouring ones of a row.

// h of rows g and g + 8 as fragments, four neighbouring ranks a lane per sixteen
template <int KS>   // sixteens of the largest rank
struct HTerms
{
  uint32_t top[KS][2][2], rest[KS][2][2];

  __device__ __forceinline__ void take(int ks, int half, const float4 &v)
  {
    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 2; ++i)
    {
      const uint32_t high = pack_bf16x2(e[2 * i], e[2 * i + 1]);
      // (an infinity has no second term)
      const float r0 = isfinite(e[2 * i]) ? e[2 * i] - __uint_as_float(high << 16) : 0.0f;
      const float r1 = isfinite(e[2 * i + 1]) ? e[2 * i + 1] - __uint_as_float(high & 0xFFFF0000u) : 0.0f;
      top[ks][half][i] = high;
      rest[ks][half][i] = pack_bf16x2(r0, r1);
    }
  }
};

// the adapter's rows of B for 32 columns, and the frozen product there
template <int KS>
struct UpColumns
{
  uint2 w[KS][4];
  float4 f[2][2];

  __device__ __forceinline__ void fetch_b(const __nv_bfloat16 *b, int rank, int col0, int out_dim)
  {
    const int lane = threadIdx.x & 31;
    const int g = lane >> 2;
    const int t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
    {
      const int n = col0 + 8 * (g >> 1) + 2 * nt + (g & 1);   // the column whose row of B this lane feeds
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
      {
        w[ks][nt] = make_uint2(0u, 0u);
        if (16 * ks + 4 * t < rank && n < out_dim)
        {
          w[ks][nt] = __ldg(reinterpret_cast<const uint2 *>(b + static_cast<int64_t>(n) * rank + 16 * ks + 4 * t));
        }
      }
    }
  }

  __device__ __forceinline__ void fetch_frozen(const float *frozen, const int32_t (&row_of)[2], int col0, int out_dim)
  {
    const int c = col0 + 8 * static_cast<int>(threadIdx.x & 3);
#pragma unroll
    for (int half = 0; half < 2; ++half)
    {
      if (row_of[half] >= 0 && c < out_dim)
      {
        const float4 *src = reinterpret_cast<const float4 *>(frozen + static_cast<int64_t>(row_of[half]) * out_dim + c);
        f[half][0] = src[0];
        f[half][1] = src[1];
      }
    }
  }

  // (rank 0, rows without an adapter: the frozen product, whatever the other rows hold)
  __device__ __forceinline__ void store(const HTerms<KS> &h, int rank, float scale, __nv_bfloat16 *y, const int32_t (&row_of)[2], int col0,
                                        int out_dim) const
  {
    float c[4][4];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
    {
      c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.0f;
      if (rank > 0)
      {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
        {
          mma_16816(c[nt], h.top[ks][0][0], h.top[ks][1][0], h.top[ks][0][1], h.top[ks][1][1], w[ks][nt].x, w[ks][nt].y);
          mma_16816(c[nt], h.rest[ks][0][0], h.rest[ks][1][0], h.rest[ks][0][1], h.rest[ks][1][1], w[ks][nt].x, w[ks][nt].y);
        }
      }
    }
    const int at = col0 + 8 * static_cast<int>(threadIdx.x & 3);
#pragma unroll
    for (int half = 0; half < 2; ++half)
    {
      if (row_of[half] >= 0 && at < out_dim)
      {
        const float4 *q = f[half];
        const int e = 2 * half;
        uint4 o;
        o.x = pack_bf16x2(fmaf(c[0][e], scale, q[0].x), fmaf(c[0][e + 1], scale, q[0].y));
        o.y = pack_bf16x2(fmaf(c[1][e], scale, q[0].z), fmaf(c[1][e + 1], scale, q[0].w));
        o.z = pack_bf16x2(fmaf(c[2][e], scale, q[1].x), fmaf(c[2][e + 1], scale, q[1].y));
        o.w = pack_bf16x2(fmaf(c[3][e], scale, q[1].z), fmaf(c[3][e + 1], scale, q[1].w));
        *reinterpret_cast<uint4 *>(y + static_cast<int64_t>(row_of[half]) * out_dim + at) = o;
      }
    }
  }
};

// y of a tile's rows and 128 * GROUPS columns, a warp GROUPS times 32.  Bound by latency (tile, then operands, then results) at few rows
// and by the frozen product's 4 bytes and y's 2 at many.
//
// A short call's block finds its rows and fetches its rows of B before it waits for the frozen product: what it reads for that was
// complete before `down`, which waited for it, let the frozen product's launch in, and with it this one.
template <int KS, int GROUPS, bool SMALL>
__global__ void __launch_bounds__(128)
bank_up_mma_kernel(const float *frozen, const int32_t *__restrict__ adapter_of_row, const caifq_lora_entry *__restrict__ entries,
                   int count, int64_t m, const BankPlan plan, __nv_bfloat16 *y, int ld, int out_dim)
{
  __shared__ int rows[kTileRows];
  __shared__ caifq_lora_entry entry_of_tile;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2;
  const int t = lane & 3;
  const int64_t tile = blockIdx.x;
  const int col0 = (static_cast<int>(blockIdx.y) * 4 + warp) * 32 * GROUPS;
  caifq_lora_entry entry;
  int32_t row_of[2];
  if constexpr (SMALL)
  {
    if (!small_tile(adapter_of_row, entries, count, static_cast<int>(m), static_cast<int>(tile), rows, entry_of_tile))
    {
      asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
      asm volatile("griddepcontrol.wait;" ::: "memory");   // (whoever follows relies on it)
      return;
    }
    entry = entry_of_tile;
    row_of[0] = rows[g];
    row_of[1] = rows[g + 8];
  }
  else
  {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    entry = plan.entry[tile];
    row_of[0] = plan.rows[tile * kTileRows + g];
    row_of[1] = plan.rows[tile * kTileRows + g + 8];
  }
  const int rank = entry.rank;
  if (rank < 0)
  {
    return;
  }
  UpColumns<KS> u[GROUPS];
#pragma unroll
  for (int i = 0; i < GROUPS; ++i)
  {
    u[i].fetch_b(static_cast<const __nv_bfloat16 *>(entry.b), rank, col0 + 32 * i, out_dim);
  }
  if constexpr (SMALL)
  {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
  }
  float4 v[KS][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
  {
#pragma unroll
    for (int half = 0; half < 2; ++half)
    {
      v[ks][half] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (row_of[half] >= 0 && 16 * ks + 4 * t < rank)
      {
        v[ks][half] = *reinterpret_cast<const float4 *>(plan.h + (tile * kTileRows + g + 8 * half) * ld + 16 * ks + 4 * t);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < GROUPS; ++i)
  {
    u[i].fetch_frozen(frozen, row_of, col0 + 32 * i, out_dim);
  }
  HTerms<KS> h;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
  {
    h.take(ks, 0, v[ks][0]);
    h.take(ks, 1, v[ks][1]);
  }
#pragma unroll
  for (int i = 0; i < GROUPS; ++i)
  {
    u[i].store(h, rank, entry.scale, y, row_of, col0 + 32 * i, out_dim);
  }
}

// Short calls with few columns to add to: both steps after the frozen product in one launch.  A cluster of a tile takes x . A^T, its
// blocks a share of the columns each; they give their sums to one another, and take a share of the columns of y.  Another launch
// less: 1024 -> 1024, one row 9.1 -> 7.7 us, 128 rows of 16 adapters 15.6 -> 13.9; 14336 -> 4096, 16 rows of 4 34.7 -> 30.3.  Many
// tiles of many columns want `up`'s small blocks, and B before the frozen product ends: 4096 -> 14336, 16 rows of 12, 25.7 and 27.2 so.
template <int NT>   // eights of the largest rank
__global__ void __launch_bounds__(256, 2)
bank_few_mma_kernel(const __nv_bfloat16 *x, const float *frozen, const int32_t *__restrict__ adapter_of_row,
                    const caifq_lora_entry *__restrict__ entries, int count, __nv_bfloat16 *y, int m, int in_dim, int out_dim, int cluster)
{
  constexpr int KS = (NT + 1) / 2;
  __shared__ float part[8][kTileRows][NT * 8 + 1];
  __shared__ __align__(16) float h_sum[kTileRows][KS * 16 + 4];
  __shared__ int rows[kTileRows];
  __shared__ caifq_lora_entry entry;
  asm volatile("griddepcontrol.wait;" : "+l"(adapter_of_row), "+l"(entries), "+l"(x)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2;
  const int t = lane & 3;
  const int rank_in_cluster = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = static_cast<int>(blockIdx.x) / cluster;
  // (every block of a cluster finds the same)
  if (!small_tile(adapter_of_row, entries, count, m, tile, rows, entry))
  {
    return;
  }
  const int rank = entry.rank;
  const int32_t row_of[2] = {rows[g], rows[g + 8]};
  const __nv_bfloat16 *b = static_cast<const __nv_bfloat16 *>(entry.b);
  const int groups = (out_dim + 31) / 32;   // of columns, a warp's work
  const int shares = cluster * static_cast<int>(gridDim.y);
  const int share = static_cast<int>(blockIdx.y) * cluster + rank_in_cluster;
  const int first = static_cast<int>(static_cast<int64_t>(groups) * share / shares);
  const int last = static_cast<int>(static_cast<int64_t>(groups) * (share + 1) / shares);
  UpColumns<KS> u;
  HTerms<KS> h{};
  int group = first + warp;
  if (group < last)
  {
    u.fetch_b(b, rank, group * 32, out_dim);
    u.fetch_frozen(frozen, row_of, group * 32, out_dim);
  }
  if (rank > 0)
  {
    h_part<NT>(x, rows, entry, in_dim, cluster, rank_in_cluster, part);
    if (cluster > 1)
    {
      cluster_sync_all();
    }
    else
    {
      __syncthreads();
    }
    for (int e = threadIdx.x; e < kTileRows * KS * 16; e += 256)
    {
      const int rr = e / (KS * 16);
      const int col = e % (KS * 16);
      float v = 0.0f;
      if (col < rank)
      {
        v = part[0][rr][col];
        if (cluster > 1)
        {
          const uint32_t mine = smem_u32(&part[0][rr][col]);
          float from[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)   // (all on their way before the first is added)
          {
            from[k] = k < cluster ? __uint_as_float(ld_shared_cluster(map_to_cta(mine, static_cast<uint32_t>(k)))) : 0.0f;
          }
          v = ((from[0] + from[1]) + (from[2] + from[3])) + ((from[4] + from[5]) + (from[6] + from[7]));
        }
      }
      h_sum[rr][col] = v;
    }
    if (cluster > 1)
    {
      cluster_sync_all();   // nobody's sums are left while they are read
    }
    else
    {
      __syncthreads();
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
    {
      h.take(ks, 0, *reinterpret_cast<const float4 *>(&h_sum[g][16 * ks + 4 * t]));
      h.take(ks, 1, *reinterpret_cast<const float4 *>(&h_sum[g + 8][16 * ks + 4 * t]));
    }
  }
  while (group < last)
  {
    const int next = group + 8;
    if constexpr (KS <= 2)   // (of rank 64 two groups do not fit the registers of two blocks an SM)
    {
      UpColumns<KS> ahead;
      if (next < last)
      {
        ahead.fetch_b(b, rank, next * 32, out_dim);
        ahead.fetch_frozen(frozen, row_of, next * 32, out_dim);
      }
      u.store(h, rank, entry.scale, y, row_of, group * 32, out_dim);
      u = ahead;
    }
    else
    {
      u.store(h, rank, entry.scale, y, row_of, group * 32, out_dim);
      if (next < last)
      {
        u.fetch_b(b, rank, next * 32, out_dim);
        u.fetch_frozen(frozen, row_of, next * 32, out_dim);
      }
    }
    group = next;
  }
}

size_t round_256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

// the plan in `scratch`, of lora_bank_scratch_bytes
BankPlan plan_in(void *scratch, int64_t tiles)
{
  char *p = static_cast<char *>(scratch);
  BankPlan plan;
  plan.entry = reinterpret_cast<caifq_lora_entry *>(p);
  p += round_256(static_cast<size_t>(tiles) * sizeof(caifq_lora_entry));
  plan.rows = reinterpret_cast<int32_t *>(p);
  p += round_256(static_cast<size_t>(tiles) * kTileRows * sizeof(int32_t));
  plan.h = reinterpret_cast<float *>(p);
  return plan;
}

int down_mma(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const void *x, int64_t m, void *scratch, cudaStream_t s)
{
  const int64_t tiles = most_tiles(m, bank.count);
  const BankPlan plan = plan_in(scratch, tiles);
  const bool small = m <= kSmallCall;
  if (!small)
  {
    CAIFQ_CHECK_CUDA(launch_dependent(bank_plan_kernel, dim3(1), dim3(1024), static_cast<size_t>(bank.count + 1) * 2 * sizeof(int), s,
                                      adapter_of_row, bank.entries, bank.count, plan, m, static_cast<int>(tiles)));
  }
  // clusters that split the columns where the tiles leave SMs without work, with at least two steps of 32 columns for every warp.
  // (4096 -> 14336 int4, 16 rows of 12 adapters: 10 us more with one block a tile; 4096 -> 4096, 48 rows of 16: 2 more)
  int cluster = 1;
  while (cluster < 8 && tiles * cluster < 2 * 148 && bank.in_dim / 32 >= 2 * cluster * 8 * 2)
  {
    cluster *= 2;
  }
  void (*down)(const __nv_bfloat16 *, const int32_t *, const caifq_lora_entry *, int, BankPlan, int, int64_t, int, int) = nullptr;
  if (bank.max_rank <= 8)
  {
    down = small ? bank_down_mma_kernel<1, true> : bank_down_mma_kernel<1, false>;
  }
  else if (bank.max_rank <= 16)
  {
    down = small ? bank_down_mma_kernel<2, true> : bank_down_mma_kernel<2, false>;
  }
  else if (bank.max_rank <= 32)
  {
    down = small ? bank_down_mma_kernel<4, true> : bank_down_mma_kernel<4, false>;
  }
  else
  {
    down = small ? bank_down_mma_kernel<8, true> : bank_down_mma_kernel<8, false>;
  }
  CAIFQ_CHECK_CUDA(launch_dependent_clusters(down, dim3(static_cast<unsigned>(tiles * cluster)), dim3(256), 0, s, cluster,
                                             static_cast<const __nv_bfloat16 *>(x), adapter_of_row, bank.entries, bank.count, plan,
                                             bank.max_rank, m, bank.in_dim, cluster));
  return CAIFQ_OK;
}

template <int KS, int GROUPS>
int up_mma_inst(const caifq_lora_bank &bank, const int32_t *adapter_of_row, int64_t m, const BankPlan &plan, int64_t tiles,
                const float *frozen, void *y, cudaStream_t s)
{
  auto kernel = m <= kSmallCall ? bank_up_mma_kernel<KS, GROUPS, true> : bank_up_mma_kernel<KS, GROUPS, false>;
  const unsigned columns = static_cast<unsigned>((bank.out_dim + 128 * GROUPS - 1) / (128 * GROUPS));
  CAIFQ_CHECK_CUDA(launch_dependent(kernel, dim3(static_cast<unsigned>(tiles), columns), dim3(128), 0, s, frozen, adapter_of_row,
                                    bank.entries, bank.count, m, plan, static_cast<__nv_bfloat16 *>(y), bank.max_rank, bank.out_dim));
  return CAIFQ_OK;
}

int up_mma(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const float *frozen, int64_t m, void *y, void *scratch,
           cudaStream_t s)
{
  const int64_t tiles = most_tiles(m, bank.count);
  const BankPlan plan = plan_in(scratch, tiles);
  if (bank.max_rank <= 16)
  {
    return up_mma_inst<1, 2>(bank, adapter_of_row, m, plan, tiles, frozen, y, s);
  }
  if (bank.max_rank <= 32)
  {
    return up_mma_inst<2, 2>(bank, adapter_of_row, m, plan, tiles, frozen, y, s);
  }
  return up_mma_inst<4, 1>(bank, adapter_of_row, m, plan, tiles, frozen, y, s);
}

// calls that bank_few_mma_kernel takes: by the tiles' columns, and by the rank where it is above 16.  (4096 -> 4096 int4, 18 tiles: rank 8 18.8 us
// and 20.0 with two launches around the product, 16 19.3 and 20.3, but 64 26.9 and 24.5; 64 tiles of rank 16 24.6 and 21.8; 4096 -> 8192, 9
// tiles: 16.2 and 16.5, 16.7 and 16.6, 23.7 and 21.6)
bool few(const caifq_lora_bank &bank, int64_t m)
{
  const int64_t sixteens = (bank.max_rank + 15) / 16;
  return m <= kSmallCall && most_tiles(m, bank.count) * bank.out_dim * sixteens <= 24 * 4096;
}

int few_mma(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const void *x, const float *frozen, int64_t m, void *y, cudaStream_t s)
{
  const int64_t tiles = most_tiles(m, bank.count);
  int cluster = 1;   // (each block a share of the columns of both)
  while (cluster < 8 && tiles * cluster < 2 * 148 && (bank.out_dim >= 256 * cluster || bank.in_dim >= 1024 * cluster))
  {
    cluster *= 2;
  }
  auto kernel = bank.max_rank <= 8
                    ? bank_few_mma_kernel<1>
                    : (bank.max_rank <= 16 ? bank_few_mma_kernel<2> : (bank.max_rank <= 32 ? bank_few_mma_kernel<4> : bank_few_mma_kernel<8>));
  // several clusters of a tile where its columns are many, each with the whole x . A^T (4096 -> 14336, 8 rows of 4: 17.5 us, 21.2 with one)
  int64_t parts = (bank.out_dim + 512 * cluster - 1) / (512 * cluster);
  const int64_t room = 4 * 148 / (tiles * cluster);
  parts = parts < room ? parts : (room < 1 ? 1 : room);
  CAIFQ_CHECK_CUDA(launch_dependent_clusters(kernel, dim3(static_cast<unsigned>(tiles * cluster), static_cast<unsigned>(parts)), dim3(256), 0, s, cluster,
                                             static_cast<const __nv_bfloat16 *>(x), frozen, adapter_of_row, bank.entries, bank.count,
                                             static_cast<__nv_bfloat16 *>(y), static_cast<int>(m), bank.in_dim, bank.out_dim, cluster));
  return CAIFQ_OK;
}

template <typename T>
int down_general(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const void *x, int64_t m, float *h, cudaStream_t s)
{
  int split = 1;
  while (split < 8 && m * bank.max_rank * split < 8 * 8 * 148 && bank.in_dim >= 256 * split)
  {
    split *= 2;
  }
  const int per = 8 / split;
  CAIFQ_CHECK_CUDA(launch_dependent(bank_down_kernel<T>, dim3(static_cast<unsigned>(m), static_cast<unsigned>((bank.max_rank + per - 1) / per)),
                                    dim3(kBankThreads), 0, s, static_cast<const T *>(x), adapter_of_row, bank.entries, bank.count,
                                    h, bank.max_rank, bank.in_dim, split));
  return CAIFQ_OK;
}

template <typename T>
int up_general(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const float *frozen, const float *h, int64_t m, void *y,
               cudaStream_t s)
{
  CAIFQ_CHECK_CUDA(launch_dependent(bank_up_kernel<T>,
                                    dim3(static_cast<unsigned>(m), static_cast<unsigned>((bank.out_dim + kBankColumns - 1) / kBankColumns)),
                                    dim3(kBankThreads), 0, s, frozen, h, adapter_of_row, bank.entries, bank.count,
                                    static_cast<T *>(y), bank.max_rank, bank.out_dim));
  return CAIFQ_OK;
}

bool on_16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// whether a call runs on the tensor core
bool tiled(const caifq_lora_bank &bank, const void *x, const void *y, const float *frozen, int64_t m)
{
  return bank.vectors != 0 && (bank.in_dim % 32) == 0 && (bank.out_dim % 8) == 0 && on_16(x) &&
         on_16(y) && on_16(frozen) && (m <= kSmallCall || bank.count <= kTableMost);
}

}  // namespace

// x . A^T of every row, and where the rows of each adapter are
size_t lora_bank_scratch_bytes(const caifq_lora_bank &bank, int64_t m)
{
  const size_t tiles = static_cast<size_t>(most_tiles(m, bank.count));
  const size_t rank = static_cast<size_t>(bank.max_rank);
  const size_t by_tile = round_256(tiles * sizeof(caifq_lora_entry)) + round_256(tiles * kTileRows * sizeof(int32_t)) +
                         tiles * kTileRows * rank * sizeof(float);
  const size_t by_row = static_cast<size_t>(m) * rank * sizeof(float);
  return round_256(bank.vectors != 0 && by_tile > by_row ? by_tile : by_row);
}

// The two launches around the frozen product, with the same arguments: x . A^T into the scratch (256-byte aligned), and
// y[m, out] = frozen[m, out] + the adapters' part; frozen (fp32) may be y itself.  m >= 1
int launch_lora_bank_down(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const void *x, const float *frozen, int64_t m,
                          const void *y, void *scratch, cudaStream_t s)
{
  if (tiled(bank, x, y, frozen, m))
  {
    return few(bank, m) ? CAIFQ_OK : down_mma(bank, adapter_of_row, x, m, scratch, s);
  }
  float *h = static_cast<float *>(scratch);
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

// frozen[m, out] = x . W^T in fp32 by bank_frozen_kernel, where it takes the call: int8 with one scale or none, int4 with groups of eights,
// rows of x on 16-byte boundaries, few of them.
// It reads the codes once for eight rows, the kernel for any cell once for 64 but by blocks of 64 x 64 that leave SMs idle where there are few:
// the time of one goes with eights of rows x columns, that of the other with its waves of two blocks an SM.  Whole call, own kernel and any
// cell, us:                        rows 32          64          96          128
//   fp32  1408 -> 1776 int4     28 / 179    52 / 183    76 / 183   101 / 185
//         2048 -> 4104 int4     81 / 259   153 / 265   221 / 269   294 / 271
//         4096 -> 14344 int4   472 / 631   917 / 642  1362 / 1294 1806 / 1313
//         4096 -> 14344 int8   283 / 474   671 / 490   894 / 969  1353 / 992
//   bf16  1408 -> 14344 int4   149 / 217   290 / 222   432 / 442   573 / 447
//         4096 -> 14344 int4   293 / 618   573 / 627   860 / 1272 1141 / 1281
//         4096 -> 14344 int8   250 / 459   510 / 465   756 / 958  1004 / 960
//   fp16  4096 -> 14344 int8   225 / 467   508 / 481   760 / 978   911 / 991
//         2048 -> 4104 int8     41 / 168    77 / 172   112 / 176   147 / 178
bool lora_bank_frozen_supported(const caifq_weight &w, const void *x, int dtype, int64_t m)
{
  const int64_t out = w.out_dim;
  const int64_t waves = ((out + 63) / 64 * ((m + 63) / 64) + 2 * 148 - 1) / (2 * 148);
  const int64_t most = (dtype == CAIFQ_F32 ? 60000 : 90000) * waves;
  return m <= 128 && (m + kFrozenRows - 1) / kFrozenRows * out <= most && (w.in_dim % 8) == 0 && on_16(x) &&
         (reinterpret_cast<uintptr_t>(w.codes) & 3u) == 0 &&
         ((w.storage == CAIFQ_I8 && (w.scales == nullptr || w.scheme == CAIFQ_PER_TENSOR)) ||
          (w.storage == CAIFQ_I4 && w.scales != nullptr && w.group_size > 0 && (w.group_size % 8) == 0));
}

namespace
{
template <typename T>
int frozen_of(const caifq_weight &w, const void *x, int64_t m, float *frozen, cudaStream_t s)
{
  auto kernel = w.storage == CAIFQ_I4 ? bank_frozen_kernel<T, true> : bank_frozen_kernel<T, false>;
  const dim3 grid(static_cast<unsigned>((w.out_dim + 7) / 8), static_cast<unsigned>((m + kFrozenRows - 1) / kFrozenRows));
  CAIFQ_CHECK_CUDA(launch_dependent(kernel, grid, dim3(kBankThreads), 0, s, static_cast<const T *>(x), static_cast<const uint8_t *>(w.codes),
                                    w.scales, frozen, m, w.in_dim, w.out_dim, w.group_size));
  return CAIFQ_OK;
}
}  // namespace

int launch_lora_bank_frozen(const caifq_weight &w, const void *x, int dtype, int64_t m, float *frozen, cudaStream_t s)
{
  switch (dtype)
  {
    case CAIFQ_F32:
      return frozen_of<float>(w, x, m, frozen, s);
    case CAIFQ_F16:
      return frozen_of<__half>(w, x, m, frozen, s);
    default:
      return frozen_of<__nv_bfloat16>(w, x, m, frozen, s);
  }
}

int launch_lora_bank_up(const caifq_lora_bank &bank, const int32_t *adapter_of_row, const void *x, const float *frozen, int64_t m,
                        void *y, void *scratch, cudaStream_t s)
{
  if (tiled(bank, x, y, frozen, m))
  {
    return few(bank, m) ? few_mma(bank, adapter_of_row, x, frozen, m, y, s) : up_mma(bank, adapter_of_row, frozen, m, y, scratch, s);
  }
  const float *h = static_cast<const float *>(scratch);
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
