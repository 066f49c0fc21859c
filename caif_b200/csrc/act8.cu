// Activations kept in 8 bits between an adapter's forward and backward pass, and the reductions over tokens that read them.
//
// A block is 32 columns of a row.  Its scale is s = 2^e, the smallest power of two (e >= -126) with max|x| <= 127 s; a code is
// rint(x / s), ties to even; the scale is stored as the byte e + 127.  A block with a value that is not finite has the byte
// 255 and codes of 0 and stands for NaN: a loss that ran off is not hidden by a checkpoint.
// Why a power of two, which costs up to one of the code's eight bits against max|x| / 127: code * s is exact in bf16 and
// fp32 (7 bits of significand), so x / s and the value need no rounding beyond the code's own and the backward pass
// multiplies the very rows that caifq_act_unpack gives; and a block's scale is one byte.
#include "umma.cuh"

namespace caifq
{

namespace
{

constexpr int kActBlock = 32;
constexpr int kActThreads = 256;

// scale byte of a block from the bits of its largest magnitude (as integers the bits of NaN lie above infinity's, and those
// above every number's)
__device__ __forceinline__ uint32_t scale_byte(uint32_t most)
{
  const uint32_t e = most >> 23;
  if (e == 255u)
  {
    return 255u;
  }
  // 127 = 1.984375 * 2^6: the largest significand that seven bits below it still hold
  const int b = static_cast<int>(e) - 6 + ((most & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);
  return b < 1 ? 1u : static_cast<uint32_t>(b);
}

// rint(v / s) in the low byte: adding 1.5 * 2^23 rounds to the nearest even integer
__device__ __forceinline__ uint32_t code_of(float v, float inverse) { return __float_as_uint(fmaf(v, inverse, 12582912.0f)); }

// 1 / s; 0 for a block that stands for NaN (finite values give codes of 0, the others NaN, which converts to 0)
__device__ __forceinline__ float inverse_of(uint32_t byte) { return byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23); }

// s; infinite for the byte 255, so that a code of 0 becomes NaN
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

template <typename T>
__device__ __forceinline__ float act_f(T v);
template <>
__device__ __forceinline__ float act_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float act_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float act_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T act_t(float v);
template <>
__device__ __forceinline__ float act_t<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half act_t<__half>(float v) { return __float2half(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 act_t<__nv_bfloat16>(float v) { return __float2bfloat16(v); }

// ---- any width, any alignment: a lane an element ----
// A warp takes sixteen neighbouring blocks of a row at a time, all on their way together (bound by latency: one after the other, 67000
// rows of 1000 bf16 took 210 us, four at a time 125).

constexpr int kActTrain = 16;

// trips of a warp over all rows; the same for every lane
struct ActTrips
{
  int blocks;       // of a row
  int trips;        // of a row
  int64_t total;

  __device__ __forceinline__ ActTrips(int64_t rows, int dim)
  {
    blocks = static_cast<int>((static_cast<int64_t>(dim) + kActBlock - 1) / kActBlock);
    trips = (blocks + kActTrain - 1) / kActTrain;
    total = rows * trips;
  }
};

template <typename T>
__global__ void __launch_bounds__(kActThreads)
act_pack_kernel(const T *x, int8_t *codes, uint8_t *scales, int64_t rows, int dim)
{
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const ActTrips k(rows, dim);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kActThreads / 32);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * (kActThreads / 32) + (threadIdx.x >> 5); i < k.total; i += step)
  {
    const int64_t row = k.trips == 1 ? i : i / k.trips;
    const int b0 = static_cast<int>(i - row * k.trips) * kActTrain;
    const int c0 = b0 * kActBlock + lane;
    const T *src = x + row * dim + c0;
    int8_t *dst = codes + row * dim + c0;
    const int left = dim - c0;   // this lane's columns from here on, every 32nd of them
    T v[kActTrain];
#pragma unroll
    for (int u = 0; u < kActTrain; ++u)
    {
      v[u] = u * kActBlock < left ? src[u * kActBlock] : act_t<T>(0.0f);
    }
    uint32_t mine = 0u;   // the scale byte of block `lane`
#pragma unroll
    for (int u = 0; u < kActTrain; ++u)
    {
      const float f = act_f<T>(v[u]);
      const uint32_t byte = scale_byte(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(f) & 0x7FFFFFFFu));
      mine = lane == u ? byte : mine;
      if (u * kActBlock < left)
      {
        dst[u * kActBlock] = static_cast<int8_t>(byte == 255u ? 0u : code_of(f, inverse_of(byte)));
      }
    }
    if (lane < kActTrain && b0 + lane < k.blocks)
    {
      scales[row * k.blocks + b0 + lane] = static_cast<uint8_t>(mine);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kActThreads)
act_unpack_kernel(const int8_t *codes, const uint8_t *scales, T *x, int64_t rows, int dim)
{
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const ActTrips k(rows, dim);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kActThreads / 32);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * (kActThreads / 32) + (threadIdx.x >> 5); i < k.total; i += step)
  {
    const int64_t row = k.trips == 1 ? i : i / k.trips;
    const int b0 = static_cast<int>(i - row * k.trips) * kActTrain;
    const int c0 = b0 * kActBlock + lane;
    const int8_t *src = codes + row * dim + c0;
    T *dst = x + row * dim + c0;
    const int left = dim - c0;
    const uint32_t mine = lane < kActTrain && b0 + lane < k.blocks ? scales[row * k.blocks + b0 + lane] : 1u;
    int8_t q[kActTrain];
#pragma unroll
    for (int u = 0; u < kActTrain; ++u)
    {
      q[u] = u * kActBlock < left ? src[u * kActBlock] : static_cast<int8_t>(0);
    }
#pragma unroll
    for (int u = 0; u < kActTrain; ++u)
    {
      const float s = scale_of(__shfl_sync(0xFFFFFFFFu, mine, u));
      if (u * kActBlock < left)
      {
        dst[u * kActBlock] = act_t<T>(static_cast<float>(q[u]) * s);
      }
    }
  }
}

unsigned act_grid(int64_t rows, int dim)
{
  const int64_t blocks = (static_cast<int64_t>(dim) + kActBlock - 1) / kActBlock;
  const int64_t warps = rows * ((blocks + kActTrain - 1) / kActTrain);
  const int64_t ctas = (warps + kActThreads / 32 - 1) / (kActThreads / 32);
  return static_cast<unsigned>(ctas < 148 * 64 ? ctas : 148 * 64);
}

// ---- rows of whole blocks on 16-byte boundaries: a thread 16 bytes of the row ----
// HBM-bound (8192 x 4096 bf16: 102 MB each way).  A thread holds kActTrip pieces so that all its loads are in flight before
// the first is used; the lanes of a block (4, or 8 of fp32) meet in two or three shuffles.  A code takes one fused multiply-add
// instead of a conversion, whose unit serves a sixteenth of a warp a cycle.

constexpr int kActTrip = 4;

// the bits of the largest magnitude of a 16-byte piece, as those of a fp32 number
template <typename T>
__device__ __forceinline__ uint32_t piece_most(const uint4 v)
{
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(T) == 4)
  {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
      m = max(m, w[i] & 0x7FFFFFFFu);
    }
    return m;
  }
  else
  {
    // two at a time as 16-bit integers: the order of magnitudes
    uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
    for (int i = 1; i < 4; ++i)
    {
      m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    }
    const uint16_t top = static_cast<uint16_t>(max(m >> 16, m & 0xFFFFu));
    return __float_as_uint(act_f<T>(*reinterpret_cast<const T *>(&top)));
  }
}

template <typename T>
__device__ __forceinline__ float piece_get(const uint32_t (&w)[4], int i)
{
  if constexpr (sizeof(T) == 4)
  {
    return __uint_as_float(w[i]);
  }
  else
  {
    const uint16_t h = static_cast<uint16_t>((i & 1) != 0 ? w[i >> 1] >> 16 : w[i >> 1]);
    return act_f<T>(*reinterpret_cast<const T *>(&h));
  }
}

// four codes a word
template <typename T>
__device__ __forceinline__ uint32_t codes_of(const uint32_t (&w)[4], int first, float inverse)
{
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
  {
    b[i] = code_of(piece_get<T>(w, first + i), inverse);
  }
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

template <typename T>
__global__ void __launch_bounds__(kActThreads)
act_pack_rows_kernel(const uint4 *x, void *codes, uint8_t *scales, int64_t pieces)
{
  constexpr int PER = 16 / sizeof(T);       // elements of a piece
  constexpr int LANES = kActBlock / PER;    // pieces of a block
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (kActThreads * kActTrip) + threadIdx.x;
  uint4 v[kActTrip];
#pragma unroll
  for (int u = 0; u < kActTrip; ++u)
  {
    const int64_t i = base + u * kActThreads;
    v[u] = i < pieces ? x[i] : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int u = 0; u < kActTrip; ++u)
  {
    const int64_t i = base + u * kActThreads;
    uint32_t most = piece_most<T>(v[u]);
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1)
    {
      most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, off));
    }
    const uint32_t byte = scale_byte(most);
    const float inverse = inverse_of(byte);
    const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
    // (a block that is not finite: codes of 0, whatever NaN would leave in the low byte)
    const uint32_t keep = byte == 255u ? 0u : 0xFFFFFFFFu;
    if (i < pieces)
    {
      if constexpr (PER == 8)
      {
        static_cast<uint2 *>(codes)[i] = make_uint2(codes_of<T>(w, 0, inverse) & keep, codes_of<T>(w, 4, inverse) & keep);
      }
      else
      {
        static_cast<uint32_t *>(codes)[i] = codes_of<T>(w, 0, inverse) & keep;
      }
      if ((threadIdx.x & (LANES - 1)) == 0)
      {
        scales[i / LANES] = static_cast<uint8_t>(byte);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kActThreads)
act_unpack_rows_kernel(const void *codes, const uint8_t *scales, uint4 *x, int64_t pieces)
{
  constexpr int PER = 16 / sizeof(T);
  constexpr int LANES = kActBlock / PER;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (kActThreads * kActTrip) + threadIdx.x;
  uint2 c[kActTrip];
  uint32_t b[kActTrip];
#pragma unroll
  for (int u = 0; u < kActTrip; ++u)
  {
    const int64_t i = base + u * kActThreads;
    c[u] = make_uint2(0u, 0u);
    b[u] = 1u;
    if (i < pieces)
    {
      if constexpr (PER == 8)
      {
        c[u] = static_cast<const uint2 *>(codes)[i];
      }
      else
      {
        c[u].x = static_cast<const uint32_t *>(codes)[i];
      }
      b[u] = scales[i / LANES];
    }
  }
#pragma unroll
  for (int u = 0; u < kActTrip; ++u)
  {
    const int64_t i = base + u * kActThreads;
    const float s = scale_of(b[u]);
    float f[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e)
    {
      // the code with its sign turned in the low mantissa of 2^23
      const uint32_t word = (e < 4 ? c[u].x : c[u].y) ^ 0x80808080u;
      f[e] = (__uint_as_float(__byte_perm(word, 0x4B000000u, 0x7440 + (e & 3))) - 8388736.0f) * s;
    }
    uint4 out;
    if constexpr (PER == 4)
    {
      out = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    else
    {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
      {
        const T lo = act_t<T>(f[2 * e]);
        const T hi = act_t<T>(f[2 * e + 1]);
        w[e] = static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(&lo)) |
               (static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(&hi)) << 16);
      }
      out = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (i < pieces)
    {
      x[i] = out;
    }
  }
}

bool whole_pieces(const void *x, const void *codes, int dim)
{
  return (dim % kActBlock) == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes)) & 15u) == 0;
}

// pieces that a launch can number
unsigned piece_grid(int64_t pieces)
{
  return static_cast<unsigned>((pieces + kActThreads * kActTrip - 1) / (kActThreads * kActTrip));
}

template <typename T>
int act_pack(const void *x, int8_t *codes, uint8_t *scales, int64_t rows, int dim, cudaStream_t s)
{
  const int64_t pieces = rows * dim / (16 / static_cast<int>(sizeof(T)));
  if (whole_pieces(x, codes, dim) && pieces <= (static_cast<int64_t>(1) << 40))
  {
    CAIFQ_CHECK_CUDA(launch_dependent(act_pack_rows_kernel<T>, dim3(piece_grid(pieces)), dim3(kActThreads), 0, s,
                                      static_cast<const uint4 *>(x), static_cast<void *>(codes), scales, pieces));
    return CAIFQ_OK;
  }
  CAIFQ_CHECK_CUDA(launch_dependent(act_pack_kernel<T>, dim3(act_grid(rows, dim)),
                                    dim3(kActThreads), 0, s, static_cast<const T *>(x), codes, scales, rows, dim));
  return CAIFQ_OK;
}

template <typename T>
int act_unpack(const int8_t *codes, const uint8_t *scales, void *x, int64_t rows, int dim, cudaStream_t s)
{
  const int64_t pieces = rows * dim / (16 / static_cast<int>(sizeof(T)));
  if (whole_pieces(x, codes, dim) && pieces <= (static_cast<int64_t>(1) << 40))
  {
    CAIFQ_CHECK_CUDA(launch_dependent(act_unpack_rows_kernel<T>, dim3(piece_grid(pieces)), dim3(kActThreads), 0, s,
                                      static_cast<const void *>(codes), scales, static_cast<uint4 *>(x), pieces));
    return CAIFQ_OK;
  }
  CAIFQ_CHECK_CUDA(launch_dependent(act_unpack_kernel<T>, dim3(act_grid(rows, dim)),
                                    dim3(kActThreads), 0, s, codes, scales, static_cast<T *>(x), rows, dim));
  return CAIFQ_OK;
}


// ---- reductions over tokens: both gradients of an adapter in one launch, and their sums over slices of tokens in a second ----
//   dB[out, r] = factor * sum_m dy[m, out] * h[m, r]        dA[r, in] = factor * sum_m dH[m, r] * x[m, in], x packed
// A slice's sums go to part[slice], dB's [out][r] and then dA's as [in][r]; gradients_kernel adds the slices in order and rounds
// once, so that equal calls give equal bits.

struct Gradients
{
  const void *dy;          // [m, out]
  const void *h;           // [m, r]
  const void *dh;          // [m, r]
  const void *dh_rest;     // in bf16: what its rounding left, as another bf16 number; null where dh is fp32
  const int8_t *x;         // [m, in]
  const uint8_t *scales;   // [m, ceil(in / 32)]
  float *part;
  void *d_b;               // with one slice: the results themselves, rounded here; else null
  void *d_a;
  float factor;
  int out, in, r;
};

// any type and width: 64 x 32 tiles of the result, fp32 multiply-adds, eight a thread for six values from shared memory.  The next
// tokens' loads are issued before this trip's products.  (32 x 32 tiles with four for four: 500 rows, 2048 columns each way, rank 64, 37 us instead of 23)
// A trip's 32 products are added up by themselves and then to the trips before (64 tokens or fewer: one chain): with one chain over a slice,
// 8192 tokens of a layer so wide that it has three slices lost 8e-5 of a sum to small terms.
constexpr int kTnWide = 64;
constexpr int kTnTile = 32;
constexpr int kTnRows = 32;
constexpr int kTnGeneralBlocks = 6;   // an SM

template <typename T, typename H, bool FEW>   // dy, h and the results; dH; so few tokens that one chain holds them
__device__ __forceinline__ void tn_general(const Gradients &j, int64_t m)
{
  constexpr int U = kTnRows * kTnWide / 256;
  constexpr int V = kTnRows * kTnTile / 256;
  __shared__ __align__(16) float su[kTnRows][kTnWide + 4];
  __shared__ __align__(16) float sv[kTnRows][kTnTile + 2];
  const int tid = threadIdx.x;
  const int tiles_b = (j.out + kTnWide - 1) / kTnWide;
  const bool is_a = static_cast<int>(blockIdx.x) >= tiles_b;
  const int wide = is_a ? j.in : j.out;   // the dimension that is not the rank
  const int c0 = (static_cast<int>(blockIdx.x) - (is_a ? tiles_b : 0)) * kTnWide;
  const int r0 = blockIdx.y * kTnTile;
  const int64_t begin = m * blockIdx.z / gridDim.z;
  const int64_t end = m * (blockIdx.z + 1) / gridDim.z;
  const int blocks = (j.in + kActBlock - 1) / kActBlock;
  const int tq = tid % 16;
  const int tp = tid / 16;
  float u[U], v[V];
  auto fetch = [&](int64_t mb) {
    const int col = c0 + tid % kTnWide;
    const int64_t row0 = mb + tid / kTnWide;
    if (is_a)
    {
#pragma unroll
      for (int i = 0; i < U; ++i)
      {
        const int64_t row = row0 + i * (256 / kTnWide);
        u[i] = row < end && col < wide ? static_cast<float>(j.x[row * wide + col]) * scale_of(j.scales[row * blocks + col / kActBlock]) : 0.0f;
      }
    }
    else
    {
#pragma unroll
      for (int i = 0; i < U; ++i)
      {
        const int64_t row = row0 + i * (256 / kTnWide);
        u[i] = row < end && col < wide ? act_f<T>(static_cast<const T *>(j.dy)[row * wide + col]) : 0.0f;
      }
    }
    const int rr = r0 + tid % kTnTile;
#pragma unroll
    for (int i = 0; i < V; ++i)
    {
      const int64_t row = mb + tid / kTnTile + i * (256 / kTnTile);
      v[i] = 0.0f;
      if (row < end && rr < j.r)
      {
        v[i] = is_a ? act_f<H>(static_cast<const H *>(j.dh)[row * j.r + rr]) : act_f<T>(static_cast<const T *>(j.h)[row * j.r + rr]);
        if constexpr (sizeof(H) == 2)
        {
          v[i] += is_a ? act_f<H>(static_cast<const H *>(j.dh_rest)[row * j.r + rr]) : 0.0f;
        }
      }
    }
  };
  float c[4][2] = {}, sum[4][2] = {};
  fetch(begin);
  for (int64_t mb = begin; mb < end; mb += kTnRows)
  {
#pragma unroll
    for (int i = 0; i < U; ++i)
    {
      su[tid / kTnWide + i * (256 / kTnWide)][tid % kTnWide] = u[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
    {
      sv[tid / kTnTile + i * (256 / kTnTile)][tid % kTnTile] = v[i];
    }
    __syncthreads();
    if (mb + kTnRows < end)
    {
      fetch(mb + kTnRows);
    }
#pragma unroll 8
    for (int r = 0; r < kTnRows; ++r)
    {
      const float4 p = *reinterpret_cast<const float4 *>(&su[r][tp * 4]);
      const float2 q = *reinterpret_cast<const float2 *>(&sv[r][tq * 2]);
      c[0][0] = fmaf(p.x, q.x, c[0][0]);
      c[0][1] = fmaf(p.x, q.y, c[0][1]);
      c[1][0] = fmaf(p.y, q.x, c[1][0]);
      c[1][1] = fmaf(p.y, q.y, c[1][1]);
      c[2][0] = fmaf(p.z, q.x, c[2][0]);
      c[2][1] = fmaf(p.z, q.y, c[2][1]);
      c[3][0] = fmaf(p.w, q.x, c[3][0]);
      c[3][1] = fmaf(p.w, q.y, c[3][1]);
    }
    if constexpr (!FEW)
    {
#pragma unroll
      for (int i = 0; i < 8; ++i)
      {
        sum[i >> 1][i & 1] += c[i >> 1][i & 1];
        c[i >> 1][i & 1] = 0.0f;
      }
    }
    __syncthreads();
  }
  float *part = j.part + static_cast<int64_t>(blockIdx.z) * (static_cast<int64_t>(j.out) + j.in) * j.r +
                (is_a ? static_cast<int64_t>(j.out) * j.r : 0);
#pragma unroll
  for (int a = 0; a < 4; ++a)
  {
#pragma unroll
    for (int b = 0; b < 2; ++b)
    {
      const int col = c0 + tp * 4 + a;
      const int rr = r0 + tq * 2 + b;
      const float total = FEW ? c[a][b] : sum[a][b];
      if (col < wide && rr < j.r)
      {
        if (j.d_b == nullptr)
        {
          part[static_cast<int64_t>(col) * j.r + rr] = total;
        }
        else if (is_a)
        {
          static_cast<T *>(j.d_a)[static_cast<int64_t>(rr) * j.in + col] = act_t<T>(total * j.factor);
        }
        else
        {
          static_cast<T *>(j.d_b)[static_cast<int64_t>(col) * j.r + rr] = act_t<T>(total * j.factor);
        }
      }
    }
  }
}

template <typename T, typename H>
__global__ void __launch_bounds__(256) act_tn_kernel(const Gradients j, int64_t m)
{
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  tn_general<T, H, false>(j, m);
}

// bf16, ranks 8, 16, 32, 64, widths of whole 128-column tiles: the tensor core, as the adapter's reductions on full rows run it (both
// operands have the token as their slow axis: tiles lie in shared memory as they come, fragments are read transposed).  A tile of
// 64 tokens x 128 columns is 16 KB of dy, or 8 KB of codes, which become bf16 numbers on the way to shared memory: code * s has
// seven bits of significand, so the products are those of the expanded rows.  dH comes as two bf16 terms, whose products with the codes meet in
// one sum (2^-16 of dH; as one term the error of dA is 2.4e-3 instead of 1.7e-3, and a caller of fp32 compute does not expect it; the second
// costs 4 us of 227 at 4096 -> 4096, 8192 tokens, rank 16, and 26 of 260 at rank 64.  More slices for dA than for dB got back 8 of these, and
// cost 3 of 131 at 14336 -> 4096, 1000 tokens, rank 16).  Bound by HBM: dy and the codes once.
constexpr int kTnColumns = 128;
constexpr int kTnTokens = 64;
constexpr int kTnPitch = kTnColumns + 8;   // bf16 elements: 272-byte rows keep the transposed reads free of conflicts

__device__ __forceinline__ void tn_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// sixteen codes and their scale byte as bf16 numbers, exactly
__device__ __forceinline__ void codes_to_bf16(const uint4 c, uint32_t byte, uint4 (&out)[2])
{
  const uint32_t s = (byte << 7) | (byte << 23);   // bf16 numbers of that exponent; infinite for 255: NaN with codes of 0
  const uint4 p = expand_int8x8(make_uint2(c.x, c.y));
  const uint4 q = expand_int8x8(make_uint2(c.z, c.w));
  out[0] = make_uint4(mul_bf16x2(p.x, s), mul_bf16x2(p.y, s), mul_bf16x2(p.z, s), mul_bf16x2(p.w, s));
  out[1] = make_uint4(mul_bf16x2(q.x, s), mul_bf16x2(q.y, s), mul_bf16x2(q.z, s), mul_bf16x2(q.w, s));
}

// blocks an SM: the accumulators of large ranks leave room for two
template <int NT>
constexpr int kTnBlocks = NT <= 2 ? 4 : 2;

template <int NT>   // rank / 8
__global__ void __launch_bounds__(256, kTnBlocks<NT>) act_tn_mma_kernel(const Gradients j, int64_t m)
{
  constexpr int R = 8 * NT;
  __shared__ __align__(16) __nv_bfloat16 su[kTnTokens][kTnPitch];
  __shared__ __align__(16) __nv_bfloat16 sv[2][kTnTokens][R + 8];   // (h, or dH and what its rounding left)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x;
  // a warp 16 columns and all ranks, or, of large ranks, 32 columns and half of them, so that the thin operand crosses shared memory half as often
  constexpr int WC = NT >= 4 ? 2 : 1;
  constexpr int NW = NT / WC;
  const int col_w = (tid >> 5) % (8 / WC) * WC * 16;
  const int rank_w = (tid >> 5) / (8 / WC) * NW * 8;
  const int lane = tid & 31;
  const int g = lane >> 2;
  const int t = lane & 3;
  const int tiles_b = j.out / kTnColumns;
  const bool is_a = static_cast<int>(blockIdx.x) >= tiles_b;
  const int c0 = (static_cast<int>(blockIdx.x) - (is_a ? tiles_b : 0)) * kTnColumns;
  const int wide = is_a ? j.in : j.out;
  const int64_t per = ((m + gridDim.y - 1) / gridDim.y + kTnTokens - 1) / kTnTokens * kTnTokens;
  const int64_t begin = per * blockIdx.y;
  const int64_t end = begin + per < m ? begin + per : m;
  const __nv_bfloat16 *v = static_cast<const __nv_bfloat16 *>(is_a ? j.dh : j.h);
  const __nv_bfloat16 *v_rest = static_cast<const __nv_bfloat16 *>(j.dh_rest);
  constexpr int THIN = kTnTokens * NT;             // 16-byte pieces of a tile of the thin operand
  constexpr int RV = (2 * THIN + 255) / 256;
  const int thin = is_a ? 2 * THIN : THIN;
  float c[WC][NW][4] = {};
  // the next tile's loads are issued before this one's products: 16-byte pieces of dy (four a thread) or of codes (two, with
  // their scale bytes), and of the thin operand
  uint4 ru[4];
  uint32_t rs[2];
  uint4 rv[RV];
  auto fetch = [&](int64_t mb) {
    if (is_a)
    {
#pragma unroll
      for (int i = 0; i < 2; ++i)
      {
        const int e = tid + i * 256;
        const int64_t row = mb + (e >> 3);
        const int col = c0 + (e & 7) * 16;
        ru[i] = make_uint4(0u, 0u, 0u, 0u);
        rs[i] = 1u;
        if (row < end)
        {
          ru[i] = *reinterpret_cast<const uint4 *>(j.x + row * wide + col);
          rs[i] = j.scales[row * (wide / kActBlock) + col / kActBlock];
        }
      }
    }
    else
    {
#pragma unroll
      for (int i = 0; i < 4; ++i)
      {
        const int e = tid + i * 256;
        const int64_t row = mb + (e >> 4);
        ru[i] = make_uint4(0u, 0u, 0u, 0u);
        if (row < end)
        {
          ru[i] = *reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(j.dy) + row * wide + c0 + (e & 15) * 8);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < RV; ++i)
    {
      const int e = tid + i * 256;
      rv[i] = make_uint4(0u, 0u, 0u, 0u);
      if (e < thin && mb + e % THIN / NT < end)
      {
        rv[i] = *reinterpret_cast<const uint4 *>((e < THIN ? v : v_rest) + (mb + e % THIN / NT) * R + (e % NT) * 8);
      }
    }
  };
  if (begin < end)
  {
    fetch(begin);
  }
  for (int64_t mb = begin; mb < end; mb += kTnTokens)
  {
    if (is_a)
    {
#pragma unroll
      for (int i = 0; i < 2; ++i)
      {
        const int e = tid + i * 256;
        uint4 o[2];
        codes_to_bf16(ru[i], rs[i], o);
        uint4 *dst = reinterpret_cast<uint4 *>(&su[e >> 3][(e & 7) * 16]);
        dst[0] = o[0];
        dst[1] = o[1];
      }
    }
    else
    {
#pragma unroll
      for (int i = 0; i < 4; ++i)
      {
        const int e = tid + i * 256;
        *reinterpret_cast<uint4 *>(&su[e >> 4][(e & 15) * 8]) = ru[i];
      }
    }
#pragma unroll
    for (int i = 0; i < RV; ++i)
    {
      const int e = tid + i * 256;
      if (e < thin)
      {
        *reinterpret_cast<uint4 *>(&sv[e / THIN][e % THIN / NT][(e % NT) * 8]) = rv[i];
      }
    }
    __syncthreads();
    if (mb + kTnTokens < end)
    {
      fetch(mb + kTnTokens);
    }
#pragma unroll
    for (int k16 = 0; k16 < kTnTokens / 16; ++k16)
    {
      // rows of the product: this warp's columns, 16 at a time; lane l addresses row (l & 7) of 8 x 8 tile (l >> 3)
      const int tile = lane >> 3;
      uint32_t a[WC][4];
#pragma unroll
      for (int i = 0; i < WC; ++i)
      {
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(a[i][0]), "=r"(a[i][1]), "=r"(a[i][2]), "=r"(a[i][3])
                     : "r"(smem_u32(&su[k16 * 16 + (tile >> 1) * 8 + (lane & 7)][col_w + i * 16 + (tile & 1) * 8])));
      }
      auto multiply = [&](int plane) {
#pragma unroll
        for (int nt = 0; nt < NW; ++nt)
        {
          uint32_t b0, b1;
          asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
                       : "=r"(b0), "=r"(b1)
                       : "r"(smem_u32(&sv[plane][k16 * 16 + (lane & 15)][rank_w + nt * 8])));
#pragma unroll
          for (int i = 0; i < WC; ++i)
          {
            tn_mma(c[i][nt], a[i][0], a[i][1], a[i][2], a[i][3], b0, b1);
          }
        }
      };
      multiply(0);
      if (is_a)
      {
        multiply(1);
      }
    }
    __syncthreads();
  }
  float *part = j.part + static_cast<int64_t>(blockIdx.y) * (static_cast<int64_t>(j.out) + j.in) * R +
                (is_a ? static_cast<int64_t>(j.out) * R : 0);
#pragma unroll
  for (int i = 0; i < WC * NW; ++i)
  {
#pragma unroll
    for (int half = 0; half < 2; ++half)
    {
      const int64_t col = c0 + col_w + i / NW * 16 + g + 8 * half;
      const int rr = rank_w + i % NW * 8 + 2 * t;
      const float lo = c[i / NW][i % NW][2 * half], hi = c[i / NW][i % NW][2 * half + 1];
      if (j.d_b == nullptr)
      {
        *reinterpret_cast<float2 *>(part + col * R + rr) = make_float2(lo, hi);
      }
      else if (is_a)
      {
        __nv_bfloat16 *d_a = static_cast<__nv_bfloat16 *>(j.d_a) + static_cast<int64_t>(rr) * j.in + col;
        d_a[0] = __float2bfloat16(lo * j.factor);
        d_a[j.in] = __float2bfloat16(hi * j.factor);
      }
      else
      {
        __nv_bfloat16 *d_b = static_cast<__nv_bfloat16 *>(j.d_b) + col * R + rr;
        d_b[0] = __float2bfloat16(lo * j.factor);
        d_b[1] = __float2bfloat16(hi * j.factor);
      }
    }
  }
}

// dH[m, r] = dy . B for the same adapters, with the transposed copy bt[r, out] of B: as two bf16 terms, and times `mul` / *div in bf16, padded to
// 64 columns, as the extra k-block of the product that gives dx.  A block takes 32 rows, so that bt crosses the SM's cache once for 32 rows and not once for
// 16 (8192 x 4096, rank 16: it is as many bytes as 16 rows of dy); eight warps split the columns, in 16-byte pieces straight into
// fragments (the order of the columns inside a fragment is the same for both operands).
template <int NT>
__global__ void __launch_bounds__(256, NT <= 2 ? 3 : 2)
act_nt_mma_kernel(const __nv_bfloat16 *dy, const __nv_bfloat16 *bt, __nv_bfloat16 *dh, __nv_bfloat16 *rest, __nv_bfloat16 *padded, float mul,
                  const float *div, int64_t m, int out)
{
  constexpr int R = 8 * NT;
  __shared__ float part[8][16][R + 1];
  asm volatile("griddepcontrol.wait;" : "+l"(dy), "+l"(bt), "+l"(div)::"memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2;
  const int t = lane & 3;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * 32;
  const int steps = out / 32;
  const int begin = steps * warp / 8;
  const int end = steps * (warp + 1) / 8;
  const uint4 *src[4];
  bool live[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
  {
    live[i] = row0 + g + 8 * i < m;
    src[i] = reinterpret_cast<const uint4 *>(dy + (live[i] ? row0 + g + 8 * i : 0) * out) + t;
  }
  const uint4 *b_row = reinterpret_cast<const uint4 *>(bt + static_cast<int64_t>(g) * out) + t;
  float c[2][NT][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
  {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
    {
      c[i][nt][0] = c[i][nt][1] = c[i][nt][2] = c[i][nt][3] = 0.0f;
    }
  }
#pragma unroll 2
  for (int st = begin; st < end; ++st)
  {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
      v[i] = live[i] ? __ldg(src[i] + st * 4) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
    {
      const uint4 w = __ldg(b_row + static_cast<int64_t>(nt) * out + st * 4);
#pragma unroll
      for (int i = 0; i < 2; ++i)
      {
        tn_mma(c[i][nt], v[2 * i].x, v[2 * i + 1].x, v[2 * i].y, v[2 * i + 1].y, w.x, w.y);
        tn_mma(c[i][nt], v[2 * i].z, v[2 * i + 1].z, v[2 * i].w, v[2 * i + 1].w, w.z, w.w);
      }
    }
  }
  const float factor = div != nullptr ? mul / __ldg(div) : mul;
#pragma unroll
  for (int i = 0; i < 2; ++i)   // sixteen rows at a time
  {
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
    {
      part[warp][g][nt * 8 + 2 * t] = c[i][nt][0];
      part[warp][g][nt * 8 + 2 * t + 1] = c[i][nt][1];
      part[warp][g + 8][nt * 8 + 2 * t] = c[i][nt][2];
      part[warp][g + 8][nt * 8 + 2 * t + 1] = c[i][nt][3];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * 32; e += 256)
    {
      const int64_t row = row0 + 16 * i + (e >> 5);
      const int col = (e & 31) * 2;
      if (row < m)
      {
        uint32_t pad = 0u;
        if (col < R)
        {
          float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int w = 0; w < 8; ++w)
          {
            sum.x += part[w][e >> 5][col];
            sum.y += part[w][e >> 5][col + 1];
          }
          const uint32_t top = pack_bf16x2(sum.x, sum.y);
          *reinterpret_cast<uint32_t *>(dh + row * R + col) = top;
          *reinterpret_cast<uint32_t *>(rest + row * R + col) = rest_bf16x2(sum.x, sum.y, top);
          pad = pack_bf16x2(sum.x * factor, sum.y * factor);
        }
        *reinterpret_cast<uint32_t *>(padded + row * 64 + col) = pad;
      }
    }
  }
}

// the slices' sums, rounded once: [out][r] as it lies, [in][r] turned to [r, in]; `block` of 256 sums
struct GradientSums
{
  const float *part;
  void *d_b;
  void *d_a;
  float factor;
  int dtype, slices, in, r;
  int64_t n_b;
};

__device__ __forceinline__ void gradient_sums(const GradientSums &j, int64_t block)
{
  const int64_t n = j.n_b + static_cast<int64_t>(j.in) * j.r;
  const int64_t i = block * 256 + threadIdx.x;
  if (i >= n)
  {
    return;
  }
  float s = 0.0f;
#pragma unroll 4
  for (int z = 0; z < j.slices; ++z)
  {
    s += j.part[static_cast<int64_t>(z) * n + i];
  }
  if (i < j.n_b)
  {
    store_from_float(j.d_b, i, j.dtype, s * j.factor);
  }
  else
  {
    const int64_t e = i - j.n_b;
    store_from_float(j.d_a, (e % j.r) * j.in + e / j.r, j.dtype, s * j.factor);
  }
}

__global__ void __launch_bounds__(256) gradients_kernel(const GradientSums j)
{
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  gradient_sums(j, blockIdx.x);
}

// ---- what the general form of the backward pass multiplies by itself ----

constexpr int kDhChunk = 1024;

// dH[m, r] = dy . B, fp32: a block a row.  B's rows lie one behind the other, so the block reads it as one run of numbers and a
// thread always meets the same column of it; the row of dy waits in shared memory.
template <typename T>
__global__ void __launch_bounds__(256)
dh_row_kernel(const T *dy, const T *b, float *dh, int64_t m, int out, int r)
{
  __shared__ float row[kDhChunk];
  __shared__ float sums[256];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x;
  const int64_t at = blockIdx.x;
  for (int j0 = 0; j0 < r; j0 += 256)
  {
    const int width = r - j0 < 256 ? r - j0 : 256;   // columns of this trip
    const int groups = 256 / width;                  // rows of B at a time
    const int j = tid % width;
    const int group = tid / width;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // (sixteen loads on their way, four chains of additions)
    for (int c0 = 0; c0 < out; c0 += kDhChunk)
    {
      const int n = out - c0 < kDhChunk ? out - c0 : kDhChunk;
      __syncthreads();   // the chunk before has been read
      for (int i = tid; i < n; i += 256)
      {
        row[i] = act_f<T>(dy[at * out + c0 + i]);
      }
      __syncthreads();
      if (group < groups)
      {
        int o = group;
        for (; o + 15 * groups < n; o += 16 * groups)
        {
          float w[16];
#pragma unroll
          for (int u = 0; u < 16; ++u)
          {
            w[u] = act_f<T>(b[static_cast<int64_t>(c0 + o + u * groups) * r + j0 + j]);
          }
#pragma unroll
          for (int u = 0; u < 16; ++u)
          {
            s[u & 3] = fmaf(row[o + u * groups], w[u], s[u & 3]);
          }
        }
        for (; o < n; o += groups)
        {
          s[0] = fmaf(row[o], act_f<T>(b[static_cast<int64_t>(c0 + o) * r + j0 + j]), s[0]);
        }
      }
    }
    __syncthreads();
    sums[tid] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (tid < width)
    {
      float v = 0.0f;
      for (int g0 = 0; g0 < groups; g0 += 16)   // (up to 256 of them, for a rank of 1: sixteen at a time by themselves)
      {
        float some = 0.0f;
        for (int i = g0; i < groups && i < g0 + 16; ++i)
        {
          some += sums[i * width + tid];
        }
        v += some;
      }
      dh[at * r + j0 + tid] = v;
    }
  }
}

// The same where B is large: a cluster four or eight rows, its blocks a share of the columns each; a number of B serves those rows, and
// the blocks' sums are added in order.  64 products of a row are added up by themselves and then to those before (one chain of every other
// product of 14336 lost 2e-4 of a sum to small terms).
constexpr int kDhPart = 512;

template <typename T, int kDhRows>   // 4 or 8
__global__ void __launch_bounds__(256)
dh_kernel(const T *dy, const T *b, float *dh, int64_t m, int out, int r, int cluster)
{
  __shared__ __align__(16) float row[kDhPart][kDhRows];   // (a number of B meets four rows' with one load)
  __shared__ float sums[kDhRows][256];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x;
  const int rank = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / cluster) * kDhRows;
  const int begin = static_cast<int>(static_cast<int64_t>(out) * rank / cluster);
  const int end = static_cast<int>(static_cast<int64_t>(out) * (rank + 1) / cluster);
  for (int j0 = 0; j0 < r; j0 += 256)
  {
    const int width = r - j0 < 256 ? r - j0 : 256;   // columns of this trip
    const int groups = 256 / width;                  // rows of B at a time
    const int j = tid % width;
    const int group = tid / width;
    constexpr int CHAINS = 8 / kDhRows;   // of a row: eight in all, so that multiply-adds follow one another
    float s[kDhRows][CHAINS] = {}, sum[kDhRows] = {};
    auto gather = [&]() {
#pragma unroll
      for (int q = 0; q < kDhRows; ++q)
      {
        sum[q] += CHAINS == 2 ? s[q][0] + s[q][CHAINS - 1] : s[q][0];
        s[q][0] = s[q][CHAINS - 1] = 0.0f;
      }
    };
    for (int c0 = begin; c0 < end; c0 += kDhPart)
    {
      const int n = end - c0 < kDhPart ? end - c0 : kDhPart;
      __syncthreads();   // the chunk before has been read
      for (int i = tid; i < kDhRows * kDhPart; i += 256)
      {
        const int rr = i / kDhPart;
        const int c = i % kDhPart;
        row[c][rr] = row0 + rr < m && c < n ? act_f<T>(dy[(row0 + rr) * out + c0 + c]) : 0.0f;
      }
      __syncthreads();
      if (group < groups)
      {
        auto meet = [&](int at, float w, int chain) {
#pragma unroll
          for (int q = 0; q < kDhRows; q += 4)
          {
            const float4 v = *reinterpret_cast<const float4 *>(&row[at][q]);
            s[q][chain] = fmaf(v.x, w, s[q][chain]);
            s[q + 1][chain] = fmaf(v.y, w, s[q + 1][chain]);
            s[q + 2][chain] = fmaf(v.z, w, s[q + 2][chain]);
            s[q + 3][chain] = fmaf(v.w, w, s[q + 3][chain]);
          }
        };
        int o = group;
        const T *src = b + static_cast<int64_t>(c0 + o) * r + j0 + j;
        const int64_t step = static_cast<int64_t>(groups) * r;
        int trip = 0;
        for (; o + 15 * groups < n; o += 16 * groups, src += 16 * step)
        {
          T w[16];   // (all on their way before the first is used)
#pragma unroll
          for (int u = 0; u < 16; ++u)
          {
            w[u] = src[u * step];
          }
#pragma unroll
          for (int u = 0; u < 16; ++u)
          {
            meet(o + u * groups, act_f<T>(w[u]), u % CHAINS);
          }
          if ((++trip & 3) == 0)
          {
            gather();
          }
        }
        for (; o < n; o += groups, src += step)
        {
          meet(o, act_f<T>(*src), 0);
        }
        gather();
      }
    }
    __syncthreads();
#pragma unroll
    for (int rr = 0; rr < kDhRows; ++rr)
    {
      sums[rr][tid] = sum[rr];
    }
    __syncthreads();
    // a thread adds the groups of one row and column; in place, where its own first group lies
    for (int e = tid; e < kDhRows * width; e += 256)
    {
      float v = 0.0f;
      for (int i = 0; i < groups; ++i)
      {
        v += sums[e / width][i * width + e % width];
      }
      sums[e / width][e % width] = v;
    }
    if (cluster > 1)
    {
      cluster_sync_all();
    }
    else
    {
      __syncthreads();
    }
    for (int e = rank * 256 + tid; e < kDhRows * width; e += cluster * 256)
    {
      const int rr = e / width;
      float v = sums[rr][e % width];
      if (cluster > 1)
      {
        const uint32_t mine = smem_u32(&sums[rr][e % width]);
        float from[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)   // (all on their way before the first is added)
        {
          from[k] = k < cluster ? __uint_as_float(ld_shared_cluster(map_to_cta(mine, static_cast<uint32_t>(k)))) : 0.0f;
        }
        v = ((from[0] + from[1]) + (from[2] + from[3])) + ((from[4] + from[5]) + (from[6] + from[7]));
      }
      if (row0 + rr < m)
      {
        dh[(row0 + rr) * r + j0 + e % width] = v;
      }
    }
    if (cluster > 1)
    {
      cluster_sync_all();   // nobody's sums are written again, or left, while they are read
    }
  }
}

// dx[m, in] = factor * dH . A, a thread a column of ROWS rows, which share A's numbers; `block` of ROWS rows' 256 columns.  64 products are
// added up by themselves and then to those before (one chain over 1024 ranks lost 3e-5 of a sum to small terms).
template <typename T, int ROWS>
__device__ __forceinline__ void dx_general(const float *dh, const T *a, T *dx, float factor, int64_t m, int in, int r, int64_t block)
{
  __shared__ __align__(16) float row[256][ROWS];
  const int parts = (in + 255) / 256;   // blocks of ROWS rows
  const int64_t at = block / parts * ROWS;
  const int c = static_cast<int>(block % parts) * 256 + static_cast<int>(threadIdx.x);
  float s[ROWS] = {}, sum[ROWS] = {};
  for (int j0 = 0; j0 < r; j0 += 256)
  {
    const int n = r - j0 < 256 ? r - j0 : 256;
    __syncthreads();
    for (int e = threadIdx.x; e < n * ROWS; e += 256)
    {
      const int64_t rr = at + e / n;
      row[e % n][e / n] = rr < m ? dh[rr * r + j0 + e % n] : 0.0f;
    }
    __syncthreads();
    if (c < in)
    {
      auto meet = [&](int k, float w) {
        if constexpr (ROWS == 1)
        {
          s[0] = fmaf(row[k][0], w, s[0]);
        }
        else
        {
#pragma unroll
          for (int q = 0; q < ROWS; q += 4)
          {
            const float4 v = *reinterpret_cast<const float4 *>(&row[k][q]);
            s[q] = fmaf(v.x, w, s[q]);
            s[q + 1] = fmaf(v.y, w, s[q + 1]);
            s[q + 2] = fmaf(v.z, w, s[q + 2]);
            s[q + 3] = fmaf(v.w, w, s[q + 3]);
          }
        }
      };
      const T *src = a + static_cast<int64_t>(j0) * in + c;
      for (int k = 0; k < n;)
      {
        const int stop = n - k < 64 ? n : k + 64;
        for (; ROWS > 1 && k + 16 <= stop; k += 16, src += static_cast<int64_t>(16) * in)
        {
          T w[16];   // (all on their way before the first is used)
#pragma unroll
          for (int u = 0; u < 16; ++u)
          {
            w[u] = src[static_cast<int64_t>(u) * in];
          }
#pragma unroll
          for (int u = 0; u < 16; ++u)
          {
            meet(k + u, act_f<T>(w[u]));
          }
        }
#pragma unroll 8
        for (; k < stop; ++k, src += in)
        {
          meet(k, act_f<T>(*src));
        }
#pragma unroll
        for (int q = 0; q < ROWS; ++q)
        {
          sum[q] += s[q];
          s[q] = 0.0f;
        }
      }
    }
  }
#pragma unroll
  for (int q = 0; q < ROWS; ++q)
  {
    if (c < in && at + q < m)
    {
      dx[(at + q) * in + c] = act_t<T>(sum[q] * factor);
    }
  }
}

// The sums (the first blocks), and dx, which needs none of them, in one launch
template <typename T, int ROWS>
__global__ void __launch_bounds__(256)
gradients_dx_kernel(const GradientSums j, int sum_blocks, const float *dh, const T *a, T *dx, int64_t m)
{
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (static_cast<int>(blockIdx.x) < sum_blocks)
  {
    gradient_sums(j, blockIdx.x);
    return;
  }
  dx_general<T, ROWS>(dh, a, dx, j.factor, m, j.in, j.r, static_cast<int64_t>(blockIdx.x) - sum_blocks);
}

// Few tokens: the reductions, of one slice, and dx in one launch
template <typename T>
__global__ void __launch_bounds__(256)
act_tn_dx_kernel(const Gradients j, int64_t m, int tiles, const T *a, T *dx)
{
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (static_cast<int>(blockIdx.x) < tiles)
  {
    tn_general<T, float, true>(j, m);
  }
  else if (blockIdx.y == 0)
  {
    dx_general<T, 1>(static_cast<const float *>(j.dh), a, dx, j.factor, m, j.in, j.r, static_cast<int64_t>(blockIdx.x) - tiles);
  }
}

// slices of tokens: as many as one wave of `blocks` an SM holds, no slice without tokens
int tn_slices(int64_t m, int64_t tiles, int tokens, int blocks)
{
  int64_t n = 148 * blocks / tiles;
  const int64_t most = (m + tokens - 1) / tokens;
  n = n > most ? most : n;
  return static_cast<int>(n < 1 ? 1 : n);
}

int64_t general_tiles(int out, int in, int r)
{
  return static_cast<int64_t>((out + kTnWide - 1) / kTnWide + (in + kTnWide - 1) / kTnWide) * ((r + kTnTile - 1) / kTnTile);
}

// So few tokens make one slice, whose sums are rounded where they are made, a launch less.  The whole pass, tensor core: 4096 -> 4096 int8,
// 64 rows 35.9 -> 33.4 us, 128 rows 36.7 -> 34.7, 200 rows 36.5 and 36.2 so.  Multiply-adds (one chain of a sum: 64 tokens at most), fp32: 2048 ->
// 2048, rank 64, 64 rows 35.6 -> 31.7; 1024 -> 1024, rank 16, 33 rows 20.5 -> 18.6, 64 rows 21.3 -> 20.5; 256 -> 256, rank 8, 17.5 and 17.7, 18.1 and 18.2.
bool one_slice(bool tensor, int64_t m) { return m <= (tensor ? 128 : 64); }

}  // namespace

int launch_act_pack(const void *x, int dtype, int8_t *codes, uint8_t *scales, int64_t rows, int dim, cudaStream_t s)
{
  if (rows <= 0)
  {
    return CAIFQ_OK;
  }
  switch (dtype)
  {
    case CAIFQ_F32:
      return act_pack<float>(x, codes, scales, rows, dim, s);
    case CAIFQ_F16:
      return act_pack<__half>(x, codes, scales, rows, dim, s);
    default:
      return act_pack<__nv_bfloat16>(x, codes, scales, rows, dim, s);
  }
}

int launch_act_unpack(const int8_t *codes, const uint8_t *scales, void *x, int dtype, int64_t rows, int dim, cudaStream_t s)
{
  if (rows <= 0)
  {
    return CAIFQ_OK;
  }
  switch (dtype)
  {
    case CAIFQ_F32:
      return act_unpack<float>(codes, scales, x, rows, dim, s);
    case CAIFQ_F16:
      return act_unpack<__half>(codes, scales, x, rows, dim, s);
    default:
      return act_unpack<__nv_bfloat16>(codes, scales, x, rows, dim, s);
  }
}

// fp32 scratch of launch_act_gradients; never less for more rows
size_t act_gradients_scratch_bytes(int64_t m, int out, int in, int r)
{
  const int64_t general = tn_slices(m, general_tiles(out, in, r), kTnRows, kTnGeneralBlocks);
  const int64_t tiled = tn_slices(m, (out + in + kTnColumns - 1) / kTnColumns, kTnTokens, r <= 16 ? kTnBlocks<2> : kTnBlocks<8>);
  return static_cast<size_t>(general > tiled ? general : tiled) * (static_cast<size_t>(out) + in) * r * sizeof(float);
}

namespace
{
template <typename T>
int launch_tn_dx(const Gradients &j, const void *a, void *dx, int64_t m, cudaStream_t s)
{
  const int tiles = (j.out + kTnWide - 1) / kTnWide + (j.in + kTnWide - 1) / kTnWide;
  const int64_t blocks = tiles + m * ((j.in + 255) / 256);
  CAIFQ_CHECK_ARG(blocks <= 0x7FFFFFFF, "LoRA backward on packed rows: %lld rows of %d columns are too many for its general form",
                  static_cast<long long>(m), j.in);
  CAIFQ_CHECK_CUDA(launch_dependent(act_tn_dx_kernel<T>, dim3(static_cast<unsigned>(blocks), (j.r + kTnTile - 1) / kTnTile), dim3(256), 0, s,
                                    j, m, tiles, static_cast<const T *>(a), static_cast<T *>(dx)));
  return CAIFQ_OK;
}

template <typename T>
int launch_gradients_dx(const GradientSums &j, int64_t sum_blocks, const float *dh, const void *a, void *dx, int64_t m, cudaStream_t s)
{
  // eight rows a block where that many blocks are left: A's numbers come from L2 once for eight (500 rows, 2048 columns, rank 64: 42 us by
  // single rows)
  const int parts = (j.in + 255) / 256;
  const bool eight = m * parts >= 8 * 148;
  const int64_t blocks = sum_blocks + (eight ? (m + 7) / 8 : m) * parts;
  CAIFQ_CHECK_ARG(blocks <= 0x7FFFFFFF, "LoRA backward on packed rows: %lld rows of %d columns are too many for its general form",
                  static_cast<long long>(m), j.in);
  CAIFQ_CHECK_CUDA(launch_dependent(eight ? gradients_dx_kernel<T, 8> : gradients_dx_kernel<T, 1>, dim3(static_cast<unsigned>(blocks)), dim3(256),
                                    0, s, j, static_cast<int>(sum_blocks), dh, static_cast<const T *>(a), static_cast<T *>(dx), m));
  return CAIFQ_OK;
}
}  // namespace

// d_b[out, r] = factor * dy^T . h and d_a[r, in] = factor * (dh + dh_rest)^T . x, x packed, dh_rest for dh in bf16 alone; with dx (dh is fp32
// then) dx[m, in] = factor * dh . a too.  m >= 1; dy, h, a, d_b, d_a, dx in dtype
int launch_act_gradients(const void *dy, const void *h, const void *dh, const void *dh_rest, int dh_dtype, const int8_t *x, const uint8_t *scales,
                         void *d_b, void *d_a, const void *a, void *dx, int dtype, float factor, float *scratch, int64_t m, int out,
                         int in, int r, cudaStream_t s)
{
  auto on_16 = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const bool tensor = dtype == CAIFQ_BF16 && dh_dtype == CAIFQ_BF16 && (r == 8 || r == 16 || r == 32 || r == 64) && (out % kTnColumns) == 0 &&
                      (in % kTnColumns) == 0 && on_16(dy) && on_16(h) && on_16(dh) && on_16(dh_rest) && on_16(x);
  const bool direct = one_slice(tensor, m);
  const Gradients j{dy, h, dh, dh_rest, x, scales, scratch, direct ? d_b : nullptr, direct ? d_a : nullptr, factor, out, in, r};
  int slices = 0;
  if (tensor)
  {
    const int tiles = (out + in) / kTnColumns;
    slices = direct ? 1 : tn_slices(m, tiles, kTnTokens, r <= 16 ? kTnBlocks<2> : kTnBlocks<8>);
    auto kernel = r == 8 ? act_tn_mma_kernel<1>
                         : (r == 16 ? act_tn_mma_kernel<2> : (r == 32 ? act_tn_mma_kernel<4> : act_tn_mma_kernel<8>));
    CAIFQ_CHECK_CUDA(launch_dependent(kernel, dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(slices)), dim3(256), 0, s, j, m));
  }
  else if (direct && dx != nullptr)
  {
    switch (dtype)
    {
      case CAIFQ_F32:
        return launch_tn_dx<float>(j, a, dx, m, s);
      case CAIFQ_F16:
        return launch_tn_dx<__half>(j, a, dx, m, s);
      default:
        return launch_tn_dx<__nv_bfloat16>(j, a, dx, m, s);
    }
  }
  else
  {
    slices = direct ? 1 : tn_slices(m, general_tiles(out, in, r), kTnRows, kTnGeneralBlocks);
    const dim3 grid((out + kTnWide - 1) / kTnWide + (in + kTnWide - 1) / kTnWide, (r + kTnTile - 1) / kTnTile,
                    static_cast<unsigned>(slices));
    auto kernel = dtype == CAIFQ_F32 ? act_tn_kernel<float, float>
                                     : (dtype == CAIFQ_F16 ? act_tn_kernel<__half, float>
                                                           : (dh_dtype == CAIFQ_BF16 ? act_tn_kernel<__nv_bfloat16, __nv_bfloat16>
                                                                                     : act_tn_kernel<__nv_bfloat16, float>));
    CAIFQ_CHECK_CUDA(launch_dependent(kernel, grid, dim3(256), 0, s, j, m));
  }
  if (direct && dx == nullptr)
  {
    return CAIFQ_OK;
  }
  const int64_t n = (static_cast<int64_t>(out) + in) * r;
  const int64_t blocks = (n + 255) / 256;
  const GradientSums sums{scratch, d_b, d_a, factor, dtype, slices, in, r, static_cast<int64_t>(out) * r};
  if (dx == nullptr)
  {
    CAIFQ_CHECK_CUDA(launch_dependent(gradients_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, sums));
    return CAIFQ_OK;
  }
  switch (dtype)
  {
    case CAIFQ_F32:
      return launch_gradients_dx<float>(sums, blocks, static_cast<const float *>(dh), a, dx, m, s);
    case CAIFQ_F16:
      return launch_gradients_dx<__half>(sums, blocks, static_cast<const float *>(dh), a, dx, m, s);
    default:
      return launch_gradients_dx<__nv_bfloat16>(sums, blocks, static_cast<const float *>(dh), a, dx, m, s);
  }
}

// dh[m, r] = dy . bt^T in bf16, rest[m, r] what that rounding left, and padded[m, 64] = bf16(dh * mul / *div): bf16 operands on 16-byte
// boundaries, r 8, 16, 32 or 64, out a
// multiple of 32, m >= 1
int launch_act_nt(const void *dy, const void *bt, void *dh, void *rest, void *padded, float mul, const float *div, int64_t m, int out, int r,
                  cudaStream_t s)
{
  auto kernel = r == 8 ? act_nt_mma_kernel<1>
                       : (r == 16 ? act_nt_mma_kernel<2> : (r == 32 ? act_nt_mma_kernel<4> : act_nt_mma_kernel<8>));
  CAIFQ_CHECK_CUDA(launch_dependent(kernel, dim3(static_cast<unsigned>((m + 31) / 32)), dim3(256), 0, s,
                                    static_cast<const __nv_bfloat16 *>(dy), static_cast<const __nv_bfloat16 *>(bt),
                                    static_cast<__nv_bfloat16 *>(dh), static_cast<__nv_bfloat16 *>(rest), static_cast<__nv_bfloat16 *>(padded), mul, div, m, out));
  return CAIFQ_OK;
}

namespace
{
template <typename T>
int launch_dh_of(const void *dy, const void *b, float *dh, int64_t m, int out, int r, cudaStream_t s)
{
  // A block a row where a thread then reads up to 64 numbers of B: four rows a block, and clusters, cost 2 us and more there (64 rows,
  // 1024 columns, rank 16), and save 30 of 91 where it would read 480 (152 rows, 1920 columns, rank 64)
  const bool large = static_cast<int64_t>(out) * r > 64 * 256;
  // (eight rows: half the reading of B, where enough blocks are left)
  const bool eight = large && m >= 8 * 32;
  const int64_t groups = eight ? (m + 7) / 8 : (m + 3) / 4;
  int cluster = 1;
  while (large && cluster < 8 && groups * cluster < 4 * 148 && static_cast<int64_t>(out) * r > static_cast<int64_t>(64 * 256) * cluster)
  {
    cluster *= 2;
  }
  if (!large)
  {
    CAIFQ_CHECK_CUDA(launch_dependent(dh_row_kernel<T>, dim3(static_cast<unsigned>(m)), dim3(256), 0, s, static_cast<const T *>(dy),
                                      static_cast<const T *>(b), dh, m, out, r));
    return CAIFQ_OK;
  }
  CAIFQ_CHECK_CUDA(launch_dependent_clusters(eight ? dh_kernel<T, 8> : dh_kernel<T, 4>, dim3(static_cast<unsigned>(groups * cluster)), dim3(256), 0, s, cluster,
                                             static_cast<const T *>(dy), static_cast<const T *>(b), dh, m, out, r, cluster));
  return CAIFQ_OK;
}
}  // namespace

// dh[m, r] (fp32) = dy . b, dy and b in dtype
int launch_dh(const void *dy, const void *b, float *dh, int dtype, int64_t m, int out, int r, cudaStream_t s)
{
  switch (dtype)
  {
    case CAIFQ_F32:
      return launch_dh_of<float>(dy, b, dh, m, out, r, s);
    case CAIFQ_F16:
      return launch_dh_of<__half>(dy, b, dh, m, out, r, s);
    default:
      return launch_dh_of<__nv_bfloat16>(dy, b, dh, m, out, r, s);
  }
}

}  // namespace caifq
