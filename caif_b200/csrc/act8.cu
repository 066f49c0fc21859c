// Activations kept in 8 bits between an adapter's forward and backward pass, and the reductions over tokens that read them.
//
// A block is 32 columns of a row.  Its scale is s = 2^e, the smallest power of two (e >= -126) with max|x| <= 127 s; a code is
// rint(x / s), ties to even; the scale is stored as the byte e + 127.  A block with a value that is not finite has the byte
// 255 and codes of 0 and stands for NaN: a loss that ran off is not hidden by a checkpoint.
// Why a power of two, which costs up to one of the code's eight bits against max|x| / 127: code * s is exact in bf16 and
// fp32 (7 bits of significand), so x / s and the value need no rounding beyond the code's own and the backward pass
// multiplies the very rows that caifq_act_unpack gives; and a block's scale is one byte.
#include "common.cuh"

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

// ---- any width, any alignment: a warp a block, a lane an element ----

template <typename T>
__global__ void __launch_bounds__(kActThreads)
act_pack_kernel(const T *x, int8_t *codes, uint8_t *scales, int64_t rows, int dim)
{
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int blocks = (dim + kActBlock - 1) / kActBlock;
  const int64_t total = rows * blocks;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * (kActThreads / 32);
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * (kActThreads / 32) + (threadIdx.x >> 5); b < total; b += stride)
  {
    const int64_t row = b / blocks;
    const int c = static_cast<int>(b - row * blocks) * kActBlock + lane;
    const bool live = c < dim;
    const float v = live ? act_f<T>(x[row * dim + c]) : 0.0f;
    const uint32_t byte = scale_byte(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v) & 0x7FFFFFFFu));
    if (live)
    {
      codes[row * dim + c] = static_cast<int8_t>(__float2int_rn(v * inverse_of(byte)));
    }
    if (lane == 0)
    {
      scales[b] = static_cast<uint8_t>(byte);
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
  const int blocks = (dim + kActBlock - 1) / kActBlock;
  const int64_t total = rows * blocks;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * (kActThreads / 32);
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * (kActThreads / 32) + (threadIdx.x >> 5); b < total; b += stride)
  {
    const int64_t row = b / blocks;
    const int c = static_cast<int>(b - row * blocks) * kActBlock + lane;
    if (c < dim)
    {
      x[row * dim + c] = act_t<T>(static_cast<float>(codes[row * dim + c]) * scale_of(scales[b]));
    }
  }
}

unsigned act_grid(int64_t blocks)
{
  const int64_t ctas = (blocks + kActThreads / 32 - 1) / (kActThreads / 32);
  return static_cast<unsigned>(ctas < 148 * 64 ? ctas : 148 * 64);
}

// ---- rows of whole blocks on 16-byte boundaries: a thread 16 bytes of the row ----
// HBM-bound (8192 x 4096 bf16: 102 MB each way).  A thread holds kActTrip pieces so that all its loads are in flight before
// the first is used; the lanes of a block (4, or 8 of fp32) meet in two or three shuffles.  A code is the low byte of
// x / s + 1.5 * 2^23, which rounds to the nearest even integer: one fused multiply-add instead of a conversion, whose unit
// takes a sixteenth of a warp a cycle.

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
  constexpr float kRound = 12582912.0f;   // 1.5 * 2^23
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
  {
    b[i] = __float_as_uint(fmaf(piece_get<T>(w, first + i), inverse, kRound));
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
  CAIFQ_CHECK_CUDA(launch_dependent(act_pack_kernel<T>, dim3(act_grid(rows * ((dim + kActBlock - 1) / kActBlock))),
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
  CAIFQ_CHECK_CUDA(launch_dependent(act_unpack_kernel<T>, dim3(act_grid(rows * ((dim + kActBlock - 1) / kActBlock))),
                                    dim3(kActThreads), 0, s, codes, scales, static_cast<T *>(x), rows, dim));
  return CAIFQ_OK;
}


// ---- reductions over tokens, any type: C[p, q] = factor * sum_m U[m, p] * V[m, q] ----
// V may be packed rows.  gridDim.z slices the tokens; a slice's sums go to part[slice][p][q] and tn_finish_kernel adds the
// slices in order and rounds once.

constexpr int kTnTile = 32;
constexpr int kTnRows = 32;

struct TnJob
{
  const void *u;           // [m, p]
  const void *v;           // [m, q], or codes
  const uint8_t *v_scales; // null: v holds floats
  float *part;
  int u_dtype, v_dtype;
  int p, q;
};

__global__ void __launch_bounds__(256) act_tn_kernel(const TnJob j, int64_t m)
{
  __shared__ float su[kTnRows][kTnTile + 1];
  __shared__ float sv[kTnRows][kTnTile + 1];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x;
  const int p0 = blockIdx.y * kTnTile;
  const int q0 = blockIdx.x * kTnTile;
  const int64_t begin = m * blockIdx.z / gridDim.z;
  const int64_t end = m * (blockIdx.z + 1) / gridDim.z;
  const int blocks = (j.q + kActBlock - 1) / kActBlock;
  const int tq = tid % 16;
  const int tp = tid / 16;
  float c[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
  for (int64_t mb = begin; mb < end; mb += kTnRows)
  {
    for (int e = tid; e < kTnRows * kTnTile; e += 256)
    {
      const int col = e % kTnTile;
      const int64_t row = mb + e / kTnTile;
      float u = 0.0f, v = 0.0f;
      if (row < end && p0 + col < j.p)
      {
        u = load_as_float(j.u, row * j.p + p0 + col, j.u_dtype);
      }
      if (row < end && q0 + col < j.q)
      {
        const int64_t at = row * j.q + q0 + col;
        v = j.v_scales != nullptr
                ? static_cast<float>(static_cast<const int8_t *>(j.v)[at]) * scale_of(j.v_scales[row * blocks + (q0 + col) / kActBlock])
                : load_as_float(j.v, at, j.v_dtype);
      }
      su[e / kTnTile][col] = u;
      sv[e / kTnTile][col] = v;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kTnRows; ++r)
    {
      const float u0 = su[r][tp * 2];
      const float u1 = su[r][tp * 2 + 1];
      const float v0 = sv[r][tq * 2];
      const float v1 = sv[r][tq * 2 + 1];
      c[0][0] = fmaf(u0, v0, c[0][0]);
      c[0][1] = fmaf(u0, v1, c[0][1]);
      c[1][0] = fmaf(u1, v0, c[1][0]);
      c[1][1] = fmaf(u1, v1, c[1][1]);
    }
    __syncthreads();
  }
  float *part = j.part + static_cast<int64_t>(blockIdx.z) * j.p * j.q;
#pragma unroll
  for (int a = 0; a < 2; ++a)
  {
#pragma unroll
    for (int b = 0; b < 2; ++b)
    {
      const int gp = p0 + tp * 2 + a;
      const int gq = q0 + tq * 2 + b;
      if (gp < j.p && gq < j.q)
      {
        part[static_cast<int64_t>(gp) * j.q + gq] = c[a][b];
      }
    }
  }
}

__global__ void __launch_bounds__(256)
tn_finish_kernel(const float *part, void *out, int dtype, float factor, int slices, int64_t n)
{
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n)
  {
    float s = 0.0f;
#pragma unroll 4
    for (int z = 0; z < slices; ++z)
    {
      s += part[static_cast<int64_t>(z) * n + i];
    }
    store_from_float(out, i, dtype, s * factor);
  }
}

int tn_slices(int64_t m, int p, int q)
{
  const int64_t tiles = static_cast<int64_t>((p + kTnTile - 1) / kTnTile) * ((q + kTnTile - 1) / kTnTile);
  int64_t n = (148 * 4 + tiles - 1) / tiles;
  const int64_t most = (m + kTnRows - 1) / kTnRows;
  n = n > most ? most : n;
  n = n > 64 ? 64 : n;
  return static_cast<int>(n < 1 ? 1 : n);
}

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

// fp32 scratch of launch_act_tn
size_t act_tn_scratch_bytes(int64_t m, int p, int q)
{
  return static_cast<size_t>(tn_slices(m, p, q)) * static_cast<size_t>(p) * static_cast<size_t>(q) * sizeof(float);
}

// out[p, q] = factor * sum over tokens of u[m, p] * v[m, q]; v_scales != null: v is packed rows.  m >= 1
int launch_act_tn(const void *u, int u_dtype, const void *v, int v_dtype, const uint8_t *v_scales, void *out, int out_dtype,
                  float factor, float *scratch, int64_t m, int p, int q, cudaStream_t s)
{
  const int slices = tn_slices(m, p, q);
  const TnJob job{u, v, v_scales, scratch, u_dtype, v_dtype, p, q};
  const dim3 grid((q + kTnTile - 1) / kTnTile, (p + kTnTile - 1) / kTnTile, static_cast<unsigned>(slices));
  CAIFQ_CHECK_CUDA(launch_dependent(act_tn_kernel, grid, dim3(256), 0, s, job, m));
  const int64_t n = static_cast<int64_t>(p) * q;
  CAIFQ_CHECK_CUDA(launch_dependent(tn_finish_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, s,
                                    static_cast<const float *>(scratch), out, out_dtype, factor, slices, n));
  return CAIFQ_OK;
}

}  // namespace caifq
