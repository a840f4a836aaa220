// Microscaled 4-bit floating point: matrices whose elements are 4 bits (sign, two bits of exponent, one of mantissa:
// 0, 0.5, 1, 1.5, 2, 3, 4, 6) with one power of two for each block of 32 elements of a row, and products of two such matrices.
//
// The definition.  For a block with the largest magnitude a, the scale is 2^(s - 127), s = max(0, floor(log2 a) + 125), so that
// a lies in [4, 8) units; an element is x / scale rounded to the nearest level, ties to the even code, what exceeds 6 becoming
// 6.  A block with an infinity or a NaN has s = 255, which stands for NaN.  Division by a power of two is exact, so every
// implementation gives the same bits.
//
// Layout.  Codes: [rows][k / 2] bytes, element 2 i in the low half.  Scales: in the order in which the tensor core wants them in
// tensor memory: tiles of 128 rows x 128 of k, 512 bytes each, tile (rt, kt) at (rt * ceil(k / 128) + kt) * 512, the byte of
// (row, block) at (row % 32) * 16 + (row % 128 / 32) * 4 + block % 4; rows are padded to 256, so that a copy of two tiles of
// rows stays inside.  A gated matrix (gate rows [0, O), up rows [O, 2 O)) keeps row i of the gate in row 2 i and row i of the
// up half in row 2 i + 1: the two numbers of an output then lie in neighbouring lanes of the accumulator.
#include <cuda.h>
#include <type_traits>
#include "common.cuh"

typedef __nv_bfloat16 bf16;
constexpr int MX_BLOCK = 32;

// ---------------------------------------------------------------------------------------------
// Rounding of rows to 4 bits, and the values that the bits stand for
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t mx_scale_byte(float amax_or_bits_max) {
  const uint32_t f = __float_as_uint(amax_or_bits_max) >> 23;          // the exponent field of a number without its sign
  return f == 255u ? 255u : (f >= 2u ? f - 2u : 0u);
}
__device__ __forceinline__ float mx_inverse_scale(uint32_t s) {        // 2^(127 - s), s = 0 .. 252 (255: any)
  return __uint_as_float((254u - (s > 253u ? 253u : s)) << 23);
}
// Eight scaled numbers to eight codes (the first in the lowest four bits).
__device__ __forceinline__ uint32_t mx_codes8(const float (&v)[8], float inv) {
  uint32_t r;
  asm("{\n .reg .b8 b0, b1, b2, b3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      " mov.b32 %0, {b0, b1, b2, b3};\n}\n"
      : "=r"(r) : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv),
        "f"(v[6] * inv), "f"(v[7] * inv));
  return r;
}
__host__ __device__ __forceinline__ size_t mx_scale_at(int row, int block, int k_tiles) {
  return ((size_t)(row >> 7) * k_tiles + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// 16 numbers as the words they come in, and their largest magnitude as float32 bits.
template <typename T> struct MxSixteen;
template <> struct MxSixteen<bf16> {
  uint4 w[2];
  __device__ __forceinline__ void load(const bf16* p) {
    w[0] = reinterpret_cast<const uint4*>(p)[0];
    w[1] = reinterpret_cast<const uint4*>(p)[1];
  }
  __device__ __forceinline__ uint32_t word(int i) const { const uint4& x = w[i >> 2]; return (i & 3) == 0 ? x.x : (i & 3) == 1 ? x.y : (i & 3) == 2 ? x.z : x.w; }
  __device__ __forceinline__ uint32_t amax_bits() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __vmaxu2(m, word(i) & 0x7fff7fffu);
    return max(m << 16, m & 0xffff0000u);
  }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? word(i >> 1) & 0xffff0000u : word(i >> 1) << 16); }
};
template <> struct MxSixteen<float> {
  float4 w[4];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const float4*>(p)[i];
  }
  __device__ __forceinline__ float at(int i) const { const float4& x = w[i >> 2]; return (i & 3) == 0 ? x.x : (i & 3) == 1 ? x.y : (i & 3) == 2 ? x.z : x.w; }
  __device__ __forceinline__ uint32_t amax_bits() const {
    // magnitudes compared as integers: a NaN is larger than infinity, and neither is lost
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(at(i)) & 0x7fffffffu);
    return m;
  }
};

// Two neighbouring lanes have a block: 16 elements (32 or 64 bytes of input, 8 of output) each.  8 lanes have the four blocks whose
// scales lie in one 32-bit word.  The columns of a row are spread over the grid's x; a thread has PER rows, all of them requested
// at once (a large matrix: one row per thread is a load's latency per CTA of little work).  Bound by memory: 24,576 x 4,096 of bfloat16 38 us,
// 6.7 TB/s, and the way back 40 us, 6.4 TB/s.
// early: the next kernel may begin at once.  The product that rounds its rows with this kernel reads them behind its wait; but what may become a
// product's matrix is read before that wait, so nothing may begin ahead of these writes but mx4_written_kernel (nor ahead of other kernels' writes: ifb_mx4_written).
template <typename T, int PER>
__global__ void __launch_bounds__(256)
mx4_quantize_kernel(const T* x, long long row_stride, uint8_t* codes, uint8_t* scales, int rows, int k, int gated_rows, int early) {
  ifb_pdl_wait();
  if (early) ifb_pdl_trigger();
  const int k_tiles = (k + 127) / 128;
  const int e = (blockIdx.x * 256 + threadIdx.x) * 16;                 // of the row's elements, padded to 128
  const uint32_t lanes = __ballot_sync(0xffffffffu, e < k_tiles * 128);
  if (e >= k_tiles * 128) return;                                      // 8 lanes leave together
  const int row0 = blockIdx.y * PER;                                   // of the result
  const bool in = e < k;
  MxSixteen<T> v[PER];
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int row = min(row0 + p, rows - 1), from = gated_rows ? (row & 1) * gated_rows + (row >> 1) : row;
    v[p].load(x + (size_t)from * row_stride + (in ? e : 0));
  }
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int row = row0 + p;
    uint32_t m = v[p].amax_bits();
    m = max(m, __shfl_xor_sync(lanes, m, 1));
    const uint32_t s = mx_scale_byte(__uint_as_float(m));
    uint32_t word = (in ? s : 0u) << ((threadIdx.x & 6) * 4);
    word |= __shfl_xor_sync(lanes, word, 2);
    word |= __shfl_xor_sync(lanes, word, 4);
    if (row >= rows) continue;
    if (in) {
      const float inv = mx_inverse_scale(s);
      float a[8], b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) { a[i] = v[p].at(i); b[i] = v[p].at(8 + i); }
      *reinterpret_cast<uint2*>(codes + (size_t)row * (k / 2) + e / 2) = make_uint2(mx_codes8(a, inv), mx_codes8(b, inv));
    }
    if ((threadIdx.x & 7) == 0) *reinterpret_cast<uint32_t*>(scales + mx_scale_at(row, e / MX_BLOCK, k_tiles)) = word;
  }
  if (PER == 1 && !early) __threadfence();
}

// The values of eight codes in pairs of bfloat16, which holds them exactly.  The bits "ee m" of a code at the lowest end of a bfloat16's
// exponent and the top of its fraction are the code's magnitude times 2^-126, subnormal numbers included, so two products with
// powers of two (2^126, and the scale) are the value.
__device__ __forceinline__ uint32_t mx_times(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("mul.rn.bf16x2 %0, %1, %2;\n" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
__device__ __forceinline__ void mx_values8(uint32_t c, uint32_t s, uint32_t (&v)[4]) {
  const uint32_t one = s == 255u ? 0x7fffu : s ? s << 7 : 0x0040u, scale = one * 0x00010001u;      // 2^(s - 127); 255: NaN
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t n = c >> (8 * i), x = (n & 15u) | (n & 0xf0u) << 12;
    v[i] = mx_times(mx_times((x & 0x00070007u) << 6 | (x & 0x00080008u) << 12, 0x7e807e80u), scale);
  }
}
template <typename T> __device__ __forceinline__ void mx_store8(T* p, const uint32_t (&v)[4]);
template <> __device__ __forceinline__ void mx_store8<bf16>(bf16* p, const uint32_t (&v)[4]) { *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]); }
template <> __device__ __forceinline__ void mx_store8<float>(float* p, const uint32_t (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    reinterpret_cast<uint4*>(p)[i] = make_uint4(v[2 * i] << 16, v[2 * i] & 0xffff0000u, v[2 * i + 1] << 16, v[2 * i + 1] & 0xffff0000u);
}
template <typename T, int PER>                                          // (the numbers, too, may be the matrix of a product)
__global__ void __launch_bounds__(256)
mx4_values_kernel(const uint8_t* codes, const uint8_t* scales, T* out, int rows, int k, int gated_rows, int early) {
  ifb_pdl_wait();
  if (early) ifb_pdl_trigger();
  const int e = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (e >= k) return;
  const int row0 = blockIdx.y * PER, k_tiles = (k + 127) / 128;
  uint32_t c[PER];
  uint32_t s[PER];
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int row = min(row0 + p, rows - 1);
    c[p] = *reinterpret_cast<const uint32_t*>(codes + (size_t)row * (k / 2) + e / 2);
    s[p] = scales[mx_scale_at(row, e / MX_BLOCK, k_tiles)];
  }
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int row = row0 + p;
    if (row >= rows) break;
    const int to = gated_rows ? (row & 1) * gated_rows + (row >> 1) : row;
    uint32_t v[4];
    mx_values8(c[p], s[p], v);
    mx_store8<T>(out + (size_t)to * k + e, v);
  }
  if (PER == 1) __threadfence();
}
// What a matrix's kernel ends with: the kernel after this one begins when all that went before is complete and visible.  Small matrices have no
// trigger and a fence per thread in its place (8 rows of 4,096: 3.5 us, 2.5 without; a launch is 2 us of the host's); for large ones that
// would keep their CTAs waiting (24,576 x 4,096 there and back: 89 us, 82 with this kernel, 81 with neither).
__global__ void mx4_written_kernel() {
  ifb_pdl_wait();
  ifb_pdl_trigger();
}
static int mx_written(cudaStream_t stream) { return ifb_launch(mx4_written_kernel, dim3(1), dim3(32), 0, stream); }
// For matrices that other kernels wrote.
IFB_EXPORT int ifb_mx4_written(void* stream) { return mx_written((cudaStream_t)stream); }

static int mx_sizes(int rows, int k, int gated) {
  if (rows < 1 || k < MX_BLOCK || k % MX_BLOCK || (gated && (rows & 1))) return IFB_ERR_SIZE;
  return IFB_OK;
}

constexpr int MX_GRID_ROWS = 65535 / 256 * 256;      // a grid has at most 65,535 rows; whole tiles of rows, whole pairs
// Rows per thread: four where that still gives every SM several CTAs, or where a grid would not have the rows; the one row of a float32 matrix is as
// many bytes in flight as two of bfloat16.  One and four, bfloat16: 8 rows of 4,096 1.9 and 2.5 us, 512 rows 2.8 both, 2,048 rows 5.4 and 4.9,
// 24,576 rows 50.3 and 39.0 (there and back 126 and 80); float32: 2,048 rows 7.2 and 7.8, 8,192 rows 27.1 and 26.4.
static int mx_rows_per_thread(int rows, int k, int dtype) {
  return (long long)rows * k >= (long long)ifb_sm_count() * (dtype == IFB_F32 ? 131072 : 32768) || rows > MX_GRID_ROWS ? 4 : 1;
}

template <typename T, int PER>
static int mx_quantize_launch(const void* x, long long row_stride, void* codes, void* scales, int rows, int k, int gated, int early, cudaStream_t stream) {
  // (a gated matrix has its rows from two places, so one launch has to hold it)
  if (gated && (rows + PER - 1) / PER > MX_GRID_ROWS) return IFB_ERR_SIZE;
  for (long long r0 = 0; r0 < rows; r0 += (long long)MX_GRID_ROWS * PER) {
    const int n = (int)(rows - r0 < (long long)MX_GRID_ROWS * PER ? rows - r0 : (long long)MX_GRID_ROWS * PER);
    const dim3 grid(((k + 127) / 128 * 8 + 255) / 256, (n + PER - 1) / PER);
    const int e = ifb_launch(mx4_quantize_kernel<T, PER>, grid, dim3(256), 0, stream, (const T*)x + (size_t)r0 * row_stride, row_stride,
                             (uint8_t*)codes + (size_t)r0 * (k / 2), (uint8_t*)scales + (size_t)(r0 / 128) * ((k + 127) / 128) * 512, n, k,
                             gated ? rows / 2 : 0, early || PER > 1);
    if (e) return e;
  }
  return PER > 1 && !early ? mx_written(stream) : IFB_OK;
}
static int mx_quantize(const void* x, int dtype, long long row_stride, void* codes, void* scales, int rows, int k, int gated, int early, void* stream) {
  const int bad = mx_sizes(rows, k, gated);
  if (bad) return bad;
  const int esize = dtype == IFB_F32 ? 4 : 2;
  if (dtype != IFB_F32 && dtype != IFB_BF16) return IFB_ERR_DTYPE;
  if ((((uintptr_t)x) | ((uintptr_t)codes) | ((uintptr_t)scales) | (uintptr_t)(row_stride * esize)) & 15) return IFB_ERR_ALIGN;
  cudaStream_t st = (cudaStream_t)stream;
  if (mx_rows_per_thread(rows, k, dtype) == 4)
    return dtype == IFB_F32 ? mx_quantize_launch<float, 4>(x, row_stride, codes, scales, rows, k, gated, early, st)
                            : mx_quantize_launch<bf16, 4>(x, row_stride, codes, scales, rows, k, gated, early, st);
  return dtype == IFB_F32 ? mx_quantize_launch<float, 1>(x, row_stride, codes, scales, rows, k, gated, early, st)
                          : mx_quantize_launch<bf16, 1>(x, row_stride, codes, scales, rows, k, gated, early, st);
}
IFB_EXPORT int ifb_mx4_quantize(const void* x, int dtype, long long row_stride, void* codes, void* scales, int rows, int k, int gated,
                                void* stream) {
  return mx_quantize(x, dtype, row_stride, codes, scales, rows, k, gated, 0, stream);
}

template <typename T, int PER>
static int mx_values_launch(const void* codes, const void* scales, void* out, int rows, int k, int gated, cudaStream_t stream) {
  if (gated && (rows + PER - 1) / PER > MX_GRID_ROWS) return IFB_ERR_SIZE;
  for (long long r0 = 0; r0 < rows; r0 += (long long)MX_GRID_ROWS * PER) {
    const int n = (int)(rows - r0 < (long long)MX_GRID_ROWS * PER ? rows - r0 : (long long)MX_GRID_ROWS * PER);
    const dim3 grid((k / 8 + 255) / 256, (n + PER - 1) / PER);
    const int e = ifb_launch(mx4_values_kernel<T, PER>, grid, dim3(256), 0, stream, (const uint8_t*)codes + (size_t)r0 * (k / 2),
                             (const uint8_t*)scales + (size_t)(r0 / 128) * ((k + 127) / 128) * 512, (T*)out + (size_t)r0 * k, n, k, gated ? rows / 2 : 0,
                             (int)(PER > 1));
    if (e) return e;
  }
  return PER > 1 ? mx_written(stream) : IFB_OK;
}
IFB_EXPORT int ifb_mx4_values(const void* codes, const void* scales, void* out, int dtype, int rows, int k, int gated, void* stream) {
  const int bad = mx_sizes(rows, k, gated);
  if (bad) return bad;
  if (dtype != IFB_F32 && dtype != IFB_BF16) return IFB_ERR_DTYPE;
  if ((((uintptr_t)out) | ((uintptr_t)codes) | ((uintptr_t)scales)) & 15) return IFB_ERR_ALIGN;
  cudaStream_t st = (cudaStream_t)stream;
  if (mx_rows_per_thread(rows, k, dtype) == 4)
    return dtype == IFB_F32 ? mx_values_launch<float, 4>(codes, scales, out, rows, k, gated, st) : mx_values_launch<bf16, 4>(codes, scales, out, rows, k, gated, st);
  return dtype == IFB_F32 ? mx_values_launch<float, 1>(codes, scales, out, rows, k, gated, st) : mx_values_launch<bf16, 1>(codes, scales, out, rows, k, gated, st);
}

// ---------------------------------------------------------------------------------------------
// The product: out[n, o] = sum_k x[n, k] w[o, k] of two microscaled matrices, by tcgen05.mma of kind mxf4, which multiplies
// 4-bit elements, applies both blocks' scales and adds in float32.
//
// The features are the 128 rows of the accumulator (its lanes), the tokens its columns, so that a step of few tokens wastes
// nothing of the instruction but its width, and one kernel serves one token and a prompt.  A CTA owns 128 rows of w by NT
// tokens.  Per 256 of k, a stage: 128 bytes of every row (one swizzle row) of both operands by TMA, and their scale tiles (512
// bytes per 128 x 128) by bulk copies; the issuing thread copies the scales on to tensor memory (tcgen05.cp, 32 lanes x 16
// bytes, repeated for the four quarters of the lanes) into columns that belong to the stage, then issues four products of k =
// 64.  Rows and k beyond the matrices are zeros.
//   warp 0: producer; warp 1: copies scales and issues products; warps 2 ..: epilogue, a quarter of the lanes each (warp % 4).
// SPLITS: where tiles are few, the k range of a tile is shared by a cluster of CTAs along z, which add their accumulators
// through distributed shared memory in the order of their ranks.
// What does not depend on the kernel before this one, the matrix, is requested before the wait for it.
// ROUND: the rows come as numbers, and the epilogue's warps, idle until then, round a stage's 256 of k of them (a thread a block
// of 32) into the stage, where TMA would have put them: every CTA rounds all rows of its part of k, which for few rows is little
// beside its part of the matrix, and a launch and a trip through memory are saved.  The numbers are requested some stages ahead
// (one ahead: 8 rows of 12,288 by 4,096 11.1 us, four 8.3; with a kernel of its own for the rounding 8.9).  From 33 rows on the
// rounding takes longer than the matrix (24,576 x 4,096: 25 us, 15.5 with the kernel of its own).
// What bounds it: few tokens, the matrix's bytes and what a CTA does beside them, its start, its first stages and the sum over its cluster (8 rows
// of 12,288 by 4,096: 8.2 us, 3.3 TB/s; 33 rows by gate and up of 12,288 x 4,096, rows rounded first: 15.6 us, 3.5 TB/s, 192 tiles at once of which 44 SMs have two; 1 row of 1,024 by
// 4,096: 3.3 us, latency).
// Waits are bounded: after a limit a thread records a code in `*err`, raises the CTA's abort flag, and all fall through to the
// end, where the tensor memory is given back.
// ---------------------------------------------------------------------------------------------
constexpr int MX_KSTAGE = 256;
constexpr int MX_A_BYTES = 128 * 128;
constexpr uint32_t MX_SPIN_LIMIT = 1u << 22;

__device__ __forceinline__ uint32_t mx_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mx_mbar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(mx_smem(bar)), "r"(count));
}
__device__ __forceinline__ void mx_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(mx_smem(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mx_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
  unsigned long long t0 = 0;
  for (uint32_t i = 0; i < MX_SPIN_LIMIT; ++i) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(mx_smem(bar)), "r"(parity) : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
    if (ifb_wait_expired(i, t0)) break;
  }
  *abort_flag = 1;
  atomicExch(err, code);
  return false;
}
__device__ __forceinline__ void mx_tma_2d(uint32_t smem, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
               ::"r"(smem), "l"(map), "r"(mx_smem(bar)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void mx_bulk(uint32_t smem, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
               ::"r"(smem), "l"(src), "r"(bytes), "r"(mx_smem(bar)) : "memory");
}
__device__ __forceinline__ bool mx_elect() {
  uint32_t pred;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(pred));
  return pred != 0;
}
// K-major rows of 128 bytes in the 128-byte swizzle, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t mx_desc(uint32_t smem) {
  return (uint64_t)((smem >> 4) & 0x3FFF) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// 32 rows of 16 bytes one after the other: groups of 8 rows 128 bytes apart, no swizzle.
__device__ __forceinline__ uint64_t mx_scale_desc(uint32_t smem) {
  return (uint64_t)((smem >> 4) & 0x3FFF) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}
__device__ __forceinline__ void mx_copy_scales(uint32_t tmem, uint32_t smem) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n" ::"r"(tmem), "l"(mx_scale_desc(smem)) : "memory");
}
__device__ __forceinline__ void mx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
               " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc) : "memory");
}
__device__ __forceinline__ void mx_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(mx_smem(bar)) : "memory");
}
__device__ __forceinline__ void mx_tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
}

template <int NT_, int STAGES_> struct MxCfg {
  static constexpr int NT = NT_, STAGES = STAGES_;
  static constexpr int B_BYTES = NT * 128;
  static constexpr int SA = MX_A_BYTES + B_BYTES, SB = SA + 1024, STAGE_BYTES = SB + 1024;      // where the scales lie
  static constexpr int S_COLS = 16;                                    // columns of a stage's scales
  static constexpr int COLS = NT + STAGES * S_COLS;
  static constexpr int TMEM = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  static constexpr int EPI_WARPS = NT >= 128 ? 8 : 4, THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024;
  static_assert(COLS <= 512 && STAGE_BYTES % 1024 == 0, "tensor memory and alignment");
  static_assert(NT <= 128 && STAGES * STAGE_BYTES >= NT * 128 * 4, "one tile of the tokens' scales; the float32 tile of a shared k range lies in the stages");
  // 4-bit elements of both operands (format 1), scales as powers of two, M = 128, N = NT, k = 64, both K-major
  static constexpr uint32_t IDESC = (1u << 7) | (1u << 10) | ((uint32_t)(NT >> 3) << 17) | (1u << 23) | ((uint32_t)(128 >> 4) << 24);
};

struct MxProduct {
  const uint8_t* x_scales;
  const uint8_t* w_scales;
  void* out;
  int rows, k, w_rows, out_features, unary, per_split;                 // per_split: stages of a CTA
  const void* x;                                                       // rows that the kernel rounds itself (ROUND)
  long long x_row;
};

// 32 numbers of a row as 16 bytes of codes and the scale's byte.
__device__ __forceinline__ uint4 mx_round32(const uint32_t (&w)[16], uint32_t& s) {      // pairs of bfloat16
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  m = max(m & 0xffffu, m >> 16);
  s = mx_scale_byte(__uint_as_float(m << 16));
  const float inv = mx_inverse_scale(s);
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(w[4 * i + j] << 16);
      v[2 * j + 1] = __uint_as_float(w[4 * i + j] & 0xffff0000u);
    }
    c[i] = mx_codes8(v, inv);
  }
  return make_uint4(c[0], c[1], c[2], c[3]);
}
__device__ __forceinline__ uint4 mx_round32(const uint32_t (&w)[32], uint32_t& s) {      // float32
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = max(m, w[i] & 0x7fffffffu);
  s = mx_scale_byte(__uint_as_float(m));
  const float inv = mx_inverse_scale(s);
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[8 * i + j]);
    c[i] = mx_codes8(v, inv);
  }
  return make_uint4(c[0], c[1], c[2], c[3]);
}

// What becomes of a sum.  The function is chosen at compile time, or is one call: copies of every function's code for every
// element of an unrolled loop are fetched by every SM (33 rows of gated 4,096 x 12,288: 38 us then, 20 so, before other steps).
//   MX_PLAIN: nothing; MX_SILU: silu(gate) * up with the hardware's exp2 and reciprocal (relative error about 2^-21; outputs of
//   16 bits); MX_UNARY, MX_GATED: any function of common.cuh.
enum { MX_PLAIN, MX_SILU, MX_UNARY, MX_GATED };
__device__ __noinline__ float mx_unary_call(float y, int kind) { return ifb_unary(y, kind); }
__device__ __noinline__ float mx_gate_call(float g, int kind) { return ifb_gate_act(g, kind); }
template <int EPI> __device__ __forceinline__ float mx_gate(float g, float u, int unary) {
  if (EPI == MX_GATED) return mx_gate_call(g, unary) * u;
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(e) : "f"(-1.4426950408889634f * g));
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(1.f + e));
  return g * r * u;
}
template <int EPI> __device__ __forceinline__ float mx_apply(float y, int unary) { return EPI == MX_UNARY ? mx_unary_call(y, unary) : y; }

template <typename C, int EPI, typename TO, typename TX>
__global__ void __launch_bounds__(C::THREADS)
mx4_linear_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, MxProduct p, int* err) {
  constexpr bool GATED = EPI == MX_SILU || EPI == MX_GATED;
  constexpr bool ROUND = !std::is_same<TX, void>::value;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ uint64_t full[C::STAGES], empty[C::STAGES], ready;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const uint32_t base = (mx_smem(raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int o0 = blockIdx.x * 128, n0 = blockIdx.y * C::NT;
  const int k_tiles = (p.k + 127) / 128, stages = (p.k + MX_KSTAGE - 1) / MX_KSTAGE;
  const int s0 = blockIdx.z * p.per_split, s1 = min(stages, s0 + p.per_split);
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) { mx_mbar_init(&full[i], ROUND ? 1 + 32 * C::EPI_WARPS : 1); mx_mbar_init(&empty[i], 1); }
    mx_mbar_init(&ready, 1);
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(mx_smem(&tmem_slot)), "r"(C::TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const uint32_t tmem = *(volatile uint32_t*)&tmem_slot;

  if (warp == 0) {
    // the matrix of the first stages before the wait, the tokens after it
    auto bytes = [&](int s) { return (uint32_t)min(2, k_tiles - 2 * s) * 512u; };      // of one tile of rows' scales
    auto load_w = [&](int s, int i) {
      const uint32_t at = base + i * C::STAGE_BYTES;
      mx_expect_tx(&full[i], ROUND ? MX_A_BYTES + bytes(s) : MX_A_BYTES + C::B_BYTES + bytes(s) * 2);
      mx_tma_2d(at, &w_map, &full[i], s * 64, o0);
      mx_bulk(at + C::SA, p.w_scales + ((size_t)(o0 >> 7) * k_tiles + 2 * s) * 512, bytes(s), &full[i]);
    };
    auto load_x = [&](int s, int i) {
      const uint32_t at = base + i * C::STAGE_BYTES;
      mx_tma_2d(at + MX_A_BYTES, &x_map, &full[i], s * 64, n0);
      mx_bulk(at + C::SB, p.x_scales + ((size_t)(n0 >> 7) * k_tiles + 2 * s) * 512, bytes(s), &full[i]);
    };
    const int ahead = min(C::STAGES, s1 - s0);
    if (mx_elect())
      for (int i = 0; i < ahead; ++i) load_w(s0 + i, i);
    __syncwarp();
    ifb_pdl_wait();
    ifb_pdl_trigger();
    if (!ROUND && mx_elect())
      for (int i = 0; i < ahead; ++i) load_x(s0 + i, i);
    __syncwarp();
    for (int s = s0 + ahead; s < s1; ++s) {
      const int j = s - s0, i = j % C::STAGES;
      if (!mx_wait(&empty[i], ((j / C::STAGES) & 1) ^ 1, abort_flag, err, 701)) break;
      if (mx_elect()) { load_w(s, i); if (!ROUND) load_x(s, i); }
      __syncwarp();
    }
  } else {
    ifb_pdl_wait();
    if constexpr (ROUND) {
      if (warp >= 2) {
        // a thread's blocks lie THREADS apart; AHEAD stages' numbers are under way
        constexpr int THREADS = 32 * C::EPI_WARPS, PER = C::NT * 8 / THREADS, W = sizeof(TX) == 2 ? 16 : 32;
        constexpr int AHEAD = PER * W <= 16 ? 4 : PER * W <= 32 ? 2 : 1;
        const int tid = threadIdx.x - 64;
        uint32_t ring[AHEAD][PER][W];
        auto request = [&](int s, uint32_t (&w)[PER][W]) {
#pragma unroll
          for (int b = 0; b < PER; ++b) {
            const int at = tid + b * THREADS, row = at >> 3, e = (s * 8 + (at & 7)) * MX_BLOCK;
            const bool in = row < p.rows && e < p.k;
            const uint4* src = reinterpret_cast<const uint4*>((const TX*)p.x + (size_t)(in ? row : 0) * p.x_row + (in ? e : 0));
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
              const uint4 v = in ? src[i] : make_uint4(0, 0, 0, 0);
              w[b][4 * i] = v.x; w[b][4 * i + 1] = v.y; w[b][4 * i + 2] = v.z; w[b][4 * i + 3] = v.w;
            }
          }
        };
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) request(s0 + q, ring[q]);      // (beyond the part of k: read and not used, or zeros)
        bool go = true;
        for (int s8 = s0; s8 < s1 && go; s8 += AHEAD)
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
          const int s = s8 + q;
          if (s >= s1) break;
          const int j = s - s0, i = j % C::STAGES;
          uint4 codes[PER];
          uint32_t scale[PER];
#pragma unroll
          for (int b = 0; b < PER; ++b) codes[b] = mx_round32(ring[q][b], scale[b]);
          if (s + AHEAD < s1) request(s + AHEAD, ring[q]);
          if (j >= C::STAGES && !mx_wait(&empty[i], ((j / C::STAGES) & 1) ^ 1, abort_flag, err, 704)) { go = false; break; }
          unsigned char* const at_b = raw + (base - mx_smem(raw)) + i * C::STAGE_BYTES + MX_A_BYTES;
          unsigned char* const at_s = raw + (base - mx_smem(raw)) + i * C::STAGE_BYTES + C::SB;
#pragma unroll
          for (int b = 0; b < PER; ++b) {
            const int at = tid + b * THREADS, row = at >> 3, block = at & 7;
            *reinterpret_cast<uint4*>(at_b + row * 128 + ((block ^ (row & 7)) << 4)) = codes[b];
            at_s[(block >> 2) * 512 + (row & 31) * 16 + (row >> 5) * 4 + (block & 3)] = (unsigned char)scale[b];
          }
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(mx_smem(&full[i])) : "memory");
        }
      }
    }
    if (warp == 1) {
      for (int s = s0; s < s1; ++s) {
        const int j = s - s0, i = j % C::STAGES;
        if (!mx_wait(&full[i], (j / C::STAGES) & 1, abort_flag, err, 702)) break;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        if (mx_elect()) {
          const uint32_t at = base + i * C::STAGE_BYTES, sc = tmem + C::NT + i * C::S_COLS;
          const int tiles = min(2, k_tiles - 2 * s), products = min(4, (p.k - s * MX_KSTAGE + 63) / 64);
          for (int t = 0; t < tiles; ++t) {
            mx_copy_scales(sc + t * 4, at + C::SA + t * 512);
            mx_copy_scales(sc + 8 + t * 4, at + C::SB + t * 512);
          }
          const uint64_t a = mx_desc(at), b = mx_desc(at + MX_A_BYTES);
#pragma unroll
          for (int m = 0; m < 4; ++m)
            if (m < products) {
              const uint32_t id = (uint32_t)(m & 1) * 2;               // which two of the four scales of a word
              mx_mma(tmem, a + m * 2, b + m * 2, C::IDESC | (id << 4) | (id << 29), sc + (m >> 1) * 4, sc + 8 + (m >> 1) * 4,
                     (j | m) != 0);
            }
          mx_commit(&empty[i]);
        }
        __syncwarp();
      }
      if (mx_elect()) mx_commit(&ready);
      __syncwarp();
    }
  }
  const bool ok = mx_wait(&ready, 0, abort_flag, err, 703);
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const int splits = gridDim.z;
  TO* out = (TO*)p.out;
  if (warp >= 2 && ok && splits == 1) {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    constexpr int PER = C::NT / (C::EPI_WARPS / 4);                    // tokens of a warp
    const int row = o0 + quarter * 32 + lane;                          // of w
    for (int c = half * PER; c < (half + 1) * PER; c += 16) {
      if (n0 + c >= p.rows) break;                                     // warp-uniform
      uint32_t v[16];
      mx_tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + c, v);
      if (GATED) {
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const uint32_t other = __shfl_xor_sync(0xffffffffu, lane & 1 ? v[j] : v[j + 1], 1);
          const int token = n0 + c + j + (lane & 1);
          const float y = lane & 1 ? mx_gate<EPI>(__uint_as_float(other), __uint_as_float(v[j + 1]), p.unary)
                                   : mx_gate<EPI>(__uint_as_float(v[j]), __uint_as_float(other), p.unary);
          if (row < p.w_rows && token < p.rows) out[(size_t)token * p.out_features + (row >> 1)] = from_f32<TO>(y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (row < p.w_rows && n0 + c + j < p.rows)
            out[(size_t)(n0 + c + j) * p.out_features + row] = from_f32<TO>(mx_apply<EPI>(__uint_as_float(v[j]), p.unary));
      }
    }
  }
  if (splits > 1) {
    float* mine = reinterpret_cast<float*>(raw + (base - mx_smem(raw)));      // [tokens][128]
    if (warp >= 2 && ok) {
      const int quarter = warp & 3, half = (warp - 2) >> 2;
      constexpr int PER = C::NT / (C::EPI_WARPS / 4);
      for (int c = half * PER; c < (half + 1) * PER; c += 16) {
        uint32_t v[16];
        mx_tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + c, v);
#pragma unroll
        for (int j = 0; j < 16; ++j) mine[(c + j) * 128 + quarter * 32 + lane] = __uint_as_float(v[j]);
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    const int tokens = min(C::NT, p.rows - n0);
    // two rows of w (one output, if gated) per thread and turn, the ranks' numbers added in their order
    const int step = splits * C::THREADS;
    auto put = [&](int i, float2 sum) {
      const int row = o0 + (i & 63) * 2;
      TO* to = out + (size_t)(n0 + (i >> 6)) * p.out_features;
      if (GATED) {
        if (row < p.w_rows) to[row >> 1] = from_f32<TO>(mx_gate<EPI>(sum.x, sum.y, p.unary));
      } else {
        if (row < p.w_rows) to[row] = from_f32<TO>(mx_apply<EPI>(sum.x, p.unary));
        if (row + 1 < p.w_rows) to[row + 1] = from_f32<TO>(mx_apply<EPI>(sum.y, p.unary));
      }
    };
    auto from = [&](int r) {
      uint32_t remote;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"(mx_smem(mine)), "r"(r));
      return remote;
    };
    auto get = [](float2& f, uint32_t remote) {
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];\n" : "=f"(f.x), "=f"(f.y) : "r"(remote) : "memory");
    };
    if constexpr (C::NT == 16) {                                        // one or two turns in all
      for (int i = blockIdx.z * C::THREADS + threadIdx.x; i < tokens * 64; i += step) {
        float2 sum = make_float2(0.f, 0.f);
        for (int r = 0; r < splits; ++r) {
          float2 f;
          get(f, from(r) + i * 8);
          sum.x += f.x;
          sum.y += f.y;
        }
        put(i, sum);
      }
    } else {
      // the numbers of four ranks and TURN turns are requested together (one by one: 128 rows of 1,024, shared by two, 7.0 us for 5.5)
      constexpr int TURN = C::NT >= 64 ? 4 : 2;
      for (int i0 = blockIdx.z * C::THREADS + threadIdx.x; i0 < tokens * 64; i0 += TURN * step) {
        float2 sum[TURN];
#pragma unroll
        for (int u = 0; u < TURN; ++u) sum[u] = make_float2(0.f, 0.f);
        for (int r0 = 0; r0 < splits; r0 += 4) {
          float2 f[4][TURN];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (r0 + r >= splits) break;
            const uint32_t remote = from(r0 + r);
#pragma unroll
            for (int u = 0; u < TURN; ++u) get(f[r][u], remote + min(i0 + u * step, tokens * 64 - 1) * 8);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (r0 + r >= splits) break;
#pragma unroll
            for (int u = 0; u < TURN; ++u) { sum[u].x += f[r][u].x; sum[u].y += f[r][u].y; }
          }
        }
#pragma unroll
        for (int u = 0; u < TURN; ++u)
          if (i0 + u * step < tokens * 64) put(i0 + u * step, sum[u]);
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
  }
  if (!ok) for (int i = 0; i < 2000; ++i) __nanosleep(1000);           // copies in flight land
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(C::TMEM) : "memory");
  }
}

// Clusters of s CTAs that find SMs at a time (33 of four, not 37: a cluster stays in one part of the device).
template <typename K> static int mx_clusters(K kernel, cudaLaunchConfig_t cfg, int s) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = s;
  cfg.gridDim.z = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
  return n;
}
template <typename C, int EPI, typename TO, typename TX>
static int mx_launch(const CUtensorMap& xm, const CUtensorMap& wm, MxProduct p, int splits, int* err, cudaStream_t stream) {
  auto kernel = mx4_linear_kernel<C, EPI, TO, TX>;
  IFB_ALLOW_SMEM(kernel, C::SMEM);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.w_rows + 127) / 128, (p.rows + C::NT - 1) / C::NT, 1);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  const int stages = (p.k + MX_KSTAGE - 1) / MX_KSTAGE, tiles = cfg.gridDim.x * cfg.gridDim.y;
  if (!splits) {
    // The k range of a tile is shared by up to four CTAs, if all find an SM at once, in as many stages of a CTA and, for the sum, two to four more as are
    // the fewest.  (8 rows, k = 4,096, on 1, 2, 3, 4 CTAs: 16 tiles 8.1, 6.4, 5.7 and 4.7 us, 36 tiles 8.0, 6.4, 5.9 and, in two rounds, 9.2, 48 tiles 8.4,
    // 6.8, 11.5 and 10.2; 128 rows: 16 tiles 8.8, 7.3, 7.1, 6.3, 48 tiles 9.0, 7.9, 14.3, 13.3; k = 1,024, 48 tiles: 8 rows 3.8, 4.3, 4.3, 7.8.
    // More than four leave SMs without one: 16 tiles of 128 rows, k = 2,048, eight 8.8.)
    static int clusters[IFB_MAX_DEVICES][5] = {};
    int dev = 0, least = stages;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= IFB_MAX_DEVICES) return IFB_ERR_ARG;
    splits = 1;
    for (int s = 4; s > 1; --s) {
      int& fit = clusters[dev][s];
      if (!fit) fit = 1 + mx_clusters(kernel, cfg, s);
      const int cost = (stages + s - 1) / s + (s == 4 ? (C::NT == 32 ? 2 : 3) : C::NT <= 32 ? 2 : 4);
      if (tiles < fit && cost < least) { splits = s; least = cost; }
    }
  }
  if (splits < 1 || splits > 8 || splits > stages) return IFB_ERR_ARG;
  p.per_split = (stages + splits - 1) / splits;
  splits = (stages + p.per_split - 1) / p.per_split;                   // every CTA has a stage
  cfg.gridDim.z = splits;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = splits;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ifb_pdl_enabled() ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, xm, wm, p, err);
  if (e != cudaSuccess) { cudaGetLastError(); return -(int)e; }
  return IFB_OK;
}
template <typename C, typename TX>
static int mx_launch_any(const CUtensorMap& xm, const CUtensorMap& wm, const MxProduct& p, bool gated, int dtype, int splits, int* err,
                         cudaStream_t stream) {
  if (dtype == IFB_F32) {
    if (gated) return mx_launch<C, MX_GATED, float, TX>(xm, wm, p, splits, err, stream);
    return p.unary ? mx_launch<C, MX_UNARY, float, TX>(xm, wm, p, splits, err, stream) : mx_launch<C, MX_PLAIN, float, TX>(xm, wm, p, splits, err, stream);
  }
  if (gated) return p.unary ? mx_launch<C, MX_GATED, bf16, TX>(xm, wm, p, splits, err, stream) : mx_launch<C, MX_SILU, bf16, TX>(xm, wm, p, splits, err, stream);
  return p.unary ? mx_launch<C, MX_UNARY, bf16, TX>(xm, wm, p, splits, err, stream) : mx_launch<C, MX_PLAIN, bf16, TX>(xm, wm, p, splits, err, stream);
}

// ---------------------------------------------------------------------------------------------
// The product of many rows, over pairs of SMs: a cluster of two CTAs owns 256 rows of w by 256 tokens.  Each CTA brings 128 rows
// of either operand (and the scales of its rows of w and of all 256 tokens), one tcgen05.mma of the pair (M = 256), issued by the
// first CTA, multiplies out of both shared memories into both tensor memories, where a CTA finds its 128 rows of w.  What bounds
// these products is the bytes that reach an SM: 8 KB for the 128 cycles of 128 x 256 x 64, where a CTA alone would bring 12 (2,048 rows by gate
// and up of 12,288 x 4,096: 89 us with the rows' rounding, 4.6 PFLOP/s, 103 in the long run, at the clocks of the power limit; the tensor pipe busy for 63 % of the time, 46 bytes a cycle into an SM; by
// CTAs alone 150).
// Persistent, one accumulator (the scales leave no room for two): the epilogue's warps take it to registers at once (256
// columns in some hundred cycles) and let the next tile's products begin, which run while they finish and store.
// The "full" barriers are the first CTA's and count both CTAs' bytes; "empty" and "accumulator ready" are each CTA's own, by
// multicast commits; "accumulator read" is the first CTA's and counts all sixteen warps.
// STAGED (rows of the output on 16 bytes): a half of the epilogue's warps lays its 128 tokens out in shared memory, rows of 128 bytes
// in the swizzle, and one thread stores them by TMA: whole lines, which clip at the output's ends; stores of a number per lane, 64
// bytes of a row each, took 13 of 95 us (gate and up of 12,288 x 4,096, 2,048 rows).
// ---------------------------------------------------------------------------------------------
constexpr int MXP_STAGES = 5;
constexpr int MXP_B = MX_A_BYTES, MXP_SA = 2 * MX_A_BYTES, MXP_SB = MXP_SA + 1024, MXP_STAGE = MXP_SB + 2048;      // where things lie in a stage
constexpr int MXP_STAGING = 16384;       // of each half of the epilogue's warps
constexpr int MXP_SMEM = MXP_STAGES * MXP_STAGE + 2 * MXP_STAGING + 1024;
constexpr int MXP_S_COLS = 24, MXP_TMEM = 512, MXP_THREADS = 320;
static_assert(256 + MXP_STAGES * MXP_S_COLS <= MXP_TMEM && MXP_STAGE % 1024 == 0 && MXP_SMEM <= 227 * 1024, "pair sizes");
constexpr uint32_t MXP_IDESC = (1u << 7) | (1u << 10) | ((uint32_t)(256 >> 3) << 17) | (1u << 23) | ((uint32_t)(256 >> 4) << 24);

__device__ __forceinline__ uint32_t mx_peer(const void* p, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(mx_smem(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void mx_tma_pair(uint32_t smem, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
               ::"r"(smem), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void mx_copy_scales_pair(uint32_t tmem, uint32_t smem) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n" ::"r"(tmem), "l"(mx_scale_desc(smem)) : "memory");
}
__device__ __forceinline__ void mx_mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
               " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc) : "memory");
}
__device__ __forceinline__ void mx_commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
               ::"r"(mx_smem(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void mx_tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}

__device__ __forceinline__ void mx_tma_store(const CUtensorMap* map, uint32_t smem, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];\n" ::"l"(map), "r"(smem), "r"(x), "r"(y) : "memory");
}

template <int EPI, typename TO, bool STAGED>
__global__ void __launch_bounds__(MXP_THREADS, 1)
mx4_pair_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap xs_map,
                const __grid_constant__ CUtensorMap ws_map, const __grid_constant__ CUtensorMap out_map, MxProduct p, int token_tiles, int tiles, int* err) {
  constexpr bool GATED = EPI == MX_SILU || EPI == MX_GATED;
  constexpr int FEATURES = GATED ? 64 : 128, BOXES = FEATURES * (int)sizeof(TO) / 128, PASS = 128 / BOXES;      // of a CTA; a pass's tokens
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ uint64_t full[MXP_STAGES], empty[MXP_STAGES], acc_full, acc_empty;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const uint32_t base = (mx_smem(raw) + 1023u) & ~1023u;                // the same offset in both CTAs
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, rank = blockIdx.x & 1;
  const int stages = (p.k + MX_KSTAGE - 1) / MX_KSTAGE, k_tiles = (p.k + 127) / 128;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < MXP_STAGES; ++i) { mx_mbar_init(&full[i], 1); mx_mbar_init(&empty[i], 1); }
    mx_mbar_init(&acc_full, 1);
    mx_mbar_init(&acc_empty, 16);
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(mx_smem(&tmem_slot)), "r"(MXP_TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");      // both CTAs' barriers exist
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const uint32_t tmem = *(volatile uint32_t*)&tmem_slot;

  if (warp == 0) {
    // producer, in both CTAs; the matrix of the first tile's first stages before the wait for the kernel that rounds the rows
    auto load_w = [&](int t, int s, int i) {
      const uint32_t at = base + i * MXP_STAGE, bar = mx_peer(&full[i], 0);
      const int o0 = t / token_tiles * 256 + rank * 128;
      if (rank == 0) mx_expect_tx(&full[i], 2 * MXP_STAGE);
      mx_tma_pair(at, &w_map, bar, s * 64, o0);
      mx_tma_pair(at + MXP_SA, &ws_map, bar, 0, (o0 >> 7) * k_tiles + 2 * s);
    };
    auto load_x = [&](int t, int s, int i) {
      const uint32_t at = base + i * MXP_STAGE, bar = mx_peer(&full[i], 0);
      const int n0 = t % token_tiles * 256;
      mx_tma_pair(at + MXP_B, &x_map, bar, s * 64, n0 + rank * 128);
      mx_tma_pair(at + MXP_SB, &xs_map, bar, 0, (n0 >> 7) * k_tiles + 2 * s);
      mx_tma_pair(at + MXP_SB + 1024, &xs_map, bar, 0, ((n0 >> 7) + 1) * k_tiles + 2 * s);
    };
    const int ahead = first < tiles ? min(MXP_STAGES, stages) : 0;
    if (mx_elect())
      for (int i = 0; i < ahead; ++i) load_w(first, i, i);
    __syncwarp();
    ifb_pdl_wait();
    ifb_pdl_trigger();
    if (mx_elect())
      for (int i = 0; i < ahead; ++i) load_x(first, i, i);
    __syncwarp();
    int g = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step)
      for (int s = 0; s < stages; ++s, ++g) {
        if (g < ahead) continue;
        const int i = g % MXP_STAGES;
        if (g >= MXP_STAGES && !mx_wait(&empty[i], ((g / MXP_STAGES) & 1) ^ 1, abort_flag, err, 711)) { ok = false; break; }
        if (mx_elect()) { load_w(t, s, i); load_x(t, s, i); }
        __syncwarp();
      }
  } else if (warp == 1) {
    bool ok = rank == 0;
    int g = 0, n = 0;
    for (int t = first; t < tiles && ok; t += step, ++n) {
      if (n > 0) ok = mx_wait(&acc_empty, (n - 1) & 1, abort_flag, err, 714);
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      for (int s = 0; s < stages && ok; ++s, ++g) {
        const int i = g % MXP_STAGES;
        ok = mx_wait(&full[i], (g / MXP_STAGES) & 1, abort_flag, err, 712);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        if (mx_elect()) {
          const uint32_t at = base + i * MXP_STAGE, sc = tmem + 256 + i * MXP_S_COLS;
          const int products = min(4, (p.k - s * MX_KSTAGE + 63) / 64);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (2 * h < products) {
              mx_copy_scales_pair(sc + h * 4, at + MXP_SA + h * 512);
              mx_copy_scales_pair(sc + 8 + h * 8, at + MXP_SB + h * 512);
              mx_copy_scales_pair(sc + 8 + h * 8 + 4, at + MXP_SB + 1024 + h * 512);
            }
          const uint64_t a = mx_desc(at), b = mx_desc(at + MXP_B);
#pragma unroll
          for (int m = 0; m < 4; ++m)
            if (m < products) {
              const uint32_t id = (uint32_t)(m & 1) * 2;
              mx_mma_pair(tmem, a + m * 2, b + m * 2, MXP_IDESC | (id << 4) | (id << 29), sc + (m >> 1) * 4, sc + 8 + (m >> 1) * 8, (s | m) != 0);
            }
          mx_commit_pair(&empty[i]);
          if (s == stages - 1) mx_commit_pair(&acc_full);
        }
        __syncwarp();
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    TO* out = (TO*)p.out;
    int n = 0;
    ifb_pdl_wait();                                                     // (the kernel before may still read what this one writes)
    for (int t = first; t < tiles; t += step, ++n) {
      const int row = t / token_tiles * 256 + rank * 128 + quarter * 32 + lane, n0 = t % token_tiles * 256 + half * 128;
      const bool ok = __all_sync(0xffffffffu, mx_wait(&acc_full, n & 1, abort_flag, err, 713)) != 0;
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      uint32_t v[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) mx_tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + half * 128 + c * 32, v + c * 32);
      asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        const uint32_t bar = mx_peer(&acc_empty, 0);
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
      }
      if constexpr (STAGED) {
        const uint32_t staging = base + MXP_STAGES * MXP_STAGE + half * MXP_STAGING;
        const int feature = GATED ? quarter * 16 + (lane >> 1) : quarter * 32 + lane, byte = feature * (int)sizeof(TO);
        const uint32_t at = staging + (byte >> 7) * (PASS * 128) + (byte & 15);
        const int chunk = (byte >> 4) & 7;
        const bool first_thread = ((warp - 2) & 3) == 0 && lane == 0;
#pragma unroll
        for (int pass = 0; pass < BOXES; ++pass) {
          if (first_thread) asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");      // the pass before has been read
          asm volatile("bar.sync %0, 128;\n" ::"r"(1 + half) : "memory");
#pragma unroll
          for (int j = 0; j < PASS; j += 2) {
            auto put = [&](int token, float y) {
              const uint32_t to = at + token * 128 + ((chunk ^ (token & 7)) << 4);
              if (sizeof(TO) == 2) {
                const __nv_bfloat16 b = __float2bfloat16_rn(y);
                asm volatile("st.shared.u16 [%0], %1;\n" ::"r"(to), "h"(*reinterpret_cast<const uint16_t*>(&b)) : "memory");
              } else {
                asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(to), "f"(y) : "memory");
              }
            };
            const uint32_t v0 = v[pass * PASS + j], v1 = v[pass * PASS + j + 1];
            if (GATED) {
              const uint32_t other = __shfl_xor_sync(0xffffffffu, lane & 1 ? v0 : v1, 1);
              put(j + (lane & 1), lane & 1 ? mx_gate<EPI>(__uint_as_float(other), __uint_as_float(v1), p.unary)
                                           : mx_gate<EPI>(__uint_as_float(v0), __uint_as_float(other), p.unary));
            } else {
              put(j, mx_apply<EPI>(__uint_as_float(v0), p.unary));
              put(j + 1, mx_apply<EPI>(__uint_as_float(v1), p.unary));
            }
          }
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
          asm volatile("bar.sync %0, 128;\n" ::"r"(1 + half) : "memory");
          if (first_thread) {
            const int x0 = (t / token_tiles * 256 + rank * 128) / (GATED ? 2 : 1), y0 = n0 + pass * PASS;
#pragma unroll
            for (int b = 0; b < BOXES; ++b)
              if (y0 < p.rows && x0 + b * (128 / (int)sizeof(TO)) < p.out_features)
                mx_tma_store(&out_map, staging + b * (PASS * 128), x0 * (int)sizeof(TO) / 2 + b * 64, y0);
            asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
          }
        }
        continue;
      }
      TO* to = out + (size_t)n0 * p.out_features;
#pragma unroll
      for (int j = 0; j < 128; j += 2) {
        if (GATED) {
          const uint32_t other = __shfl_xor_sync(0xffffffffu, lane & 1 ? v[j] : v[j + 1], 1);
          const float y = lane & 1 ? mx_gate<EPI>(__uint_as_float(other), __uint_as_float(v[j + 1]), p.unary)
                                   : mx_gate<EPI>(__uint_as_float(v[j]), __uint_as_float(other), p.unary);
          if (row < p.w_rows && n0 + j + (lane & 1) < p.rows) to[(size_t)(j + (lane & 1)) * p.out_features + (row >> 1)] = from_f32<TO>(y);
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (row < p.w_rows && n0 + j + e < p.rows) to[(size_t)(j + e) * p.out_features + row] = from_f32<TO>(mx_apply<EPI>(__uint_as_float(v[j + e]), p.unary));
        }
      }
    }
  }
  if (STAGED) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");      // (of the threads that stored)
  if (*abort_flag) for (int i = 0; i < 2000; ++i) __nanosleep(1000);    // copies in flight land
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");      // neither CTA leaves while the other needs its memory
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(MXP_TMEM) : "memory");
  }
}

template <int EPI, typename TO, bool STAGED>
static int mx_launch_pair(const CUtensorMap (&m)[5], const MxProduct& p, int* err, cudaStream_t stream) {
  auto kernel = mx4_pair_kernel<EPI, TO, STAGED>;
  IFB_ALLOW_SMEM(kernel, MXP_SMEM);
  const int token_tiles = (p.rows + 255) / 256, tiles = token_tiles * ((p.w_rows + 255) / 256), pairs = ifb_sm_count() / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (tiles < pairs ? tiles : pairs));
  cfg.blockDim = dim3(MXP_THREADS);
  cfg.dynamicSmemBytes = MXP_SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ifb_pdl_enabled() ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, m[0], m[1], m[2], m[3], m[4], p, token_tiles, tiles, err);
  if (e != cudaSuccess) { cudaGetLastError(); return -(int)e; }
  return IFB_OK;
}
// The output by TMA where its rows begin on 16 bytes.
template <int EPI, typename TO>
static int mx_launch_pair_out(CUtensorMap (&m)[5], const MxProduct& p, int* err, cudaStream_t stream) {
  constexpr int FEATURES = EPI == MX_SILU || EPI == MX_GATED ? 64 : 128, BOXES = FEATURES * (int)sizeof(TO) / 128;
  const unsigned long long bytes = (unsigned long long)p.out_features * sizeof(TO), d[2] = {bytes / 2, (unsigned long long)p.rows}, s[1] = {bytes};
  const unsigned box[2] = {64, 128 / BOXES};
  if (bytes % 16 || ((uintptr_t)p.out & 15) || ifb_tensor_map_bf16(&m[4], p.out, 2, d, s, box)) {
    m[4] = m[0];                                                        // not looked at
    return mx_launch_pair<EPI, TO, false>(m, p, err, stream);
  }
  return mx_launch_pair<EPI, TO, true>(m, p, err, stream);
}
static int mx_launch_pair_any(CUtensorMap (&m)[5], const MxProduct& p, bool gated, int dtype, int* err, cudaStream_t stream) {
  if (dtype == IFB_F32) {
    if (gated) return mx_launch_pair_out<MX_GATED, float>(m, p, err, stream);
    return p.unary ? mx_launch_pair_out<MX_UNARY, float>(m, p, err, stream) : mx_launch_pair_out<MX_PLAIN, float>(m, p, err, stream);
  }
  if (gated) return p.unary ? mx_launch_pair_out<MX_GATED, bf16>(m, p, err, stream) : mx_launch_pair_out<MX_SILU, bf16>(m, p, err, stream);
  return p.unary ? mx_launch_pair_out<MX_UNARY, bf16>(m, p, err, stream) : mx_launch_pair_out<MX_PLAIN, bf16>(m, p, err, stream);
}

// x: [rows][k], w: [w_rows][k] (twice the out features if the epilogue is gated).  x_dtype IFB_F32 or IFB_BF16: `x` has numbers, rows
// x_row elements apart; up to ifb_mx4_round_rows rows are rounded within the product, more of them first, into x_codes and
// x_scales (whose room is the caller's; neither is looked at otherwise).  x_dtype -1: x_codes and x_scales have been rounded.
// epilogue: as in the other products.  nt, splits: 0, or (for measurements) tokens of a tile and CTAs that share its k range.
constexpr int MX_ROUND_ROWS = 32;
IFB_EXPORT int ifb_mx4_round_rows(int dtype) { return dtype == IFB_F32 ? MX_ROUND_ROWS / 2 : MX_ROUND_ROWS; }
IFB_EXPORT int ifb_mx4_linear(const void* x, int x_dtype, long long x_row, void* x_codes, void* x_scales, const void* w_codes, const void* w_scales,
                              void* out, int out_dtype, int rows, int k, int w_rows, int epilogue, int nt, int splits, void* err, void* stream) {
  const bool gated = epilogue & 1;
  const int unary = epilogue >> 4;
  int bad = mx_sizes(rows, k, 0);
  if (bad) return bad;
  if (w_rows < 1 || (gated && (w_rows & 1))) return IFB_ERR_SIZE;
  if ((epilogue & 14) || unary > IFB_UNARY_LAST) return IFB_ERR_ARG;
  if (out_dtype != IFB_F32 && out_dtype != IFB_BF16) return IFB_ERR_DTYPE;
  if (x_dtype != -1 && x_dtype != IFB_F32 && x_dtype != IFB_BF16) return IFB_ERR_DTYPE;
  if ((((uintptr_t)x_codes) | ((uintptr_t)x_scales) | ((uintptr_t)w_codes) | ((uintptr_t)w_scales)) & 15) return IFB_ERR_ALIGN;
  const bool round = x_dtype != -1 && rows <= (x_dtype == IFB_F32 ? MX_ROUND_ROWS / 2 : MX_ROUND_ROWS);
  if (round && ((((uintptr_t)x) | (uintptr_t)(x_row * (x_dtype == IFB_F32 ? 4 : 2))) & 15)) return IFB_ERR_ALIGN;
  if (!round && (!x_codes || !x_scales)) return IFB_ERR_ARG;
  if (!round && x_dtype != -1) {
    bad = mx_quantize(x, x_dtype, x_row, x_codes, x_scales, rows, k, 0, 1, stream);
    if (bad) return bad;
  }
  // Pairs of SMs (tiles of 256 x 256) from the second round of tiles of 128 x 128 on, where their rounds are fewer; theirs is 1.3 times as long.
  // (24,576 x 4,096: 64 rows 19.5 us and 20.0 over pairs, 256 rows 30.3 and 23.7; 4,096 x 4,096, 193 rows: 8.7 and 13.4.)
  const long long tiles1 = (long long)((w_rows + 127) / 128) * ((rows + 127) / 128), tiles2 = (long long)((w_rows + 255) / 256) * ((rows + 255) / 256);
  const int sms = ifb_sm_count(), pairs = sms / 2;
  const bool many = rows > 128 && tiles1 > sms && 4 * ((tiles2 + pairs - 1) / pairs) <= 3 * ((tiles1 + sms - 1) / sms);
  const bool pair = nt ? nt == 256 : many;
  if (!nt || round) nt = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
  if (nt < rows && nt < 128) return IFB_ERR_ARG;
  const MxProduct p = {(const uint8_t*)x_scales, (const uint8_t*)w_scales, out, rows, k, w_rows, gated ? w_rows / 2 : w_rows, unary, 0, x, x_row};
  // the maps see pairs of bytes as one number of 16 bits: only widths and strides in bytes count
  const unsigned long long xd[2] = {(unsigned long long)k / 4, (unsigned long long)rows}, xs[1] = {(unsigned long long)k / 2};
  const unsigned long long wd[2] = {(unsigned long long)k / 4, (unsigned long long)w_rows}, ws[1] = {(unsigned long long)k / 2};
  const unsigned xb[2] = {64, pair ? 128u : (unsigned)nt}, wb[2] = {64, 128};
  CUtensorMap xm, wm;
  bad = ifb_tensor_map_bf16(&wm, w_codes, 2, wd, ws, wb);
  if (bad) return bad;
  cudaStream_t st = (cudaStream_t)stream;
  int* e = (int*)err;
  if (round) {
    if (x_dtype == IFB_F32) return mx_launch_any<MxCfg<16, 6>, float>(wm, wm, p, gated, out_dtype, splits, e, st);      // (16 rows at most)
    return nt == 16 ? mx_launch_any<MxCfg<16, 6>, bf16>(wm, wm, p, gated, out_dtype, splits, e, st)
                    : mx_launch_any<MxCfg<32, 6>, bf16>(wm, wm, p, gated, out_dtype, splits, e, st);
  }
  bad = ifb_tensor_map_bf16(&xm, x_codes, 2, xd, xs, xb);
  if (bad) return bad;
  if (pair) {
    // scale tiles as rows of 512 bytes
    const unsigned long long k_tiles = (unsigned long long)(k + 127) / 128, sd[1] = {512};
    const unsigned long long xsd[2] = {256, k_tiles * 2 * ((rows + 255) / 256)}, wsd[2] = {256, k_tiles * 2 * ((w_rows + 255) / 256)};
    const unsigned sb[2] = {256, 2};
    CUtensorMap m[5] = {xm, wm};
    bad = ifb_tensor_map_bf16(&m[2], x_scales, 2, xsd, sd, sb, true);
    if (!bad) bad = ifb_tensor_map_bf16(&m[3], w_scales, 2, wsd, sd, sb, true);
    return bad ? bad : mx_launch_pair_any(m, p, gated, out_dtype, e, st);
  }
  switch (nt) {
    case 16: return mx_launch_any<MxCfg<16, 6>, void>(xm, wm, p, gated, out_dtype, splits, e, st);
    case 32: return mx_launch_any<MxCfg<32, 6>, void>(xm, wm, p, gated, out_dtype, splits, e, st);
    case 64: return mx_launch_any<MxCfg<64, 4>, void>(xm, wm, p, gated, out_dtype, splits, e, st);
    case 128: return mx_launch_any<MxCfg<128, 6>, void>(xm, wm, p, gated, out_dtype, splits, e, st);
    default: return IFB_ERR_ARG;
  }
}
