// MXFP4 operands (OCP Microscaling Formats v1.0, section 5 and 6.3): e2m1
// codes, two to a byte (even column in the low nibble), and one e8m0 scale
// byte per 32 columns of a row.
//
//   scale exponent  E = floor(log2 max|v|) - 2   (2 = the exponent of e2m1's 6)
//   stored byte     E + 127, at least 0; 255 (NaN) where the block holds an
//                   infinity or a NaN; 0 for a block of zeros
//   code            e2m1(v * 2^-E), to nearest even, saturating at 6
//
// Every factor is a power of two, so v * 2^-E is exact and codes and scales
// are the same on any machine that follows the definition.
//
// Scales are stored in tiles of 128 rows x 4 blocks (512 bytes), tile
// [row / 128][block / 4], byte (row % 32) * 16 + (row % 128) / 32 * 4 +
// block % 4 inside it: the order in which the tensor core wants them in TMEM
// (32 lanes of 16 bytes), so that the product copies tiles without shuffling.
// Bytes of rows and blocks beyond the matrix are 0.
#include <cuda_fp4.h>

#include "host.cuh"
#include "ptx.cuh"

namespace swiglu {
namespace {

constexpr int kBlock = 32;          // columns that share a scale
constexpr int kTileRows = 128;
constexpr int kTileBytes = 512;
constexpr int kQuantCols = 256;     // columns of one CTA: a warp covers a row of them, 8 a thread
constexpr int kQuantThreads = 256;

// Eight consecutive values of a row.
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack_bf16x2(w[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
  f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                            pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

__device__ __forceinline__ float power_of_two(int field) { return __uint_as_float(static_cast<uint32_t>(field) << 23); }

// 2^(byte - 127): byte 0 is the subnormal 2^-127, byte 255 a NaN.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return byte == 0 ? __uint_as_float(0x00400000u) : byte == 255 ? __uint_as_float(0x7fc00000u) : power_of_two(byte);
}

// Two e2m1 codes (low nibble first) as f32.
__device__ __forceinline__ float2 e2m1x2_value(uint32_t byte) {
  const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(byte), __NV_E2M1);
  return __half22float2(__half2(h));
}

// One CTA: 128 rows x 256 columns, two scale tiles. A warp reads 256 columns
// of one row (512 bytes of bf16), eight rows in flight a thread; four lanes
// share a block, and the tiles' bytes leave together, so that no scale byte is
// written alone.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_mxfp4_kernel(const T* __restrict__ src,
                                                                       uint8_t* __restrict__ dst,
                                                                       uint8_t* __restrict__ scale, long long rows,
                                                                       int cols, int tiles_k) {
  __shared__ __align__(16) uint8_t tile[2 * kTileBytes];
  const int lane = static_cast<int>(lane_id()), warp = static_cast<int>(warp_id());
  const long long r0 = blockIdx.y * static_cast<long long>(kTileRows);
  const int c0 = blockIdx.x * kQuantCols + lane * 8;
  const bool in_cols = c0 < cols;  // cols is a multiple of 32: whole groups of 8
  reinterpret_cast<uint32_t*>(tile)[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float f[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long long r = r0 + (half * 8 + i) * 8 + warp;
      if (in_cols && r < rows) load8(src + r * cols + c0, f[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int rt = (half * 8 + i) * 8 + warp;
      const long long r = r0 + rt;
      const bool in = in_cols && r < rows;
      uint32_t top = 0;  // |v| compares as an integer; a NaN is above infinity
      if (in) {
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[i][e]) & 0x7fffffffu);
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (!in) continue;
      const int field = static_cast<int>(top >> 23);  // 127 + floor(log2 max), 0 below the normals
      const int byte = field == 255 ? 255 : max(field - 2, 0);
      const float inv = power_of_two(254 - min(byte, 253));
      uint32_t out = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __nv_fp4x2_storage_t v = __nv_cvt_float2_to_fp4x2(
            make_float2(f[i][2 * e] * inv, f[i][2 * e + 1] * inv), __NV_E2M1, cudaRoundNearest);
        out |= static_cast<uint32_t>(v) << (8 * e);
      }
      *reinterpret_cast<uint32_t*>(dst + r * (cols / 2) + c0 / 2) = out;
      if ((lane & 3) == 0) {
        const int b = lane >> 2;  // block 0..7 of this CTA's columns
        tile[(b >> 2) * kTileBytes + (rt & 31) * 16 + (rt >> 5) * 4 + (b & 3)] = static_cast<uint8_t>(byte);
      }
    }
  }
  __syncthreads();
  const int t = 2 * blockIdx.x + (threadIdx.x >> 5);
  if (threadIdx.x < 64 && t < tiles_k) {
    uint8_t* to = scale + (blockIdx.y * static_cast<long long>(tiles_k) + t) * kTileBytes;
    reinterpret_cast<uint4*>(to)[threadIdx.x & 31] = reinterpret_cast<const uint4*>(tile)[threadIdx.x];
  }
}

template <typename T>
__global__ void __launch_bounds__(kQuantThreads) dequantize_mxfp4_kernel(const uint8_t* __restrict__ src,
                                                                         const uint8_t* __restrict__ scale,
                                                                         T* __restrict__ dst, long long rows, int cols,
                                                                         int tiles_k) {
  __shared__ __align__(16) uint8_t tile[2 * kTileBytes];
  const int lane = static_cast<int>(lane_id()), warp = static_cast<int>(warp_id());
  const long long r0 = blockIdx.y * static_cast<long long>(kTileRows);
  const int c0 = blockIdx.x * kQuantCols + lane * 8;
  const int t = 2 * blockIdx.x + (threadIdx.x >> 5);
  if (threadIdx.x < 64 && t < tiles_k) {
    const uint8_t* from = scale + (blockIdx.y * static_cast<long long>(tiles_k) + t) * kTileBytes;
    reinterpret_cast<uint4*>(tile)[threadIdx.x] = __ldg(reinterpret_cast<const uint4*>(from) + (threadIdx.x & 31));
  }
  const bool in_cols = c0 < cols;
  uint32_t q[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const long long r = r0 + i * 8 + warp;
    if (in_cols && r < rows) q[i] = __ldg(reinterpret_cast<const uint32_t*>(src + r * (cols / 2) + c0 / 2));
  }
  __syncthreads();
  if (!in_cols) return;
  const int b = lane >> 2;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int rt = i * 8 + warp;
    const long long r = r0 + rt;
    if (r >= rows) break;
    const float s = scale_value(tile[(b >> 2) * kTileBytes + (rt & 31) * 16 + (rt >> 5) * 4 + (b & 3)]);
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 v = e2m1x2_value((q[i] >> (8 * e)) & 0xffu);
      f[2 * e] = v.x * s;
      f[2 * e + 1] = v.y * s;
    }
    store8(dst + r * cols + c0, f);
  }
}

// C = A . B^T from the decoded values, f32 accumulation: 64 x 64 outputs a
// CTA, one block of 32 along K at a time.
__device__ __forceinline__ void decode_rows(const uint8_t* q, const uint8_t* scale, long long rows, long long r0, int K,
                                            int tiles_k, int kb, float (*to)[kBlock + 1]) {
  // 64 rows x 16 bytes: a thread decodes 4 bytes of one row.
  const int rr = threadIdx.x >> 2, part = threadIdx.x & 3;
  const long long r = r0 + rr;
  uint32_t codes = 0;
  float s = 0.0f;
  if (r < rows) {
    codes = *reinterpret_cast<const uint32_t*>(q + r * (K / 2) + kb * 16 + part * 4);
    s = scale_value(scale[((r / kTileRows) * tiles_k + kb / 4) * kTileBytes + (r % 32) * 16 + (r % kTileRows) / 32 * 4 +
                          kb % 4]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 v = e2m1x2_value((codes >> (8 * e)) & 0xffu);
    to[rr][part * 8 + 2 * e] = v.x * s;
    to[rr][part * 8 + 2 * e + 1] = v.y * s;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) matmul_mxfp4_kernel(const uint8_t* aq, const uint8_t* as, const uint8_t* bq,
                                                           const uint8_t* bs, T* c, int M, int N, int K, int tiles_k) {
  __shared__ float a[64][kBlock + 1], b[64][kBlock + 1];
  const long long m0 = blockIdx.y * 64ll, n0 = blockIdx.x * 64ll;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int kb = 0; kb < K / kBlock; ++kb) {
    __syncthreads();
    decode_rows(aq, as, M, m0, K, tiles_k, kb, a);
    decode_rows(bq, bs, N, n0, K, tiles_k, kb, b);
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < kBlock; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += a[ty + 16 * i][k] * b[tx + 16 * j][k];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < M && n < N) {
        if constexpr (sizeof(T) == 4) c[m * N + n] = acc[i][j];
        else c[m * N + n] = __float2bfloat16_rn(acc[i][j]);
      }
    }
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_mx(const char* what, int64_t rows, int64_t cols) {
  if (int rc = check_dims(what, rows, cols, 0)) return rc;
  if (cols % kBlock)
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "%s: %lld columns are not a multiple of 32", what, (long long)cols);
  if ((rows + kTileRows - 1) / kTileRows > 65535)
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "%s: more than 8,388,480 rows", what);
  return SWIGLU_OK;
}

dim3 quant_grid(int64_t rows, int64_t cols) {
  return dim3(static_cast<unsigned>((cols + kQuantCols - 1) / kQuantCols),
              static_cast<unsigned>((rows + kTileRows - 1) / kTileRows));
}

int op_quantize(const void* src, void* dst, void* scale, int64_t rows, int64_t cols, int dtype, cudaStream_t st) {
  if (int rc = check_mx("quantize_mxfp4", rows, cols)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (rows == 0 || cols == 0) return SWIGLU_OK;
  if (!src || !dst || !scale) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned16(src) || !aligned16(dst) || !aligned16(scale))
    return fail(SWIGLU_ERR_MISALIGNED, "quantize_mxfp4: pointers must be 16-byte aligned");
  DeviceInfo* d;
  if (int rc = current_device(&d)) return rc;
  const int tiles_k = static_cast<int>((cols + 127) / 128);
  if (dtype == SWIGLU_F32)
    quantize_mxfp4_kernel<float><<<quant_grid(rows, cols), kQuantThreads, 0, st>>>(
        static_cast<const float*>(src), static_cast<uint8_t*>(dst), static_cast<uint8_t*>(scale), rows,
        static_cast<int>(cols), tiles_k);
  else
    quantize_mxfp4_kernel<__nv_bfloat16><<<quant_grid(rows, cols), kQuantThreads, 0, st>>>(
        static_cast<const __nv_bfloat16*>(src), static_cast<uint8_t*>(dst), static_cast<uint8_t*>(scale), rows,
        static_cast<int>(cols), tiles_k);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, "quantize_mxfp4 launch");
}

int op_dequantize(const void* q, const void* scale, void* dst, int64_t rows, int64_t cols, int dtype,
                  cudaStream_t st) {
  if (int rc = check_mx("dequantize_mxfp4", rows, cols)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (rows == 0 || cols == 0) return SWIGLU_OK;
  if (!q || !dst || !scale) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned16(q) || !aligned16(dst) || !aligned16(scale))
    return fail(SWIGLU_ERR_MISALIGNED, "dequantize_mxfp4: pointers must be 16-byte aligned");
  DeviceInfo* d;
  if (int rc = current_device(&d)) return rc;
  const int tiles_k = static_cast<int>((cols + 127) / 128);
  if (dtype == SWIGLU_F32)
    dequantize_mxfp4_kernel<float><<<quant_grid(rows, cols), kQuantThreads, 0, st>>>(
        static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scale), static_cast<float*>(dst), rows,
        static_cast<int>(cols), tiles_k);
  else
    dequantize_mxfp4_kernel<__nv_bfloat16><<<quant_grid(rows, cols), kQuantThreads, 0, st>>>(
        static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scale), static_cast<__nv_bfloat16*>(dst), rows,
        static_cast<int>(cols), tiles_k);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, "dequantize_mxfp4 launch");
}

int op_matmul(const void* aq, const void* a_scale, const void* bq, const void* b_scale, void* c, int64_t M, int64_t N,
              int64_t K, int out_dtype, cudaStream_t st) {
  if (int rc = check_mx("matmul_mxfp4", M, K)) return rc;
  if (int rc = check_mx("matmul_mxfp4", N, K)) return rc;
  if (int rc = check_dtype(out_dtype)) return rc;
  if (K <= 0) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "K must be positive");
  if (int rc = check_mult8("N", N)) return rc;
  if (M == 0 || N == 0) return SWIGLU_OK;
  if (!aq || !a_scale || !bq || !b_scale || !c) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned16(aq) || !aligned16(a_scale) || !aligned16(bq) || !aligned16(b_scale) || !aligned16(c))
    return fail(SWIGLU_ERR_MISALIGNED, "matmul_mxfp4: pointers must be 16-byte aligned");
  DeviceInfo* d;
  if (int rc = current_device(&d)) return rc;
  const dim3 grid(static_cast<unsigned>((N + 63) / 64), static_cast<unsigned>((M + 63) / 64));
  if (grid.y > 65535) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "matmul_mxfp4: M=%lld is too large", (long long)M);
  const int tiles_k = static_cast<int>((K + 127) / 128);
  const auto *a = static_cast<const uint8_t*>(aq), *as = static_cast<const uint8_t*>(a_scale);
  const auto *b = static_cast<const uint8_t*>(bq), *bs = static_cast<const uint8_t*>(b_scale);
  if (out_dtype == SWIGLU_F32)
    matmul_mxfp4_kernel<float><<<grid, 256, 0, st>>>(a, as, b, bs, static_cast<float*>(c), (int)M, (int)N, (int)K,
                                                     tiles_k);
  else
    matmul_mxfp4_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a, as, b, bs, static_cast<__nv_bfloat16*>(c), (int)M,
                                                             (int)N, (int)K, tiles_k);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, "matmul_mxfp4 launch");
}

}  // namespace
}  // namespace swiglu

using namespace swiglu;

extern "C" {

int swiglu_b200_quantize_mxfp4(const void* src, void* dst, void* scale, int64_t rows, int64_t cols, int dtype,
                               void* stream) {
  return op_quantize(src, dst, scale, rows, cols, dtype, static_cast<cudaStream_t>(stream));
}

int swiglu_b200_dequantize_mxfp4(const void* q, const void* scale, void* dst, int64_t rows, int64_t cols, int dtype,
                                 void* stream) {
  return op_dequantize(q, scale, dst, rows, cols, dtype, static_cast<cudaStream_t>(stream));
}

int swiglu_b200_matmul_mxfp4(const void* aq, const void* a_scale, const void* bq, const void* b_scale, void* c,
                             int64_t M, int64_t N, int64_t K, int out_dtype, void* stream) {
  return op_matmul(aq, a_scale, bq, b_scale, c, M, N, K, out_dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
