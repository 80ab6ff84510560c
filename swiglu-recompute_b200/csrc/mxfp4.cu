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
#include "tc_mxfp4.cuh"

namespace swiglu {
namespace {

constexpr int kBlock = 32;          // columns that share a scale
constexpr int kTileRows = 128;
constexpr int kTileBytes = kMxTileBytes;
constexpr int kQuantCols = 256;     // columns of one CTA: a warp covers a row of them, 8 a thread
constexpr int kQuantThreads = 256;

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

// One CTA: 128 rows x 256 columns, two scale tiles. A warp takes a row at a time,
// 16 bytes a lane (bf16: all 256 columns, four lanes a block; f32: twice 128,
// eight lanes a block), several rows in flight; the scale bytes are collected in
// shared memory and leave as whole tiles, none is written alone.
template <typename T>
struct MxLanes {
  static constexpr int E = 16 / sizeof(T);             // elements of a lane
  static constexpr int GROUPS = kQuantCols / (32 * E); // loads that make the 256 columns
  static constexpr int LANES = kBlock / E;             // lanes that share a block
  static constexpr int BATCH = 8 / GROUPS;             // rows in flight
};

// |v| as an integer compares as |v|, and a NaN is above infinity: the exponent
// field of the largest of a lane's elements.
template <typename T>
__device__ __forceinline__ uint32_t top_exponent(const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m >> 23;
  } else {
    const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu),
                                __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16) >> 7;
  }
}

template <typename T>
__global__ void __launch_bounds__(kQuantThreads, 4) quantize_mxfp4_kernel(const T* __restrict__ src,
                                                                          uint8_t* __restrict__ dst,
                                                                          uint8_t* __restrict__ scale, long long rows,
                                                                          int cols, int tiles_k) {
  using L = MxLanes<T>;
  __shared__ __align__(16) uint8_t tile[2 * kTileBytes];
  const int lane = static_cast<int>(lane_id()), warp = static_cast<int>(warp_id());
  const long long r0 = blockIdx.y * static_cast<long long>(kTileRows) + warp;
  const int c0 = blockIdx.x * kQuantCols + lane * L::E;
  reinterpret_cast<uint32_t*>(tile)[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll 1
  for (int i0 = 0; i0 < 16 && r0 + i0 * 8 < rows; i0 += L::BATCH) {
    uint4 u[L::BATCH][L::GROUPS];
#pragma unroll
    for (int i = 0; i < L::BATCH; ++i) {
#pragma unroll
      for (int g = 0; g < L::GROUPS; ++g) {
        const long long r = r0 + (i0 + i) * 8;
        const int c = c0 + g * 32 * L::E;
        u[i][g] = make_uint4(0, 0, 0, 0);
        if (r < rows && c < cols) u[i][g] = __ldg(reinterpret_cast<const uint4*>(src + r * cols + c));
      }
    }
#pragma unroll
    for (int i = 0; i < L::BATCH; ++i) {
#pragma unroll
      for (int g = 0; g < L::GROUPS; ++g) {
        const long long r = r0 + (i0 + i) * 8;
        const int c = c0 + g * 32 * L::E;
        uint32_t field = top_exponent<T>(u[i][g]);  // 127 + floor(log2 max), 0 below the normals
#pragma unroll
        for (int o = 1; o < L::LANES; o *= 2) field = max(field, __shfl_xor_sync(0xffffffffu, field, o));
        if (r >= rows || c >= cols) continue;  // cols is a multiple of 32: a block is inside or not
        const int byte = field == 255 ? 255 : max(static_cast<int>(field) - 2, 0);
        const float inv = power_of_two(254 - min(byte, 253));
        const uint32_t w[4] = {u[i][g].x, u[i][g].y, u[i][g].z, u[i][g].w};
        uint32_t out = 0;
#pragma unroll
        for (int e = 0; e < L::E / 2; ++e) {
          float2 v;
          if constexpr (sizeof(T) == 4) v = make_float2(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
          else v = unpack_bf16x2(w[e]);
          const __nv_fp4x2_storage_t q =
              __nv_cvt_float2_to_fp4x2(make_float2(v.x * inv, v.y * inv), __NV_E2M1, cudaRoundNearest);
          out |= static_cast<uint32_t>(q) << (8 * e);
        }
        uint8_t* to = dst + r * (cols / 2) + c / 2;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(out);
        else *reinterpret_cast<uint32_t*>(to) = out;
        if (lane % L::LANES == 0) {
          const int b = (c - static_cast<int>(blockIdx.x) * kQuantCols) / kBlock;  // 0..7 of this CTA's blocks
          const int rt = (i0 + i) * 8 + warp;
          tile[(b >> 2) * kTileBytes + (rt & 31) * 16 + (rt >> 5) * 4 + (b & 3)] = static_cast<uint8_t>(byte);
        }
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
__global__ void __launch_bounds__(kQuantThreads, 4) dequantize_mxfp4_kernel(const uint8_t* __restrict__ src,
                                                                            const uint8_t* __restrict__ scale,
                                                                            T* __restrict__ dst, long long rows,
                                                                            int cols, int tiles_k) {
  using L = MxLanes<T>;
  __shared__ __align__(16) uint8_t tile[2 * kTileBytes];
  const int lane = static_cast<int>(lane_id()), warp = static_cast<int>(warp_id());
  const long long r0 = blockIdx.y * static_cast<long long>(kTileRows) + warp;
  const int c0 = blockIdx.x * kQuantCols + lane * L::E;
  const int t = 2 * blockIdx.x + (threadIdx.x >> 5);
  if (threadIdx.x < 64 && t < tiles_k) {
    const uint8_t* from = scale + (blockIdx.y * static_cast<long long>(tiles_k) + t) * kTileBytes;
    reinterpret_cast<uint4*>(tile)[threadIdx.x] = __ldg(reinterpret_cast<const uint4*>(from) + (threadIdx.x & 31));
  }
  uint32_t q[16][L::GROUPS];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int g = 0; g < L::GROUPS; ++g) {
      const long long r = r0 + i * 8;
      const int c = c0 + g * 32 * L::E;
      if (r < rows && c < cols) {
        const uint8_t* from = src + r * (cols / 2) + c / 2;
        if constexpr (sizeof(T) == 4) q[i][g] = __ldg(reinterpret_cast<const uint16_t*>(from));
        else q[i][g] = __ldg(reinterpret_cast<const uint32_t*>(from));
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int g = 0; g < L::GROUPS; ++g) {
      const long long r = r0 + i * 8;
      const int c = c0 + g * 32 * L::E;
      if (r >= rows || c >= cols) continue;
      const int b = (c - static_cast<int>(blockIdx.x) * kQuantCols) / kBlock, rt = i * 8 + warp;
      const float s = scale_value(tile[(b >> 2) * kTileBytes + (rt & 31) * 16 + (rt >> 5) * 4 + (b & 3)]);
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < L::E / 2; ++e) {
        const float2 v = e2m1x2_value((q[i][g] >> (8 * e)) & 0xffu);
        if constexpr (sizeof(T) == 4) {
          w[2 * e] = __float_as_uint(v.x * s);
          w[2 * e + 1] = __float_as_uint(v.y * s);
        } else {
          w[e] = pack_bf16x2(v.x * s, v.y * s);
        }
      }
      *reinterpret_cast<uint4*>(dst + r * cols + c) = make_uint4(w[0], w[1], w[2], w[3]);
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

// Scale tiles as rows of 32-bit cells, one row per 128 rows of the matrix; a
// box is the two tiles of a stage.
int make_map_scales(CUtensorMap* m, const void* ptr, int64_t rows, int64_t K, const char* what) {
  EncodeTiledFn fn;
  if (int rc = get_encode_fn(&fn)) return rc;
  const cuuint64_t tiles_k = static_cast<cuuint64_t>((K + 127) / 128);
  const cuuint64_t dims[2] = {tiles_k * (kMxTileBytes / 4), static_cast<cuuint64_t>((rows + 127) / 128)};
  const cuuint64_t strides[1] = {tiles_k * kMxTileBytes};
  const cuuint32_t box[2] = {kMxScaleBytes / 4, 1};
  const cuuint32_t es[2] = {1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(ptr), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SWIGLU_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (CUresult %d)", what, (int)r);
  return SWIGLU_OK;
}

// How a product runs: on 256 x 256 pair tiles, or on 128 x nt tiles with
// clusters of `parts` CTAs along K.
struct MxPlan {
  bool pair;
  int nt, parts;
};

// Times in us, fitted to measurements of every form on one B200 (148 SMs) over
// 40 shapes (M 1..4096, N 128..28672, K 512..28672), most within 15 %:
//   pair     5.2 + rounds * (0.37 a k-block + 1)
//   cluster  per wave of two CTAs an SM, start and end, 0.35..0.43 a k-block of
//            a CTA (half as much again while two share an SM), and the join
// e.g. 256 x 3584 x 3584: pair 10.6, 128 columns on one CTA 12.6, on two 10.6;
// 333 x 1000 x 14336: pair 24.3, 128 on one 29.2, on four 12.6, on eight 12.4;
// 1024 x 3584 x 3584: pair 11.0, 128 on one 15.3; 1 x 3584 x 14336: 16 columns
// on one CTA 23.0, on two 14.3, on four 10.1, on eight 9.5.
MxPlan plan_matmul(int64_t M, int64_t N, int64_t K, int sms) {
  struct Width {
    int nt;
    float start, block, join[4];  // join: 1, 2, 4, 8 CTAs
  };
  constexpr Width kWidths[] = {{16, 3.3f, 0.345f, {0.0f, 0.7f, 1.2f, 2.2f}},
                               {32, 3.6f, 0.355f, {0.0f, 1.0f, 1.6f, 3.0f}},
                               {64, 4.4f, 0.36f, {0.0f, 1.5f, 2.4f, 4.4f}},
                               {128, 6.0f, 0.43f, {0.0f, 1.5f, 2.4f, 4.4f}}};
  const int64_t num_kb = (K + kMxStageK - 1) / kMxStageK, tiles_w = (N + 127) / 128;
  MxPlan best{true, 256, 1};
  const int64_t pairs = sms / 2;
  const int64_t rounds = ((M + 255) / 256 * ((N + 255) / 256) + pairs - 1) / pairs;
  float best_us = 4.2f + static_cast<float>(rounds) * (0.37f * static_cast<float>(num_kb) + 1.0f);
  if (M <= 64) best_us = 1e30f;  // three quarters of a pair tile would be padding
  for (const Width& w : kWidths) {
    // A narrow tile holds all rows: a second one would start inside a scale tile.
    if (w.nt < 128 && M > w.nt) continue;
    const int64_t tiles = tiles_w * ((M + w.nt - 1) / w.nt);
    for (int i = 0, parts = 1; i < 4 && parts <= num_kb; ++i, parts *= 2) {
      const int64_t ctas = tiles * parts, waves = (ctas + 2 * sms - 1) / (2 * sms);
      const float blocks = static_cast<float>((num_kb + parts - 1) / parts) * (ctas > sms ? 1.5f : 1.0f);
      const float us = static_cast<float>(waves) * (w.start + w.block * blocks + w.join[i]);
      if (us < best_us) {
        best_us = us;
        best = MxPlan{false, w.nt, parts};
      }
    }
  }
  return best;
}

int usable_sms(const DeviceInfo& d) {
  const int sms = d.sms - sm_reserve();
  return sms < 2 ? 2 : sms;
}

template <int NT, bool F32>
int launch_cluster(const MxClusterParams& p, const MxPlan& plan, cudaStream_t st) {
  using Cfg = MxClusterCfg<NT, F32>;
  constexpr auto kern = mx_gemm_cluster_kernel<Cfg>;
  KernelState& ks = kernel_state<kern>();
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(ks.ready.load() & (1ull << dev))) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
    if (e != cudaSuccess) return cuda_fail(e, "matmul_mxfp4 launch");
    ks.ready.fetch_or(1ull << dev);
  }
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = pair_launch_config(attr, Cfg::NUM_THREADS, Cfg::SMEM_BYTES, st);
  attr[0].val.clusterDim.x = plan.parts;
  cfg.gridDim = dim3(static_cast<unsigned>((p.N + 127) / 128 * p.tiles_x * plan.parts));
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, "matmul_mxfp4 launch");
}

template <bool F32>
int run_cluster(MxClusterParams& p, const MxPlan& plan, cudaStream_t st) {
  switch (plan.nt) {
    case 16: return launch_cluster<16, F32>(p, plan, st);
    case 32: return launch_cluster<32, F32>(p, plan, st);
    case 64: return launch_cluster<64, F32>(p, plan, st);
    default: return launch_cluster<128, F32>(p, plan, st);
  }
}

template <bool F32>
int run_pair(MxParams& p, const DeviceInfo& d, cudaStream_t st) {
  using Cfg = MxCfg<F32>;
  return launch_pair<mx_gemm_pair_kernel<Cfg>>(p, p.tiles_m * p.tiles_n, Cfg::NUM_THREADS, Cfg::SMEM_BYTES, d, st,
                                               "matmul_mxfp4 launch");
}

int check_matmul(int64_t M, int64_t N, int64_t K) {
  if (int rc = check_mx("matmul_mxfp4", M, K)) return rc;
  if (int rc = check_mx("matmul_mxfp4", N, K)) return rc;
  if (K <= 0) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "K must be positive");
  if (int rc = check_mult8("N", N)) return rc;
  if (((M + 255) / 256) * ((N + 255) / 256) > 0x7fffffff)
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "matmul_mxfp4: M=%lld, N=%lld make too many tiles", (long long)M,
                (long long)N);
  return SWIGLU_OK;
}

int op_matmul(const void* aq, const void* a_scale, const void* bq, const void* b_scale, void* c, int64_t M, int64_t N,
              int64_t K, int out_dtype, cudaStream_t st) {
  if (int rc = check_matmul(M, N, K)) return rc;
  if (int rc = check_dtype(out_dtype)) return rc;
  if (M == 0 || N == 0) return SWIGLU_OK;
  if (!aq || !a_scale || !bq || !b_scale || !c) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned16(aq) || !aligned16(a_scale) || !aligned16(bq) || !aligned16(b_scale) || !aligned16(c))
    return fail(SWIGLU_ERR_MISALIGNED, "matmul_mxfp4: pointers must be 16-byte aligned");
  DeviceInfo* d;
  if (int rc = current_device(&d)) return rc;
  const bool f32 = out_dtype == SWIGLU_F32;
  const MxPlan plan = plan_matmul(M, N, K, usable_sms(*d));
  if (!plan.pair) {
    MxClusterParams p{};
    if (int rc = make_map_bytes(&p.tmW, bq, K / 2, N, K / 2, 128, "B (MXFP4)")) return rc;
    if (int rc = make_map_bytes(&p.tmX, aq, K / 2, M, K / 2, plan.nt, "A (MXFP4)")) return rc;
    if (int rc = make_map_scales(&p.tmWs, b_scale, N, K, "B scales")) return rc;
    if (int rc = make_map_scales(&p.tmXs, a_scale, M, K, "A scales")) return rc;
    p.out = c;
    p.M = (int)M, p.N = (int)N, p.K = (int)K;
    p.tiles_x = (int)((M + plan.nt - 1) / plan.nt);
    p.status = d->status;
    return f32 ? run_cluster<true>(p, plan, st) : run_cluster<false>(p, plan, st);
  }
  MxParams p{};
  if (int rc = make_map_bytes(&p.tmA, aq, K / 2, M, K / 2, 128, "A (MXFP4)")) return rc;
  if (int rc = make_map_bytes(&p.tmB, bq, K / 2, N, K / 2, 128, "B (MXFP4)")) return rc;
  if (int rc = make_map_scales(&p.tmAs, a_scale, M, K, "A scales")) return rc;
  if (int rc = make_map_scales(&p.tmBs, b_scale, N, K, "B scales")) return rc;
  if (int rc = make_store_map(&p.tmC, c, N, M, N, f32)) return rc;
  p.M = (int)M, p.N = (int)N, p.K = (int)K;
  p.tiles_m = (int)((M + 255) / 256), p.tiles_n = (int)((N + 255) / 256);
  p.group_m = 16;
  p.status = d->status;
  return f32 ? run_pair<true>(p, *d, st) : run_pair<false>(p, *d, st);
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
