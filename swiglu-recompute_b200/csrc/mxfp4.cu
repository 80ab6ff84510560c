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
constexpr int kQuantRows = 64;      // and its rows
constexpr int kQuantThreads = 256;

__device__ __forceinline__ float power_of_two(int field) { return __uint_as_float(static_cast<uint32_t>(field) << 23); }

// 2^(byte - 127) as two bf16: byte 0 is the subnormal 2^-127, byte 255 a NaN.
__device__ __forceinline__ uint32_t scale_bf16x2(uint32_t byte) {
  const uint32_t s = byte == 0 ? 0x0040u : byte == 255 ? 0x7fc0u : byte << 7;
  return s | (s << 16);
}

// Eight e2m1 codes as bf16 pairs: the seven bits above the sign of a code's value
// are looked up by byte permutation (two tables of eight bytes), which takes half
// the instructions of converting through f16 and f32.
__device__ __forceinline__ void e2m1x8_bf16(uint32_t codes, uint32_t (&out)[4]) {
  constexpr uint32_t kHigh0 = 0x3f3f3f00u, kHigh1 = 0x40404040u;  // 0 0.5 1 1.5 | 2 3 4 6
  constexpr uint32_t kLow0 = 0xc0800000u, kLow1 = 0xc0804000u;
  const uint32_t sel = codes & 0x77777777u;
  const uint32_t even = (codes << 4) & 0x80808080u, odd = codes & 0x80808080u;  // sign bits of codes 0 2 4 6, 1 3 5 7
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // codes 4h .. 4h + 3
    const uint32_t pick = h ? sel >> 16 : sel;
    const uint32_t high = __byte_perm(kHigh0, kHigh1, pick) | __byte_perm(even, odd, h ? 0x7362 : 0x5140);
    const uint32_t low = __byte_perm(kLow0, kLow1, pick);
    out[2 * h] = __byte_perm(low, high, 0x5140);
    out[2 * h + 1] = __byte_perm(low, high, 0x7362);
  }
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// One CTA: 64 rows x 256 columns, half of two scale tiles (whole tiles left 13 % of
// the last round of CTAs idle at 28672 x 3584). A warp takes a row at a time, 16
// bytes a lane (bf16: all 256 columns, four lanes a block; f32: twice 128, eight
// lanes a block), several rows in flight; the scale bytes are collected in shared
// memory and leave eight at a time.
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

// Where a CTA works, and its scale bytes: [tile of two][row % 32][row / 32 of two][block].
struct QuantBlock {
  long long r0;   // first row
  int c0, warp, lane;
  long long tile; // first scale tile
  int half;       // which two of the tile's four groups of 32 rows
  int tiles;      // scale tiles inside the matrix: 1 or 2

  __device__ __forceinline__ QuantBlock(int cols, int tiles_k) {
    const int col_blocks = (cols + kQuantCols - 1) / kQuantCols;
    const long long rb = blockIdx.x / col_blocks;
    const int cb = static_cast<int>(blockIdx.x % col_blocks);
    r0 = rb * kQuantRows;
    c0 = cb * kQuantCols;
    warp = static_cast<int>(warp_id());
    lane = static_cast<int>(lane_id());
    tile = rb / 2 * tiles_k + 2 * cb;
    half = static_cast<int>(rb % 2);
    tiles = min(2, tiles_k - 2 * cb);
  }
  __device__ __forceinline__ static int byte_of(int row, int block) {
    return (block >> 2) * 256 + (row & 31) * 8 + (row >> 5) * 4 + (block & 3);
  }
  // Thread t < 32 * tiles moves eight bytes of tile t / 32.
  __device__ __forceinline__ long long at() const {
    return (tile + (threadIdx.x >> 5)) * kTileBytes + (threadIdx.x & 31) * 16 + half * 8;
  }
};

template <typename T, bool WHOLE>
__device__ __forceinline__ void quantize_rows(const QuantBlock& q, const T* src, uint8_t* dst, uint8_t* bytes,
                                              long long rows, int cols) {
  using L = MxLanes<T>;
  const long long r0 = q.r0 + q.warp, at0 = r0 * cols + q.c0 + q.lane * L::E;
  const long long step = 8ll * cols;
#pragma unroll 1
  for (int i0 = 0; i0 < 8; i0 += L::BATCH) {
    uint4 u[L::BATCH][L::GROUPS];
#pragma unroll
    for (int i = 0; i < L::BATCH; ++i) {
#pragma unroll
      for (int g = 0; g < L::GROUPS; ++g) {
        const bool in = WHOLE || (r0 + (i0 + i) * 8 < rows && q.c0 + (g * 32 + q.lane) * L::E < cols);
        u[i][g] = make_uint4(0, 0, 0, 0);
        // Read once: f32 with the streaming hint 69.0 us at 28672 x 3584, without 70.3;
        // bf16 47.1 and 42.4.
        const uint4* from = reinterpret_cast<const uint4*>(src + at0 + (i0 + i) * step + g * 32 * L::E);
        if (in) u[i][g] = sizeof(T) == 4 ? __ldcs(from) : *from;
      }
    }
#pragma unroll
    for (int i = 0; i < L::BATCH; ++i) {
#pragma unroll
      for (int g = 0; g < L::GROUPS; ++g) {
        uint32_t field = top_exponent<T>(u[i][g]);  // 127 + floor(log2 max), 0 below the normals
#pragma unroll
        for (int o = 1; o < L::LANES; o *= 2) field = max(field, __shfl_xor_sync(0xffffffffu, field, o));
        // cols is a multiple of 32: a block is inside or not
        if (!WHOLE && !(r0 + (i0 + i) * 8 < rows && q.c0 + (g * 32 + q.lane) * L::E < cols)) continue;
        const int byte = field == 255 ? 255 : max(static_cast<int>(field) - 2, 0);
        const float inv = power_of_two(254 - min(byte, 253));
        const uint32_t w[4] = {u[i][g].x, u[i][g].y, u[i][g].z, u[i][g].w};
        uint32_t out = 0;
#pragma unroll
        for (int e = 0; e < L::E / 2; ++e) {
          float2 v;
          if constexpr (sizeof(T) == 4) v = make_float2(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
          else v = unpack_bf16x2(w[e]);
          const __nv_fp4x2_storage_t code =
              __nv_cvt_float2_to_fp4x2(__fmul2_rn(v, make_float2(inv, inv)), __NV_E2M1, cudaRoundNearest);
          out |= static_cast<uint32_t>(code) << (8 * e);
        }
        uint8_t* to = dst + (at0 + (i0 + i) * step + g * 32 * L::E) / 2;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(out);
        else *reinterpret_cast<uint32_t*>(to) = out;
        if (q.lane % L::LANES == 0)
          bytes[QuantBlock::byte_of((i0 + i) * 8 + q.warp, (g * 32 + q.lane) / L::LANES)] = static_cast<uint8_t>(byte);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kQuantThreads, 4) quantize_mxfp4_kernel(const T* src, uint8_t* dst,
                                                                          uint8_t* scale, long long rows, int cols,
                                                                          int tiles_k) {
  wait_for_previous();
  __shared__ __align__(16) uint8_t bytes[512];
  const QuantBlock q(cols, tiles_k);
  if (threadIdx.x < 128) reinterpret_cast<uint32_t*>(bytes)[threadIdx.x] = 0;
  __syncthreads();
  // Blocks wholly inside the matrix skip the checks.
  if (q.r0 + kQuantRows <= rows && q.c0 + kQuantCols <= cols)
    quantize_rows<T, true>(q, src, dst, bytes, rows, cols);
  else
    quantize_rows<T, false>(q, src, dst, bytes, rows, cols);
  __syncthreads();
  if (threadIdx.x < 32 * q.tiles)
    *reinterpret_cast<uint2*>(scale + q.at()) = reinterpret_cast<const uint2*>(bytes)[threadIdx.x];
}

template <typename T, bool WHOLE>
__device__ __forceinline__ void dequantize_rows(const QuantBlock& q, const uint8_t* src, uint2 tile, uint8_t* bytes,
                                                T* dst, long long rows, int cols) {
  using L = MxLanes<T>;
  const long long r0 = q.r0 + q.warp, at0 = r0 * cols + q.c0 + q.lane * L::E;
  const long long step = 8ll * cols;
  uint32_t codes[8][L::GROUPS];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int g = 0; g < L::GROUPS; ++g) {
      if (!WHOLE && !(r0 + i * 8 < rows && q.c0 + (g * 32 + q.lane) * L::E < cols)) continue;
      const uint8_t* from = src + (at0 + i * step + g * 32 * L::E) / 2;
      if constexpr (sizeof(T) == 4) codes[i][g] = __ldcs(reinterpret_cast<const uint16_t*>(from));
      else codes[i][g] = __ldcs(reinterpret_cast<const uint32_t*>(from));
    }
  }
  if (threadIdx.x < 64) reinterpret_cast<uint2*>(bytes)[threadIdx.x] = tile;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int g = 0; g < L::GROUPS; ++g) {
      if (!WHOLE && !(r0 + i * 8 < rows && q.c0 + (g * 32 + q.lane) * L::E < cols)) continue;
      const uint32_t s = scale_bf16x2(bytes[QuantBlock::byte_of(i * 8 + q.warp, (g * 32 + q.lane) / L::LANES)]);
      uint32_t w[4];
      e2m1x8_bf16(codes[i][g], w);
      if constexpr (sizeof(T) == 4) {  // four codes
        const uint32_t a = mul_bf16x2(w[0], s), b = mul_bf16x2(w[1], s);
        w[0] = a << 16, w[1] = a & 0xffff0000u, w[2] = b << 16, w[3] = b & 0xffff0000u;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = mul_bf16x2(w[e], s);
      }
      *reinterpret_cast<uint4*>(dst + at0 + i * step + g * 32 * L::E) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// Five blocks an SM for bf16: at four (50 registers) 28672 x 3584 takes 47.3 us
// instead of 42.4. f32 needs its 64 registers.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 2 ? 5 : 4)
    dequantize_mxfp4_kernel(const uint8_t* src, const uint8_t* scale, T* dst, long long rows, int cols, int tiles_k) {
  wait_for_previous();
  __shared__ __align__(16) uint8_t bytes[512];
  const QuantBlock q(cols, tiles_k);
  uint2 tile = make_uint2(0, 0);
  if (threadIdx.x < 32 * q.tiles) tile = *reinterpret_cast<const uint2*>(scale + q.at());
  if (q.r0 + kQuantRows <= rows && q.c0 + kQuantCols <= cols)
    dequantize_rows<T, true>(q, src, tile, bytes, dst, rows, cols);
  else
    dequantize_rows<T, false>(q, src, tile, bytes, dst, rows, cols);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// The kernels round rows and columns up to whole tiles (256 at most) in ints.
constexpr int64_t kMaxDim = 0x7fffffffLL - 255;

int check_mx(const char* what, int64_t rows, int64_t cols) {
  if (int rc = check_dims(what, rows, cols, 0)) return rc;
  if (rows > kMaxDim || cols > kMaxDim)
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "%s: at most %lld rows and columns", what, (long long)kMaxDim);
  if (cols % kBlock)
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "%s: %lld columns are not a multiple of 32", what, (long long)cols);
  const int64_t blocks = (rows + kQuantRows - 1) / kQuantRows * ((cols + kQuantCols - 1) / kQuantCols);
  if (blocks > 0x7ffffffe) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "%s: the matrix is too large", what);
  return SWIGLU_OK;
}

// Whole scale tiles: an even number of row blocks, so that the bytes of rows
// beyond the matrix are written too.
unsigned quant_grid(int64_t rows, int64_t cols) {
  return static_cast<unsigned>((rows + kTileRows - 1) / kTileRows * 2 * ((cols + kQuantCols - 1) / kQuantCols));
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
  const auto to = static_cast<uint8_t*>(dst), scales = static_cast<uint8_t*>(scale);
  const unsigned grid = quant_grid(rows, cols);
  const int k = static_cast<int>(cols);
  if (dtype == SWIGLU_F32)
    launch_after(quantize_mxfp4_kernel<float>, grid, kQuantThreads, 0, st, static_cast<const float*>(src), to, scales,
                 rows, k, tiles_k);
  else
    launch_after(quantize_mxfp4_kernel<__nv_bfloat16>, grid, kQuantThreads, 0, st,
                 static_cast<const __nv_bfloat16*>(src), to, scales, rows, k, tiles_k);
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
  const auto codes = static_cast<const uint8_t*>(q), scales = static_cast<const uint8_t*>(scale);
  const unsigned grid = quant_grid(rows, cols);
  const int k = static_cast<int>(cols);
  if (dtype == SWIGLU_F32)
    launch_after(dequantize_mxfp4_kernel<float>, grid, kQuantThreads, 0, st, codes, scales, static_cast<float*>(dst),
                 rows, k, tiles_k);
  else
    launch_after(dequantize_mxfp4_kernel<__nv_bfloat16>, grid, kQuantThreads, 0, st, codes, scales,
                 static_cast<__nv_bfloat16*>(dst), rows, k, tiles_k);
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
//   pair     4.2 + rounds * (0.37 a k-block + 1)
//   cluster  per wave of two CTAs an SM, start and end, 0.35..0.43 a k-block of
//            a CTA (half as much again while two share an SM), and the join
// Measured, e.g. 256 x 3584 x 3584: pair 10.6, 128 columns on one CTA 12.6, on two 10.6;
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

// The second launch attribute of a cluster kernel that begins with
// wait_for_previous().
void after_previous(cudaLaunchAttribute* attr, cudaLaunchConfig_t& cfg) {
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
}

template <int NT, bool F32>
int launch_cluster(const MxClusterParams& p, const MxPlan& plan, cudaStream_t st) {
  using Cfg = MxClusterCfg<NT, F32>;
  constexpr auto kern = mx_gemm_cluster_kernel<Cfg>;
  if (int rc = opt_in_smem<kern>(Cfg::SMEM_BYTES, "matmul_mxfp4 launch")) return rc;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = pair_launch_config(attr, Cfg::NUM_THREADS, Cfg::SMEM_BYTES, st);
  attr[0].val.clusterDim.x = plan.parts;
  after_previous(attr, cfg);
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

template <class Cfg>
int run_pair(MxParams& p, const DeviceInfo& d, cudaStream_t st) {
  constexpr auto kern = mx_gemm_pair_kernel<Cfg>;
  int cap = 0;
  if (int rc = pair_capacity<kern>(Cfg::NUM_THREADS, Cfg::SMEM_BYTES, d, &cap, "matmul_mxfp4 launch")) return rc;
  const int tiles = p.tiles_m * p.tiles_n;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = pair_launch_config(attr, Cfg::NUM_THREADS, Cfg::SMEM_BYTES, st);
  cfg.gridDim = dim3(2 * (tiles < cap ? tiles : cap));
  after_previous(attr, cfg);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, "matmul_mxfp4 launch");
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
  return f32 ? run_pair<MxCfg<true>>(p, *d, st) : run_pair<MxCfg<false>>(p, *d, st);
}

// Whether GEMM1 + SwiGLU runs as one launch: where its product takes pair tiles.
bool swiglu_fused(int64_t M, int64_t K, int64_t H, int sms) { return plan_matmul(M, 2 * H, K, sms).pair; }

int check_swiglu(int64_t M, int64_t K, int64_t H, int layout) {
  if (int rc = check_dims("fused_matmul_swiglu_mxfp4", M, K, H)) return rc;
  if (layout != SWIGLU_LAYOUT_STD && layout != SWIGLU_LAYOUT_PACKED128)
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "unknown layout %d", layout);
  if (H <= 0 || H % 128)
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "H=%lld must be a positive multiple of 128", (long long)H);
  return check_matmul(M, 2 * H, K);
}

int op_swiglu(const void* xq, const void* x_scale, const void* wq, const void* w_scale, void* preact, void* h,
              int64_t M, int64_t K, int64_t H, int layout, cudaStream_t st) {
  if (int rc = check_swiglu(M, K, H, layout)) return rc;
  if (M == 0) return SWIGLU_OK;
  if (!xq || !x_scale || !wq || !w_scale || (!preact && !h)) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned16(xq) || !aligned16(x_scale) || !aligned16(wq) || !aligned16(w_scale) || !aligned16(preact) ||
      !aligned16(h))
    return fail(SWIGLU_ERR_MISALIGNED, "fused_matmul_swiglu_mxfp4: pointers must be 16-byte aligned");
  DeviceInfo* d;
  if (int rc = current_device(&d)) return rc;
  if (!swiglu_fused(M, K, H, usable_sms(*d))) {
    if (!preact)
      return fail(SWIGLU_ERR_INVALID_ARGUMENT, "fused_matmul_swiglu_mxfp4: this size needs preact (see the plan query)");
    if (int rc = op_matmul(xq, x_scale, wq, w_scale, preact, M, 2 * H, K, SWIGLU_BF16, st)) return rc;
    return h ? swiglu_b200_forward_logic(preact, h, M, H, SWIGLU_BF16, layout, st) : SWIGLU_OK;
  }
  MxParams p{};
  if (int rc = make_map_bytes(&p.tmA, xq, K / 2, M, K / 2, 128, "x (MXFP4)")) return rc;
  if (int rc = make_map_bytes(&p.tmB, wq, K / 2, 2 * H, K / 2, 128, "W1 (MXFP4)")) return rc;
  if (int rc = make_map_scales(&p.tmAs, x_scale, M, K, "x scales")) return rc;
  if (int rc = make_map_scales(&p.tmBs, w_scale, 2 * H, K, "W1 scales")) return rc;
  if (preact) {
    if (int rc = make_store_map(&p.tmC, preact, 2 * H, M, 2 * H, false)) return rc;
  }
  if (h) {
    if (int rc = make_store_map(&p.tmD, h, H, M, H, false)) return rc;
  }
  p.M = (int)M, p.N = (int)(2 * H), p.K = (int)K, p.H = (int)H, p.layout = layout;
  p.store_preact = preact != nullptr, p.store_h = h != nullptr;
  p.tiles_m = (int)((M + 255) / 256), p.tiles_n = (int)(H / 128);
  p.group_m = 16;
  p.status = d->status;
  return run_pair<MxCfg<false, true>>(p, *d, st);
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

int swiglu_b200_fused_matmul_swiglu_mxfp4_plan(int64_t M, int64_t K, int64_t H, int num_sms, int* fused) {
  if (int rc = check_swiglu(M, K, H, SWIGLU_LAYOUT_STD)) return rc;
  if (!fused) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  if (num_sms < 1) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "num_sms must be positive");
  const int sms = num_sms - sm_reserve();
  *fused = swiglu_fused(M, K, H, sms < 2 ? 2 : sms) ? 1 : 0;
  return SWIGLU_OK;
}

int swiglu_b200_fused_matmul_swiglu_mxfp4(const void* xq, const void* x_scale, const void* w1q, const void* w1_scale,
                                          void* preact, void* h, int64_t M, int64_t K, int64_t H, int layout,
                                          void* stream) {
  return op_swiglu(xq, x_scale, w1q, w1_scale, preact, h, M, K, H, layout, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
