// Residual RMS norm in front of the SwiGLU block, and its gradient.
//
//   s = x + residual (rounded to the stream's type and stored), or s = x
//   rstd = (mean_j s_j^2 + eps)^(-1/2)
//   y = s * rstd * weight                                     (stream's type)
//   or e4m3: A = max_j |s_j w_j|, q_j = e4m3(s_j w_j * 448 / A),
//            scale = A * rstd / 448
//
// In the e4m3 form rstd cancels inside q, so the row's maximum is taken over
// s w together with the sum of squares: one statistics pass instead of two.
//
//   g = dy * weight
//   dx = rstd * (g - s * rstd^2 * mean_j(g_j s_j)) + ds
//   dweight_j = sum over rows of dy_j s_j rstd
//
// Statistics, products and sums are f32; each output is rounded once. s is
// rounded before its statistics are taken, so that forward and backward (which
// reads the stored s) see the same stream.
#include "host.cuh"
#include "ptx.cuh"

namespace swiglu {
namespace {

constexpr float kE4m3Max = 448.0f;

// 16 bytes of T as f32.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
};

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& u, float (&f)[Vec<T>::N]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(w[i]);
    } else {
      const float2 v = unpack_bf16x2(w[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&f)[Vec<T>::N]) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else return __float2bfloat16_rn(v);
}

__device__ __forceinline__ uint8_t e4m3_byte(float v) { return static_cast<uint8_t>(e4m3x2(v, 0.0f) & 0xffu); }

// Sum and maximum over the threads that share a row: one warp, or the block.
// Every thread gets the result; the order of the sum is fixed.
__device__ __forceinline__ void row_reduce(float& sum, float& top, int warps, float2* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (warps == 1) return;
  const int lane = static_cast<int>(lane_id()), warp = static_cast<int>(warp_id());
  if (lane == 0) scratch[warp] = make_float2(sum, top);
  __syncthreads();
  const float2 v = lane < warps ? scratch[lane] : make_float2(0.0f, 0.0f);
  sum = v.x;
  top = v.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
}

struct FwdParams {
  const void* x;
  const void* residual;  // may be null
  const void* weight;
  void* y;               // stream's type, or e4m3 bytes
  float* row_scale;      // e4m3 only
  void* s;               // written when residual is given
  float* rstd;
  long long rows;
  int cols;
  float eps;
};

// Row factors from the statistics: rstd, the factor that takes s w to e4m3
// (clamped, so that a row of tiny values gives 0 * finite and not 0 * inf),
// and the stored scale: 1 for an all-zero row, NaN where the row holds one.
__device__ __forceinline__ void row_factors(float sum, float top, const FwdParams& p, float& rstd, float& qs,
                                            float& scale) {
  rstd = rsqrtf(sum / static_cast<float>(p.cols) + p.eps);
  qs = top > 0.0f ? fminf(kE4m3Max / top, 3.4028234e38f) : 1.0f;
  scale = top > 0.0f ? top * rstd / kE4m3Max : (rstd == rstd ? 1.0f : rstd);
}

// Any width and alignment: a block per row, one element per thread at a time;
// the second pass reads the row (or the s just written by the same thread)
// again from L1 / L2.
template <typename T, typename W, bool E4M3>
__global__ void __launch_bounds__(512) rmsnorm_fwd_any_kernel(const FwdParams p) {
  __shared__ float2 scratch[16];
  const long long base = blockIdx.x * static_cast<long long>(p.cols);
  const T* x = static_cast<const T*>(p.x) + base;
  const T* r = p.residual ? static_cast<const T*>(p.residual) + base : nullptr;
  T* s = static_cast<T*>(p.s) + base;
  const W* w = static_cast<const W*>(p.weight);
  float sum = 0.0f, top = 0.0f;
  for (int j = threadIdx.x; j < p.cols; j += blockDim.x) {
    float v = to_f32(x[j]);
    if (r) {
      const T t = from_f32<T>(v + to_f32(r[j]));
      s[j] = t;
      v = to_f32(t);
    }
    sum += v * v;
    if constexpr (E4M3) top = fmaxf(top, fabsf(v * to_f32(w[j])));
  }
  row_reduce(sum, top, blockDim.x >> 5, scratch);
  float rstd, qs, scale;
  row_factors(sum, top, p, rstd, qs, scale);
  if (threadIdx.x == 0) {
    p.rstd[blockIdx.x] = rstd;
    if constexpr (E4M3) p.row_scale[blockIdx.x] = scale;
  }
  const T* src = r ? s : x;
  for (int j = threadIdx.x; j < p.cols; j += blockDim.x) {
    const float v = to_f32(src[j]), f = to_f32(w[j]);
    if constexpr (E4M3) static_cast<uint8_t*>(p.y)[base + j] = e4m3_byte(v * f * qs);
    else static_cast<T*>(p.y)[base + j] = from_f32<T>(v * rstd * f);
  }
}

struct BwdParams {
  const void* dy;
  const void* s;
  const void* weight;
  const float* rstd;
  const void* ds;     // may be null
  void* dx;
  float* dot;         // [rows]: sum_j g_j s_j
  float* partial;     // [chunks, cols]
  void* dweight;
  long long rows;
  int cols;
  int chunks;         // row chunks of the column pass
  int rows_per_chunk;
};

// dot_r = sum_j dy_j w_j s_j, a block per row.
template <typename T, typename W>
__global__ void __launch_bounds__(512) rmsnorm_bwd_dot_kernel(const BwdParams p) {
  __shared__ float2 scratch[16];
  const long long base = blockIdx.x * static_cast<long long>(p.cols);
  const T* dy = static_cast<const T*>(p.dy) + base;
  const T* s = static_cast<const T*>(p.s) + base;
  const W* w = static_cast<const W*>(p.weight);
  float sum = 0.0f, top = 0.0f;
  for (int j = threadIdx.x; j < p.cols; j += blockDim.x) sum += to_f32(dy[j]) * to_f32(w[j]) * to_f32(s[j]);
  row_reduce(sum, top, blockDim.x >> 5, scratch);
  if (threadIdx.x == 0) p.dot[blockIdx.x] = sum;
}

// A thread per column walks a chunk of rows: dx, and its part of dweight.
template <typename T, typename W>
__global__ void __launch_bounds__(256) rmsnorm_bwd_cols_kernel(const BwdParams p) {
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= p.cols) return;
  const float w = to_f32(static_cast<const W*>(p.weight)[j]);
  const float inv = 1.0f / static_cast<float>(p.cols);
  const long long r0 = blockIdx.y * static_cast<long long>(p.rows_per_chunk);
  const long long r1 = min(r0 + p.rows_per_chunk, p.rows);
  float acc = 0.0f;
  for (long long r = r0; r < r1; ++r) {
    const long long at = r * p.cols + j;
    const float dy = to_f32(static_cast<const T*>(p.dy)[at]), s = to_f32(static_cast<const T*>(p.s)[at]);
    const float rstd = p.rstd[r];
    const float c = p.dot[r] * inv * rstd * rstd;
    float dx = rstd * (dy * w - s * c);
    if (p.ds) dx += to_f32(static_cast<const T*>(p.ds)[at]);
    static_cast<T*>(p.dx)[at] = from_f32<T>(dx);
    acc += dy * s * rstd;
  }
  p.partial[blockIdx.y * static_cast<long long>(p.cols) + j] = acc;
}

// dweight = sum of the chunks' parts, in a fixed order: 32 columns a block,
// 32 threads along the chunks of each.
template <typename W>
__global__ void __launch_bounds__(1024) rmsnorm_dweight_kernel(const float* partial, W* dweight, int cols, int chunks) {
  __shared__ float part[32][33];
  const int j = blockIdx.x * 32 + threadIdx.x;
  float acc = 0.0f;
  if (j < cols) {
    for (int c = threadIdx.y; c < chunks; c += 32) acc += partial[c * static_cast<long long>(cols) + j];
  }
  part[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  acc = part[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  const int k = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && k < cols) dweight[k] = from_f32<W>(acc);
}

int check_norm(const char* what, int64_t rows, int64_t cols, int dtype, int weight_dtype) {
  if (int rc = check_dims(what, rows, cols, 0)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_dtype(weight_dtype)) return rc;
  if (cols == 0) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "%s: a row must have at least one column", what);
  return SWIGLU_OK;
}

bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int threads_for(int64_t items, int most) {
  int64_t t = (items + 31) / 32 * 32;
  return static_cast<int>(t < 32 ? 32 : t > most ? most : t);
}

template <typename T, typename W, bool E4M3>
int launch_fwd(const FwdParams& p, cudaStream_t st) {
  rmsnorm_fwd_any_kernel<T, W, E4M3><<<static_cast<unsigned>(p.rows), threads_for(p.cols, 512), 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, "rmsnorm forward launch");
}

int op_rmsnorm_fwd(FwdParams p, int64_t rows, int64_t cols, int dtype, int weight_dtype, bool e4m3, cudaStream_t st) {
  if (int rc = check_norm("rmsnorm_fwd", rows, cols, dtype, weight_dtype)) return rc;
  if (!(p.eps >= 0.0f)) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "rmsnorm_fwd: eps must not be negative");
  if (rows == 0) return SWIGLU_OK;
  if (!p.x || !p.weight || !p.y || !p.rstd || (p.residual && !p.s) || (e4m3 && !p.row_scale))
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  const uintptr_t es = dtype == SWIGLU_F32 ? 4 : 2, ws = weight_dtype == SWIGLU_F32 ? 4 : 2;
  if (!aligned(p.x, es) || !aligned(p.residual, es) || !aligned(p.s, es) || !aligned(p.weight, ws) ||
      !aligned(p.rstd, 4) || !aligned(p.row_scale, 4) || !aligned(p.y, e4m3 ? 1 : es))
    return fail(SWIGLU_ERR_MISALIGNED, "rmsnorm_fwd: a pointer is not aligned to its element");
  DeviceInfo* d;
  if (int rc = current_device(&d)) return rc;
  p.rows = rows;
  p.cols = static_cast<int>(cols);
#define SWIGLU_NORM(T, W) (e4m3 ? launch_fwd<T, W, true>(p, st) : launch_fwd<T, W, false>(p, st))
  if (dtype == SWIGLU_F32)
    return weight_dtype == SWIGLU_F32 ? SWIGLU_NORM(float, float) : SWIGLU_NORM(float, __nv_bfloat16);
  return weight_dtype == SWIGLU_F32 ? SWIGLU_NORM(__nv_bfloat16, float) : SWIGLU_NORM(__nv_bfloat16, __nv_bfloat16);
#undef SWIGLU_NORM
}

// Row chunks of the column pass: enough that the blocks of all chunks fill the
// device a few times, at least 16 rows each.
void plan_bwd(int64_t rows, int64_t cols, int sms, int* chunks, int* rows_per_chunk) {
  const int64_t col_blocks = (cols + 255) / 256;
  int64_t want = (8 * static_cast<int64_t>(sms) + col_blocks - 1) / col_blocks;
  int64_t per = (rows + want - 1) / want;
  if (per < 16) per = 16;
  *rows_per_chunk = static_cast<int>(per);
  *chunks = static_cast<int>((rows + per - 1) / per);
}

template <typename T, typename W>
int launch_bwd(BwdParams& p, const DeviceInfo& d, cudaStream_t st) {
  rmsnorm_bwd_dot_kernel<T, W><<<static_cast<unsigned>(p.rows), threads_for(p.cols, 512), 0, st>>>(p);
  rmsnorm_bwd_cols_kernel<T, W><<<dim3((p.cols + 255) / 256, p.chunks), 256, 0, st>>>(p);
  rmsnorm_dweight_kernel<W><<<(p.cols + 31) / 32, dim3(32, 32), 0, st>>>(p.partial, static_cast<W*>(p.dweight), p.cols,
                                                                         p.chunks);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, "rmsnorm backward launch");
}

// Floats of the workspace: the rows' dots, then the chunks' parts of dweight.
int64_t bwd_floats(int64_t rows, int64_t cols, int chunks) { return rows + static_cast<int64_t>(chunks) * cols; }

int op_rmsnorm_bwd(BwdParams p, int64_t rows, int64_t cols, int dtype, int weight_dtype, float* workspace,
                   int64_t workspace_floats, cudaStream_t st) {
  if (int rc = check_norm("rmsnorm_bwd", rows, cols, dtype, weight_dtype)) return rc;
  if (!p.dweight) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  DeviceInfo* d;
  if (rows == 0) {  // no row: the weight's gradient is an empty sum
    if (int rc = current_device(&d)) return rc;
    const cudaError_t e = cudaMemsetAsync(p.dweight, 0, cols * (weight_dtype == SWIGLU_F32 ? 4 : 2), st);
    return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, "rmsnorm_bwd");
  }
  if (!p.dy || !p.s || !p.weight || !p.rstd || !p.dx || !workspace)
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  const uintptr_t es = dtype == SWIGLU_F32 ? 4 : 2, ws = weight_dtype == SWIGLU_F32 ? 4 : 2;
  if (!aligned(p.dy, es) || !aligned(p.s, es) || !aligned(p.ds, es) || !aligned(p.dx, es) || !aligned(p.weight, ws) ||
      !aligned(p.dweight, ws) || !aligned(p.rstd, 4) || !aligned(workspace, 16))
    return fail(SWIGLU_ERR_MISALIGNED, "rmsnorm_bwd: a pointer is not aligned to its element (workspace: 16 bytes)");
  if (int rc = current_device(&d)) return rc;
  p.rows = rows;
  p.cols = static_cast<int>(cols);
  plan_bwd(rows, cols, d->sms, &p.chunks, &p.rows_per_chunk);
  if (workspace_floats < bwd_floats(rows, cols, p.chunks))
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "rmsnorm_bwd: workspace of %lld floats, %lld needed",
                (long long)workspace_floats, (long long)bwd_floats(rows, cols, p.chunks));
  p.dot = workspace;
  p.partial = workspace + rows;
  if (dtype == SWIGLU_F32)
    return weight_dtype == SWIGLU_F32 ? launch_bwd<float, float>(p, *d, st) : launch_bwd<float, __nv_bfloat16>(p, *d, st);
  return weight_dtype == SWIGLU_F32 ? launch_bwd<__nv_bfloat16, float>(p, *d, st)
                                    : launch_bwd<__nv_bfloat16, __nv_bfloat16>(p, *d, st);
}

}  // namespace
}  // namespace swiglu

using namespace swiglu;

extern "C" {

int swiglu_b200_rmsnorm_fwd(const void* x, const void* residual, const void* weight, void* y, void* s, float* rstd,
                            int64_t rows, int64_t cols, const float* eps, int dtype, int weight_dtype, void* stream) {
  if (!eps) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  FwdParams p{x, residual, weight, y, nullptr, s, rstd, 0, 0, *eps};
  return op_rmsnorm_fwd(p, rows, cols, dtype, weight_dtype, false, static_cast<cudaStream_t>(stream));
}

int swiglu_b200_rmsnorm_fwd_e4m3(const void* x, const void* residual, const void* weight, void* q, float* row_scale,
                                 void* s, float* rstd, int64_t rows, int64_t cols, const float* eps, int dtype,
                                 int weight_dtype, void* stream) {
  if (!eps) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  FwdParams p{x, residual, weight, q, row_scale, s, rstd, 0, 0, *eps};
  return op_rmsnorm_fwd(p, rows, cols, dtype, weight_dtype, true, static_cast<cudaStream_t>(stream));
}

int swiglu_b200_rmsnorm_bwd_workspace(int64_t rows, int64_t cols, int num_sms, int64_t* floats) {
  if (int rc = check_dims("rmsnorm_bwd_workspace", rows, cols, num_sms)) return rc;
  if (!floats) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  if (cols == 0 || num_sms == 0) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "cols and num_sms must be positive");
  int chunks = 0, per = 0;
  if (rows) plan_bwd(rows, cols, num_sms, &chunks, &per);
  *floats = bwd_floats(rows, cols, chunks);
  return SWIGLU_OK;
}

int swiglu_b200_rmsnorm_bwd(const void* dy, const void* s, const void* weight, const float* rstd, const void* ds,
                            void* dx, void* dweight, float* workspace, int64_t workspace_floats, int64_t rows,
                            int64_t cols, int dtype, int weight_dtype, void* stream) {
  BwdParams p{dy, s, weight, rstd, ds, dx, nullptr, nullptr, dweight, 0, 0, 0, 0};
  return op_rmsnorm_bwd(p, rows, cols, dtype, weight_dtype, workspace, workspace_floats,
                        static_cast<cudaStream_t>(stream));
}

}  // extern "C"
