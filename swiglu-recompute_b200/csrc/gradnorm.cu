// Global norm over a list of gradients, and clipping by it.
//
//   norm = sqrt(sum over all tensors of g^2)
//   out  = g * min(1, max_norm / (norm + 1e-6))          (in place, or to `out`)
//
// The tensors of a launch travel in its parameters (no copy to the device):
// each is cut into chunks, and a persistent grid walks the chunks of all of
// them. The squares of a thread's 64 (bf16) or 32 (f32) values are summed in
// f32 and everything above that in f64, in an order that depends on sizes
// only. A thread whose f32 sum leaves the range where f32 squares are safe
// (values around 1e19 or 1e-15) squares its values again in f64; one whose values
// are all zeros, told by their bits, is done.
#include <algorithm>
#include <new>
#include <vector>

#include "host.cuh"
#include "ptx.cuh"

namespace swiglu {
namespace {

constexpr int kTableTensors = 112;  // one launch's table stays below 4 KB of parameters
constexpr int kGradThreads = 256;
constexpr int kGradSlots = 8;       // 16-byte slots per thread and chunk
constexpr int kGradBlocks = 4;      // per SM
constexpr int kChunkSlots = kGradThreads * kGradSlots;

struct GradTable {
  const void* in[kTableTensors];
  void* out[kTableTensors];
  long long size[kTableTensors];         // elements
  int first_chunk[kTableTensors + 1];
  uint8_t f32[kTableTensors];
  int count;
};
static_assert(sizeof(GradTable) <= 3900, "launch parameters");

// 16-byte slots that a tensor touches, counted from the 16-byte boundary at or
// below its first element.
__host__ __device__ __forceinline__ long long slots_of(const void* p, long long bytes) {
  return (static_cast<long long>(reinterpret_cast<uintptr_t>(p) % 16) + bytes + 15) / 16;
}

__device__ __forceinline__ int tensor_of(const GradTable& t, int chunk) {
  int lo = 0, hi = t.count - 1;  // the last tensor whose first chunk is at or before `chunk`
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first_chunk[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A thread's slots of one chunk of tensor k. Slots wholly inside the tensor are
// 16-byte words; in the others, at its ends, elements outside are zeros.
template <typename T>
struct ChunkSlots {
  static constexpr int N = 16 / sizeof(T);
  const T* base;
  long long size, e0;  // the tensor's elements; the first element of this thread's first slot
  bool whole;          // all slots of the chunk (any thread's) are inside

  __device__ __forceinline__ ChunkSlots(const GradTable& t, int k, int chunk) {
    base = static_cast<const T*>(t.in[k]);
    size = t.size[k];
    const int head = static_cast<int>(reinterpret_cast<uintptr_t>(base) % 16 / sizeof(T));
    const long long c0 = static_cast<long long>(chunk - t.first_chunk[k]) * (kChunkSlots * N) - head;
    whole = c0 >= 0 && c0 + kChunkSlots * N <= size;
    e0 = c0 + static_cast<long long>(threadIdx.x) * N;
  }
  __device__ __forceinline__ long long at(int i) const { return e0 + i * (kGradThreads * N); }
  __device__ __forceinline__ bool inside(int i) const { return at(i) >= 0 && at(i) + N <= size; }
  __device__ __forceinline__ uint4 load_one(int i) const {
    if (inside(i)) return *reinterpret_cast<const uint4*>(base + at(i));
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (at(i) + e < 0 || at(i) + e >= size) continue;
      if constexpr (sizeof(T) == 4) w[e] = __float_as_uint(base[at(i) + e]);
      else w[e / 2] |= static_cast<uint32_t>(__bfloat16_as_ushort(base[at(i) + e])) << (16 * (e & 1));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void load(uint4 (&u)[kGradSlots]) const {
    if (whole) {
      const uint4* p = reinterpret_cast<const uint4*>(base + e0);
#pragma unroll
      for (int i = 0; i < kGradSlots; ++i) u[i] = p[i * kGradThreads];
    } else {
#pragma unroll
      for (int i = 0; i < kGradSlots; ++i) u[i] = load_one(i);
    }
  }
  __device__ static __forceinline__ void values(const uint4& u, float (&f)[N]) {
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
};

template <typename T>
__device__ __forceinline__ double chunk_squares(const GradTable& t, int k, int chunk) {
  constexpr int N = ChunkSlots<T>::N;
  const ChunkSlots<T> slots(t, k, chunk);
  uint4 u[kGradSlots];
  slots.load(u);
  float2 sum[2] = {};  // packed f32x2 arithmetic
#pragma unroll
  for (int i = 0; i < kGradSlots; ++i) {
    float f[N];
    ChunkSlots<T>::values(u[i], f);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      const float2 v = make_float2(f[2 * e], f[2 * e + 1]);
      sum[e & 1] = __ffma2_rn(v, v, sum[e & 1]);
    }
  }
  const float total = (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
  if (total >= 1e-30f && total <= 1e37f) return static_cast<double>(total);
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < kGradSlots; ++i) bits |= u[i].x | u[i].y | u[i].z | u[i].w;
  if ((bits & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu)) == 0) return 0.0;
  double exact = 0.0;
#pragma unroll 1
  for (int i = 0; i < kGradSlots; ++i) {  // read again, so that the usual path keeps no values
    float f[N];
    ChunkSlots<T>::values(slots.load_one(i), f);
#pragma unroll
    for (int e = 0; e < N; ++e) exact += static_cast<double>(f[e]) * static_cast<double>(f[e]);
  }
  return exact;
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kGradThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane_id() == 0) part[warp_id()] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < kGradThreads / 32; ++i) v += part[i];
  return v;
}

__global__ void __launch_bounds__(kGradThreads, kGradBlocks)
    grad_squares_kernel(const __grid_constant__ GradTable t, double* partial) {
  wait_for_previous();
  double sum = 0.0;
  const int chunks = t.first_chunk[t.count];
  int k = blockIdx.x < chunks ? tensor_of(t, blockIdx.x) : 0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    while (c >= t.first_chunk[k + 1]) ++k;
    sum += t.f32[k] ? chunk_squares<float>(t, k, c) : chunk_squares<__nv_bfloat16>(t, k, c);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__device__ __forceinline__ double total_norm(const double* partial, int count) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < count; i += kGradThreads) sum += partial[i];
  return sqrt(block_sum(sum));
}

__global__ void __launch_bounds__(kGradThreads) grad_norm_kernel(const double* partial, int count, float* norm) {
  wait_for_previous();
  const double n = total_norm(partial, count);
  if (threadIdx.x == 0) *norm = static_cast<float>(n);
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const GradTable& t, int k, int chunk, float factor) {
  constexpr int N = ChunkSlots<T>::N;
  const ChunkSlots<T> slots(t, k, chunk);
  T* out = static_cast<T*>(t.out[k]);
  const bool same = (reinterpret_cast<uintptr_t>(slots.base) ^ reinterpret_cast<uintptr_t>(out)) % 16 == 0;
  uint4 u[kGradSlots];
  slots.load(u);
#pragma unroll
  for (int i = 0; i < kGradSlots; ++i) {
    float f[N];
    ChunkSlots<T>::values(u[i], f);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      const float2 v = __fmul2_rn(make_float2(f[2 * e], f[2 * e + 1]), make_float2(factor, factor));
      f[2 * e] = v.x;
      f[2 * e + 1] = v.y;
    }
    const long long at = slots.at(i);
    if (same && (slots.whole || slots.inside(i))) {
      uint4 r;
      if constexpr (sizeof(T) == 4) {
        r = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      } else {
        r = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                       pack_bf16x2(f[6], f[7]));
      }
      *reinterpret_cast<uint4*>(out + at) = r;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (at + e >= 0 && at + e < slots.size) {
          if constexpr (sizeof(T) == 4) out[at + e] = f[e];
          else out[at + e] = __float2bfloat16_rn(f[e]);
        }
      }
    }
  }
}

// Scales one launch's tensors. The norm comes from `count` partial sums (each
// block adds them up for itself; the first writes it to norm_out) or, with
// count == 0, from *norm_in. Chunks are walked from the last to the first: the
// squares pass ended there, so that part is still in L2.
__global__ void __launch_bounds__(kGradThreads, kGradBlocks)
    grad_scale_kernel(const __grid_constant__ GradTable t, const double* partial, int count, const float* norm_in,
                      float* norm_out, double max_norm) {
  wait_for_previous();
  const double n = count ? total_norm(partial, count) : static_cast<double>(*norm_in);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = static_cast<float>(n);
  double ratio = max_norm / (n + 1e-6);
  if (ratio > 1.0) ratio = 1.0;  // a NaN norm stays one, and reaches every gradient
  const float factor = static_cast<float>(ratio);
  const int last = t.first_chunk[t.count] - 1 - static_cast<int>(blockIdx.x);
  int k = last >= 0 ? tensor_of(t, last) : 0;
  for (int c = last; c >= 0; c -= gridDim.x) {
    while (c < t.first_chunk[k]) --k;
    if (factor == 1.0f && t.out[k] == t.in[k]) continue;  // x * 1 in place
    if (t.f32[k]) chunk_scale<float>(t, k, c, factor);
    else chunk_scale<__nv_bfloat16>(t, k, c, factor);
  }
}

// Blocks of a launch: as many as are resident at once.
int grad_grid(int chunks, int sms) {
  const int most = sms * kGradBlocks;
  return chunks < most ? (chunks < 1 ? 1 : chunks) : most;
}

int64_t launches_of(int64_t count) { return (count + kTableTensors - 1) / kTableTensors; }

// Fills one launch's table with tensors [k0, ...) and returns how many it took.
int64_t fill_table(GradTable& t, const void* const* grads, void* const* outs, const int64_t* sizes, const int* dtypes,
                   int64_t k0, int64_t count) {
  int n = 0;
  int64_t chunks = 0, k = k0;
  for (; k < count && n < kTableTensors; ++k) {
    if (sizes[k] == 0) continue;
    const int64_t es = dtypes[k] == SWIGLU_F32 ? 4 : 2;
    const int64_t add = (slots_of(grads[k], sizes[k] * es) + kChunkSlots - 1) / kChunkSlots;
    if (chunks + add > 0x3fffffff) break;  // chunk numbers are ints
    t.in[n] = grads[k];
    t.out[n] = outs ? outs[k] : nullptr;
    t.size[n] = sizes[k];
    t.f32[n] = dtypes[k] == SWIGLU_F32;
    t.first_chunk[n] = static_cast<int>(chunks);
    chunks += add;
    ++n;
  }
  t.first_chunk[n] = static_cast<int>(chunks);
  t.count = n;
  return k - k0;
}

int check_grads(const char* what, const void* const* grads, void* const* outs, bool need_outs, const int64_t* sizes,
                const int* dtypes, int64_t count) {
  if (count < 0 || !fits_int(count)) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "%s: bad tensor count", what);
  if (count && (!grads || !sizes || !dtypes || (need_outs && !outs)))
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  for (int64_t k = 0; k < count; ++k) {
    if (int rc = check_dtype(dtypes[k])) return rc;
    if (sizes[k] < 0 || sizes[k] > (1ll << 40))
      return fail(SWIGLU_ERR_INVALID_ARGUMENT, "%s: tensor %lld has a bad size", what, (long long)k);
    if (sizes[k] == 0) continue;
    if (!grads[k] || (need_outs && !outs[k])) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
    const uintptr_t es = dtypes[k] == SWIGLU_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(grads[k]) % es || (need_outs && reinterpret_cast<uintptr_t>(outs[k]) % es))
      return fail(SWIGLU_ERR_MISALIGNED, "%s: tensor %lld is not aligned to its element", what, (long long)k);
  }
  return SWIGLU_OK;
}

// A tensor that is written may share memory with no other one: its elements
// would be scaled twice, or read after they were written.
int check_disjoint(const void* const* grads, void* const* outs, const int64_t* sizes, const int* dtypes,
                   int64_t count) {
  struct Range {
    uintptr_t begin, end;
    bool written;
  };
  std::vector<Range> all;
  all.reserve(2 * count);
  for (int64_t k = 0; k < count; ++k) {
    const uintptr_t bytes = static_cast<uintptr_t>(sizes[k]) * (dtypes[k] == SWIGLU_F32 ? 4 : 2);
    if (!bytes) continue;
    const uintptr_t o = reinterpret_cast<uintptr_t>(outs[k]), g = reinterpret_cast<uintptr_t>(grads[k]);
    all.push_back({o, o + bytes, true});
    if (g != o) all.push_back({g, g + bytes, false});
  }
  std::sort(all.begin(), all.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  uintptr_t any = 0, written = 0;
  for (const Range& r : all) {
    if (r.begin < (r.written ? any : written))
      return fail(SWIGLU_ERR_INVALID_ARGUMENT, "a gradient that is written overlaps another tensor of the call");
    any = std::max(any, r.end);
    if (r.written) written = std::max(written, r.end);
  }
  return SWIGLU_OK;
}

// Squares of every launch's tensors; *parts = partial sums written.
int launch_squares(const void* const* grads, const int64_t* sizes, const int* dtypes, int64_t count,
                   double* workspace, int64_t workspace_doubles, const DeviceInfo& d, int* parts, cudaStream_t st) {
  *parts = 0;
  for (int64_t k = 0; k < count;) {
    GradTable t;
    k += fill_table(t, grads, nullptr, sizes, dtypes, k, count);
    if (t.count == 0) continue;
    const int grid = grad_grid(t.first_chunk[t.count], d.sms);
    if (*parts + grid > workspace_doubles)
      return fail(SWIGLU_ERR_INVALID_ARGUMENT, "workspace of %lld doubles is too small", (long long)workspace_doubles);
    launch_after(grad_squares_kernel, grid, kGradThreads, 0, st, t, workspace + *parts);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "grad norm launch");
    *parts += grid;
  }
  return SWIGLU_OK;
}

int launch_scale(const void* const* grads, void* const* outs, const int64_t* sizes, const int* dtypes, int64_t count,
                 const double* partial, int parts, const float* norm_in, float* norm_out, double max_norm,
                 const DeviceInfo& d, cudaStream_t st) {
  bool wrote = false;
  for (int64_t k = 0; k < count;) {
    GradTable t;
    k += fill_table(t, grads, outs, sizes, dtypes, k, count);
    if (t.count == 0) continue;
    launch_after(grad_scale_kernel, grad_grid(t.first_chunk[t.count], d.sms), kGradThreads, 0, st, t, partial, parts,
                 norm_in, wrote ? nullptr : norm_out, max_norm);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "gradient scaling launch");
    wrote = true;
  }
  return SWIGLU_OK;
}

int zero_norm(float* norm, cudaStream_t st) {
  const cudaError_t e = cudaMemsetAsync(norm, 0, sizeof(float), st);
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, "grad norm");
}

int op_grad_norm(const void* const* grads, const int64_t* sizes, const int* dtypes, int64_t count, double* workspace,
                 int64_t workspace_doubles, float* norm, cudaStream_t st) {
  if (int rc = check_grads("grad_norm", grads, nullptr, false, sizes, dtypes, count)) return rc;
  if (!norm || !workspace) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  DeviceInfo* d;
  if (int rc = current_device(&d)) return rc;
  int parts = 0;
  if (int rc = launch_squares(grads, sizes, dtypes, count, workspace, workspace_doubles, *d, &parts, st)) return rc;
  if (parts == 0) return zero_norm(norm, st);
  launch_after(grad_norm_kernel, 1, kGradThreads, 0, st, workspace, parts, norm);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, "grad norm launch");
}

int check_max_norm(double max_norm) {
  if (!(max_norm >= 0.0)) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "max_norm must not be negative");
  return SWIGLU_OK;
}

int op_clip(const void* const* grads, void* const* outs, const int64_t* sizes, const int* dtypes, int64_t count,
            double max_norm, double* workspace, int64_t workspace_doubles, float* norm, cudaStream_t st) {
  if (int rc = check_grads("clip_grad_norm", grads, outs, true, sizes, dtypes, count)) return rc;
  if (int rc = check_max_norm(max_norm)) return rc;
  if (!norm || !workspace) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  if (int rc = check_disjoint(grads, outs, sizes, dtypes, count)) return rc;
  DeviceInfo* d;
  if (int rc = current_device(&d)) return rc;
  int parts = 0;
  if (int rc = launch_squares(grads, sizes, dtypes, count, workspace, workspace_doubles, *d, &parts, st)) return rc;
  if (parts == 0) return zero_norm(norm, st);
  return launch_scale(grads, outs, sizes, dtypes, count, workspace, parts, nullptr, norm, max_norm, *d, st);
}

int op_scale_by_norm(const void* const* grads, void* const* outs, const int64_t* sizes, const int* dtypes,
                     int64_t count, const float* norm, double max_norm, cudaStream_t st) {
  if (int rc = check_grads("clip_grads_by_norm", grads, outs, true, sizes, dtypes, count)) return rc;
  if (int rc = check_max_norm(max_norm)) return rc;
  if (!norm) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  if (int rc = check_disjoint(grads, outs, sizes, dtypes, count)) return rc;
  DeviceInfo* d;
  if (int rc = current_device(&d)) return rc;
  return launch_scale(grads, outs, sizes, dtypes, count, nullptr, 0, norm, nullptr, max_norm, *d, st);
}

// The lists are checked with the C++ library's containers: no exception of
// theirs leaves the C interface.
template <class F>
int guarded(F f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "out of host memory");
  }
}

}  // namespace
}  // namespace swiglu

using namespace swiglu;

extern "C" {

int swiglu_b200_grad_norm_workspace(int64_t count, int num_sms, int64_t* doubles) {
  if (int rc = check_dims("grad_norm_workspace", count, num_sms, 0)) return rc;
  if (!doubles) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  const int64_t n = launches_of(count) * num_sms * kGradBlocks;
  *doubles = n > 0 ? n : 1;
  return SWIGLU_OK;
}

int swiglu_b200_grad_norm(const void* const* grads, const int64_t* sizes, const int* dtypes, int64_t count,
                          double* workspace, int64_t workspace_doubles, float* norm, void* stream) {
  return op_grad_norm(grads, sizes, dtypes, count, workspace, workspace_doubles, norm,
                      static_cast<cudaStream_t>(stream));
}

int swiglu_b200_clip_grad_norm(const void* const* grads, void* const* outs, const int64_t* sizes, const int* dtypes,
                               int64_t count, const double* max_norm, double* workspace, int64_t workspace_doubles,
                               float* norm, void* stream) {
  if (!max_norm) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  return guarded([&] {
    return op_clip(grads, outs, sizes, dtypes, count, *max_norm, workspace, workspace_doubles, norm,
                   static_cast<cudaStream_t>(stream));
  });
}

int swiglu_b200_clip_grads_by_norm(const void* const* grads, void* const* outs, const int64_t* sizes,
                                   const int* dtypes, int64_t count, const float* norm, const double* max_norm,
                                   void* stream) {
  if (!max_norm) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "null pointer");
  return guarded([&] {
    return op_scale_by_norm(grads, outs, sizes, dtypes, count, norm, *max_norm, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
