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

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else return __float2bfloat16_rn(v);
}

__device__ __forceinline__ uint8_t e4m3_byte(float v) { return static_cast<uint8_t>(e4m3x2(v, 0.0f) & 0xffu); }

// 16 bytes of T, as loaded.
template <typename T>
constexpr int kV = 16 / sizeof(T);

template <typename T>
__device__ __forceinline__ void get16(const uint4& u, float (&f)[kV<T>]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      const float2 v = unpack_bf16x2(w[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    } else {
      f[i] = __uint_as_float(w[i]);
    }
  }
}
// The same as pairs.
template <typename T>
__device__ __forceinline__ void pairs16(const uint4& u, float2 (&f)[kV<T> / 2]) {
  float v[kV<T>];
  get16<T>(u, v);
#pragma unroll
  for (int i = 0; i < kV<T> / 2; ++i) f[i] = make_float2(v[2 * i], v[2 * i + 1]);
}
template <typename T>
__device__ __forceinline__ uint4 set16(const float (&f)[kV<T>]) {
  if constexpr (sizeof(T) == 2)
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  else
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

template <typename T>
__device__ __forceinline__ uint4 unpairs16(const float2 (&f)[kV<T> / 2]) {
  float v[kV<T>];
#pragma unroll
  for (int i = 0; i < kV<T> / 2; ++i) {
    v[2 * i] = f[i].x;
    v[2 * i + 1] = f[i].y;
  }
  return set16<T>(v);
}

// Rows whose length is no multiple of a pack (SHIFT): the packs stay on the
// tensor's 16-byte grid, so a row starts `head` elements inside its first one.
// Pack k holds the row's elements k * V - head and on; in the first and the last
// some belong to a neighbouring row or lie behind the tensor: those count as
// zeros and are neither read nor written. (Reading the whole pack and masking
// it, where the tensor has it, was slower: 5000 x 4099 f32 52 -> 59 us, its
// gradient 85 -> 125.)
template <typename T, bool SHIFT>
struct RowPacks {
  static constexpr int V = kV<T>;
  long long base;  // the row's first element
  int cols, head, packs;

  __device__ __forceinline__ RowPacks(long long row, int c)
      : base(row * c), cols(c), head(SHIFT ? static_cast<int>(row * c % V) : 0),
        packs((c + head + V - 1) / V) {}
  __device__ __forceinline__ bool edge(int k) const { return SHIFT && (k * V < head || k * V - head + V > cols); }
  __device__ __forceinline__ bool inside(int k, int e) const {
    const int j = k * V - head + e;
    return j >= 0 && j < cols;
  }
  __device__ __forceinline__ uint4 load(const T* p, int k) const {
    const long long at = base - head + static_cast<long long>(k) * V;
    if (!edge(k)) return *reinterpret_cast<const uint4*>(p + at);
    float f[V];
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = inside(k, e) ? to_f32(p[at + e]) : 0.0f;
    return set16<T>(f);
  }
  // Zeros in place of what does not belong to the row.
  __device__ __forceinline__ uint4 masked(const uint4& u, int k) const {
    float f[V];
    get16<T>(u, f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = inside(k, e) ? f[e] : 0.0f;
    return set16<T>(f);
  }
  __device__ __forceinline__ void store(T* p, int k, const uint4& u) const {
    const long long at = base - head + static_cast<long long>(k) * V;
    if (!edge(k)) {
      *reinterpret_cast<uint4*>(p + at) = u;
    } else {
      float f[V];
      get16<T>(u, f);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (inside(k, e)) p[at + e] = from_f32<T>(f[e]);
    }
  }
  __device__ __forceinline__ void store_e4m3(uint8_t* p, int k, const float (&f)[V]) const {
    const long long at = base - head + static_cast<long long>(k) * V;
    if (!edge(k)) {
      uint32_t w[V / 4];
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        w[i] = e4m3x2(f[4 * i], f[4 * i + 1]) | (e4m3x2(f[4 * i + 2], f[4 * i + 3]) << 16);
      if constexpr (V == 4) *reinterpret_cast<uint32_t*>(p + at) = w[0];
      else *reinterpret_cast<uint2*>(p + at) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (inside(k, e)) p[at + e] = e4m3_byte(f[e]);
    }
  }
  // The weight of pack k's elements.
  template <typename W>
  __device__ __forceinline__ void weight(const W* w, int k, float (&f)[V]) const {
    if constexpr (SHIFT) {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = inside(k, e) ? to_f32(w[k * V - head + e]) : 0.0f;
    } else if constexpr (V * sizeof(W) == 8) {
      const uint2 u = *reinterpret_cast<const uint2*>(w + k * V);
      const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
      f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
    } else {
#pragma unroll
      for (int i = 0; i < V / kV<W>; ++i) {
        float g[kV<W>];
        get16<W>(*reinterpret_cast<const uint4*>(w + k * V + i * kV<W>), g);
#pragma unroll
        for (int e = 0; e < kV<W>; ++e) f[i * kV<W> + e] = g[e];
      }
    }
  }
};

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

// Row factors from the statistics: rstd, the factors that take s w to e4m3, and
// the stored scale: 1 for an all-zero row, NaN where the row holds one. 448 / top
// leaves f32 below top = 1.3e-36, so such rows are first multiplied by `lift`
// (exact), and the scale rounds once, at its end.
__device__ __forceinline__ void row_factors(float sum, float top, const FwdParams& p, float& rstd, float& lift,
                                            float& qs, float& scale) {
  rstd = rsqrtf(sum / static_cast<float>(p.cols) + p.eps);
  const bool tiny = top > 0.0f && top < 0x1p-100f;
  lift = tiny ? 0x1p100f : 1.0f;
  top *= lift;
  qs = top > 0.0f ? kE4m3Max / top : 1.0f;
  scale = top > 0.0f ? top * rstd / kE4m3Max * (tiny ? 0x1p-100f : 1.0f) : (rstd == rstd ? 1.0f : rstd);
}

// A row in registers: blockDim.x threads hold VPT packs each, all loaded before
// the first is used; blockDim.y rows a block where a warp holds a row (then no
// thread waits for another warp), one otherwise. One pass over memory.
constexpr int kRowThreads = 1024;  // that a row may take, at 64 registers each

template <typename T, typename W, bool E4M3, int VPT, bool SHIFT>
__global__ void __launch_bounds__(kRowThreads) rmsnorm_fwd_row_kernel(const FwdParams p) {
  wait_for_previous();
  constexpr int V = kV<T>;
  __shared__ float2 scratch[32];
  const long long row = blockIdx.x * static_cast<long long>(blockDim.y) + threadIdx.y;
  if (row >= p.rows) return;
  const RowPacks<T, SHIFT> rp(row, p.cols);
  const W* w = static_cast<const W*>(p.weight);
  uint4 a[VPT], b[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int k = static_cast<int>(threadIdx.x + i * blockDim.x);
    if (k < rp.packs) a[i] = rp.load(static_cast<const T*>(p.x), k);
  }
  if (p.residual) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int k = static_cast<int>(threadIdx.x + i * blockDim.x);
      if (k < rp.packs) b[i] = rp.load(static_cast<const T*>(p.residual), k);
    }
  }
  // The kernel comes close to issuing an instruction every cycle (75 % of the slots
  // for bf16 in scalar form), hence the packed f32x2 arithmetic.
  constexpr int P = V / 2;
  float2 sum2 = make_float2(0.0f, 0.0f);
  float top = 0.0f;
  float sw[E4M3 ? VPT : 1][V];  // s w, kept for the e4m3 output
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int k = static_cast<int>(threadIdx.x + i * blockDim.x);
    if (k >= rp.packs) continue;
    float2 v[P];
    pairs16<T>(a[i], v);
    if (p.residual) {
      float2 r[P];
      pairs16<T>(b[i], r);
#pragma unroll
      for (int e = 0; e < P; ++e) v[e] = __fadd2_rn(v[e], r[e]);
      a[i] = unpairs16<T>(v);
      rp.store(static_cast<T*>(p.s), k, a[i]);
      pairs16<T>(a[i], v);
    }
    if constexpr (E4M3) {
      rp.weight(w, k, sw[i]);
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float2 m = __fmul2_rn(make_float2(sw[i][2 * e], sw[i][2 * e + 1]), v[e]);
        sw[i][2 * e] = m.x;
        sw[i][2 * e + 1] = m.y;
        top = fmaxf(top, fmaxf(fabsf(m.x), fabsf(m.y)));
      }
    }
#pragma unroll
    for (int e = 0; e < P; ++e) sum2 = __ffma2_rn(v[e], v[e], sum2);
  }
  float sum = sum2.x + sum2.y;
  row_reduce(sum, top, blockDim.x >> 5, scratch);
  float rstd, lift, qs, scale;
  row_factors(sum, top, p, rstd, lift, qs, scale);
  if (threadIdx.x == 0) {
    p.rstd[row] = rstd;
    if constexpr (E4M3) p.row_scale[row] = scale;
  }
  if constexpr (E4M3) {
    if (lift != 1.0f) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (static_cast<int>(threadIdx.x + i * blockDim.x) >= rp.packs) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) sw[i][e] *= lift;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int k = static_cast<int>(threadIdx.x + i * blockDim.x);
    if (k >= rp.packs) continue;
    if constexpr (E4M3) {
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float2 m = __fmul2_rn(make_float2(sw[i][2 * e], sw[i][2 * e + 1]), make_float2(qs, qs));
        sw[i][2 * e] = m.x;
        sw[i][2 * e + 1] = m.y;
      }
      rp.store_e4m3(static_cast<uint8_t*>(p.y), k, sw[i]);
    } else {
      float2 v[P];
      float f[V];
      pairs16<T>(a[i], v);
      rp.weight(w, k, f);
#pragma unroll
      for (int e = 0; e < P; ++e)
        v[e] = __fmul2_rn(__fmul2_rn(v[e], make_float2(rstd, rstd)), make_float2(f[2 * e], f[2 * e + 1]));
      rp.store(static_cast<T*>(p.y), k, unpairs16<T>(v));
    }
  }
}

// Any width and alignment: a block per row, one element per thread at a time;
// the second pass reads the row (or the s just written by the same thread)
// again from L1 / L2.
template <typename T, typename W, bool E4M3>
__global__ void __launch_bounds__(512) rmsnorm_fwd_any_kernel(const FwdParams p) {
  wait_for_previous();
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
  float rstd, lift, qs, scale;
  row_factors(sum, top, p, rstd, lift, qs, scale);
  if (threadIdx.x == 0) {
    p.rstd[blockIdx.x] = rstd;
    if constexpr (E4M3) p.row_scale[blockIdx.x] = scale;
  }
  const T* src = r ? s : x;
  for (int j = threadIdx.x; j < p.cols; j += blockDim.x) {
    const float v = to_f32(src[j]), f = to_f32(w[j]);
    if constexpr (E4M3) static_cast<uint8_t*>(p.y)[base + j] = e4m3_byte(v * f * lift * qs);
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
  int period;         // rows after which a row's 16-byte offset repeats
  int stages;         // rows in the shared-memory ring
  uint32_t* status;   // device error word
};

// Threads of a backward row, and the registers its three loads take: up to 12,
// two blocks of 512 threads fit an SM; up to 24, the next row's loads fit too. (The
// compiler reports spills for bf16 rows: one shifted pack 20 bytes a thread, two
// packs 16, four packs 64 to 324; none for f32.)
constexpr int kBwdThreads = 512;
template <int VPT>
constexpr int kBwdLoadRegs = 12 * VPT;

// One pass: a thread keeps its columns over all the rows of its block, so the
// weight is read once and dweight's part stays in registers; the next row's
// packs are in flight while a row's dot product is summed over the block
// (blockDim.y rows a block where a warp holds a row). Each block leaves one part
// of dweight. SHIFT: the heads of row r and r + period are alike (period =
// V / gcd(cols, V)), so a block takes rows of one residue class and its threads'
// columns stay the same.
template <typename T, typename W, int VPT, bool SHIFT>
__global__ void __launch_bounds__(kBwdThreads, kBwdLoadRegs<VPT> <= 12 ? 2 : 1)
    rmsnorm_bwd_row_kernel(const BwdParams p) {
  wait_for_previous();
  constexpr int V = kV<T>;
  __shared__ float2 scratch[2][32];
  __shared__ float parts[VPT == 1 ? 8 * 32 * V : 1];  // warp rows: [warp][pack element]
  const T* dy = static_cast<const T*>(p.dy);
  const T* s = static_cast<const T*>(p.s);
  const T* ds = static_cast<const T*>(p.ds);
  T* dx = static_cast<T*>(p.dx);
  const float inv = 1.0f / static_cast<float>(p.cols);
  // Rows first, first + step, ... of this warp or block.
  const int period = SHIFT ? p.period : 1;
  const long long lane_row = (blockIdx.x / period) * static_cast<long long>(blockDim.y) + threadIdx.y;
  long long row = lane_row * period + blockIdx.x % period;
  const long long step = static_cast<long long>(gridDim.x / period) * blockDim.y * period;
  const RowPacks<T, SHIFT> first(blockIdx.x % period, p.cols);  // head and packs of every row here
  float w[VPT][V], acc[VPT][V];
  bool in[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int k = static_cast<int>(threadIdx.x + i * blockDim.x);
    in[i] = k < first.packs;
    if (in[i]) first.weight(static_cast<const W*>(p.weight), k, w[i]);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[i][e] = 0.0f;
  }
  struct Row {
    uint4 dy[VPT], s[VPT], ds[VPT];
    float rstd;
  };
  auto load = [&](long long r, Row& to) {
    const RowPacks<T, SHIFT> rp(r, p.cols);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int k = static_cast<int>(threadIdx.x + i * blockDim.x);
      if (in[i]) {
        to.dy[i] = rp.load(dy, k);
        to.s[i] = rp.load(s, k);
        if (ds) to.ds[i] = rp.load(ds, k);
      }
    }
    to.rstd = p.rstd[r];
  };
  constexpr bool kAhead = kBwdLoadRegs<VPT> <= 24;
  Row cur, next;
  if (kAhead && row < p.rows) load(row, cur);
  int buf = 0;
  for (; row < p.rows; row += step) {
    if constexpr (kAhead) {
      if (row + step < p.rows) load(row + step, next);
    } else {
      load(row, cur);
    }
    float dot = 0.0f, unused = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (!in[i]) continue;
      float g[V], v[V];
      get16<T>(cur.dy[i], g);
      get16<T>(cur.s[i], v);
#pragma unroll
      for (int e = 0; e < V; ++e) dot += g[e] * w[i][e] * v[e];
    }
    row_reduce(dot, unused, blockDim.x >> 5, scratch[buf]);
    buf ^= 1;  // a warp may still be reading the other half
    const float c = dot * inv * cur.rstd * cur.rstd;
    const RowPacks<T, SHIFT> rp(row, p.cols);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (!in[i]) continue;
      float g[V], v[V], d[V];
      get16<T>(cur.dy[i], g);
      get16<T>(cur.s[i], v);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        d[e] = cur.rstd * (g[e] * w[i][e] - v[e] * c);
        acc[i][e] += g[e] * v[e] * cur.rstd;
      }
      if (ds) {
        get16<T>(cur.ds[i], g);
#pragma unroll
        for (int e = 0; e < V; ++e) d[e] += g[e];
      }
      rp.store(dx, static_cast<int>(threadIdx.x + i * blockDim.x), set16<T>(d));
    }
    if constexpr (kAhead) cur = next;
  }
  float* part = p.partial + blockIdx.x * static_cast<long long>(p.cols);
  if constexpr (VPT == 1) {
    if (blockDim.y > 1) {
      if (in[0]) {
#pragma unroll
        for (int e = 0; e < V; ++e) parts[(threadIdx.y * 32 + threadIdx.x) * V + e] = acc[0][e];
      }
      __syncthreads();
      for (int j = threadIdx.y * 32 + threadIdx.x; j < p.cols; j += 32 * blockDim.y) {
        float sum = 0.0f;
        for (int y = 0; y < static_cast<int>(blockDim.y); ++y) sum += parts[y * 32 * V + j + first.head];
        part[j] = sum;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int k = static_cast<int>(threadIdx.x + i * blockDim.x);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (in[i] && first.inside(k, e)) part[k * V - first.head + e] = acc[i][e];
  }
}

// The same for rows that a block shares (more than a warp): rows arrive through a
// ring of `stages` rows in shared memory, filled by bulk copies, so that what is
// in flight does not depend on the registers left (11136 x 3584 bf16: registers
// 60.5 us, ring 56.1; 16384 x 8192: 192, 162; 5000 x 16384: 208, 120; 11136 x 3584
// f32: 136, 96). SHIFT: a copy takes the row's packs on the 16-byte grid, its
// neighbours' elements included; they are masked where they are read.
constexpr int kMaxStages = 8;

template <typename T, typename W, int VPT, bool SHIFT>
__global__ void __launch_bounds__(kBwdThreads, 1) rmsnorm_bwd_ring_kernel(const BwdParams p) {
  wait_for_previous();
  constexpr int V = kV<T>;
  extern __shared__ __align__(128) uint8_t ring[];  // [stage][dy, s, ds][packs]
  __shared__ uint64_t full[kMaxStages];
  __shared__ float sums[2][32];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  // This block's rows all have the same head: the grid is a multiple of the period.
  const long long row0 = blockIdx.x, step = gridDim.x;
  const RowPacks<T, SHIFT> first(row0, p.cols);
  const int packs = first.packs, warps = static_cast<int>(blockDim.x >> 5);
  const uint32_t row_bytes = static_cast<uint32_t>(packs) * 16;
  const uint32_t stage_bytes = row_bytes * (p.ds ? 3 : 2);
  // The tensor may end inside the last pack of its last row: that pack is not
  // copied, its owner reads the elements themselves.
  auto cut = [&](long long row) {
    return SHIFT && row * p.cols - first.head + static_cast<long long>(packs) * V > p.rows * p.cols;
  };
  auto fill = [&](int stage, long long row) {  // one thread
    if (row >= p.rows) return;
    const long long at = (row * p.cols - first.head) * static_cast<long long>(sizeof(T));
    const uint32_t bytes = cut(row) ? row_bytes - 16 : row_bytes;
    uint8_t* to = ring + stage * stage_bytes;
    mbar_arrive_expect_tx(&full[stage], bytes * (p.ds ? 3 : 2));
    bulk_load(to, static_cast<const uint8_t*>(p.dy) + at, bytes, &full[stage]);
    bulk_load(to + row_bytes, static_cast<const uint8_t*>(p.s) + at, bytes, &full[stage]);
    if (p.ds) bulk_load(to + 2 * row_bytes, static_cast<const uint8_t*>(p.ds) + at, bytes, &full[stage]);
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) mbar_init(&full[i], 1);
    *abort_flag = 0;
    fence_barrier_init();
    for (int i = 0; i < p.stages; ++i) fill(i, row0 + i * step);
  }
  // Pairs of columns: the arithmetic is on packed f32x2 instructions (the kernel
  // is bound by the instructions it issues, 67 % of the slots without them).
  constexpr int P = V / 2;
  float2 w[VPT][P], acc[VPT][P];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int k = static_cast<int>(threadIdx.x + i * blockDim.x);
    float f[V] = {};
    if (k < packs) first.weight(static_cast<const W*>(p.weight), k, f);
#pragma unroll
    for (int e = 0; e < P; ++e) {
      w[i][e] = make_float2(f[2 * e], f[2 * e + 1]);
      acc[i][e] = make_float2(0.0f, 0.0f);
    }
  }
  __syncthreads();
  const float inv = 1.0f / static_cast<float>(p.cols);
  int stage = 0, buf = 0;
  uint32_t parity = 0;
  float next_rstd = row0 < p.rows ? p.rstd[row0] : 0.0f;
  for (long long row = row0; row < p.rows; row += step) {
    const RowPacks<T, SHIFT> rp(row, p.cols);
    const float rstd = next_rstd;
    const float2 rstd2 = make_float2(rstd, rstd);
    if (row + step < p.rows) next_rstd = p.rstd[row + step];
    const bool ok = mbar_wait(&full[stage], parity, abort_flag, p.status, kErrTimeoutProducer);
    const uint4* at = reinterpret_cast<const uint4*>(ring + stage * stage_bytes);
    // Four packs stay as loaded and are taken apart twice: as f32, bf16 would need 32
    // registers more. The compiler reports 24 bytes of spills a thread for bf16 even
    // so (shifted 72), none for f32.
    constexpr bool kKeep = VPT <= 2;
    float2 g[kKeep ? VPT : 1][P], v[kKeep ? VPT : 1][P];
    uint4 dys[kKeep ? 1 : VPT], ss[kKeep ? 1 : VPT], ds[VPT];
    float2 dot2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int k = static_cast<int>(threadIdx.x + i * blockDim.x);
      if (k >= packs) continue;
      const int m = kKeep ? i : 0;
      uint4 a = at[k], b = at[packs + k];
      if (p.ds) ds[i] = at[2 * packs + k];
      if (SHIFT && first.edge(k)) {
        if (k + 1 == packs && cut(row)) {
          a = rp.load(static_cast<const T*>(p.dy), k);
          b = rp.load(static_cast<const T*>(p.s), k);
          if (p.ds) ds[i] = rp.load(static_cast<const T*>(p.ds), k);
        } else {
          a = first.masked(a, k);
          b = first.masked(b, k);
        }
      }
      if constexpr (!kKeep) dys[i] = a, ss[i] = b;
      pairs16<T>(a, g[m]);
      pairs16<T>(b, v[m]);
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float2 gv = __fmul2_rn(g[m][e], v[m][e]);
        dot2 = __ffma2_rn(gv, w[i][e], dot2);
        acc[i][e] = __ffma2_rn(gv, rstd2, acc[i][e]);
      }
    }
    float dot = dot2.x + dot2.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (lane_id() == 0) sums[buf][warp_id()] = dot;
    // Everybody has read the stage after this barrier, and knows whether it came.
    if (__syncthreads_or(!ok)) break;
    if (threadIdx.x == 0) fill(stage, row + p.stages * step);
    dot = static_cast<int>(lane_id()) < warps ? sums[buf][lane_id()] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    buf ^= 1;  // a warp may still be reading the other half
    const float c = -(dot * inv * rstd * rstd) * rstd;
    const float2 c2 = make_float2(c, c);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int k = static_cast<int>(threadIdx.x + i * blockDim.x);
      if (k >= packs) continue;
      const int m = kKeep ? i : 0;
      if constexpr (!kKeep) {
        pairs16<T>(dys[i], g[m]);
        pairs16<T>(ss[i], v[m]);
      }
      float2 d[P] = {};
      if (p.ds) pairs16<T>(ds[i], d);
#pragma unroll
      for (int e = 0; e < P; ++e) {
        d[e] = __ffma2_rn(v[m][e], c2, d[e]);
        d[e] = __ffma2_rn(__fmul2_rn(g[m][e], rstd2), w[i][e], d[e]);
      }
      rp.store(static_cast<T*>(p.dx), k, unpairs16<T>(d));
    }
    if (++stage == p.stages) {
      stage = 0;
      parity ^= 1;
    }
  }
  if (*abort_flag) {
    // A copy never came: let the others land before the shared memory goes.
    if (threadIdx.x == 0) {
      volatile int never = 0;
      for (int i = 0; i < p.stages; ++i)
        if (i != stage) mbar_wait(&full[i], i < stage ? parity ^ 1 : parity, &never, p.status, kErrTimeoutTeardown);
    }
    __syncthreads();
  }
  float* part = p.partial + blockIdx.x * static_cast<long long>(p.cols);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int k = static_cast<int>(threadIdx.x + i * blockDim.x);
    if (k >= packs) continue;
#pragma unroll
    for (int e = 0; e < P; ++e) {
      if (!SHIFT || first.inside(k, 2 * e)) part[k * V - first.head + 2 * e] = acc[i][e].x;
      if (!SHIFT || first.inside(k, 2 * e + 1)) part[k * V - first.head + 2 * e + 1] = acc[i][e].y;
    }
  }
}

// The pair of kernels for any width and alignment. dot_r = sum_j dy_j w_j s_j, a
// block per row.
template <typename T, typename W>
__global__ void __launch_bounds__(512) rmsnorm_bwd_dot_kernel(const BwdParams p) {
  wait_for_previous();
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
  wait_for_previous();
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

// dweight = sum of the chunks' parts, in a fixed order: 32 columns a block, 128
// threads along the chunks for each four of them, so that a thread's few loads
// are all in flight at once (with 32 threads along the chunks the sum of 296
// parts of 3584 columns took 7 us).
template <typename W>
__global__ void __launch_bounds__(1024) rmsnorm_dweight_kernel(const float* partial, W* dweight, int cols, int chunks) {
  wait_for_previous();
  __shared__ float part[128][33];
  const int tx = static_cast<int>(threadIdx.x & 7), ty = static_cast<int>(threadIdx.x >> 3);
  const int j = blockIdx.x * 32 + tx * 4;
  float acc[4] = {};
  if (j < cols) {
    const bool whole = cols % 4 == 0;  // every part's row then starts on the 16-byte grid
#pragma unroll 4
    for (int c = ty; c < chunks; c += 128) {
      const float* p = partial + c * static_cast<long long>(cols) + j;
      if (whole) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        acc[0] += v.x, acc[1] += v.y, acc[2] += v.z, acc[3] += v.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j + i < cols) acc[i] += p[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[ty][tx * 4 + i] = acc[i];
  __syncthreads();
  const int lane = static_cast<int>(lane_id()), k = static_cast<int>(warp_id());
  float sum = (part[lane][k] + part[lane + 32][k]) + (part[lane + 64][k] + part[lane + 96][k]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int col = blockIdx.x * 32 + k;
  if (lane == 0 && col < cols) dweight[col] = from_f32<W>(sum);
}

// The kernels step through a row's columns in ints, up to 1024 at a time.
constexpr int64_t kMaxCols = 0x7fffffffLL - 1024;
int check_cols(const char* what, int64_t cols) {
  if (cols > kMaxCols)
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "%s: at most %lld columns", what, (long long)kMaxCols);
  return SWIGLU_OK;
}

int check_norm(const char* what, int64_t rows, int64_t cols, int dtype, int weight_dtype) {
  if (int rc = check_dims(what, rows, cols, 0)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_dtype(weight_dtype)) return rc;
  if (cols == 0) return fail(SWIGLU_ERR_INVALID_ARGUMENT, "%s: a row must have at least one column", what);
  return check_cols(what, cols);
}

bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int threads_for(int64_t items, int most) {
  int64_t t = (items + 31) / 32 * 32;
  return static_cast<int>(t < 32 ? 32 : t > most ? most : t);
}

// Packs that a row touches at most, and the rows after which its offset on the
// 16-byte grid repeats.
template <typename T, bool SHIFT>
int64_t most_packs(int64_t cols) {
  return SHIFT ? (cols + 2 * kV<T> - 2) / kV<T> : cols / kV<T>;
}
template <typename T>
int row_period(int64_t cols) {
  int period = 1;
  while (period * cols % kV<T>) period *= 2;
  return period;
}

template <typename T, typename W, bool E4M3, int VPT, bool SHIFT>
bool launch_row(const FwdParams& p, cudaStream_t st) {
  const int64_t threads = (most_packs<T, SHIFT>(p.cols) + VPT - 1) / VPT;
  if (threads > kRowThreads) return false;
  const int x = threads_for(threads, kRowThreads);
  const dim3 block(x, x == 32 ? 4 : 1);
  const unsigned grid = static_cast<unsigned>((p.rows + block.y - 1) / block.y);
  launch_after(rmsnorm_fwd_row_kernel<T, W, E4M3, VPT, SHIFT>, grid, block, 0, st, p);
  return true;
}

// Packs a thread, in GB/s on one B200 (bf16, residual): 60000 x 512 one 6507, two
// 6420, four 5915 (e4m3 out 5099, 5972, 4616); 11136 x 3584 one 6054, two 6418,
// four 6368; 16384 x 8192 one 6126, two 6355, four 6824.
template <typename T, typename W, bool E4M3, bool SHIFT>
bool launch_rows(const FwdParams& p, cudaStream_t st) {
  return (p.cols <= 32 * kV<T> && launch_row<T, W, E4M3, 1, SHIFT>(p, st)) ||
         (p.cols <= 512 * kV<T> && launch_row<T, W, E4M3, 2, SHIFT>(p, st)) ||
         launch_row<T, W, E4M3, 4, SHIFT>(p, st);
}

// Tensors on the 16-byte grid move in packs, shifted ones where rows are no whole
// packs; tensors off the grid, and rows too long for a block's registers, take the
// looping kernel (11136 x 3584 e4m3: 135 us against 45).
template <typename T, typename W, bool E4M3>
int launch_fwd(const FwdParams& p, cudaStream_t st) {
  constexpr int V = kV<T>;
  const bool grid16 = aligned(p.x, 16) && aligned(p.residual, 16) && aligned(p.s, 16) && aligned(p.y, E4M3 ? V : 16);
  const bool whole = p.cols % V == 0 && aligned(p.weight, V * sizeof(W) < 16 ? V * sizeof(W) : 16);
  const bool done =
      grid16 && (whole ? launch_rows<T, W, E4M3, false>(p, st) : launch_rows<T, W, E4M3, true>(p, st));
  if (!done)
    launch_after(rmsnorm_fwd_any_kernel<T, W, E4M3>, static_cast<unsigned>(p.rows), threads_for(p.cols, 512), 0, st, p);
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

// Blocks the row kernel may have: two an SM at 8192 columns, eight from 2048 down.
int64_t most_bwd_blocks(int64_t rows, int64_t cols, int sms) {
  int64_t per_sm = 16384 / cols;
  per_sm = per_sm < 1 ? 1 : per_sm > 8 ? 8 : per_sm;
  return rows < per_sm * sms ? rows : per_sm * sms;
}

template <typename T, typename W, int VPT, bool SHIFT>
bool launch_bwd_row(BwdParams& p, const DeviceInfo& d, cudaStream_t st) {
  const int64_t threads = (most_packs<T, SHIFT>(p.cols) + VPT - 1) / VPT;
  if (threads > kBwdThreads) return false;
  const int x = threads_for(threads, kBwdThreads);
  const dim3 block(x, x == 32 && VPT == 1 ? 8 : 1);
  int per_sm = (kBwdLoadRegs<VPT> <= 12 ? 1024 : 512) / static_cast<int>(x * block.y);
  int64_t grid = static_cast<int64_t>(d.sms) * per_sm;
  const int64_t most = most_bwd_blocks(p.rows, p.cols, d.sms);
  if (grid > most) grid = most;
  p.period = SHIFT ? row_period<T>(p.cols) : 1;
  grid = grid / p.period * p.period;  // as many blocks for every residue class
  if (grid == 0) return false;
  // No more than one block for every blockDim.y rows of a class.
  const int64_t class_rows = (p.rows + p.period - 1) / p.period;
  const int64_t needed = (class_rows + block.y - 1) / block.y * p.period;
  p.chunks = static_cast<int>(grid > needed ? needed : grid);
  // Not placed early: the blocks, fewer than fit an SM, would gather on the SMs
  // that drain first (60000 x 512 bf16: 56 us against 78).
  rmsnorm_bwd_row_kernel<T, W, VPT, SHIFT><<<p.chunks, block, 0, st>>>(p);
  return true;
}

// At least two rows in the ring: 210 KB of shared memory an SM over the blocks its
// registers hold.
template <typename T, typename W, int VPT, bool SHIFT>
bool launch_bwd_ring(BwdParams& p, const DeviceInfo& d, cudaStream_t st) {
  const int64_t packs = most_packs<T, SHIFT>(p.cols), threads = (packs + VPT - 1) / VPT;
  // Fewer packs: registers. (60000 x 512 bf16, 64 packs: registers 55.8 us, ring
  // 67.2. Shifted bf16 rows favour the ring earlier: 40000 x 331 registers 98 us, ring
  // 75; f32 rows do not: 20000 x 501 31.5, 36.8.)
  const int fewest = SHIFT && sizeof(T) == 2 ? 40 : 128;
  if (packs < fewest || threads > kBwdThreads) return false;
  const int x = threads_for(threads, kBwdThreads);
  int64_t per_sm = kBwdThreads / x;
  const int64_t most = most_bwd_blocks(p.rows, p.cols, d.sms);
  if (per_sm * d.sms > most) per_sm = (most + d.sms - 1) / d.sms;
  const int64_t stage_bytes = packs * 16 * (p.ds ? 3 : 2);
  int64_t stages = 210 * 1024 / per_sm / stage_bytes;
  if (stages < 2) return false;
  p.stages = static_cast<int>(stages > kMaxStages ? kMaxStages : stages);
  int64_t grid = per_sm * d.sms < most ? per_sm * d.sms : most;
  p.period = SHIFT ? row_period<T>(p.cols) : 1;
  grid = grid / p.period * p.period;
  if (grid == 0 || p.rows < 3 * grid) return false;  // a ring pays once a block has several rows to go through
  p.chunks = static_cast<int>(grid);
  constexpr auto kern = rmsnorm_bwd_ring_kernel<T, W, VPT, SHIFT>;
  if (opt_in_smem<kern>(212 * 1024, "rmsnorm backward launch")) return false;
  launch_after(kern, p.chunks, x, p.stages * stage_bytes, st, p);
  return true;
}

template <typename T, typename W, bool SHIFT>
bool launch_bwd_rows(BwdParams& p, const DeviceInfo& d, cudaStream_t st) {
  // Two packs a thread first: 11136 x 3584 bf16 56.5 us (four 60.9; one took 59.5, and
  // no shape that two packs refuse).
  return launch_bwd_ring<T, W, 2, SHIFT>(p, d, st) || launch_bwd_ring<T, W, 4, SHIFT>(p, d, st) ||
         launch_bwd_row<T, W, 1, SHIFT>(p, d, st) || launch_bwd_row<T, W, 2, SHIFT>(p, d, st) ||
         launch_bwd_row<T, W, 4, SHIFT>(p, d, st);
}

template <typename T, typename W>
int launch_bwd(BwdParams& p, const DeviceInfo& d, cudaStream_t st) {
  constexpr int V = kV<T>;
  const bool grid16 = aligned(p.dy, 16) && aligned(p.s, 16) && aligned(p.ds, 16) && aligned(p.dx, 16);
  const bool whole = p.cols % V == 0 && aligned(p.weight, V * sizeof(W) < 16 ? V * sizeof(W) : 16);
  const int chunks = p.chunks;
  const bool done =
      grid16 && (whole ? launch_bwd_rows<T, W, false>(p, d, st) : launch_bwd_rows<T, W, true>(p, d, st));
  if (!done) p.chunks = chunks;
  if (!done) {
    launch_after(rmsnorm_bwd_dot_kernel<T, W>, static_cast<unsigned>(p.rows), threads_for(p.cols, 512), 0, st, p);
    launch_after(rmsnorm_bwd_cols_kernel<T, W>, dim3((p.cols + 255) / 256, p.chunks), 256, 0, st, p);
  }
  launch_after(rmsnorm_dweight_kernel<W>, (p.cols + 31) / 32, 1024, 0, st, p.partial,
               static_cast<W*>(p.dweight), p.cols, p.chunks);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, "rmsnorm backward launch");
}

// Floats of the workspace: the rows' dots (a multiple of four), then the parts of
// dweight of whichever kernels run.
int64_t dot_floats(int64_t rows) { return (rows + 3) / 4 * 4; }
int64_t bwd_floats(int64_t rows, int64_t cols, int sms) {
  if (rows == 0) return 0;
  int chunks, per;
  plan_bwd(rows, cols, sms, &chunks, &per);
  const int64_t blocks = most_bwd_blocks(rows, cols, sms);
  return dot_floats(rows) + (blocks > chunks ? blocks : chunks) * cols;
}

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
  if (workspace_floats < bwd_floats(rows, cols, d->sms))
    return fail(SWIGLU_ERR_INVALID_ARGUMENT, "rmsnorm_bwd: workspace of %lld floats, %lld needed",
                (long long)workspace_floats, (long long)bwd_floats(rows, cols, d->sms));
  p.status = d->status;
  p.dot = workspace;
  p.partial = workspace + dot_floats(rows);
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
  if (int rc = check_cols("rmsnorm_bwd_workspace", cols)) return rc;
  *floats = bwd_floats(rows, cols, num_sms);
  return SWIGLU_OK;
}

int swiglu_b200_rmsnorm_bwd(const void* dy, const void* s, const void* weight, const float* rstd, const void* ds,
                            void* dx, void* dweight, float* workspace, int64_t workspace_floats, int64_t rows,
                            int64_t cols, int dtype, int weight_dtype, void* stream) {
  BwdParams p{dy, s, weight, rstd, ds, dx, nullptr, nullptr, dweight, 0, 0, 0, 0, 1, 0, nullptr};
  return op_rmsnorm_bwd(p, rows, cols, dtype, weight_dtype, workspace, workspace_floats,
                        static_cast<cudaStream_t>(stream));
}

}  // extern "C"
