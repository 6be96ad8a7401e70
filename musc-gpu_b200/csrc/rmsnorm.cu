// Residual add + root-mean-square norm, the norm of blocks that keep no mean:
//
//   h[row] = x[row] + delta[row]              (kept in x, rounded to x's type)
//   y[row] = h / sqrt(mean(h^2) + eps) * weight
//
// with y in 32 or 16 bits or in e4m3 with one scale for a row or for a group of its columns
// (scale = amax |y| / 448, stored values = y / scale).  It stands beside add_layernorm
// (models/backbone/open_clip/transformer.py:236-249 has the blocks' residual adds).
//
// One read of x and delta, one write of x and y: memory bounds it.  A row's sums of squares
// and h itself stay in 32 bits and in registers between the two uses, so h is normalised
// before it is rounded to x's type.  A row goes to as many threads as give each at most four
// runs of eight columns (a warp up to 1024 columns); eight columns of a run are consecutive,
// which makes a 16-byte access of them and keeps a group of 128 columns on 16 neighbouring
// lanes, whose shuffles find its amax.
#include "common.cuh"

#include <cuda_fp8.h>

namespace musc {
namespace rms {

constexpr int RUN = 8;        // consecutive columns of a thread
constexpr int MAX_RUNS = 4;   // runs of a thread: 32 values in registers
constexpr int MAX_THREADS = 1024;
constexpr int WARP_ROWS = 4;  // rows of a CTA where a row is one warp's
constexpr float E4M3_MAX = 448.0f;
constexpr float MIN_SCALE = 1.17549435e-38f;  // 2^-126: its reciprocal is finite, rows of zeros stay zeros

struct Params {
  void* x;
  const void* delta;
  const float* weight;
  void* out;
  float* scales;
  long long rows, x_stride, delta_stride, out_stride;
  int channels, group, groups;  // group 0: one scale for the row
  int out_dtype;
  float eps;
};

// Eight columns from c on, those past the row as zeros.
template <typename T, bool VEC>
__device__ __forceinline__ void load_run(const T* row, int c, int channels, float (&v)[RUN]) {
  if (VEC) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 raw = *reinterpret_cast<const uint4*>(row + c);
      const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < RUN; ++i) v[i] = static_cast<float>(t[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < RUN; ++i) v[i] = c + i < channels ? static_cast<float>(row[c + i]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, bool VEC>
__device__ __forceinline__ void store_run(T* row, int c, int channels, const float (&v)[RUN]) {
  if (VEC) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(row + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 raw;
      T* t = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int i = 0; i < RUN; ++i) t[i] = narrow<T>(v[i]);
      *reinterpret_cast<uint4*>(row + c) = raw;
    }
  } else {
#pragma unroll
    for (int i = 0; i < RUN; ++i)
      if (c + i < channels) row[c + i] = narrow<T>(v[i]);
  }
}

template <bool VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* row, int c, int channels, const float (&v)[RUN], float factor) {
  uint2 raw;
  __nv_fp8x2_storage_t* t = reinterpret_cast<__nv_fp8x2_storage_t*>(&raw);
#pragma unroll
  for (int i = 0; i < RUN / 2; ++i)
    t[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * factor, v[2 * i + 1] * factor), __NV_SATFINITE, __NV_E4M3);
  if (VEC) {
    *reinterpret_cast<uint2*>(row + c) = raw;
  } else {
    const uint8_t* b = reinterpret_cast<const uint8_t*>(&raw);
#pragma unroll
    for (int i = 0; i < RUN; ++i)
      if (c + i < channels) row[c + i] = b[i];
  }
}

// Reduction over a row's threads: a warp, or the whole CTA through shared memory.
template <bool WARP, typename Op>
__device__ __forceinline__ float row_reduce(float v, Op op, float* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (WARP) return v;
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[lane < warps ? lane : 0];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_down_sync(0xffffffffu, v, o);
    if (lane + o < warps) v = op(v, other);
  }
  return __shfl_sync(0xffffffffu, v, 0);
}

// WARP: a row is one warp's, WARP_ROWS rows a CTA; otherwise a row is the CTA's.
template <typename XT, typename DT, bool VEC, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * WARP_ROWS : MAX_THREADS) add_rmsnorm_kernel(const Params p) {
  __shared__ float shared[2][32];
  const long long row = WARP ? (long long)blockIdx.x * WARP_ROWS + (threadIdx.x >> 5) : (long long)blockIdx.x;
  if (row >= p.rows) return;  // uniform over a row's threads
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int step = (WARP ? 32 : blockDim.x) * RUN;
  XT* x = static_cast<XT*>(p.x) + row * p.x_stride;
  const DT* delta = static_cast<const DT*>(p.delta) + row * p.delta_stride;
  float v[MAX_RUNS][RUN];
  float sum = 0.f;
#pragma unroll
  for (int r = 0; r < MAX_RUNS; ++r) {
    const int c = r * step + tid * RUN;
    if (c < p.channels) load_run<XT, VEC>(x, c, p.channels, v[r]);
  }
  if (p.delta) {
#pragma unroll
    for (int r = 0; r < MAX_RUNS; ++r) {
      const int c = r * step + tid * RUN;
      if (c < p.channels) {
        float d[RUN];
        load_run<DT, VEC>(delta, c, p.channels, d);
#pragma unroll
        for (int i = 0; i < RUN; ++i) v[r][i] += d[i];
        store_run<XT, VEC>(x, c, p.channels, v[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < MAX_RUNS; ++r) {
    if (r * step + tid * RUN < p.channels) {
#pragma unroll
      for (int i = 0; i < RUN; ++i) sum = fmaf(v[r][i], v[r][i], sum);
    }
  }
  sum = row_reduce<WARP>(sum, [](float a, float b) { return a + b; }, shared[0]);
  const float rstd = rsqrtf(sum / (float)p.channels + p.eps);
  float top = 0.f;  // of the row
#pragma unroll
  for (int r = 0; r < MAX_RUNS; ++r) {
    const int c = r * step + tid * RUN;
    if (c < p.channels) {
      float w[RUN];
      load_run<float, VEC>(p.weight, c, p.channels, w);
#pragma unroll
      for (int i = 0; i < RUN; ++i) v[r][i] = v[r][i] * rstd * w[i];
      if (p.out_dtype == MUSC_B200_F32) store_run<float, VEC>(static_cast<float*>(p.out) + row * p.out_stride, c, p.channels, v[r]);
      else if (p.out_dtype == MUSC_B200_F16) store_run<__half, VEC>(static_cast<__half*>(p.out) + row * p.out_stride, c, p.channels, v[r]);
      else if (p.out_dtype == MUSC_B200_BF16) store_run<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16*>(p.out) + row * p.out_stride, c, p.channels, v[r]);
    } else {
#pragma unroll
      for (int i = 0; i < RUN; ++i) v[r][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < RUN; ++i) top = fmaxf(top, fabsf(v[r][i]));
  }
  if (p.out_dtype != MUSC_B200_E4M3) return;
  uint8_t* out = static_cast<uint8_t*>(p.out) + row * p.out_stride;
  float* scales = p.scales + row * p.groups;
  if (p.group == 0) {
    top = row_reduce<WARP>(top, [](float a, float b) { return fmaxf(a, b); }, shared[1]);
    const float scale = fmaxf(top / E4M3_MAX, MIN_SCALE);
    if (tid == 0) scales[0] = scale;
#pragma unroll
    for (int r = 0; r < MAX_RUNS; ++r) {
      const int c = r * step + tid * RUN;
      if (c < p.channels) store_e4m3<VEC>(out, c, p.channels, v[r], 1.0f / scale);
    }
  } else {
    const int lanes = p.group / RUN;  // 4 to 32 neighbouring lanes hold a group
#pragma unroll
    for (int r = 0; r < MAX_RUNS; ++r) {
      const int c = r * step + tid * RUN;
      if (r * step >= p.channels) break;  // uniform over the row's threads
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < RUN; ++i) m = fmaxf(m, fabsf(v[r][i]));
      for (int o = lanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float scale = fmaxf(m / E4M3_MAX, MIN_SCALE);
      if (c < p.channels) {
        if (tid % lanes == 0) scales[c / p.group] = scale;
        store_e4m3<VEC>(out, c, p.channels, v[r], 1.0f / scale);
      }
    }
  }
}

template <typename XT, typename DT, bool VEC>
int launch_rows(const Params& p, cudaStream_t s) {
  if (p.channels <= 32 * RUN * MAX_RUNS) {
    const long long grid = (p.rows + WARP_ROWS - 1) / WARP_ROWS;
    add_rmsnorm_kernel<XT, DT, VEC, true><<<(unsigned)grid, 32 * WARP_ROWS, 0, s>>>(p);
  } else {
    int threads = 64;
    while (threads * RUN * MAX_RUNS < p.channels) threads *= 2;
    add_rmsnorm_kernel<XT, DT, VEC, false><<<(unsigned)p.rows, threads, 0, s>>>(p);
  }
  return check_launch("add_rmsnorm_kernel");
}

template <typename XT>
int launch_delta(const Params& p, int delta_dtype, bool vec, cudaStream_t s) {
  if (delta_dtype == MUSC_B200_F32) return vec ? launch_rows<XT, float, true>(p, s) : launch_rows<XT, float, false>(p, s);
  if (delta_dtype == MUSC_B200_F16) return vec ? launch_rows<XT, __half, true>(p, s) : launch_rows<XT, __half, false>(p, s);
  return vec ? launch_rows<XT, __nv_bfloat16, true>(p, s) : launch_rows<XT, __nv_bfloat16, false>(p, s);
}

int size_of(int dtype) { return dtype == MUSC_B200_F32 ? 4 : dtype == MUSC_B200_E4M3 ? 1 : 2; }

}  // namespace rms
}  // namespace musc

using namespace musc;

extern "C" int musc_b200_add_rmsnorm(void* x, int x_dtype, const void* delta, int delta_dtype, const float* weight,
                                     float eps, void* out, int out_dtype, float* scales, int group, long long rows,
                                     int channels, long long x_stride, long long delta_stride, long long out_stride,
                                     musc_b200_stream stream) {
  using namespace rms;
  const auto wide = [](int t) { return t == MUSC_B200_F32 || t == MUSC_B200_F16 || t == MUSC_B200_BF16; };
  if (!wide(x_dtype) || (delta && !wide(delta_dtype)))
    return fail(MUSC_B200_ERR_INVALID, "add_rmsnorm: x and delta must be f32, f16 or bf16");
  if (!wide(out_dtype) && out_dtype != MUSC_B200_E4M3)
    return fail(MUSC_B200_ERR_INVALID, "add_rmsnorm: out dtype must be f32, f16, bf16 or e4m3");
  if (rows < 0 || rows > 0x7FFFFFFFLL || channels <= 0 || channels > MAX_THREADS * RUN * MAX_RUNS)
    return fail(MUSC_B200_ERR_INVALID, "add_rmsnorm: 0 <= rows < 2^31 and 1 <= channels <= 32768");
  if (!(eps >= 0.f)) return fail(MUSC_B200_ERR_INVALID, "add_rmsnorm: eps must not be negative");
  if (group != 0 && (out_dtype != MUSC_B200_E4M3 || (group != 32 && group != 64 && group != 128 && group != 256)))
    return fail(MUSC_B200_ERR_INVALID, "add_rmsnorm: group must be 0 (the row), or 32, 64, 128 or 256 for an e4m3 output");
  if (rows == 0) return MUSC_B200_OK;
  if (!x || !weight || !out || (out_dtype == MUSC_B200_E4M3 && !scales))
    return fail(MUSC_B200_ERR_INVALID, "add_rmsnorm: null pointer");
  if (rows > 1 && (x_stride < channels || out_stride < channels || (delta && delta_stride < channels)))
    return fail(MUSC_B200_ERR_INVALID, "add_rmsnorm: row strides must hold a row's channels");
  struct Span {
    uintptr_t at;
    long long bytes, stride;
    int size;
  };
  const auto span = [&](const void* ptr, long long stride, int size) {
    return Span{reinterpret_cast<uintptr_t>(ptr), ((rows - 1) * stride + channels) * size, rows > 1 ? stride * size : 0, size};
  };
  const Span sx = span(x, x_stride, size_of(x_dtype)), so = span(out, out_stride, size_of(out_dtype));
  const Span sw = {reinterpret_cast<uintptr_t>(weight), channels * 4LL, 0, 4};
  const Span sd = delta ? span(delta, delta_stride, size_of(delta_dtype)) : sx;
  bool vec = channels % RUN == 0;
  for (const Span& s : {sx, so, sw, sd}) {
    const int align = s.size == 1 ? 8 : 16;  // of a run: eight bytes of e4m3, 16-byte vectors else
    if (s.at % s.size != 0) return fail(MUSC_B200_ERR_INVALID, "add_rmsnorm: pointers must be aligned to their element");
    vec = vec && s.at % align == 0 && s.stride % align == 0;
  }
  const auto meet = [](const Span& a, const Span& b) {
    return a.at < b.at + (uintptr_t)b.bytes && b.at < a.at + (uintptr_t)a.bytes;
  };
  const Span sc = {reinterpret_cast<uintptr_t>(scales), rows * 4 * (group ? (channels + group - 1) / group : 1), 0, 4};
  const bool eight = out_dtype == MUSC_B200_E4M3;
  if (meet(so, sx) || (delta && (meet(so, sd) || meet(sx, sd))) ||
      (eight && (meet(sc, sx) || meet(sc, so) || (delta && meet(sc, sd)))))
    return fail(MUSC_B200_ERR_INVALID, "add_rmsnorm: x, delta, out and scales must not overlap");
  MUSC_TRY(require_sm100());
  Params p;
  p.x = x, p.delta = delta, p.weight = weight, p.out = out, p.scales = scales;
  p.rows = rows, p.x_stride = x_stride, p.delta_stride = delta_stride, p.out_stride = out_stride;
  p.channels = channels, p.group = group, p.groups = group ? (channels + group - 1) / group : 1;
  p.out_dtype = out_dtype, p.eps = eps;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (x_dtype == MUSC_B200_F32) return launch_delta<float>(p, delta_dtype, vec, s);
  if (x_dtype == MUSC_B200_F16) return launch_delta<__half>(p, delta_dtype, vec, s);
  return launch_delta<__nv_bfloat16>(p, delta_dtype, vec, s);
}
