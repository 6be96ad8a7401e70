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
// before it is rounded to x's type.  A row goes to a warp (up to 1024 columns) or to a CTA of
// 256 to 1024 threads; a CTA walks over rows and loads the next one before it works on this one, so that
// loads are in flight during the reductions.  Where rows start on 16 bytes a thread takes runs of eight
// consecutive columns: 16-byte accesses, and a group of 128 columns on 16 neighbouring lanes, whose
// shuffles find its amax.  Otherwise consecutive threads take consecutive columns, a warp's 32 at a
// time, and a group's amax is that of its slices of 32.
#include "common.cuh"

#include <cuda_fp8.h>

#include <algorithm>

namespace musc {
namespace rms {

constexpr int RUN = 8;        // consecutive columns of a thread
constexpr int MAX_CHANNELS = 32768;
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

__device__ __forceinline__ float reciprocal(float x) {  // of a scale: off by 2^-23, e4m3 rounds at 2^-4
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Column of a thread's value i of run r.
template <bool VEC>
__device__ __forceinline__ int column(int r, int i, int tid, int threads) {
  return VEC ? (r * threads + tid) * RUN + i : (r * RUN + i) * threads + tid;
}

// A run as it lies in memory.
template <typename T>
struct Raw {
  uint4 w[sizeof(T) * RUN / 16];
};

template <typename E, bool VEC>
__device__ __forceinline__ void load_run(Raw<E>& raw, const E* row, int r, int tid, int threads, int channels) {
  if (VEC) {
    const uint4* src = reinterpret_cast<const uint4*>(row + column<VEC>(r, 0, tid, threads));
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) raw.w[i] = src[i];
  } else {
    E* v = reinterpret_cast<E*>(raw.w);
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
      const int c = column<VEC>(r, i, tid, threads);
      v[i] = c < channels ? row[c] : E(0.f);
    }
  }
}

template <typename E>
__device__ __forceinline__ void widen(const Raw<E>& raw, float (&v)[RUN]) {
  const E* t = reinterpret_cast<const E*>(raw.w);
#pragma unroll
  for (int i = 0; i < RUN; ++i) v[i] = static_cast<float>(t[i]);
}

template <typename E>
__device__ __forceinline__ E narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename E, bool VEC>
__device__ __forceinline__ void store_run(E* row, int r, int tid, int threads, int channels, const float (&v)[RUN]) {
  if (VEC) {
    Raw<E> raw;
    E* t = reinterpret_cast<E*>(raw.w);
#pragma unroll
    for (int i = 0; i < RUN; ++i) t[i] = narrow<E>(v[i]);
    uint4* dst = reinterpret_cast<uint4*>(row + column<VEC>(r, 0, tid, threads));
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) dst[i] = raw.w[i];
  } else {
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
      const int c = column<VEC>(r, i, tid, threads);
      if (c < channels) row[c] = narrow<E>(v[i]);
    }
  }
}

// Eight values of e4m3, each value times its factor (one factor for a run of consecutive columns).
template <bool VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* row, int r, int tid, int threads, int channels, const float (&v)[RUN],
                                           const float (&factor)[RUN]) {
  uint2 raw;
  __nv_fp8x2_storage_t* t = reinterpret_cast<__nv_fp8x2_storage_t*>(&raw);
#pragma unroll
  for (int i = 0; i < RUN / 2; ++i)
    t[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * factor[2 * i], v[2 * i + 1] * factor[2 * i + 1]), __NV_SATFINITE,
                                    __NV_E4M3);
  if (VEC) {
    *reinterpret_cast<uint2*>(row + column<VEC>(r, 0, tid, threads)) = raw;
  } else {
    const uint8_t* b = reinterpret_cast<const uint8_t*>(&raw);
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
      const int c = column<VEC>(r, i, tid, threads);
      if (c < channels) row[c] = b[i];
    }
  }
}

// Reduction over a row's threads: a warp, or the whole CTA through shared memory.
template <bool WARP, typename Op>
__device__ __forceinline__ float row_reduce(float v, Op op, float* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (WARP) return v;
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
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

// A row is a warp's, WARP_ROWS rows a CTA, or a CTA's; a thread has at most RUNS runs of it.
// CTAs that fit an SM, by which the compiler bounds the registers of a thread.  A vectorised row of a
// warp: three of 128 threads with the weights in registers (5480 rows of 1024 in 12.0 us; with four, or
// with the weights read again for every row, 13 us).  A vectorised row of a CTA: 64 registers, so that
// two of 512 fit, weights read again (16389 rows of 4096 in 75 us; with 83 registers and the weights kept 93 us).
template <bool VEC, int T>
constexpr int MIN_CTAS = T == 0 || T == 512 ? 2 : T == 1024 ? 1 : T == 256 ? 4 : 3;

// T: threads of a row, 0: the CTA's, at most 512.
template <typename XT, typename DT, bool VEC, int T, int RUNS>
__global__ void __launch_bounds__(T == 32 ? 32 * WARP_ROWS : T ? T : 512, MIN_CTAS<VEC, T>) add_rmsnorm_kernel(const Params p) {
  constexpr bool WARP = T == 32;
  __shared__ float shared[2][2][32];  // [parity of the row][sum or amax][warp]
  __shared__ float slice_top[VEC ? 1 : (WARP ? WARP_ROWS : 1)][VEC ? 1 : (WARP ? 32 : 1024)];  // of 32 columns; then of groups
  const int threads = T ? T : blockDim.x;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int sub = WARP ? threadIdx.x >> 5 : 0;
  const long long step = WARP ? (long long)gridDim.x * WARP_ROWS : (long long)gridDim.x;
  long long row = WARP ? (long long)blockIdx.x * WARP_ROWS + sub : (long long)blockIdx.x;
  const auto mine = [&](int r) { return column<VEC>(r, 0, tid, threads) < p.channels; };  // the run has a column of the row
  Raw<XT> next_x[RUNS];
  Raw<DT> next_d[RUNS];
  const auto load = [&](long long at) {
    const XT* x = static_cast<const XT*>(p.x) + at * p.x_stride;
    const DT* d = static_cast<const DT*>(p.delta) + at * p.delta_stride;
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
      if (mine(r)) load_run<XT, VEC>(next_x[r], x, r, tid, threads, p.channels);
    if (p.delta) {
#pragma unroll
      for (int r = 0; r < RUNS; ++r)
        if (mine(r)) load_run<DT, VEC>(next_d[r], d, r, tid, threads, p.channels);
    }
  };
  constexpr bool AHEAD = VEC && (RUNS == 2 || WARP);  // elsewhere registers for a second row would cost more than it gives
  if (AHEAD && row < p.rows) load(row);
  constexpr bool KEEP = VEC && WARP;  // the thread's weights, the same for every row
  Raw<float> weight[KEEP ? RUNS : 1];
  if (KEEP) {
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
      if (mine(r)) load_run<float, VEC>(weight[KEEP ? r : 0], p.weight, r, tid, threads, p.channels);
  }
  for (int parity = 0; row < p.rows; row += step, parity ^= 1) {  // uniform over a row's threads
    if (!AHEAD) load(row);
    float v[RUNS][RUN];
    XT* x = static_cast<XT*>(p.x) + row * p.x_stride;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
      if (mine(r)) {
        widen(next_x[r], v[r]);
        if (p.delta) {
          float d[RUN];
          widen(next_d[r], d);
#pragma unroll
          for (int i = 0; i < RUN; ++i) v[r][i] += d[i];
          store_run<XT, VEC>(x, r, tid, threads, p.channels, v[r]);
        }
#pragma unroll
        for (int i = 0; i < RUN; ++i) sum = fmaf(v[r][i], v[r][i], sum);
      } else {
#pragma unroll
        for (int i = 0; i < RUN; ++i) v[r][i] = 0.f;
      }
    }
    if (AHEAD && row + step < p.rows) load(row + step);
    sum = row_reduce<WARP>(sum, [](float a, float b) { return a + b; }, shared[parity][0]);
    const float rstd = rsqrtf(sum / (float)p.channels + p.eps);
    float top = 0.f;  // of the row
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
      if (mine(r)) {
        if (!KEEP) load_run<float, VEC>(weight[0], p.weight, r, tid, threads, p.channels);
        float w[RUN];
        widen(weight[KEEP ? r : 0], w);
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
          v[r][i] = v[r][i] * rstd * w[i];
          if (!VEC && column<VEC>(r, i, tid, threads) >= p.channels) v[r][i] = 0.f;  // no value, also where rstd is not finite
        }
        const long long at = row * p.out_stride;
        if (p.out_dtype == MUSC_B200_F32) store_run<float, VEC>(static_cast<float*>(p.out) + at, r, tid, threads, p.channels, v[r]);
        else if (p.out_dtype == MUSC_B200_F16) store_run<__half, VEC>(static_cast<__half*>(p.out) + at, r, tid, threads, p.channels, v[r]);
        else if (p.out_dtype == MUSC_B200_BF16) store_run<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16*>(p.out) + at, r, tid, threads, p.channels, v[r]);
#pragma unroll
        for (int i = 0; i < RUN; ++i) top = fmaxf(top, fabsf(v[r][i]));
      }
    }
    if (p.out_dtype != MUSC_B200_E4M3) continue;
    uint8_t* out = static_cast<uint8_t*>(p.out) + row * p.out_stride;
    float* scales = p.scales + row * p.groups;
    const auto scale_of = [](float m) { return fmaxf(m * (1.f / E4M3_MAX), MIN_SCALE); };
    float factor[RUN];
    if (p.group == 0) {
      top = row_reduce<WARP>(top, [](float a, float b) { return fmaxf(a, b); }, shared[parity][1]);
      const float scale = scale_of(top);
      if (tid == 0) scales[0] = scale;
#pragma unroll
      for (int i = 0; i < RUN; ++i) factor[i] = reciprocal(scale);
#pragma unroll
      for (int r = 0; r < RUNS; ++r)
        if (mine(r)) store_e4m3<VEC>(out, r, tid, threads, p.channels, v[r], factor);
    } else if (VEC) {
      const int lanes = p.group / RUN;  // 4 to 32 neighbouring lanes hold a group
#pragma unroll
      for (int r = 0; r < RUNS; ++r) {
        if (r * threads * RUN >= p.channels) break;  // uniform over the row's threads
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < RUN; ++i) m = fmaxf(m, fabsf(v[r][i]));
        for (int o = lanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float scale = scale_of(m);
        if (mine(r)) {
          if (tid % lanes == 0) scales[column<VEC>(r, 0, tid, threads) / p.group] = scale;
#pragma unroll
          for (int i = 0; i < RUN; ++i) factor[i] = reciprocal(scale);
          store_e4m3<VEC>(out, r, tid, threads, p.channels, v[r], factor);
        }
      }
    } else {
      // Slice k, columns 32 k to 32 k + 31, is a warp's; a group is group / 32 slices.
      const int warps = threads >> 5, warp = tid >> 5, lane = tid & 31;
#pragma unroll
      for (int r = 0; r < RUNS; ++r)
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
          const float m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(v[r][i]), 0.f))));
          if (lane == 0) slice_top[sub][(r * RUN + i) * warps + warp] = m;
        }
      const int in_group = p.group / 32, slices = RUNS * RUN * warps;
      const auto sync = [] {
        if (WARP) __syncwarp();
        else __syncthreads();
      };
      sync();
      // A thread's share of the groups: scales out, reciprocals in the place of each group's first slice.
      for (int g = tid; g < p.groups; g += threads) {
        float m = 0.f;
        for (int k = g * in_group; k < min((g + 1) * in_group, slices); ++k) m = fmaxf(m, slice_top[sub][k]);
        const float scale = scale_of(m);
        scales[g] = scale;
        slice_top[sub][g * in_group] = reciprocal(scale);
      }
      sync();
#pragma unroll
      for (int r = 0; r < RUNS; ++r) {
#pragma unroll
        for (int i = 0; i < RUN; ++i) factor[i] = slice_top[sub][((r * RUN + i) * warps + warp) & ~(in_group - 1)];
        store_e4m3<VEC>(out, r, tid, threads, p.channels, v[r], factor);
      }
      sync();  // the next row's slices come after these have been read
    }
  }
}

constexpr int THREADS_PER_SM = 4096;  // of a grid: about two waves

template <typename XT, typename DT, bool VEC, int T, int RUNS>
int launch_as(const Params& p, int threads, cudaStream_t s) {
  const long long ctas = T == 32 ? (p.rows + WARP_ROWS - 1) / WARP_ROWS : p.rows;
  // As many rows for every CTA, few enough CTAs that most of them walk over several.
  const long long most = (long long)sm_count() * std::max(1, THREADS_PER_SM / threads);
  const long long each = (ctas + most - 1) / most;
  add_rmsnorm_kernel<XT, DT, VEC, T, RUNS><<<(unsigned)((ctas + each - 1) / each), threads, 0, s>>>(p);
  return check_launch("add_rmsnorm_kernel");
}

template <typename XT, typename DT, bool VEC>
int launch_rows(const Params& p, cudaStream_t s) {
  if (p.channels <= 32 * 4 * RUN) return launch_as<XT, DT, VEC, 32, 4>(p, 32 * WARP_ROWS, s);
  const int runs = (p.channels + RUN - 1) / RUN;
  if constexpr (VEC) {
    if (runs <= 2 * 512) return launch_as<XT, DT, VEC, 0, 2>(p, ((runs + 1) / 2 + 31) / 32 * 32, s);
  } else {  // a column of its own for every value: their distances are constants
    if (runs <= 2 * 256) return launch_as<XT, DT, VEC, 256, 2>(p, 256, s);
    if (runs <= 2 * 512) return launch_as<XT, DT, VEC, 512, 2>(p, 512, s);
  }
  if (runs <= 2 * 1024) return launch_as<XT, DT, VEC, 1024, 2>(p, 1024, s);
  return launch_as<XT, DT, VEC, 1024, 4>(p, 1024, s);
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
  if (rows < 0 || rows > 0x7FFFFFFFLL || channels <= 0 || channels > MAX_CHANNELS)
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
  if (eight && sc.at % 4 != 0) return fail(MUSC_B200_ERR_INVALID, "add_rmsnorm: scales must be aligned to 4 bytes");
  if (meet(so, sx) || meet(so, sw) || (delta && meet(sx, sw)) || (delta && (meet(so, sd) || meet(sx, sd))) ||
      (eight && (meet(sc, sx) || meet(sc, so) || meet(sc, sw) || (delta && meet(sc, sd)))))
    return fail(MUSC_B200_ERR_INVALID, "add_rmsnorm: x, delta, weight, out and scales must not overlap");
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
