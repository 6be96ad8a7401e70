// Masked attention of few query rows against many keys (masked.cuh has the operator): one
// CTA per query row, key head and split of the row's keys.
//
// A row's keys and values are read once for all query heads of their group, and nothing else
// is large: memory bounds it.  The group's heads are the 16 rows of the tensor core's
// m16n8k16 products (a larger group takes several CTAs): S = Q K^T over 16 keys and the head
// dimension, then O += P V, at 2 x 16 x 16 x D operations per 64 D bytes far below what the
// tensor cores give.  Each of the CTA's warps takes every WARPS-th run of 16 keys through a
// ring of its own that cp.async fills STAGES runs ahead, so no barrier stands between a
// warp's loads and their use; keys past the row's interval are filled with zeros by the copy
// itself (a masked value that is NaN never reaches a product).  The warps' and the splits'
// sums are joined at the end by their maxima: up to eight splits form a cluster and read each
// other's sums from shared memory (one launch, no workspace), more leave theirs to combine_kernel.
#include "masked.cuh"
#include "tc.cuh"

#include <algorithm>

namespace musc {
namespace masked {
namespace {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int KEYS = 16;    // keys of a warp's step
constexpr int STAGES = 2;   // steps in flight per warp: WARPS x STAGES x 64 D bytes a CTA
constexpr int HEADS = 16;   // query heads of a CTA
// Splits.  Three waves of what is resident (148 SMs x 3 CTAs) even out documents of differing lengths:
// 32 tokens over 8192 keys in 116 us, 132 with one wave.  Where several rows of a document read its keys
// from L2, one wave keeps them together: 2 rows over 6390 keys in 32 us, 38 with three.
constexpr int TARGET_SINGLE = 1332, TARGET_SEVERAL = 444;
constexpr int MIN_KEYS = 256;       // of a split: 465 keys in one take 15 us, in two 21
constexpr int CLUSTER_KEYS = 4096;  // more keys per split than this, and more than a cluster's splits are taken
constexpr float RESCALE = 8.f;  // log2 by which a running maximum may lag behind before sums are rescaled

template <int D>
struct Smem {
  union {
    uint4 ring[WARPS][STAGES][2][KEYS * D / 8];  // K and V rows of a step, 16-byte chunks swizzled by row
    float o[WARPS][HEADS][D + 4];
  };
  float ml[WARPS][HEADS][2];
  float sums[HEADS][D];        // of the CTA, for its cluster
  float2 sums_ml[HEADS];
};

__device__ __forceinline__ uint32_t cluster_address(const void* p, uint32_t rank) {
  return tc::mapa(tc::smem_u32(p), rank);
}
__device__ __forceinline__ float2 load_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <bool FP16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (FP16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool FP16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (FP16) {
    __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&t);
  }
  __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&t);
}

// Eight finished dimensions of a head.
template <bool FP16>
__device__ __forceinline__ void store_eight(const Params& p, long long row, int column, const float (&acc)[8], float inv) {
  uint4 packed;
  packed.x = pack2<FP16>(acc[0] * inv, acc[1] * inv), packed.y = pack2<FP16>(acc[2] * inv, acc[3] * inv);
  packed.z = pack2<FP16>(acc[4] * inv, acc[5] * inv), packed.w = pack2<FP16>(acc[6] * inv, acc[7] * inv);
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * p.out_stride + column) = packed;
}

template <int D, bool FP16, bool CLUSTER>
__global__ void __launch_bounds__(THREADS) rows_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>(smem_raw);
  constexpr int CHUNKS = D / 8;  // 16-byte chunks of a key
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Neighbouring CTAs take neighbouring rows: those of one document share its keys in L2.
  long long unit = blockIdx.x / p.splits;
  const int split = (int)(blockIdx.x - unit * p.splits);
  const long long row = unit % p.q_rows;
  unit /= p.q_rows;
  const int kv_head = (int)(unit % p.kv_heads), block = (int)(unit / p.kv_heads);
  const int head0 = kv_head * p.group + block * HEADS;
  const int n_heads = min(HEADS, p.group - block * HEADS);
  const int doc = find_document_warp(p, row);
  if (doc < 0) return;  // uniform over the CTA and its cluster
  const Interval iv = row_interval(p, doc, row);
  // This split's share of the interval, in whole steps.
  const long long steps = (iv.hi - iv.lo + KEYS - 1) / KEYS;
  const long long first = steps * split / p.splits, last = steps * (split + 1) / p.splits;
  const uint16_t* k_base = static_cast<const uint16_t*>(p.k) + kv_head * D;
  const uint16_t* v_base = static_cast<const uint16_t*>(p.v) + kv_head * D;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(&sm.ring[warp][0][0][0]));
  constexpr uint32_t HALF = KEYS * D * 2;  // bytes of a step's K (or V)
  // The warp's i-th step is step first + warp + i * WARPS.
  const auto load = [&](long long step, int stage) {
    if (step < last) {
      const long long key0 = iv.lo + step * KEYS;
#pragma unroll
      for (int i = 0; i < KEYS * CHUNKS / 32; ++i) {
        const int c = i * 32 + lane, key = c / CHUNKS, chunk = c % CHUNKS;
        const bool take = key0 + key < iv.hi;
        const long long at = take ? key0 + key : iv.lo;
        const uint32_t dst = ring + stage * 2 * HALF + key * (D * 2) + ((chunk ^ (key & 7)) << 4);
        cp_async16(dst, k_base + at * p.k_stride + chunk * 8, take);
        cp_async16(dst + HALF, v_base + at * p.v_stride + chunk * 8, take);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load(first + warp + s * WARPS, s);

  // Query heads as the A operand: row r = head0 + r, zeros past the group.
  uint32_t qa[D / 16][4];
  {
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + row * p.q_stride + (long long)head0 * D;
    const int r = lane >> 2, c = (lane & 3) * 2;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      const uint16_t* a = q + r * D + t * 16 + c;
      const uint16_t* b = a + 8 * D;
      qa[t][0] = r < n_heads ? *reinterpret_cast<const uint32_t*>(a) : 0u;
      qa[t][1] = r + 8 < n_heads ? *reinterpret_cast<const uint32_t*>(b) : 0u;
      qa[t][2] = r < n_heads ? *reinterpret_cast<const uint32_t*>(a + 8) : 0u;
      qa[t][3] = r + 8 < n_heads ? *reinterpret_cast<const uint32_t*>(b + 8) : 0u;
    }
  }
  const bool capped = p.cap > 0.f;
  const float scale2 = p.scale * LOG2E, cap2 = p.cap * LOG2E;
  const float factor = capped ? p.scale / p.cap : 0.f;
  float slope2[2] = {0.f, 0.f};
  if (p.slopes) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = (lane >> 2) + 8 * h;
      if (r < n_heads) slope2[h] = __ldg(p.slopes + head0 + r) * LOG2E;
    }
  }

  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // rows lane / 4 and lane / 4 + 8; l of this lane's keys
  int stage = 0;
  for (long long step = first + warp; step < last; step += WARPS) {
    load(step + (STAGES - 1) * WARPS, (stage + STAGES - 1) % STAGES);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const uint32_t kt = ring + stage * 2 * HALF, vt = kt + HALF;
    float s[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      // matrices: keys 0-7 and 8-15 of dims 16 t .. 16 t + 7, then of the next eight dims
      const int key = (lane & 7) + ((lane >> 3) & 1) * 8, chunk = t * 2 + (lane >> 4);
      uint32_t b[4];
      ldmatrix4(b, kt + key * (D * 2) + ((chunk ^ (key & 7)) << 4));
      mma16816<FP16>(s[0], qa[t], b[0], b[2]);
      mma16816<FP16>(s[1], qa[t], b[1], b[3]);
    }
    // Scores of keys key0 + {0, 1} and key0 + 8 + {0, 1}, key0 of this lane.
    const long long key0 = iv.lo + step * KEYS + (lane & 3) * 2;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const long long key = key0 + n * 8 + (e & 1);
        float z = capped ? capped_log2(s[n][e], factor, cap2) : s[n][e] * scale2;
        if (p.slopes) z = fmaf(-slope2[e >> 1], (float)llabs(key - iv.pos), z);
        z = key < iv.hi ? z : -INFINITY;
        s[n][e] = z;
        top[e >> 1] = fmaxf(top[e >> 1], z);
      }
    bool rescale = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      rescale = rescale || top[h] > m[h] + RESCALE;
    }
    if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float m_new = fmaxf(m[h], top[h]);
        const float a = m[h] == -INFINITY ? 0.f : ex2(m[h] - m_new);
        m[h] = m_new;
        l[h] *= a;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[n][2 * h] *= a, o[n][2 * h + 1] *= a;
      }
    }
    float e[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ref = m[i >> 1] == -INFINITY ? 0.f : m[i >> 1] - RAISE<FP16>;
        e[n][i] = ex2(s[n][i] - ref);
        l[i >> 1] += e[n][i];
      }
    const uint32_t pa[4] = {pack2<FP16>(e[0][0], e[0][1]), pack2<FP16>(e[0][2], e[0][3]),
                            pack2<FP16>(e[1][0], e[1][1]), pack2<FP16>(e[1][2], e[1][3])};
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      // matrices: keys 0-7 and 8-15 of dims 16 t .. 16 t + 7, then of the next eight dims
      const int key = (lane & 7) + ((lane >> 3) & 1) * 8, chunk = t * 2 + (lane >> 4);
      uint32_t b[4];
      ldmatrix4_trans(b, vt + key * (D * 2) + ((chunk ^ (key & 7)) << 4));
      mma16816<FP16>(o[2 * t], pa, b[0], b[1]);
      mma16816<FP16>(o[2 * t + 1], pa, b[2], b[3]);
    }
    __syncwarp();  // every lane is done with the stage that the next step's load fills
    stage = (stage + 1) % STAGES;
  }
  cp_async_wait<0>();
  __syncthreads();  // the rings' memory becomes the warps' sums
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    const int r = (lane >> 2) + 8 * h;
    if ((lane & 3) == 0) sm.ml[warp][r][0] = m[h], sm.ml[warp][r][1] = l[h];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      *reinterpret_cast<float2*>(&sm.o[warp][r][n * 8 + (lane & 3) * 2]) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n_heads * (D / 8); e += THREADS) {
    const int r = e / (D / 8), d = e % (D / 8) * 8;
    float common = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) common = fmaxf(common, sm.ml[w][r][0]);
    float acc[8], total = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = split_weight(sm.ml[w][r][0], common);
      total = fmaf(f, sm.ml[w][r][1], total);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = fmaf(f, sm.o[w][r][d + i], acc[i]);
    }
    if (CLUSTER) {
      if (d == 0) sm.sums_ml[r] = partial_ml(common, total, iv.hi > iv.lo);
#pragma unroll
      for (int i = 0; i < 8; ++i) sm.sums[r][d + i] = acc[i];
    } else if (p.splits == 1) {
      store_eight<FP16>(p, row, (head0 + r) * D + d, acc, inverse_sum(total, iv.hi > iv.lo));
    } else {
      const long long at = (split * p.q_rows + row) * p.heads + head0 + r;
      if (d == 0) p.part_ml[at] = partial_ml(common, total, iv.hi > iv.lo);
      if (total != 0.f) {
        *reinterpret_cast<float4*>(p.part + at * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        *reinterpret_cast<float4*>(p.part + at * D + d + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      }
    }
  }
  if (CLUSTER) {
    // Every CTA of the cluster joins its share of the heads' dimensions, eight at a time.
    tc::cluster_sync();
    for (int e = split * THREADS + threadIdx.x; e < n_heads * (D / 8); e += p.splits * THREADS) {
      const int r = e / (D / 8), d = e % (D / 8) * 8;
      float2 ml[MAX_CLUSTER];
      float common = -INFINITY, total = 0.f, acc[8];
#pragma unroll
      for (int c = 0; c < MAX_CLUSTER; ++c) {
        ml[c] = c < p.splits ? load_cluster2(cluster_address(&sm.sums_ml[r], c)) : make_float2(-INFINITY, 0.f);
        common = fmaxf(common, ml[c].x);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll
      for (int c = 0; c < MAX_CLUSTER; ++c) {
        const float f = split_weight(ml[c].x, common);
        total = fmaf(f, ml[c].y, total);
        if (c >= p.splits || ml[c].y == 0.f) continue;
        const uint32_t from = cluster_address(&sm.sums[r][d], c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 o = load_cluster2(from + i * 8);
          acc[2 * i] = fmaf(f, o.x, acc[2 * i]), acc[2 * i + 1] = fmaf(f, o.y, acc[2 * i + 1]);
        }
      }
      store_eight<FP16>(p, row, (head0 + r) * D + d, acc, inverse_sum(total, common != -INFINITY));
    }
    tc::cluster_sync();  // no CTA leaves while another reads its sums
  }
}

template <int D, bool FP16, bool CLUSTER>
int launch_as(const Params& p, long long grid, cudaStream_t s) {
  constexpr auto kernel = rows_kernel<D, FP16, CLUSTER>;
  MUSC_TRY(opt_in_smem<kernel>(sizeof(Smem<D>)));
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)grid);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = sizeof(Smem<D>);
  config.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CLUSTER ? p.splits : 1;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = CLUSTER ? 1 : 0;
  MUSC_CUDA(cudaLaunchKernelEx(&config, kernel, p));
  return MUSC_B200_OK;
}

template <int D, bool FP16>
int launch(const Params& p, cudaStream_t s) {
  const long long grid = p.q_rows * p.kv_heads * ((p.group + HEADS - 1) / HEADS) * p.splits;
  if (grid > 0x7FFFFFFFLL) return fail(MUSC_B200_ERR_INVALID, "masked_attention: too many rows and heads");
  if (p.splits > 1 && p.splits <= MAX_CLUSTER) return launch_as<D, FP16, true>(p, grid, s);
  return launch_as<D, FP16, false>(p, grid, s);
}

}  // namespace

int rows_splits(long long units, long long keys, bool single) {
  const long long target = single ? TARGET_SINGLE : TARGET_SEVERAL;
  const long long want = (target + units - 1) / units;
  const long long splits = std::max<long long>(1, std::min<long long>(std::min<long long>(want, keys / MIN_KEYS), 64));
  return (int)(splits > MAX_CLUSTER && keys <= MAX_CLUSTER * CLUSTER_KEYS ? MAX_CLUSTER : splits);
}

int rows_launch(const Params& p, int head_dim, bool fp16, cudaStream_t s) {
  if (head_dim == 64) return fp16 ? launch<64, true>(p, s) : launch<64, false>(p, s);
  return fp16 ? launch<128, true>(p, s) : launch<128, false>(p, s);
}

}  // namespace masked
}  // namespace musc
