// Masked attention of few query rows against many keys (masked.cuh has the operator): one
// CTA per block of rows of a document, key head and split of the keys.
//
// Keys and values are read once for a block's rows and all query heads of their group, and nothing
// else is large: memory bounds it.  The group's heads, for as many consecutive rows of a document as fit
// (5 rows over 2985 keys of 20 requests, 8/2 heads x 128, in 24.5 us, 35 when each row read the keys for itself), are the
// 16 rows of the tensor core's m16n8k16 products (a larger group takes several CTAs): S = Q K^T over 16
// keys and the head dimension, then O += P V, at 2 x 16 x 16 x D operations per 64 D bytes far below
// what the tensor cores give.  Each of the CTA's warps takes every WARPS-th run of 16 keys through a
// ring of its own that cp.async fills STAGES runs ahead, so no barrier stands between a
// warp's loads and their use; keys past the rows' interval are filled with zeros by the copy
// itself (a masked value that is NaN never reaches a product).  Under a causal mask the last keys
// (fewer than 16) are seen by some of the block's rows only: they are a step of their own, and if a value
// there is not finite the block's rows are taken again key by key.  The warps' and the splits'
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
constexpr int HEADS = 16;   // rows of the products: rows x query heads of a CTA
constexpr int MAX_SPLITS = 64;  // combine_kernel's two a lane
constexpr float RESCALE = 8.f;  // log2 by which a running maximum may lag behind before sums are rescaled

// CTAs of an SM: 73 KB of shared memory at D = 128, 128 registers a thread at D = 64.
template <int D>
constexpr int RESIDENT = D == 64 ? 4 : 3;

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

// Eight finished dimensions of a head.
template <bool FP16>
__device__ __forceinline__ void store_eight(const Params& p, long long row, int column, const float (&acc)[8], float inv) {
  uint4 packed;
  packed.x = pack2<FP16>(acc[0] * inv, acc[1] * inv), packed.y = pack2<FP16>(acc[2] * inv, acc[3] * inv);
  packed.z = pack2<FP16>(acc[4] * inv, acc[5] * inv), packed.w = pack2<FP16>(acc[6] * inv, acc[7] * inv);
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * p.out_stride + column) = packed;
}

// Document and first row of a block of rows, by a converged warp; -1: it holds no row.  The lanes count the
// documents whose blocks begin at or before this one.
template <bool SEVERAL>
__device__ __forceinline__ int find_block(const Params& p, long long block, long long& row) {
  const int size = SEVERAL ? p.block_rows : 1;
  if (!p.q_offsets) {
    const int per_doc = (int)((p.q_len + size - 1) / size), doc = (int)(block / per_doc);
    row = doc * p.q_len + (block - (long long)doc * per_doc) * size;
    return doc;
  }
  const auto begin = [&](int d) {
    const int first = row_offset(p, d);
    return SEVERAL ? (long long)(first / size) + d : (long long)first;
  };
  int doc;  // the last document that begins at or before the block
  if (p.documents > 1024) {
    int lo = -1, hi = p.documents;  // begin(lo) <= block < begin(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (begin(mid) <= block) lo = mid;
      else hi = mid;
    }
    doc = lo;
  } else {  // one load's time
    const int lane = threadIdx.x & 31;
    int before = 0;
#pragma unroll 8
    for (int i = lane; i < p.documents; i += 32) before += begin(i) <= block ? 1 : 0;
    doc = (int)__reduce_add_sync(0xffffffffu, before) - 1;
  }
  if (doc < 0) return -1;
  row = SEVERAL ? row_offset(p, doc) + (block - begin(doc)) * size : block;
  return row >= 0 && row < row_offset(p, doc + 1) ? doc : -1;  // below 0: offsets out of order
}

// The form with clusters keeps the compiler's own choice of registers (168 at D = 128): with the bound that the form
// without them needs (170 registers else, two CTAs an SM), 32 tokens over 8192 keys take 1.5 % longer.
template <int D, bool FP16, bool CLUSTER, bool SEVERAL>
__global__ void __launch_bounds__(THREADS, CLUSTER ? 0 : RESIDENT<D>) rows_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>(smem_raw);
  constexpr int CHUNKS = D / 8;  // 16-byte chunks of a key
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Neighbouring CTAs take neighbouring rows: those of one document share its keys in L2.
  long long unit = blockIdx.x / p.splits;
  const int split = (int)(blockIdx.x - unit * p.splits);
  const long long row_block = unit % p.row_blocks;
  unit /= p.row_blocks;
  const int kv_head = (int)(unit % p.kv_heads), block = (int)(unit / p.kv_heads);
  const int head0 = kv_head * p.group + block * HEADS;
  const int n_heads = min(HEADS, p.group - block * HEADS);
  long long row;
  const int doc = find_block<SEVERAL>(p, row_block, row);
  if (doc < 0) return;  // uniform over the CTA and its cluster
  const Interval iv = row_interval(p, doc, row);
  const int n_tokens = SEVERAL ? (int)min((long long)p.block_rows, iv.rows_left) : 1;
  const int n_rows = n_tokens * n_heads;  // row r: token r / n_heads, head r % n_heads
  // Keys that all of them see, in whole steps; then those that only the later ones do (fewer than a step).
  const int lo = (int)iv.lo, common = (int)iv.hi, end = (int)interval_end(p, iv, n_tokens - 1);
  const int main_steps = (common - lo + KEYS - 1) / KEYS, steps = main_steps + (SEVERAL && end > common ? 1 : 0);
  const int first = (int)((long long)steps * split / p.splits), last = (int)((long long)steps * (split + 1) / p.splits);
  const auto step_key = [&](int step) { return !SEVERAL || step < main_steps ? lo + step * KEYS : common; };
  const uint16_t* k_base = static_cast<const uint16_t*>(p.k) + kv_head * D;
  const uint16_t* v_base = static_cast<const uint16_t*>(p.v) + kv_head * D;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(&sm.ring[warp][0][0][0]));
  constexpr uint32_t HALF = KEYS * D * 2;  // bytes of a step's K (or V)
  // The warp's i-th step is step first + warp + i * WARPS.
  const auto load = [&](int step, int stage) {
    if (step < last) {
      const int key0 = step_key(step), stop = !SEVERAL || step < main_steps ? common : end;
#pragma unroll
      for (int i = 0; i < KEYS * CHUNKS / 32; ++i) {
        const int c = i * 32 + lane, key = c / CHUNKS, chunk = c % CHUNKS;
        const bool take = key0 + key < stop;
        const long long at = take ? key0 + key : lo;
        const uint32_t dst = ring + stage * 2 * HALF + key * (D * 2) + ((chunk ^ (key & 7)) << 4);
        cp_async16(dst, k_base + at * p.k_stride + chunk * 8, take);
        cp_async16(dst + HALF, v_base + at * p.v_stride + chunk * 8, take);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load(first + warp + s * WARPS, s);

  // Queries as the A operand, zeros past the last row.  This lane's rows are lane / 4 and lane / 4 + 8.
  int token[2], head[2];
  const uint16_t* q_row[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = (lane >> 2) + 8 * h;
    token[h] = SEVERAL ? r / n_heads : 0;
    head[h] = r - token[h] * n_heads;
    q_row[h] = r < n_rows ? static_cast<const uint16_t*>(p.q) + (row + token[h]) * p.q_stride + (long long)(head0 + head[h]) * D
                          : nullptr;
  }
  uint32_t qa[D / 16][4];
#pragma unroll
  for (int t = 0; t < D / 16; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t* at = q_row[i & 1];
      qa[t][i] = at ? *reinterpret_cast<const uint32_t*>(at + t * 16 + (lane & 3) * 2 + (i >> 1) * 8) : 0u;
    }
  const bool capped = p.cap > 0.f;
  const float scale2 = p.scale * LOG2E, cap2 = p.cap * LOG2E;
  const float factor = capped ? p.scale / p.cap : 0.f;
  float slope2[2] = {0.f, 0.f};
  if (p.slopes) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (q_row[h]) slope2[h] = __ldg(p.slopes + head0 + head[h]) * LOG2E;
  }
  const int own_end[2] = {(int)interval_end(p, iv, token[0]), (int)interval_end(p, iv, token[1])};

  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // rows lane / 4 and lane / 4 + 8; l of this lane's keys
  int stage = 0;
  bool redo = false;
  for (int step = first + warp; step < last; step += WARPS) {
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
    const int key0 = step_key(step) + (lane & 3) * 2;
    const bool tail = SEVERAL && step >= main_steps;
    const int stop[2] = {tail ? own_end[0] : common, tail ? own_end[1] : common};
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + n * 8 + (e & 1);
        float z = capped ? capped_log2(s[n][e], factor, cap2) : s[n][e] * scale2;
        if (p.slopes) z = fmaf(-slope2[e >> 1], (float)llabs(key - iv.pos - token[e >> 1]), z);
        z = key < stop[e >> 1] ? z : -INFINITY;
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
      if (tail) {  // values that are not finite, beside rows that do not see them: exponent bits all ones
        constexpr uint32_t EXP = FP16 ? 0x7C007C00u : 0x7F807F80u, UNIT = FP16 ? 0x04000400u : 0x00800080u;
        if ((((b[0] & EXP) + UNIT) | ((b[1] & EXP) + UNIT) | ((b[2] & EXP) + UNIT) | ((b[3] & EXP) + UNIT)) & 0x80008000u)
          redo = true;
      }
      mma16816<FP16>(o[2 * t], pa, b[0], b[1]);
      mma16816<FP16>(o[2 * t + 1], pa, b[2], b[3]);
    }
    __syncwarp();  // every lane is done with the stage that the next step's load fills
    stage = (stage + 1) % STAGES;
  }
  cp_async_wait<0>();
  // The rings' memory becomes the warps' sums.
  if (SEVERAL) redo = __syncthreads_or(redo);
  else __syncthreads();
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
  if (redo) {
    // The rows again, each by a warp, over the keys of this split that it sees.
    constexpr int N = D / 32;
    for (int r = warp; r < n_rows; r += WARPS) {
      const int t = SEVERAL ? r / n_heads : 0, h = head0 + r - t * n_heads;
      const uint16_t* q = static_cast<const uint16_t*>(p.q) + (row + t) * p.q_stride + (long long)h * D + lane * N;
      float qf[N], acc[N], m_row = -INFINITY, l_row = 0.f;
      for (int i = 0; i < N; ++i) qf[i] = widen<FP16>(q[i]), acc[i] = 0.f;
      const float slope = p.slopes ? __ldg(p.slopes + h) * LOG2E : 0.f;
      const int main_last = min(last, main_steps);
      const int own = (int)interval_end(p, iv, t);
      if (first < main_last)
        attend_keys<D, FP16>(p, qf, kv_head, slope, iv.pos + t, step_key(first), min(step_key(main_last - 1) + KEYS, common), acc,
                             m_row, l_row);
      if (last > main_steps)
        attend_keys<D, FP16>(p, qf, kv_head, slope, iv.pos + t, step_key(max(first, main_steps)), own, acc, m_row, l_row);
      for (int w = 0; w < WARPS; ++w) {  // in the place of the first warp's sums; those carry RAISE
        for (int i = 0; i < N; ++i) sm.o[w][r][lane * N + i] = w == 0 ? acc[i] : 0.f;
        if (lane == 0) sm.ml[w][r][0] = w == 0 ? m_row + RAISE<FP16> : -INFINITY, sm.ml[w][r][1] = w == 0 ? l_row : 0.f;
      }
    }
    __syncthreads();
  }
  for (int e = threadIdx.x; e < n_rows * (D / 8); e += THREADS) {
    const int r = e / (D / 8), d = e % (D / 8) * 8;
    const int t = SEVERAL ? r / n_heads : 0, h = head0 + r - t * n_heads;
    const bool any_key = interval_end(p, iv, t) > lo;
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
      if (d == 0) sm.sums_ml[r] = partial_ml(common, total, any_key);
#pragma unroll
      for (int i = 0; i < 8; ++i) sm.sums[r][d + i] = acc[i];
    } else if (p.splits == 1) {
      store_eight<FP16>(p, row + t, h * D + d, acc, inverse_sum(total, any_key));
    } else {
      const long long at = (split * p.q_rows + row + t) * p.heads + h;
      if (d == 0) p.part_ml[at] = partial_ml(common, total, any_key);
      if (total != 0.f) {
        *reinterpret_cast<float4*>(p.part + at * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        *reinterpret_cast<float4*>(p.part + at * D + d + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      }
    }
  }
  if (CLUSTER) {
    // Every CTA of the cluster joins its share of the heads' dimensions, eight at a time.
    tc::cluster_sync();
    for (int e = split * THREADS + threadIdx.x; e < n_rows * (D / 8); e += p.splits * THREADS) {
      const int r = e / (D / 8), d = e % (D / 8) * 8, t = SEVERAL ? r / n_heads : 0;
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
      store_eight<FP16>(p, row + t, (head0 + r - t * n_heads) * D + d, acc, inverse_sum(total, common != -INFINITY));
    }
    tc::cluster_sync();  // no CTA leaves while another reads its sums
  }
}

template <int D, bool FP16, bool CLUSTER, bool SEVERAL>
int launch_as(const Params& p, long long grid, cudaStream_t s) {
  constexpr auto kernel = rows_kernel<D, FP16, CLUSTER, SEVERAL>;
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
  const long long grid = p.row_blocks * p.kv_heads * ((p.group + HEADS - 1) / HEADS) * p.splits;
  if (grid > 0x7FFFFFFFLL) return fail(MUSC_B200_ERR_INVALID, "masked_attention: too many rows and heads");
  const bool cluster = p.splits > 1 && p.splits <= MAX_CLUSTER;
  if (p.block_rows > 1)
    return cluster ? launch_as<D, FP16, true, true>(p, grid, s) : launch_as<D, FP16, false, true>(p, grid, s);
  return cluster ? launch_as<D, FP16, true, false>(p, grid, s) : launch_as<D, FP16, false, false>(p, grid, s);
}

}  // namespace

int rows_together(int group, bool several) { return several ? std::max(1, HEADS / group) : 1; }

// Splits of the keys of `units` blocks of rows: those whose time is least, by a model in keys' times
// (9 ns at D = 128) fitted to 18 shapes in 1 to 8 splits, of which it takes one within 7 % of the best.
// A CTA takes its keys, 128 to start and 20 a row for the join, once for each wave of them; a split 20
// more, the grid 130 for each fill of the GPU, and more splits than a cluster's eight a second launch
// that reads them all.
// At D = 128, bf16, keys and values of three calls in turn:
//   2 rows over 6390 keys of 7 requests, 8 key heads (56 units): 392 CTAs 35.0 us, 448 (444 are resident) 48.1
//   1 row over 553 keys of 12 requests, 16/2 heads (24 units): in one split 9.7 us, in two 8.7, in five 7.6
//   15 rows over 450 keys of 7 requests, 8 key heads (56 units): 11.2 us in one, 11.6 in two, 17.8 in seven
//   4 rows over 20000 keys of 2 requests, 16/4 heads (8 units): 41.9 us in eight, 33.6 in sixteen
//   1 row over 60000 keys, 8 key heads (8 units): 56 us in sixteen, 51 in 32, 58 in 52
int rows_splits(long long units, long long keys, int rows, int head_dim) {
  const long long resident = 148LL * (head_dim == 64 ? RESIDENT<64> : RESIDENT<128>);
  int best = 1;
  double least = 0;
  for (int splits = 1; splits <= MAX_SPLITS; ++splits) {
    const long long ctas = units * splits, waves = (ctas + resident - 1) / resident;
    const double time = (double)waves * (128 + (keys + splits - 1) / splits + (splits > 1 ? 20 * rows : 0)) +
                        130 * ctas / resident + (splits > MAX_CLUSTER ? 450 + 40 * splits : 20 * splits);
    if (splits == 1 || time < least) least = time, best = splits;
  }
  return best;
}

int rows_launch(const Params& p, int head_dim, bool fp16, cudaStream_t s) {
  if (head_dim == 64) return fp16 ? launch<64, true>(p, s) : launch<64, false>(p, s);
  return fp16 ? launch<128, true>(p, s) : launch<128, false>(p, s);
}

}  // namespace masked
}  // namespace musc
