// Masked attention of many query rows (masked.cuh has the operator): fused tcgen05 attention
// over tiles of 256 query rows x 128 keys.
//
// One CTA per (256 consecutive rows of the packed queries, head, split of the keys), 384
// threads.  Its rows need not belong to one document: every row carries its own key interval,
// and the CTA walks the union of its documents' intervals in tiles of 128 keys, so many
// short documents share a tile and a long one pays nothing for the generality.
//   warps 0-3, 4-7  softmax of query rows 0-127 and 128-255 (the two halves), one thread
//                   per row: S out of tensor memory, cap, bias, mask, running maximum and
//                   sum in 32 bits, P rounded to 16 bits back into tensor memory over S;
//   warp 8          TMA: Q once, K and V tiles through a ring;
//   warp 9          one thread issues tcgen05.mma: S_h = Q_h K^T (128 x 128 x D, both from
//                   shared memory) and O_h += P_h V (128 x D x 128, P from tensor memory).
// While one half's softmax runs, the tensor cores work for the other: the exponentials
// (16 a cycle and SM: 1024 cycles for 128 x 128) bound the kernel for D = 64 (256 cycles of
// products at the tensor cores' rate) and for D = 128 (512).  O stays in tensor memory and is
// rescaled only when a row's maximum has risen by more than 2^8 over the one in use.
//
// A masked probability is zero, but zero times a NaN or infinite value is NaN.  Keys that no
// row of the CTA sees (behind a document's last key) are zeroed in V's tile.  In tiles that a
// warp's rows see only in part the warp looks for such values in V, and where there is one
// recomputes its rows key by key at the end, skipping what they do not see: rare, slow, right.
#include "masked.cuh"
#include "tc.cuh"

#include <algorithm>
#include <mutex>

namespace musc {
namespace masked {
namespace {

constexpr int BQ = 128;    // query rows of a half (TMEM lanes)
constexpr int ROWS = 2 * BQ;
constexpr int BKV = 128;   // keys of a tile
constexpr int BLOCK_BYTES = 128 * 128;  // 128 rows x 64 elements, one swizzle block
constexpr int SOFTMAX_WARPS = 8;
constexpr int THREADS = 32 * (SOFTMAX_WARPS + 4);  // three warpgroups; two warps of the last idle
// Registers of a thread: 168 at launch (65536 / 384), of which the copying and issuing
// warpgroup gives back what the softmax ones take: 2 x 208 + 88 = 3 x 168.
constexpr int SOFTMAX_REGS = 208, OTHER_REGS = 88;
constexpr int TMEM_COLS = 512;
constexpr int S_COL = 0;     // S (and P over its first half) at columns 0 and 128
constexpr int O_COL = 256;   // O at columns 256 and 256 + D
constexpr float RESCALE = 8.f;
constexpr int SHARED_DOCS = 1024;  // offsets searched in shared memory up to this many documents
constexpr uint64_t WAIT_LIMIT_NS = 2000000000ull;

template <int D> constexpr int STAGES = D == 64 ? 4 : 2;

template <int D>
struct Smem {
  uint8_t q[2][D / 64][BLOCK_BYTES];
  uint8_t k[STAGES<D>][D / 64][BLOCK_BYTES];
  uint8_t v[STAGES<D>][D / 64][BLOCK_BYTES];
  uint64_t q_full;
  uint64_t k_full[STAGES<D>], k_empty[STAGES<D>];
  uint64_t v_full[STAGES<D>], v_empty[STAGES<D>];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t drain;
  union {
    int offsets[SHARED_DOCS + 1];  // while the rows' documents are looked up
    int2 segments[ROWS];           // then: key ranges [x, y) that the CTA walks
  };
  int lo[ROWS], hi[ROWS], doc[ROWS];
  uint32_t starts[ROWS / 32];      // rows that begin another document than the row before
  int hull[2][2];                  // per half: first key and end of all its rows' keys
  int n_segments, n_tiles;
  uint32_t tmem_base;
  int abort_flag;
};
template <int D> constexpr size_t SMEM_BYTES = sizeof(Smem<D>) + 1024;

__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* err) {
  if (tc::mbar_try_wait(bar, parity)) return true;
  const uint64_t start = global_ns();
  uint32_t iter = 0;
  while (true) {
    if (tc::mbar_try_wait(bar, parity)) return true;
    if ((++iter & 255u) == 0) {
      if (*abort_flag) return false;
      if (global_ns() - start > WAIT_LIMIT_NS) {
        *abort_flag = 1;
        atomicExch(err, MUSC_B200_ERR_TIMEOUT);
        return false;
      }
    }
  }
}

// V as the MN-major B operand in the 128-byte swizzle: 8-key groups 1024 bytes apart, blocks of
// 64 dims BLOCK_BYTES apart.
__device__ __forceinline__ uint64_t desc_v(uint32_t smem_addr) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | ((uint64_t)(BLOCK_BYTES >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
template <bool FP16> constexpr uint32_t idesc_qk() { return tc::idesc_f16(BQ, BKV, FP16 ? 0 : 1); }
template <int D, bool FP16> constexpr uint32_t idesc_pv() {
  return tc::idesc_f16(BQ, D, FP16 ? 0 : 1) | (1u << 16);  // B (V) MN-major
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

template <bool FP16>
__device__ __forceinline__ float widen(uint16_t v) {
  return FP16 ? __half2float(__ushort_as_half(v)) : __bfloat162float(__ushort_as_bfloat16(v));
}

// The tiles [first, first + left) of the CTA's walk over its segments.
struct Walk {
  const int2* segments;
  int segment, x, left;
  __device__ Walk(const int2* s, int first, int last) : segments(s), segment(0), left(last - first) {
    while (left > 0) {
      const int tiles = (s[segment].y - s[segment].x + BKV - 1) / BKV;
      if (first < tiles) break;
      first -= tiles;
      ++segment;
    }
    x = left > 0 ? s[segment].x + first * BKV : 0;
  }
  // Next tile: keys [begin, end), end - begin <= BKV.
  __device__ bool next(int& begin, int& end) {
    if (left <= 0) return false;
    --left;
    begin = x;
    const int stop = segments[segment].y;
    end = min(x + BKV, stop);
    x += BKV;
    if (x >= stop && left > 0) x = segments[++segment].x;
    return true;
  }
};

// The slow form of a warp's 32 rows, key by key over the CTA's tiles: lanes hold D / 32
// dimensions each.  row_lo .. row_pos: this lane's own row.
template <int D, bool FP16>
__device__ __forceinline__ void rows_key_by_key(const Params& p, const int2* segments, int first, int last, long long row0,
                                             int head, int row_lo, int row_hi, int row_pos, bool row_valid, int split) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const int kv_head = head / p.group;
  const float slope2 = p.slopes ? __ldg(p.slopes + head) * LOG2E : 0.f;
  for (int r = 0; r < 32; ++r) {
    const int lo = __shfl_sync(0xffffffffu, row_lo, r), hi = __shfl_sync(0xffffffffu, row_hi, r);
    const int pos = __shfl_sync(0xffffffffu, row_pos, r);
    if (!__shfl_sync(0xffffffffu, (int)row_valid, r)) continue;
    const long long row = row0 + r;
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + row * p.q_stride + (long long)head * D + lane * N;
    float qf[N], acc[N], m = -INFINITY, l = 0.f;
    for (int i = 0; i < N; ++i) qf[i] = widen<FP16>(q[i]), acc[i] = 0.f;
    Walk walk(segments, first, last);
    int begin, end;
    while (walk.next(begin, end)) {
      for (int key = max(begin, lo); key < min(end, hi); ++key) {
        const uint16_t* k = static_cast<const uint16_t*>(p.k) + key * p.k_stride + kv_head * D + lane * N;
        const uint16_t* v = static_cast<const uint16_t*>(p.v) + key * p.v_stride + kv_head * D + lane * N;
        float dot = 0.f;
        for (int i = 0; i < N; ++i) dot = fmaf(qf[i], widen<FP16>(k[i]), dot);
        dot = warp_sum(dot);
        float z = p.cap > 0.f ? capped_log2(dot, 2.f * LOG2E * p.scale / p.cap, p.cap * LOG2E) : dot * p.scale * LOG2E;
        if (p.slopes) z = fmaf(-slope2, fabsf((float)(key - pos)), z);
        const float m_new = fmaxf(m, z);
        const float a = m == -INFINITY ? 0.f : ex2(m - m_new);
        m = m_new;
        // a key whose score is -inf or has no weight left adds nothing, NaN scores add NaN
        const float e = z == -INFINITY ? 0.f : ex2(z - m);
        l = fmaf(l, a, e);
        for (int i = 0; i < N; ++i) acc[i] = fmaf(e, widen<FP16>(v[i]), acc[i] * a);
      }
    }
    const long long at = (split * p.q_rows + row) * p.heads + head;
    if (p.splits == 1) {
      const float inv = inverse_sum(l, hi > lo);
      uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.out_stride + (long long)head * D + lane * N;
      for (int i = 0; i < N; ++i) out[i] = (uint16_t)pack2<FP16>(acc[i] * inv, 0.f);
    } else {
      // sums that the other splits raised by RAISE; here they are not, so the maximum says it
      if (lane == 0) p.part_ml[at] = make_float2(m == -INFINITY ? m : m + RAISE<FP16>, l);
      for (int i = 0; i < N; ++i) p.part[at * D + lane * N + i] = acc[i];
    }
  }
}

template <int D, bool FP16, bool CAP, bool BIAS>
__global__ void __launch_bounds__(THREADS, 1)
tiles_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
             const __grid_constant__ CUtensorMap map_v, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int NB = D / 64;
  constexpr int NS = STAGES<D>;
  constexpr uint32_t TILE_BYTES = NB * BLOCK_BYTES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &sm.abort_flag;
  // Heads change fastest (those of a group share K and V in L2), then the row tiles -- the
  // last rows first, since with a causal mask they see the most keys -- then the splits.
  const int n_row_tiles = (int)((p.q_rows + ROWS - 1) / ROWS);
  int unit = blockIdx.x;
  const int head = unit % p.heads;
  unit /= p.heads;
  const int row_tile = n_row_tiles - 1 - unit % n_row_tiles, split = unit / n_row_tiles;
  const int kv_head = head / p.group;
  const long long row0 = (long long)row_tile * ROWS;

  if (threadIdx.x == 256) {
    tc::mbar_init(tc::smem_u32(&sm.q_full), 1);
    for (int s = 0; s < NS; ++s) {
      tc::mbar_init(tc::smem_u32(&sm.k_full[s]), 1);
      tc::mbar_init(tc::smem_u32(&sm.k_empty[s]), 1);
      tc::mbar_init(tc::smem_u32(&sm.v_full[s]), 1);
      tc::mbar_init(tc::smem_u32(&sm.v_empty[s]), 1);
    }
    for (int h = 0; h < 2; ++h) {
      tc::mbar_init(tc::smem_u32(&sm.s_full[h]), 1);
      tc::mbar_init(tc::smem_u32(&sm.p_full[h]), SOFTMAX_WARPS / 2);
      tc::mbar_init(tc::smem_u32(&sm.o_full[h]), 1);
    }
    tc::mbar_init(tc::smem_u32(&sm.drain), 1);
    sm.abort_flag = 0;
    sm.hull[0][0] = sm.hull[1][0] = 0x7FFFFFFF;
    sm.hull[0][1] = sm.hull[1][1] = 0;
    tc::fence_barrier_init();
    tc::prefetch_tensormap(&map_q);
    tc::prefetch_tensormap(&map_k);
    tc::prefetch_tensormap(&map_v);
  }
  if (warp == SOFTMAX_WARPS + 1) {
    tc::tmem_alloc(tc::smem_u32(&sm.tmem_base), TMEM_COLS);
    tc::tmem_relinquish();
  }

  // ------------------------------------------------ the rows' intervals and the CTA's walk
  const bool shared_offsets = p.q_offsets && p.documents <= SHARED_DOCS;
  if (shared_offsets)
    for (int i = threadIdx.x; i <= p.documents; i += THREADS) sm.offsets[i] = __ldg(p.q_offsets + i);
  __syncthreads();
  int doc = -1, lo = 0, hi = 0, pos = 0;
  if (threadIdx.x < ROWS) {
    const long long row = row0 + threadIdx.x;
    if (row < p.q_rows) {
      if (!shared_offsets) {
        doc = find_document(p, row);
      } else if (row >= sm.offsets[0] && row < sm.offsets[p.documents]) {
        int a = 0, b = p.documents;
        while (b - a > 1) {
          const int mid = (a + b) >> 1;
          if (sm.offsets[mid] <= row) a = mid;
          else b = mid;
        }
        doc = a;
      }
    }
    if (doc >= 0) {
      const Interval iv = row_interval(p, doc, row);
      lo = (int)iv.lo, hi = (int)iv.hi, pos = (int)iv.pos;
    }
    sm.lo[threadIdx.x] = lo, sm.hi[threadIdx.x] = hi, sm.doc[threadIdx.x] = doc;
    const int first = __reduce_min_sync(0xffffffffu, hi > lo ? lo : 0x7FFFFFFF);
    const int end = __reduce_max_sync(0xffffffffu, hi > lo ? hi : 0);
    if (lane == 0) {
      atomicMin(&sm.hull[warp >> 2][0], first);
      atomicMax(&sm.hull[warp >> 2][1], end);
    }
  }
  __syncthreads();
  if (threadIdx.x < ROWS) {
    const bool start = threadIdx.x == 0 || sm.doc[threadIdx.x] != sm.doc[threadIdx.x - 1];
    const uint32_t bits = __ballot_sync(0xffffffffu, start);
    if (lane == 0) sm.starts[warp] = bits;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    // Documents in the order of their rows.  A row's hi does not fall within a document, so its
    // last row here gives the document's range; ranges that touch are walked as one.
    int n = 0, tiles = 0, covered = 0, r = 0;
    while (r < ROWS) {
      int next = ROWS;
      uint32_t bits = (r & 31) == 31 ? 0u : sm.starts[r >> 5] & (0xFFFFFFFEu << (r & 31));
      for (int w = r >> 5;;) {
        if (bits) {
          next = w * 32 + __ffs(bits) - 1;
          break;
        }
        if (++w == ROWS / 32) break;
        bits = sm.starts[w];
      }
      int first = sm.lo[r];
      const int end = sm.hi[next - 1];
      if (end > first) {
        if (n > 0) first = max(first, covered);
        if (end > first) {
          if (n > 0 && first == covered) {
            sm.segments[n - 1].y = end;
          } else {
            sm.segments[n++] = make_int2(first, end);
          }
          covered = end;
        }
      }
      r = next;
    }
    for (int i = 0; i < n; ++i) tiles += (sm.segments[i].y - sm.segments[i].x + BKV - 1) / BKV;
    sm.n_segments = n;
    sm.n_tiles = tiles;
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = sm.tmem_base;
  const int first_tile = (int)((long long)sm.n_tiles * split / p.splits);
  const int last_tile = (int)((long long)sm.n_tiles * (split + 1) / p.splits);
  const int n_tiles = last_tile - first_tile;
  // Whether a half has a row that may see keys [begin, end).
  const auto needs = [&](int h, int begin, int end) { return begin < sm.hull[h][1] && end > sm.hull[h][0]; };

  if (warp >= SOFTMAX_WARPS) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
   if (warp == SOFTMAX_WARPS) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && n_tiles > 0) {
      const uint32_t qf = tc::smem_u32(&sm.q_full);
      tc::mbar_arrive_expect_tx(qf, 2 * TILE_BYTES);
      for (int h = 0; h < 2; ++h)
        for (int b = 0; b < NB; ++b)
          tc::tma_load_2d(tc::smem_u32(sm.q[h][b]), &map_q, head * D + b * 64, (int)row0 + h * BQ, qf);
      Walk walk(sm.segments, first_tile, last_tile);
      int begin, end, j = 0;
      int k_issued = 0, v_issued = 0;
      for (; walk.next(begin, end); ++j) {
        const int s = j % NS;
        const uint32_t ph = (uint32_t)(j / NS) & 1u;
        if (!wait_bounded(tc::smem_u32(&sm.k_empty[s]), ph ^ 1u, abort_flag, p.err)) break;
        const uint32_t kf = tc::smem_u32(&sm.k_full[s]);
        tc::mbar_arrive_expect_tx(kf, TILE_BYTES);
        for (int b = 0; b < NB; ++b) tc::tma_load_2d(tc::smem_u32(sm.k[s][b]), &map_k, kv_head * D + b * 64, begin, kf);
        k_issued = j + 1;
        if (!wait_bounded(tc::smem_u32(&sm.v_empty[s]), ph ^ 1u, abort_flag, p.err)) break;
        const uint32_t vf = tc::smem_u32(&sm.v_full[s]);
        tc::mbar_arrive_expect_tx(vf, TILE_BYTES);
        for (int b = 0; b < NB; ++b) tc::tma_load_2d(tc::smem_u32(sm.v[s][b]), &map_v, kv_head * D + b * 64, begin, vf);
        v_issued = j + 1;
      }
      // Let every copy this thread issued land before the CTA can exit.
      const uint64_t start = global_ns();
      while (!tc::mbar_try_wait(qf, 0) && global_ns() - start < WAIT_LIMIT_NS) {
      }
      for (int i = 0; i < NS; ++i) {
        for (int which = 0; which < 2; ++which) {
          const int t = (which ? v_issued : k_issued) - 1 - i;
          if (t < 0) continue;
          const uint32_t bar = tc::smem_u32(which ? &sm.v_full[t % NS] : &sm.k_full[t % NS]);
          const uint64_t t0 = global_ns();
          while (!tc::mbar_try_wait(bar, (uint32_t)(t / NS) & 1u) && global_ns() - t0 < WAIT_LIMIT_NS) {
          }
        }
      }
    }
   } else if (warp == SOFTMAX_WARPS + 1) {
    // ------------------------------------------------------------ MMA issuer (the warp stays together)
    if (n_tiles > 0) {
      Walk walk(sm.segments, first_tile, last_tile);
      int begin = 0, end = 0, next_begin = 0, next_end = 0;
      int sequence[2] = {0, 0};          // tiles of each half so far
      bool pending[2] = {false, false};  // a P V product of the half that no one has waited for
      const auto issue_qk = [&](int h, int s) {
        if (lane == 0) {
          const uint32_t q_addr = tc::smem_u32(sm.q[h][0]), k_addr = tc::smem_u32(sm.k[s][0]);
          const uint32_t d_tmem = tmem_base + (uint32_t)(S_COL + h * BKV);
#pragma unroll
          for (int t = 0; t < D / 16; ++t) {
            const uint32_t at = (uint32_t)((t >> 2) * BLOCK_BYTES + (t & 3) * 32);
            tc::mma_f16_ss(d_tmem, tc::desc_k_sw128(q_addr + at), tc::desc_k_sw128(k_addr + at), idesc_qk<FP16>(),
                           t ? 1u : 0u);
          }
          tc::mma_commit(tc::smem_u32(&sm.s_full[h]));
        }
        __syncwarp();
      };
      bool ok = wait_bounded(tc::smem_u32(&sm.q_full), 0, abort_flag, p.err) &&
                wait_bounded(tc::smem_u32(&sm.k_full[0]), 0, abort_flag, p.err);
      ok = __all_sync(0xffffffffu, ok);
      walk.next(begin, end);
      if (ok) {
        tc::fence_after_sync();
        for (int h = 0; h < 2; ++h)
          if (needs(h, begin, end)) issue_qk(h, 0);
        if (lane == 0) tc::mma_commit(tc::smem_u32(&sm.k_empty[0]));
        __syncwarp();
      }
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int s = j % NS, s_next = (j + 1) % NS;
        const bool more = walk.next(next_begin, next_end);
        ok = wait_bounded(tc::smem_u32(&sm.v_full[s]), (uint32_t)(j / NS) & 1u, abort_flag, p.err);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        if (end - begin < BKV) {
          // keys behind the segment: whatever lies there becomes zero before it meets P's zeros
          const int keys = BKV - (end - begin);
          for (int c = lane; c < keys * 8 * NB; c += 32) {
            const int b = c / (keys * 8), rest = c - b * keys * 8;
            *reinterpret_cast<uint4*>(sm.v[s][b] + (end - begin) * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
          }
          tc::fence_proxy_async_smem();
          __syncwarp();
        }
        bool k_ready = false;
        for (int h = 0; h < 2 && ok; ++h) {
          if (needs(h, begin, end)) {
            ok = wait_bounded(tc::smem_u32(&sm.p_full[h]), (uint32_t)sequence[h] & 1u, abort_flag, p.err);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            tc::fence_after_sync();
            if (lane == 0) {
              const uint32_t v_addr = tc::smem_u32(sm.v[s][0]);
              const uint32_t p_tmem = tmem_base + (uint32_t)(S_COL + h * BKV);
              const uint32_t d_tmem = tmem_base + (uint32_t)(O_COL + h * D);
#pragma unroll
              for (int t = 0; t < BKV / 16; ++t)
                tc::mma_f16_ts(d_tmem, p_tmem + t * 8, desc_v(v_addr + t * 2048), idesc_pv<D, FP16>(),
                               (t || sequence[h]) ? 1u : 0u);
              tc::mma_commit(tc::smem_u32(&sm.o_full[h]));
            }
            __syncwarp();
            ++sequence[h];
            pending[h] = true;
          }
          if (more && needs(h, next_begin, next_end)) {
            if (!k_ready) ok = wait_bounded(tc::smem_u32(&sm.k_full[s_next]), (uint32_t)((j + 1) / NS) & 1u, abort_flag, p.err);
            k_ready = true;
            // the next S takes the place of P: its product has to be done
            if (ok && pending[h]) {
              ok = wait_bounded(tc::smem_u32(&sm.o_full[h]), (uint32_t)(sequence[h] - 1) & 1u, abort_flag, p.err);
              pending[h] = false;
            }
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            tc::fence_after_sync();
            issue_qk(h, s_next);
          }
        }
        if (!ok) break;
        if (more && !k_ready) {  // no half needs the next tile; its stage is released all the same
          ok = wait_bounded(tc::smem_u32(&sm.k_full[s_next]), (uint32_t)((j + 1) / NS) & 1u, abort_flag, p.err);
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
        }
        if (lane == 0) {
          tc::mma_commit(tc::smem_u32(&sm.v_empty[s]));
          if (more) tc::mma_commit(tc::smem_u32(&sm.k_empty[s_next]));
        }
        __syncwarp();
        begin = next_begin, end = next_end;
      }
      if (lane == 0) {  // every product has ended before tensor memory is freed
        tc::mma_commit(tc::smem_u32(&sm.drain));
        const uint64_t start = global_ns();
        while (!tc::mbar_try_wait(tc::smem_u32(&sm.drain), 0) && global_ns() - start < WAIT_LIMIT_NS) {
        }
      }
      __syncwarp();
    }
   }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
    // ------------------------------------------------------------ softmax, one thread per row
    const int h = warp >> 2;
    const uint32_t lanes = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_tmem = lanes + (uint32_t)(S_COL + h * BKV), o_tmem = lanes + (uint32_t)(O_COL + h * D);
    const float scale2 = p.scale * LOG2E, cap2 = p.cap * LOG2E;
    const float two_over_cap2 = CAP ? 2.f * LOG2E * p.scale / p.cap : 0.f;
    const float slope2 = BIAS ? __ldg(p.slopes + head) * LOG2E : 0.f;
    float m = -INFINITY, l = 0.f;
    int sequence = 0;
    bool ok = true, redo = false;
    Walk walk(sm.segments, first_tile, last_tile);
    int begin, end;
    for (int j = 0; walk.next(begin, end); ++j) {
      if (!needs(h, begin, end)) continue;
      ok = wait_bounded(tc::smem_u32(&sm.s_full[h]), (uint32_t)sequence & 1u, abort_flag, p.err);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc::fence_after_sync();
      float s[BKV];
      {
        uint32_t raw[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) tc::tmem_ld_32x32b_x32(s_tmem + i * 32, raw[i]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < BKV; ++i) s[i] = __uint_as_float(raw[i >> 5][i & 31]);
      }
      if (CAP) {
#pragma unroll
        for (int i = 0; i < BKV; ++i) s[i] = capped_log2(s[i], two_over_cap2, cap2);
      }
      if (BIAS) {
        const float from = (float)(begin - pos);
#pragma unroll
        for (int i = 0; i < BKV; ++i) s[i] = fmaf(-slope2, fabsf(from + (float)i), CAP ? s[i] : s[i] * scale2);
      }
      const int c0 = lo - begin, c1 = min(hi, end) - begin;  // columns that this row sees
      if (!__all_sync(0xffffffffu, c0 <= 0 && c1 >= BKV)) {
#pragma unroll
        for (int i = 0; i < BKV; ++i) s[i] = i >= c0 && i < c1 ? s[i] : -INFINITY;
        // values that are not finite: exponent bits all ones
        const int st = j % NS;
        ok = wait_bounded(tc::smem_u32(&sm.v_full[st]), (uint32_t)(j / NS) & 1u, abort_flag, p.err);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        constexpr uint32_t EXP = FP16 ? 0x7C00u : 0x7F80u;
        bool found = false;
        for (int c = lane; c < (end - begin) * 8; c += 32) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint4 w = *reinterpret_cast<const uint4*>(sm.v[st][b] + c * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t x = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
              found = found || (x & EXP) == EXP || (x & (EXP << 16)) == (EXP << 16);
            }
          }
        }
        redo = redo || __any_sync(0xffffffffu, found);
      }
      float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int i = 4; i < BKV; ++i) top[i & 3] = fmaxf(top[i & 3], s[i]);
      float m_new = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      if (!CAP && !BIAS) m_new *= scale2;
      const bool rise = m_new > m + RESCALE;
      if (__any_sync(0xffffffffu, rise)) {
        float a = 1.f;
        if (rise) {
          a = m == -INFINITY ? 0.f : ex2(m - m_new);
          m = m_new;
          l *= a;
        }
        __syncwarp();
        if (sequence > 0) {
          ok = wait_bounded(tc::smem_u32(&sm.o_full[h]), (uint32_t)(sequence - 1) & 1u, abort_flag, p.err);
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
          tc::fence_after_sync();
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            uint32_t raw[32];
            tc::tmem_ld_32x32b_x32(o_tmem + i * 32, raw);
            tc::tmem_wait_ld();
#pragma unroll
            for (int t = 0; t < 32; ++t) raw[t] = __float_as_uint(__uint_as_float(raw[t]) * a);
            tc::tmem_st_32x32b_x32(o_tmem + i * 32, raw);
          }
        }
      }
      const float ref = m == -INFINITY ? 0.f : m - RAISE<FP16>;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t packed[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int at = half * 64 + 2 * i;
          const float a = ex2(CAP || BIAS ? s[at] - ref : fmaf(s[at], scale2, -ref));
          const float b = ex2(CAP || BIAS ? s[at + 1] - ref : fmaf(s[at + 1], scale2, -ref));
          sum[(2 * i) & 3] += a, sum[(2 * i + 1) & 3] += b;
          packed[i] = pack2<FP16>(a, b);
        }
        tc::tmem_st_32x32b_x32(s_tmem + half * 32, packed);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(tc::smem_u32(&sm.p_full[h]));
      ++sequence;
    }
    // ------------------------------------------------------------ output
    const int r = h * BQ + (warp & 3) * 32 + lane;
    const long long row = row0 + r;
    const bool valid = doc >= 0;
    if (ok && sequence > 0) ok = wait_bounded(tc::smem_u32(&sm.o_full[h]), (uint32_t)(sequence - 1) & 1u, abort_flag, p.err);
    if (__all_sync(0xffffffffu, ok)) {
      if (redo) {
        rows_key_by_key<D, FP16>(p, sm.segments, first_tile, last_tile, row0 + r - lane, head, lo, hi, pos, valid, split);
      } else {
        tc::fence_after_sync();
        const float inv = p.splits == 1 ? inverse_sum(l, hi > lo) : 1.f;
        const long long at = (split * p.q_rows + row) * p.heads + head;
        if (valid && p.splits > 1) p.part_ml[at] = make_float2(m, l);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t raw[32];
          __syncwarp();
          if (sequence > 0) {
            tc::tmem_ld_32x32b_x32(o_tmem + i * 32, raw);
            tc::tmem_wait_ld();
          }
          if (l == 0.f && inv == 0.f) {  // no key: whatever tensor memory holds
#pragma unroll
            for (int t = 0; t < 32; ++t) raw[t] = 0u;
          }
          if (valid && p.splits == 1) {
            uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.out_stride + (long long)head * D + i * 32;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t w[4];
#pragma unroll
              for (int t = 0; t < 4; ++t)
                w[t] = pack2<FP16>(__uint_as_float(raw[c * 8 + 2 * t]) * inv, __uint_as_float(raw[c * 8 + 2 * t + 1]) * inv);
              *reinterpret_cast<uint4*>(out + c * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else if (valid && sequence > 0) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<uint4*>(p.part + at * D + i * 32 + c * 4) =
                  make_uint4(raw[c * 4], raw[c * 4 + 1], raw[c * 4 + 2], raw[c * 4 + 3]);
          }
        }
      }
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  if (warp == SOFTMAX_WARPS + 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int D, bool FP16, bool CAP, bool BIAS>
int launch(const Params& p, cudaStream_t s) {
  const long long grid = (p.q_rows + ROWS - 1) / ROWS * p.heads * p.splits;
  if (grid > 0x7FFFFFFFLL) return fail(MUSC_B200_ERR_INVALID, "masked_attention: too many rows and heads");
  const int qw = p.heads * D, kw = p.kv_heads * D;
  CUtensorMap mq, mk, mv;
  MUSC_TRY(make_token_map(&mq, p.q, p.q_rows, qw, p.q_rows > 1 ? p.q_stride : qw, FP16));
  MUSC_TRY(make_token_map(&mk, p.k, p.kv_rows, kw, p.kv_rows > 1 ? p.k_stride : kw, FP16));
  MUSC_TRY(make_token_map(&mv, p.v, p.kv_rows, kw, p.kv_rows > 1 ? p.v_stride : kw, FP16));
  const auto kernel = tiles_kernel<D, FP16, CAP, BIAS>;
  MUSC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES<D>));
  kernel<<<(unsigned)grid, THREADS, SMEM_BYTES<D>, s>>>(mq, mk, mv, p);
  return check_launch("masked tiles_kernel");
}

template <int D, bool FP16>
int launch_form(const Params& p, cudaStream_t s) {
  if (p.cap > 0.f) return p.slopes ? launch<D, FP16, true, true>(p, s) : launch<D, FP16, true, false>(p, s);
  return p.slopes ? launch<D, FP16, false, true>(p, s) : launch<D, FP16, false, false>(p, s);
}

}  // namespace

int tiles_splits(long long units, long long kv_bound) {
  const long long want = 148 / std::max<long long>(units, 1);
  const long long most = kv_bound / (4 * BKV);  // four tiles at least for each split
  return (int)std::max<long long>(1, std::min<long long>(std::min<long long>(want, most), 32));
}

int tiles_launch(const Params& p, int head_dim, bool fp16, cudaStream_t s) {
  if (head_dim == 64) return fp16 ? launch_form<64, true>(p, s) : launch_form<64, false>(p, s);
  return fp16 ? launch_form<128, true>(p, s) : launch_form<128, false>(p, s);
}

}  // namespace masked
}  // namespace musc
