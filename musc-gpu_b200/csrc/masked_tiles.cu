// Masked attention of many query rows (masked.cuh has the operator): fused tcgen05 attention
// over tiles of 256 query rows x 64 keys.
//
// One CTA per (256 query rows, head, split of the keys), 384 threads.  Its rows need not belong
// to one document: every row carries its own key interval, and the CTA walks the union of its
// documents' intervals in tiles of 64 keys, so short documents share a row tile; long ones begin
// their own (one that holds two long documents' rows walks both their keys: nine images of 414 to
// 932 tokens, 16 heads x 64, take 58 us, 71 when tiles are cut from the packed rows; 4 x 1370 tokens 83 and 87).
//   warps 0-3, 4-7  softmax of query rows 0-127 and 128-255 (the two halves), one thread
//                   per row: S out of tensor memory, cap, bias, mask, running maximum and
//                   sum in 32 bits, P rounded to 16 bits into tensor memory beside S;
//   warp 8          TMA: Q once, K and V tiles through a ring;
//   warps 9, 10     one thread for each half issues tcgen05.mma: S_h = Q_h K^T (128 x 64 x D,
//                   both from shared memory) and O_h += P_h V (128 x D x 64, P from tensor memory);
//   warp 11         zeroes the end of V's tiles that reach past their keys, and searches V.
// While one half's softmax runs, the tensor cores work for the other.  For 64 keys the exponentials
// of both halves take 1024 cycles (16 a cycle and SM), the products 700 for D = 64 and 1350 for D = 128
// (S of 128 x 64 runs at two thirds of the rate of 128 x 128, whose S would leave no tensor memory
// for P beside it).  Measured at 8192 tokens of 16 heads, no mask, bf16, calls apart: D = 128 509 us (1080 TF/s,
// 0.64 of the measured 1693), D = 64 486 us (566 TF/s); four waves of CTAs for 3.46 waves of work.  (In a graph of
// 18 calls back to back: D = 128 556 us, D = 64 481.)  The
// special-function unit is 60 % busy, the tensor pipe 29 % (D = 64, ncu): the rest is the softmax warps'
// own chain, two of them a scheduler.  Tried and dropped, with times at D = 64 or 128: tiles of 128 keys with P over
// S (548 us), a maximum of every tile before its exponentials (no gain from leaving it out by itself, but
// it frees registers), a share of the exponentials by polynomials (8 % slower: instructions
// bound it as much), strict turns of the two halves' exponentials (no gain, and a half that is
// tiles ahead of the other cannot wait for it), one issuing thread for both halves (596 us).
//
// A masked probability is zero, but zero times a NaN or infinite value is NaN.  Keys that no
// row of the CTA sees (behind a document's last key) are zeroed in V's tile.  Tiles that some row
// may not see in whole are searched for such values, and a warp whose rows see such a tile in part
// recomputes them key by key at the end, skipping what they do not see: rare, slow, right.
#include "masked.cuh"
#include "tc.cuh"

#include <algorithm>
#include <mutex>

namespace musc {
namespace masked {
namespace {

constexpr int BQ = 128;    // query rows of a half (TMEM lanes)
constexpr int ROWS = 2 * BQ;
constexpr int BKV = 64;    // keys of a tile
constexpr int Q_BLOCK = BQ * 128, KV_BLOCK = BKV * 128;  // bytes of 64 elements (a swizzle row) of all rows
constexpr int SOFTMAX_WARPS = 8;
constexpr int THREADS = 32 * (SOFTMAX_WARPS + 4);
constexpr int TMEM_COLS = 512;
// Tensor memory: per half S (64 columns), two buffers of P (32 each) and O (D).
constexpr int s_col(int h) { return h * 64; }
constexpr int p_col(int h, int buffer) { return 128 + h * 64 + buffer * 32; }
template <int D> constexpr int o_col(int h) { return 256 + h * D; }
constexpr float P_LIMIT = 65504.f;  // largest sum of a row's stored exponentials over a tile: each fits fp16
constexpr int SHARED_DOCS = 1024;  // offsets searched in shared memory up to this many documents
constexpr uint32_t WAIT_TRIES = 1u << 20, SLEEP_NS = 2000;
template <int D> constexpr int STAGES = D == 64 ? 8 : 4;

template <int D>
struct Smem {
  uint8_t q[2][D / 64][Q_BLOCK];
  uint8_t k[STAGES<D>][D / 64][KV_BLOCK];
  uint8_t v[STAGES<D>][D / 64][KV_BLOCK];
  uint64_t q_full;
  uint64_t full[STAGES<D>], clean[STAGES<D>], empty[STAGES<D>];
  uint64_t s_full[2], s_free[2];        // per half
  uint64_t p_full[2][2], o_full[2][2];  // per half and buffer of P
  uint64_t drained[2];
  union {
    struct {                         // while the rows' documents are looked up
      int offsets[SHARED_DOCS + 1];
      uint16_t run[SHARED_DOCS];     // first document of the run that a document belongs to
    };
    int2 segments[ROWS];             // then: key ranges [x, y) that the CTA walks
  };
  int scan[2][THREADS / 32];         // of the warps: last run begun, row tiles
  int tile_doc, tile_row0, total_tiles;
  int lo[ROWS], hi[ROWS];
  uint32_t starts[ROWS / 32];      // rows that begin another document than the row before
  int hull[2][2];                  // per half: first key and end of all its rows' keys
  int common[2];                   // the keys that all rows with keys see: from, to
  int odd[STAGES<D>];              // V's tile in a stage holds values that are not finite
  int n_segments, n_tiles;
  uint32_t tmem_base;
  int abort_flag;
};
template <int D> constexpr size_t SMEM_BYTES = sizeof(Smem<D>) + 1024;

// Bounded wait: after WAIT_TRIES tries (each sleeps for up to SLEEP_NS, so at most two
// seconds in all) the CTA's abort flag is raised, which ends every other wait and is reported
// when the CTA ends.  Few instructions: the waits stand between the products and exponentials.
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
#pragma unroll 1
  for (uint32_t tries = 0; tries < WAIT_TRIES; ++tries) {
    if (tc::mbar_try_wait_for(bar, parity, SLEEP_NS)) return true;
    if (*abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}

// Waits for work in flight whether or not the CTA has given up.
__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (uint32_t tries = 0; tries < WAIT_TRIES; ++tries)
    if (tc::mbar_try_wait_for(bar, parity, SLEEP_NS)) return;
}

// Shared-memory matrix descriptors in the 128-byte swizzle, 8-row groups 1024 bytes apart.  The
// upper word is the same for every operand here; the lower one holds the address, so the
// operands of consecutive products are an addition apart.  K-major (Q, K) has no leading
// offset; V as the MN-major B operand has its blocks of 64 dims KV_BLOCK apart.
constexpr uint32_t DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo_k(uint32_t smem_addr) { return (smem_addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_lo_v(uint32_t smem_addr) {
  return (smem_addr >> 4) | ((uint32_t)(KV_BLOCK >> 4) << 16);
}
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"((uint32_t)accumulate), "r"(DESC_HI)
      : "memory");
}
// A (one row per TMEM lane) from tensor memory: a 32-bit column holds two consecutive K
// elements, so a K step of 16 is eight columns.
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"((uint32_t)accumulate), "r"(DESC_HI)
      : "memory");
}
template <bool FP16> constexpr uint32_t idesc_qk() { return tc::idesc_f16(BQ, BKV, FP16 ? 0 : 1); }
template <int D, bool FP16> constexpr uint32_t idesc_pv() {
  return tc::idesc_f16(BQ, D, FP16 ? 0 : 1) | (1u << 16);  // B (V) MN-major
}

// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// The value, as one that changes from use to use: what is computed from it stays where it is used
// instead of taking registers through the whole loop.
__device__ __forceinline__ float here(float v) {
  asm volatile("" : "+f"(v));
  return v;
}

// s -> cap2 * tanh(s / cap) for a row's tile (factor = scale / cap, cap2 = cap log2(e)).  The exact form
// takes two of the special-function unit's operations an element, and the exponential a
// third, where that unit already bounds the loop.  tanh(x) / x as a
// polynomial in x^2 takes multiply-adds instead, two elements an instruction: of degree 3
// where the warp's scores stay within |x| <= 0.4 (most do: a cap is chosen well above them),
// of degree 6 up to 1, each fitted for the least maximum error (2e-8 and 2e-8 of tanh, below
// the rounding of its evaluation).
__device__ __forceinline__ void cap_scores(float2 (&s)[BKV / 2], float factor_, float cap2_) {
  const float factor = here(factor_), cap2 = here(cap2_);
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < BKV / 2; ++i) top = max3(top, fabsf(s[i].x), fabsf(s[i].y));
  const float x_max = top * factor;
  if (__all_sync(0xffffffffu, x_max <= 0.4f)) {
    const float2 c0 = both(cap2 * TANH3[0]), c1 = both(cap2 * TANH3[1]), c2 = both(cap2 * TANH3[2]), c3 = both(cap2 * TANH3[3]);
#pragma unroll
    for (int i = 0; i < BKV / 2; ++i) {
      const float2 x = mul2(s[i], both(factor)), t = mul2(x, x);
      s[i] = mul2(x, fma2(fma2(fma2(c3, t, c2), t, c1), t, c0));
    }
  } else if (__all_sync(0xffffffffu, x_max <= 1.f)) {
    const float2 c0 = both(cap2 * 0.999999702f), c1 = both(cap2 * -0.333321303f), c2 = both(cap2 * 0.133195832f),
                 c3 = both(cap2 * -0.0532658361f), c4 = both(cap2 * 0.0199732818f), c5 = both(cap2 * -0.00595127977f),
                 c6 = both(cap2 * 0.000963771949f);
#pragma unroll
    for (int i = 0; i < BKV / 2; ++i) {
      const float2 x = mul2(s[i], both(factor)), t = mul2(x, x);
      s[i] = mul2(x, fma2(fma2(fma2(fma2(fma2(fma2(c6, t, c5), t, c4), t, c3), t, c2), t, c1), t, c0));
    }
  } else {
#pragma unroll
    for (int i = 0; i < BKV / 2; ++i) {
      s[i].x = capped_log2(s[i].x, factor, cap2);
      s[i].y = capped_log2(s[i].y, factor, cap2);
    }
  }
}

// The tiles [first, last) of the CTA's walk over its segments, one segment's end in a register.
struct Walk {
  const int2* segments;
  int segment, x, stop, left;
  __device__ __forceinline__ Walk(const int2* s, int first, int last) : segments(s), segment(0), left(last - first) {
    x = stop = 0;
    while (left > 0) {
      const int tiles = (s[segment].y - s[segment].x + BKV - 1) / BKV;
      if (first < tiles) break;
      first -= tiles;
      ++segment;
    }
    if (left > 0) x = s[segment].x + first * BKV, stop = s[segment].y;
  }
  // Next tile: keys [begin, end), end - begin <= BKV.
  __device__ __forceinline__ bool next(int& begin, int& end) {
    if (left <= 0) return false;
    --left;
    begin = x;
    end = min(x + BKV, stop);
    x += BKV;
    if (x >= stop && left > 0) {
      const int2 s = segments[++segment];
      x = s.x, stop = s.y;
    }
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
    const long long row = row0 + r;
    if (!__shfl_sync(0xffffffffu, (int)row_valid, r)) continue;
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + row * p.q_stride + (long long)head * D + lane * N;
    float qf[N], acc[N], m = -INFINITY, l = 0.f;
    for (int i = 0; i < N; ++i) qf[i] = widen<FP16>(q[i]), acc[i] = 0.f;
    Walk walk(segments, first, last);
    int begin, end;
    while (walk.next(begin, end)) {
      attend_keys<D, FP16>(p, qf, kv_head, slope2, pos, max(begin, lo), min(end, hi), acc, m, l);
    }
    const long long at = (split * p.q_rows + row) * p.heads + head;
    if (p.splits == 1) {
      const float inv = inverse_sum(l, hi > lo);
      uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.out_stride + (long long)head * D + lane * N;
      for (int i = 0; i < N; ++i) out[i] = (uint16_t)pack2<FP16>(acc[i] * inv, 0.f);
    } else {
      // sums that the other splits raised by RAISE; here they are not, so the maximum says it
      if (lane == 0) p.part_ml[at] = partial_ml(m + RAISE<FP16>, l, hi > lo);
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
  constexpr uint32_t TILE_BYTES = NB * KV_BLOCK;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &sm.abort_flag;
  // Heads change fastest (those of a group share K and V in L2), then the row tiles -- the
  // last rows first, since with a causal mask they see the most keys -- then the splits.
  int unit = blockIdx.x;
  const int head = unit % p.heads;
  unit /= p.heads;
  const int row_tile = p.row_tiles - 1 - unit % p.row_tiles, split = unit / p.row_tiles;
  const int kv_head = head / p.group;

  if (threadIdx.x == 256) {
    tc::mbar_init(tc::smem_u32(&sm.q_full), 1);
    for (int s = 0; s < NS; ++s) {
      tc::mbar_init(tc::smem_u32(&sm.full[s]), 1);
      tc::mbar_init(tc::smem_u32(&sm.clean[s]), 1);
      tc::mbar_init(tc::smem_u32(&sm.empty[s]), 2);
    }
    for (int h = 0; h < 2; ++h) {
      tc::mbar_init(tc::smem_u32(&sm.s_full[h]), 1);
      tc::mbar_init(tc::smem_u32(&sm.s_free[h]), SOFTMAX_WARPS / 2);
      for (int b = 0; b < 2; ++b) {
        tc::mbar_init(tc::smem_u32(&sm.p_full[h][b]), SOFTMAX_WARPS / 2);
        tc::mbar_init(tc::smem_u32(&sm.o_full[h][b]), 1);
      }
      tc::mbar_init(tc::smem_u32(&sm.drained[h]), 1);
    }
    sm.abort_flag = 0;
    sm.hull[0][0] = sm.hull[1][0] = 0x7FFFFFFF;
    sm.hull[0][1] = sm.hull[1][1] = 0;
    sm.common[0] = 0, sm.common[1] = 0x7FFFFFFF;
    tc::fence_barrier_init();
    tc::prefetch_tensormap(&map_q);
    tc::prefetch_tensormap(&map_k);
    tc::prefetch_tensormap(&map_v);
  }
  if (warp == SOFTMAX_WARPS + 1) {
    tc::tmem_alloc(tc::smem_u32(&sm.tmem_base), TMEM_COLS);
    tc::tmem_relinquish();
  }

  // ------------------------------------------------ the CTA's rows, their intervals and its walk
  const bool shared_offsets = p.q_offsets && p.documents <= SHARED_DOCS;
  if (shared_offsets)
    for (int i = threadIdx.x; i <= p.documents; i += THREADS) sm.offsets[i] = row_offset(p, i);
  if (threadIdx.x == 0) sm.tile_doc = -1;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  // First row, and the run of documents that the tile is cut from (-1: all rows).
  long long row0 = (long long)row_tile * ROWS;
  int run = -1, run_end = 0x7FFFFFFF;  // documents [run, run_end)
  if (p.aligned && shared_offsets && p.documents <= 32) {
    // As below, by every warp for itself: a lane for each document.
    const int d = min(lane, p.documents), from = sm.offsets[d], to = sm.offsets[min(d + 1, p.documents)];
    const int rows = max(to - from, 0), rows_before = __shfl_up_sync(0xffffffffu, rows, 1);
    const bool begins = lane < p.documents && (lane == 0 || rows >= ROWS || rows_before >= ROWS);
    const uint32_t runs = __ballot_sync(0xffffffffu, begins);
    const int mine = 31 - __clz(runs & (0xFFFFFFFFu >> (31 - lane)));  // lane 0 begins one: there is a document
    const int start = __shfl_sync(0xffffffffu, from, mine), in_run = max(from - start, 0);
    const int tiles = lane < p.documents ? (in_run + rows + ROWS - 1) / ROWS - (in_run + ROWS - 1) / ROWS : 0;
    int first = tiles;  // inclusive, then exclusive, sum
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, first, o);
      if (lane >= o) first += other;
    }
    first -= tiles;
    const uint32_t owner = __ballot_sync(0xffffffffu, row_tile >= first && row_tile < first + tiles);
    if (owner == 0) {
      run = -2;
    } else {
      const int d_tile = __ffs(owner) - 1;
      run = __shfl_sync(0xffffffffu, mine, d_tile);
      const uint32_t later = run < 31 ? runs & (0xFFFFFFFEu << run) : 0u;
      run_end = later ? __ffs(later) - 1 : p.documents;
      row0 = __shfl_sync(0xffffffffu, start + ((in_run + ROWS - 1) / ROWS + row_tile - first) * ROWS, d_tile);
    }
  } else if (p.aligned && shared_offsets) {
    // A document of ROWS rows and more is a run of its own, shorter ones that follow each other are
    // one run.  Runs are cut into tiles from their first row on: a document's tiles are those that
    // begin in it.  Each thread takes PER documents; two scans over the threads.
    constexpr int PER = (SHARED_DOCS + THREADS - 1) / THREADS;
    const int d0 = threadIdx.x * PER;
    const auto rows_of = [&](int d) { return max(sm.offsets[d + 1] - sm.offsets[d], 0); };
    int begun = -1;
    for (int d = d0; d < min(d0 + PER, p.documents); ++d)
      if (d == 0 || rows_of(d) >= ROWS || rows_of(d - 1) >= ROWS) begun = d;
    int before = begun;  // inclusive, then exclusive, maximum over the threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before = max(before, other);
    }
    if (lane == 31) sm.scan[0][warp] = before;
    before = __shfl_up_sync(0xffffffffu, before, 1);
    if (lane == 0) before = -1;
    __syncthreads();
    for (int w = 0; w < warp; ++w) before = max(before, sm.scan[0][w]);
    int tiles[PER], sum = 0, at = before;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int d = d0 + i;
      tiles[i] = 0;
      if (d < p.documents) {
        if (d == 0 || rows_of(d) >= ROWS || rows_of(d - 1) >= ROWS) at = d;
        sm.run[d] = (uint16_t)at;
        const int from = max(sm.offsets[d] - sm.offsets[at], 0);
        tiles[i] = (from + rows_of(d) + ROWS - 1) / ROWS - (from + ROWS - 1) / ROWS;
        sum += tiles[i];
      }
    }
    int first = sum;  // inclusive, then exclusive, sum over the threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, first, o);
      if (lane >= o) first += other;
    }
    if (lane == 31) sm.scan[1][warp] = first;
    first -= sum;
    __syncthreads();
    for (int w = 0; w < warp; ++w) first += sm.scan[1][w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (row_tile >= first && row_tile < first + tiles[i]) {
        const int d = d0 + i, start = sm.offsets[sm.run[d]];
        sm.tile_doc = d;
        sm.tile_row0 = start + ((max(sm.offsets[d] - start, 0) + ROWS - 1) / ROWS + row_tile - first) * ROWS;
      }
      first += tiles[i];
    }
    __syncthreads();
    run = sm.tile_doc < 0 ? -2 : sm.run[sm.tile_doc];
    row0 = sm.tile_row0;
    run_end = -1;  // not known, but which run a document belongs to
  } else if (p.aligned) {
    const int per_doc = (int)((p.q_len + ROWS - 1) / ROWS);
    run = row_tile / per_doc;
    row0 = run * p.q_len + (long long)(row_tile - run * per_doc) * ROWS;
    run_end = run + 1;
  }
  if (run == -2) {  // the grid's bound was higher than the documents' tiles
    if (warp == SOFTMAX_WARPS + 1) tc::tmem_dealloc(sm.tmem_base, TMEM_COLS);
    return;
  }
  if (threadIdx.x == 256) {  // Q is on its way while the keys are looked up
    const uint32_t full = tc::smem_u32(&sm.q_full);
    tc::mbar_arrive_expect_tx(full, 2 * NB * Q_BLOCK);
    for (int h = 0; h < 2; ++h)
      for (int b = 0; b < NB; ++b)
        tc::tma_load_2d(tc::smem_u32(sm.q[h][b]), &map_q, head * D + b * 64, (int)row0 + h * BQ, full);
  }
  // Document of a row of this tile; -1: of none, or another tile's.
  const auto document_of = [&](long long row) {
    if (row < 0 || row >= p.q_rows) return -1;
    int d = -1;
    if (!shared_offsets) {
      d = find_document(p, row);
    } else if (row >= sm.offsets[0] && row < sm.offsets[p.documents]) {
      int a = 0, b = p.documents;
      while (b - a > 1) {
        const int mid = (a + b) >> 1;
        if (sm.offsets[mid] <= row) a = mid;
        else b = mid;
      }
      d = a;
    }
    const bool here = run < 0 || d < 0 || (run_end < 0 ? sm.run[d] == run : d >= run && d < run_end);
    return here ? d : -1;
  };
  int doc = -1, lo = 0, hi = 0, pos = 0;
  if (threadIdx.x < ROWS) {
    const long long row = row0 + threadIdx.x;
    doc = document_of(row);
    int doc_before = __shfl_up_sync(0xffffffffu, doc, 1);
    if (lane == 0) doc_before = threadIdx.x == 0 ? -2 : document_of(row - 1);
    const uint32_t bits = __ballot_sync(0xffffffffu, doc != doc_before);
    if (lane == 0) sm.starts[warp] = bits;
    if (doc >= 0) {
      const Interval iv = row_interval(p, doc, row);
      lo = (int)iv.lo, hi = (int)iv.hi, pos = (int)iv.pos;
    }
    sm.lo[threadIdx.x] = lo, sm.hi[threadIdx.x] = hi;
    const int first = __reduce_min_sync(0xffffffffu, hi > lo ? lo : 0x7FFFFFFF);
    const int end = __reduce_max_sync(0xffffffffu, hi > lo ? hi : 0);
    const int all_from = __reduce_max_sync(0xffffffffu, hi > lo ? lo : 0);
    const int all_to = __reduce_min_sync(0xffffffffu, hi > lo ? hi : 0x7FFFFFFF);
    if (lane == 0) {
      atomicMin(&sm.hull[warp >> 2][0], first);
      atomicMax(&sm.hull[warp >> 2][1], end);
      atomicMax(&sm.common[0], all_from);
      atomicMin(&sm.common[1], all_to);
    }
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
  __syncthreads();
  const uint32_t tmem_base = sm.tmem_base;
  const int first_tile = (int)((long long)sm.n_tiles * split / p.splits);
  const int last_tile = (int)((long long)sm.n_tiles * (split + 1) / p.splits);
  const int n_tiles = last_tile - first_tile;

  if (warp >= SOFTMAX_WARPS) {
   if (warp == SOFTMAX_WARPS) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      Walk walk(sm.segments, first_tile, last_tile);
      int begin, end, issued = 0;
      while (walk.next(begin, end)) {
        const int s = issued % NS;
        if (!wait_bounded(tc::smem_u32(&sm.empty[s]), ((uint32_t)(issued / NS) & 1u) ^ 1u, abort_flag)) break;
        const uint32_t full = tc::smem_u32(&sm.full[s]);
        tc::mbar_arrive_expect_tx(full, 2 * TILE_BYTES);
        for (int b = 0; b < NB; ++b) {
          tc::tma_load_2d(tc::smem_u32(sm.k[s][b]), &map_k, kv_head * D + b * 64, begin, full);
          tc::tma_load_2d(tc::smem_u32(sm.v[s][b]), &map_v, kv_head * D + b * 64, begin, full);
        }
        ++issued;
      }
      // Let every copy this thread issued land before the CTA can exit.
      drain(tc::smem_u32(&sm.q_full), 0);
      for (int t = max(issued - NS, 0); t < issued; ++t) drain(tc::smem_u32(&sm.full[t % NS]), (uint32_t)(t / NS) & 1u);
    }
   } else if (warp <= SOFTMAX_WARPS + 2) {
    // ------------------------------------------------------------ MMA issuers, one thread for each
    // half.  A wait takes a place in the scheduler's queue behind up to 32 exponentials of the
    // softmax warps there, some 270 cycles even if the barrier is ready, so one thread could
    // not keep up with both halves, and each waits for as little as it can.
    if (n_tiles > 0 && tc::elect_one()) {
      const int h = warp - SOFTMAX_WARPS - 1;
      const int hull_lo = sm.hull[h][0], hull_hi = sm.hull[h][1];
      Walk walk(sm.segments, first_tile, last_tile);
      uint32_t scores = 0, outputs = 0;  // S and P V products so far
      bool ok = true;
      const uint32_t q_lo = desc_lo_k(tc::smem_u32(sm.q[h])), k_lo = desc_lo_k(tc::smem_u32(sm.k));
      const uint32_t v_lo = desc_lo_v(tc::smem_u32(sm.v));
      const uint32_t s_tmem = tmem_base + (uint32_t)s_col(h), o_tmem = tmem_base + (uint32_t)o_col<D>(h);
      const auto await = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && wait_bounded(tc::smem_u32(bar), parity & 1u, abort_flag);
      };
      int waiting = -1;  // stage of the tile whose second product has not been issued
      const auto issue_pv = [&]() {
        const uint32_t buffer = outputs & 1u;
        await(&sm.p_full[h][buffer], outputs >> 1);
        if (!ok) return;
        tc::fence_after_sync();
        const uint32_t b = v_lo + (uint32_t)waiting * (TILE_BYTES >> 4);
#pragma unroll
        for (int t = 0; t < BKV / 16; ++t)
          mma_ts(o_tmem, tmem_base + (uint32_t)p_col(h, 0) + buffer * 32u + t * 8, b + t * (2048 >> 4), idesc_pv<D, FP16>(),
                 t > 0 || outputs > 0);
        tc::mma_commit(tc::smem_u32(&sm.o_full[h][buffer]));
        tc::mma_commit(tc::smem_u32(&sm.empty[waiting]));
        ++outputs;
        waiting = -1;
      };
      await(&sm.q_full, 0);
      int begin, end;
#pragma unroll 1
      for (int j = 0; walk.next(begin, end) && ok; ++j) {
        const int s = j % NS;
        await(&sm.clean[s], (uint32_t)j / NS);
        if (begin >= hull_hi || end <= hull_lo) {  // not this half's
          if (waiting >= 0) issue_pv();
          if (ok) tc::mbar_arrive(tc::smem_u32(&sm.empty[s]));
          continue;
        }
        if (scores > 0) await(&sm.s_free[h], scores - 1);  // the softmax has read the S before
        if (!ok) break;
        tc::fence_after_sync();
        const uint32_t b = k_lo + (uint32_t)s * (TILE_BYTES >> 4);
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
          mma_ss(s_tmem, q_lo + (uint32_t)(((t >> 2) * Q_BLOCK + (t & 3) * 32) >> 4),
                 b + (uint32_t)(((t >> 2) * KV_BLOCK + (t & 3) * 32) >> 4), idesc_qk<FP16>(), t > 0);
        tc::mma_commit(tc::smem_u32(&sm.s_full[h]));  // also the end of the P V products issued before
        ++scores;
        if (waiting >= 0) issue_pv();
        waiting = s;
      }
      if (waiting >= 0) issue_pv();
      // Every product has ended before tensor memory is freed.
      tc::mma_commit(tc::smem_u32(&sm.drained[h]));
      drain(tc::smem_u32(&sm.drained[h]), 0);
    }
    __syncwarp();
   } else {
    // ------------------------------------------------------------ keys behind a segment: whatever
    // lies there in V becomes zero before it meets P's zeros
    const int common_from = sm.common[0], common_to = sm.common[1];
    Walk walk(sm.segments, first_tile, last_tile);
    int begin, end;
    for (int j = 0; walk.next(begin, end); ++j) {
      const int s = j % NS;
      const bool ok = wait_bounded(tc::smem_u32(&sm.full[s]), (uint32_t)(j / NS) & 1u, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) break;
      const int keys = BKV - (end - begin);
      if (keys > 0) {
        for (int c = lane; c < keys * 8 * NB; c += 32) {
          const int b = c / (keys * 8), rest = c - b * keys * 8;
          *reinterpret_cast<uint4*>(sm.v[s][b] + (end - begin) * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
        }
        tc::fence_proxy_async_smem();
      }
      if (begin < common_from || begin + BKV > common_to) {
        // Values that are not finite, in keys that some row may not see: all exponent bits set, so that
        // one more unit of the exponent carries into the sign, two values of a word at once.
        constexpr uint32_t EXP = FP16 ? 0x7C007C00u : 0x7F807F80u, UNIT = FP16 ? 0x04000400u : 0x00800080u;
        uint32_t carry = 0;
        for (int c = lane; c < (end - begin) * 8; c += 32) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint4 w = *reinterpret_cast<const uint4*>(sm.v[s][b] + c * 16);
            carry |= ((w.x & EXP) + UNIT) | ((w.y & EXP) + UNIT) | ((w.z & EXP) + UNIT) | ((w.w & EXP) + UNIT);
          }
        }
        carry = __reduce_or_sync(0xffffffffu, carry & 0x80008000u);
        if (lane == 0) sm.odd[s] = carry != 0;
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(tc::smem_u32(&sm.clean[s]));
    }
   }
  } else {
    // ------------------------------------------------------------ softmax, one thread per row
    const int h = warp >> 2;
    const uint32_t lanes = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_tmem = lanes + (uint32_t)s_col(h), o_tmem = lanes + (uint32_t)o_col<D>(h);
    const int hull_lo = sm.hull[h][0], hull_hi = sm.hull[h][1];
    const float scale2 = p.scale * LOG2E, cap2 = p.cap * LOG2E;
    const float factor = CAP ? p.scale / p.cap : 0.f;
    const float slope2 = BIAS ? __ldg(p.slopes + head) * LOG2E : 0.f;
    // Keys that every row of the warp sees (rows without keys do not count), and the keys that its rows stand at.
    const bool has_keys = hi > lo;
    const int all_lo = __reduce_max_sync(0xffffffffu, has_keys ? lo : 0);
    const int all_hi = __reduce_min_sync(0xffffffffu, has_keys ? hi : 0x7FFFFFFF);
    const int first_pos = __reduce_min_sync(0xffffffffu, pos), last_pos = __reduce_max_sync(0xffffffffu, pos);
    // Reference maximum of the stored exponentials, at most 2^16 below the row's own.
    float m = -INFINITY;
    float l = 0.f;
    int sequence = 0;
    bool ok = true, redo = false;
    const auto await = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && wait_bounded(tc::smem_u32(bar), parity & 1u, abort_flag);
      __syncwarp();
      tc::fence_after_sync();
    };
    Walk walk(sm.segments, first_tile, last_tile);
    int begin, end;
    for (int j = 0; walk.next(begin, end); ++j) {
      if (begin >= hull_hi || end <= hull_lo) continue;
      const uint32_t buffer = (uint32_t)sequence & 1u;
      const uint32_t p_tmem = lanes + (uint32_t)p_col(h, 0) + buffer * 32u;
      await(&sm.s_full[h], sequence);
      float2 s[BKV / 2];
      {
        uint32_t raw[2][32];
#pragma unroll
        for (int i = 0; i < 2; ++i) tc::tmem_ld_32x32b_x32(s_tmem + i * 32, raw[i]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < BKV / 2; ++i)
          s[i] = make_float2(__uint_as_float(raw[i >> 4][2 * i & 31]), __uint_as_float(raw[i >> 4][(2 * i & 31) + 1]));
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(tc::smem_u32(&sm.s_free[h]));
      if (CAP) cap_scores(s, factor, cap2);
      if (BIAS) {
        const int from = begin - pos;  // of the tile's first key, from the row's own
        const float2 unit = both(CAP ? 1.f : scale2);
        if (begin + BKV <= first_pos || begin >= last_pos) {
          // the whole tile on one side of the rows: the distance is linear in the key
          const float slope = here(begin >= last_pos ? -slope2 : slope2), base = slope * (float)from;
#pragma unroll
          for (int i = 0; i < BKV / 2; ++i)
            s[i] = fma2(s[i], unit, make_float2(fmaf(slope, (float)(2 * i), base), fmaf(slope, (float)(2 * i + 1), base)));
        } else {
#pragma unroll
          for (int i = 0; i < BKV / 2; ++i)
            s[i] = fma2(s[i], unit, make_float2(-slope2 * fabsf((float)from + (float)(2 * i)),
                                                -slope2 * fabsf((float)from + (float)(2 * i + 1))));
        }
      }
      bool visible = has_keys;
      if (begin < all_lo || begin + BKV > all_hi) {
        const int c0 = lo - begin, c1 = min(hi, end) - begin;  // columns that this row sees
#pragma unroll
        for (int i = 0; i < BKV / 2; ++i) {
          s[i].x = 2 * i >= c0 && 2 * i < c1 ? s[i].x : -INFINITY;
          s[i].y = 2 * i + 1 >= c0 && 2 * i + 1 < c1 ? s[i].y : -INFINITY;
        }
        visible = c1 > max(c0, 0);
        await(&sm.clean[j % NS], (uint32_t)j / NS);
        redo = redo || sm.odd[j % NS] != 0;
      }
      // Exponentials against the reference at hand, which the tiles before have set.  Only where a row
      // has none yet, or its sum says that it was too low for P's type, is the tile's maximum
      // taken, O rescaled and the tile done again: a maximum of every tile, which the exponentials
      // would wait for, is not needed.
      const float2 unit = both(CAP || BIAS ? 1.f : scale2);
      // This P's product of two tiles ago has ended: its thread issued it before this S.
      for (bool again = false;; again = true) {
        const float2 offset = both(m == -INFINITY ? 0.f : RAISE<FP16> - m);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t packed[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 z = CAP || BIAS ? add2(s[part * 16 + i], offset) : fma2(s[part * 16 + i], unit, offset);
            const float2 e = make_float2(ex2(z.x), ex2(z.y));
            sum[i & 1] = add2(sum[i & 1], e);
            packed[i] = pack2<FP16>(e.x, e.y);
          }
          tc::tmem_st_32x32b_x16(p_tmem + part * 16, packed);
        }
        sum[0] = add2(sum[0], sum[1]);
        const float total = sum[0].x + sum[0].y;
        const bool low = visible && (m == -INFINITY || !(total <= P_LIMIT));
        if (again || !__any_sync(0xffffffffu, low)) {
          l += total;
          break;
        }
        float top[4] = {s[0].x, s[0].y, s[1].x, s[1].y};
#pragma unroll
        for (int i = 2; i < BKV / 2; ++i) top[i & 3] = max3(top[i & 3], s[i].x, s[i].y);
        float m_new = max3(fmaxf(top[0], top[1]), top[2], top[3]);
        if (!CAP && !BIAS) m_new *= scale2;
        float a = 1.f;
        if (m_new > m) {
          a = m == -INFINITY ? 0.f : ex2(m - m_new);
          m = m_new;
          l *= a;
        }
        __syncwarp();
        if (sequence > 0) {  // once the product before has ended
          await(&sm.o_full[h][buffer ^ 1u], (sequence - 1) >> 1);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {  // sixteen columns at a time: the scores stay in registers
            uint32_t raw[16];
            tc::tmem_ld_32x32b_x16(o_tmem + i * 16, raw);
            tc::tmem_wait_ld();
#pragma unroll
            for (int t = 0; t < 16; ++t) raw[t] = __float_as_uint(__uint_as_float(raw[t]) * a);
            tc::tmem_st_32x32b_x16(o_tmem + i * 16, raw);
          }
        }
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(tc::smem_u32(&sm.p_full[h][buffer]));
      ++sequence;
    }
    // ------------------------------------------------------------ output
    const int r = h * BQ + (warp & 3) * 32 + lane;
    const long long row = row0 + r;
    const bool valid = doc >= 0;
    if (sequence > 0) await(&sm.o_full[h][(sequence - 1) & 1], (sequence - 1) >> 1);
    if (__all_sync(0xffffffffu, ok)) {
      if (redo) {
        rows_key_by_key<D, FP16>(p, sm.segments, first_tile, last_tile, row0 + r - lane, head, lo, hi, pos, valid, split);
      } else {
        tc::fence_after_sync();
        if (!has_keys) m = -INFINITY, l = 0.f;
        const float inv = p.splits == 1 ? inverse_sum(l, has_keys) : 1.f;
        const long long at = (split * p.q_rows + row) * p.heads + head;
        if (valid && p.splits > 1) p.part_ml[at] = partial_ml(m, l, has_keys);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t raw[32];
          __syncwarp();
          if (sequence > 0) {
            tc::tmem_ld_32x32b_x32(o_tmem + i * 32, raw);
            tc::tmem_wait_ld();
          }
          if (!has_keys) {  // whatever tensor memory holds
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
    if (lane == 0 && *abort_flag) atomicExch(p.err, MUSC_B200_ERR_TIMEOUT);
  }
}

template <int D, bool FP16, bool CAP, bool BIAS>
int launch(Params p, cudaStream_t s) {
  p.err = device_error_ptr();
  if (!p.err) return fail(MUSC_B200_ERR_CUDA, "masked_attention: device error word unavailable");
  const long long grid = (long long)p.row_tiles * p.heads * p.splits;
  if (grid > 0x7FFFFFFFLL) return fail(MUSC_B200_ERR_INVALID, "masked_attention: too many rows and heads");
  const int qw = p.heads * D, kw = p.kv_heads * D;
  CUtensorMap mq, mk, mv;
  MUSC_TRY(make_token_map(&mq, p.q, p.q_rows, qw, p.q_rows > 1 ? p.q_stride : qw, FP16, BQ));
  MUSC_TRY(make_token_map(&mk, p.k, p.kv_rows, kw, p.kv_rows > 1 ? p.k_stride : kw, FP16, BKV));
  MUSC_TRY(make_token_map(&mv, p.v, p.kv_rows, kw, p.kv_rows > 1 ? p.v_stride : kw, FP16, BKV));
  constexpr auto kernel = tiles_kernel<D, FP16, CAP, BIAS>;
  MUSC_TRY(opt_in_smem<kernel>(SMEM_BYTES<D>));
  kernel<<<(unsigned)grid, THREADS, SMEM_BYTES<D>, s>>>(mq, mk, mv, p);
  return check_launch("masked tiles_kernel");
}

template <int D, bool FP16>
int launch_form(const Params& p, cudaStream_t s) {
  if (p.cap > 0.f) return p.slopes ? launch<D, FP16, true, true>(p, s) : launch<D, FP16, true, false>(p, s);
  return p.slopes ? launch<D, FP16, false, true>(p, s) : launch<D, FP16, false, false>(p, s);
}

}  // namespace

// One wave of CTAs (148 SMs): a second one costs more than the finer division gives (2048 tokens of 16
// heads x 64 in 37 us, with two waves 57).  With a causal mask the last rows' CTAs take twice the mean, and long
// ones are divided for that: 8192 tokens of 4 heads x 64 in 78 us, in one piece 120; 2753 tokens of
// 16 heads x 128 in 53 us, divided 80.
int tiles_splits(long long units, long long keys, bool causal) {
  units = std::max<long long>(units, 1);
  long long splits = std::min<long long>(148 / units, keys / 256);
  if (causal) splits = std::max(splits, std::min<long long>((2 * 148 + units / 2) / units, keys / 2048));
  return (int)std::max<long long>(1, std::min<long long>(splits, MAX_TILE_SPLITS));
}

// Documents begin tiles of their own (long ones; runs of short ones share them) where they have 64 rows in
// the mean: a tile that holds the end of one long document and the start of another walks both one's keys.
bool tiles_aligned(const Params& p) {
  return p.q_offsets ? p.documents <= SHARED_DOCS && p.q_rows >= 64LL * p.documents : p.q_len >= ROWS;
}

// A bound of the row tiles: the documents' lengths are only known on the device.  Every run after the first
// adds at most one tile to the packed rows' own; there are at most two for every document of ROWS rows, and one.
long long tiles_of_rows(const Params& p) {
  const long long packed = (p.q_rows + ROWS - 1) / ROWS;
  if (!p.aligned) return packed;
  if (!p.q_offsets) return p.documents * ((p.q_len + ROWS - 1) / ROWS);
  return packed + std::min<long long>(p.documents, 2 * (p.q_rows / ROWS) + 1) - 1;
}

int tiles_launch(const Params& p, int head_dim, bool fp16, cudaStream_t s) {
  if (head_dim == 64) return fp16 ? launch_form<64, true>(p, s) : launch_form<64, false>(p, s);
  return fp16 ? launch_form<128, true>(p, s) : launch_form<128, false>(p, s);
}

}  // namespace masked
}  // namespace musc
