// Masked attention: what its kernels share.  For a query row i of a document with nq
// queries and nk keys and a key j of the same document, in 32 bits,
//
//   z = scale * q_i . k_j;   z = cap * tanh(z / cap)          (cap > 0)
//   z -= slope[head] * |i + (nk - nq) - j|                     (slopes given)
//   out_i = sum_j exp(z_ij) v_j / sum_j exp(z_ij)              over the keys that row i sees
//
// A row sees no other document's keys; with `causal` only the keys up to its own position
// i + (nk - nq), or the document's first prefix[d] keys where those reach further.  Every
// one of these masks leaves a row one interval of the packed keys, which is all that the
// kernels know of them.  A row that sees no key gets zeros.
#pragma once

#include "common.cuh"

#include <float.h>

namespace musc {
namespace masked {

struct Params {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  long long q_stride, k_stride, v_stride, out_stride;  // elements between consecutive rows
  long long q_rows, kv_rows;
  // Documents: by offsets, or (q_offsets null) equal ones of q_len rows with key slots
  // kv_pitch rows apart.
  const int* q_offsets;
  const int* kv_offsets;
  const int* kv_lengths;  // null: a slot is used whole
  const int* prefix;
  int documents;
  long long q_len, kv_len, kv_pitch;
  const float* slopes;
  int heads, kv_heads, group;  // group = heads / kv_heads
  int causal;
  float scale, cap;
  // Keys split over `splits` CTAs: unnormalised partial outputs in 32 bits
  // [split][row][head][head_dim] with each row's reference maximum and sum beside them.
  int splits;
  float* part;
  float2* part_ml;
  int* err;
  // Tile kernel: grid of row tiles, and whether documents begin their own (masked_tiles.cu).
  int row_tiles, aligned;
  // Row kernel: rows of a document that a CTA takes, and the number of such blocks of rows that are looked at.
  int block_rows;
  long long row_blocks;
};

// Keys [lo, hi) of the packed keys that a row sees, and the key its own position falls on.
// lo is the first key of the row's document.  Whatever the offsets hold, 0 <= lo <= hi <= kv_rows.
// Also the document's keys, those that every row of it sees, and the rows from this one to its last.
struct Interval {
  long long lo, hi, pos, keys, least, rows_left;
};

// End of the keys that the row `after` rows behind an interval's own sees, in the same document.
__device__ __forceinline__ long long interval_end(const Params& p, const Interval& iv, int after) {
  if (!p.causal) return iv.lo + iv.keys;
  return iv.lo + min(max(max(iv.pos + after + 1 - iv.lo, iv.least), 0LL), iv.keys);
}

// Packed rows before document d, cut to the rows there are: what an offset claims beyond them has no rows,
// and none that would move a row's position.
__device__ __forceinline__ int row_offset(const Params& p, int d) {
  return (int)min(max((long long)__ldg(p.q_offsets + d), 0LL), p.q_rows);
}

// Document of a row: the last one that begins at or before it.  -1: the row belongs to none.
__device__ __forceinline__ int find_document(const Params& p, long long row) {
  if (!p.q_offsets) return (int)(row / p.q_len);
  if (row < __ldg(p.q_offsets) || row >= __ldg(p.q_offsets + p.documents)) return -1;
  int lo = 0, hi = p.documents;  // offsets[lo] <= row < offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(p.q_offsets + mid) <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ Interval row_interval(const Params& p, int doc, long long row) {
  long long q0, nq, k0, nk;
  if (p.q_offsets) {
    q0 = row_offset(p, doc);
    nq = row_offset(p, doc + 1) - q0;
    k0 = min(max((long long)__ldg(p.kv_offsets + doc), 0LL), p.kv_rows);
    nk = min(max((long long)__ldg(p.kv_offsets + doc + 1), k0), p.kv_rows) - k0;
  } else {
    q0 = doc * p.q_len;
    nq = p.q_len;
    k0 = doc * p.kv_pitch;
    nk = p.kv_len;
  }
  if (p.kv_lengths) nk = min(max((long long)__ldg(p.kv_lengths + doc), 0LL), nk);
  Interval r;
  r.lo = k0;
  r.pos = k0 + (row - q0) + (nk - nq);
  r.keys = nk;
  r.least = p.causal && p.prefix ? __ldg(p.prefix + doc) : 0;
  r.rows_left = q0 + nq - row;
  r.hi = interval_end(p, r, 0);
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float LOG2E = 1.4426950408889634f;

// tanh(x) / x as a polynomial in x^2 for |x| <= 0.4, fitted for the least maximum error of tanh (2e-8).
__device__ constexpr float TANH3[4] = {0.999999583f, -0.333297253f, 0.13250567f, -0.0468257405f};

// cap tanh(s scale / cap) log2(e), with factor = scale / cap and cap2 = cap log2(e).  For larger x = s factor as
// cap2 - 2 cap2 / (1 + e^(2 x)), off by 2^-23 of cap2; a small x would lose its value to that, the
// more the higher the cap, and takes the polynomial.
__device__ __forceinline__ float capped_log2(float s, float factor, float cap2) {
  const float x = s * factor, t = x * x;
  const float small = cap2 * x * fmaf(fmaf(fmaf(TANH3[3], t, TANH3[2]), t, TANH3[1]), t, TANH3[0]);
  const float large = fmaf(-2.f * cap2, rcp(1.f + ex2(x * (2.f * LOG2E))), cap2);
  return fabsf(x) <= 0.4f ? small : large;
}

// log2 by which the stored exponentials are raised.  In fp16 a weight below 2^-24 of the row's
// largest would be lost; raised by 2^6 (and by what a running maximum lags, which the kernels bound so
// that sums of them stay below 65504) it keeps 2^-30.  Sums carry the same factor, which cancels.  bf16 has fp32's range.
template <bool FP16>
constexpr float RAISE = FP16 ? 6.f : 0.f;

template <bool FP16>
__device__ __forceinline__ float widen(uint16_t v) {
  return FP16 ? __half2float(__ushort_as_half(v)) : __bfloat162float(__ushort_as_bfloat16(v));
}

// Two values in one word.  Both kernels round the exponentials P this way before P V, because the tensor cores take both
// operands in one type: half a step of each (2^-11 in fp16, 2^-8 in bf16), against 64 bits 1.2 to 1.4 times the
// error that the rounding of the result alone leaves.  The sum that divides the result is of the unrounded ones.
template <bool FP16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (FP16) {
    __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&t);
  }
  __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&t);
}

// A row and head's sums over keys [first, end) by a warp, key by key: lanes hold D / 32 dimensions of q and
// of the sums.  The slow form, for rows beside values that are not finite and that they do not see.
// Index: of keys and their distances.
template <int D, bool FP16, typename Index>
__device__ __forceinline__ void attend_keys(const Params& p, const float (&q)[D / 32], int kv_head, float slope2, Index pos,
                                            int first, int end, float (&acc)[D / 32], float& m, float& l) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  for (int key = first; key < end; ++key) {
    const uint16_t* k = static_cast<const uint16_t*>(p.k) + key * p.k_stride + kv_head * D + lane * N;
    const uint16_t* v = static_cast<const uint16_t*>(p.v) + key * p.v_stride + kv_head * D + lane * N;
    float dot = 0.f;
    for (int i = 0; i < N; ++i) dot = fmaf(q[i], widen<FP16>(k[i]), dot);
    dot = warp_sum(dot);
    float z = p.cap > 0.f ? capped_log2(dot, p.scale / p.cap, p.cap * LOG2E) : dot * p.scale * LOG2E;
    if (p.slopes) z = fmaf(-slope2, fabsf((float)(key - pos)), z);
    const float m_new = fmaxf(m, z);
    const float a = m == -INFINITY ? 0.f : ex2(m - m_new);
    m = m_new;
    // a key whose score is -inf adds nothing, NaN scores add NaN
    const float e = z == -INFINITY ? 0.f : ex2(z - m);
    l = fmaf(l, a, e);
    for (int i = 0; i < N; ++i) acc[i] = fmaf(e, widen<FP16>(v[i]), acc[i] * a);
  }
}

// A split's partial result of a row and head: its reference maximum and its sum.  The maximum of a
// row that sees keys is finite even where it met none of them; (-inf, 0) says that it sees no key.
__device__ __forceinline__ float2 partial_ml(float m, float l, bool any_key) {
  return make_float2(any_key ? fmaxf(m, -FLT_MAX) : -INFINITY, l);
}

// Weight of a split's partial sums against the row's common maximum.
__device__ __forceinline__ float split_weight(float m, float common) {
  return m == -INFINITY ? 0.f : ex2(m - common);
}

// 1 / l of a finished row.  Sums of zero: a row without keys gets zeros, one whose every
// visible score is -inf gets NaN, as 0 / 0.
__device__ __forceinline__ float inverse_sum(float l, bool any_key) {
  if (l == 0.f) return any_key ? NAN : 0.f;
  return 1.f / l;
}

// The kernels' launchers, and the splits of the keys that give `units` CTAs of work enough CTAs
// when a document has about `keys` keys.
constexpr int MAX_TILE_SPLITS = 32;
constexpr int MAX_CLUSTER = 8;  // up to so many splits the row kernel joins by itself, without a workspace
int rows_launch(const Params& p, int head_dim, bool fp16, cudaStream_t stream);
int rows_together(int group, bool several);  // several: rows a document
int rows_splits(long long units, long long keys, int rows, int head_dim);  // rows: of a block's products
int tiles_launch(const Params& p, int head_dim, bool fp16, cudaStream_t stream);
int tiles_splits(long long units, long long keys, bool causal);
bool tiles_aligned(const Params& p);
long long tiles_of_rows(const Params& p);  // row tiles of the grid
int combine_launch(const Params& p, int head_dim, bool fp16, cudaStream_t stream);

}  // namespace masked
}  // namespace musc
