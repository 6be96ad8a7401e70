// Rotary positions over several axes for the queries and keys of a block: pair p of every
// head's dimensions turns by the angle positions[token][axis[p]] * frequency[p],
//
//   y0 = x0 cos a - x1 sin a,   y1 = x1 cos a + x0 sin a,
//
// where (x0, x1) are dimensions (p, p + pairs) or, in the adjacent layout, (2p, 2p + 1);
// dimensions past 2 * pairs pass through.  It takes the place of the learned positions that
// the vision tower adds to its tokens (models/backbone/open_clip/transformer.py:570-574)
// where a grid has no fixed size.
//
// Each element is read once and written once and costs three operations, so memory bounds
// it.  The angles are the same for all heads of a token: a CTA takes a few tokens, puts
// their cosines and sines into shared memory once (tokens x pairs of them, instead of a
// table in memory that would be read beside q and k), and then streams q and k in 16-byte
// vectors, the first of them on their way while the angles are computed.  The angle is formed in 64 bits and reduced to a
// fraction of a turn before it is rounded to 32: a position of 100,000 has an angle whose
// 32-bit rounding is 4e-3 of a radian.  A token takes pairs 64-bit products, 1/40 of the
// kernel's instructions at 16 + 16 heads of 64.
#include "common.cuh"

#include <algorithm>

namespace musc {
namespace rotary {

constexpr int THREADS = 256;
constexpr int MAX_TOKENS = 16;  // tokens of a CTA: 32 KB of cosines and sines at most
// A CTA takes tokens until it has this many items (of two vectors), eight a thread, and loads them
// one by one: 65001 tokens of 20 heads of 128 take 123 us; with two or four loads in flight per
// thread the registers cost more CTAs than that gives (133, 157 us), with half the items the
// angles weigh more (127 us).
constexpr int ITEMS_PER_CTA = THREADS * 8;

struct Params {
  const void* in[2];
  void* out[2];
  long long in_stride[2], out_stride[2];
  const void* positions;
  const float* frequencies;
  const int* axis;
  long long tokens;
  int heads[2];
  int head_dim, pairs, axes;
  int tokens_per_cta;
  int float_positions;
  uint32_t token_magic, head_magic;  // ceil(2^32 / items of a token, of a head); 0: divide
};

// n / d with magic = ceil(2^32 / d), exact while n * d < 2^32.
__device__ __forceinline__ int divide(int n, int d, uint32_t magic) {
  return magic ? (int)__umulhi((uint32_t)n, magic) : n / d;
}

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Cosine and sine of the CTA's tokens, [token][pair].
__device__ __forceinline__ void fill_angles(const Params& p, long long t0, int n_tok, float2* table) {
  for (int e = threadIdx.x; e < n_tok * p.pairs; e += THREADS) {
    const int t = e / p.pairs, pair = e - t * p.pairs;
    const int axis = min(max(__ldg(p.axis + pair), 0), p.axes - 1);
    const long long at = (t0 + t) * p.axes + axis;
    const double pos = p.float_positions ? (double)__ldg(static_cast<const float*>(p.positions) + at)
                                         : (double)__ldg(static_cast<const int*>(p.positions) + at);
    const double turns = pos * (double)__ldg(p.frequencies + pair) * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    table[e] = make_float2(c, s);
  }
}

template <typename T>
union Vec {
  uint4 raw;
  T v[16 / sizeof(T)];
};

// VEC: 16-byte vectors (every row, head and half starts on a 16-byte boundary); otherwise
// one element at a time, for any alignment.
template <typename T, bool ADJACENT, bool VEC>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const Params p) {
  extern __shared__ float2 table[];
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  const long long t0 = (long long)blockIdx.x * p.tokens_per_cta;
  const int n_tok = (int)min((long long)p.tokens_per_cta, p.tokens - t0);
  // Items of a head: turned ones of V pairs each, then passed-through ones of 2 V elements.
  const int turned = p.pairs / V;
  const int rest = p.head_dim - 2 * p.pairs;
  const int per_head = turned + (rest + 2 * V - 1) / (2 * V);
  const int per_token = per_head * (p.heads[0] + p.heads[1]);
  const int total = per_token * n_tok;
  constexpr int U = VEC ? 1 : 4;
  for (int e0 = threadIdx.x; e0 - (int)threadIdx.x < total; e0 += THREADS * U) {  // uniform over the CTA
    Vec<T> a[U], b[U];
    T* dst[U];
    int second[U];   // offset of the item's second half from its first
    int angle[U];    // index of its first pair's angle, -1: passes through
    int count[U];    // halves
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * THREADS;
      count[u] = 0;
      if (e < total) {
        const int t = divide(e, per_token, p.token_magic);
        const int in_token = e - t * per_token;
        int head = divide(in_token, per_head, p.head_magic);
        const int item = in_token - head * per_head;
        const int which = head >= p.heads[0] ? 1 : 0;
        if (which) head -= p.heads[0];
        int first;
        if (item < turned) {
          first = ADJACENT ? item * 2 * V : item * V;
          second[u] = ADJACENT ? V : p.pairs;
          angle[u] = t * p.pairs + item * V;
          count[u] = 2;
        } else {
          first = 2 * p.pairs + (item - turned) * 2 * V;
          second[u] = V;
          angle[u] = -1;
          count[u] = first + V < p.head_dim ? 2 : 1;
        }
        const long long at = (long long)head * p.head_dim + first;
        const long long in_stride = which ? p.in_stride[1] : p.in_stride[0];
        const long long out_stride = which ? p.out_stride[1] : p.out_stride[0];
        const T* src = static_cast<const T*>(which ? p.in[1] : p.in[0]) + (t0 + t) * in_stride + at;
        dst[u] = static_cast<T*>(which ? p.out[1] : p.out[0]) + (t0 + t) * out_stride + at;
        if (VEC) {
          a[u].raw = *reinterpret_cast<const uint4*>(src);
          if (count[u] == 2) b[u].raw = *reinterpret_cast<const uint4*>(src + second[u]);
        } else {
          a[u].v[0] = src[0];
          if (count[u] == 2) b[u].v[0] = src[second[u]];
        }
      }
    }
    if (e0 == (int)threadIdx.x) {  // while the first items are on their way
      fill_angles(p, t0, n_tok, table);
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (count[u] == 0) continue;
      if (angle[u] >= 0) {
        const float2* cs = table + angle[u];
        if (ADJACENT && VEC) {  // a holds the pairs of the first V / 2 angles, b those of the others
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            const float2 c0 = cs[i], c1 = cs[V / 2 + i];
            const float x0 = to_float(a[u].v[2 * i]), x1 = to_float(a[u].v[2 * i + 1]);
            const float y0 = to_float(b[u].v[2 * i]), y1 = to_float(b[u].v[2 * i + 1]);
            a[u].v[2 * i] = from_float<T>(x0 * c0.x - x1 * c0.y);
            a[u].v[2 * i + 1] = from_float<T>(x1 * c0.x + x0 * c0.y);
            b[u].v[2 * i] = from_float<T>(y0 * c1.x - y1 * c1.y);
            b[u].v[2 * i + 1] = from_float<T>(y1 * c1.x + y0 * c1.y);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float2 c = cs[i];
            const float x0 = to_float(a[u].v[i]), x1 = to_float(b[u].v[i]);
            a[u].v[i] = from_float<T>(x0 * c.x - x1 * c.y);
            b[u].v[i] = from_float<T>(x1 * c.x + x0 * c.y);
          }
        }
      }
      if (VEC) {
        *reinterpret_cast<uint4*>(dst[u]) = a[u].raw;
        if (count[u] == 2) *reinterpret_cast<uint4*>(dst[u] + second[u]) = b[u].raw;
      } else {
        dst[u][0] = a[u].v[0];
        if (count[u] == 2) dst[u][second[u]] = b[u].v[0];
      }
    }
  }
}

template <typename T>
int launch(const Params& p, bool adjacent, bool vec, unsigned grid, size_t smem, cudaStream_t s) {
  if (adjacent && vec) rotary_kernel<T, true, true><<<grid, THREADS, smem, s>>>(p);
  else if (adjacent) rotary_kernel<T, true, false><<<grid, THREADS, smem, s>>>(p);
  else if (vec) rotary_kernel<T, false, true><<<grid, THREADS, smem, s>>>(p);
  else rotary_kernel<T, false, false><<<grid, THREADS, smem, s>>>(p);
  return check_launch("rotary_kernel");
}

// A block of `tokens` rows of `width` elements, `stride` apart.
struct Block {
  const char* base;
  long long stride, width, span;  // bytes
};

// Whether two blocks have an element in common.  Blocks of one stride are compared by
// columns (q and k are often column slices of one projection); other overlaps count as common.
bool overlap(const Block& a, const Block& b) {
  if (a.base + a.span <= b.base || b.base + b.span <= a.base) return false;
  if (a.stride != b.stride || a.stride == 0) return true;
  const long long diff = b.base > a.base ? b.base - a.base : a.base - b.base;
  const long long col = diff % a.stride;
  const bool b_right = b.base > a.base;  // the block to the right starts `col` bytes into the other's rows
  const long long left = b_right ? a.width : b.width, right = b_right ? b.width : a.width;
  return col < left || col + right > a.stride;
}

}  // namespace rotary
}  // namespace musc

using namespace musc;

extern "C" int musc_b200_rotary(const void* q, const void* k, void* q_out, void* k_out, int dtype, long long tokens,
                                int heads, int kv_heads, int head_dim, long long q_stride, long long k_stride,
                                long long q_out_stride, long long k_out_stride, const void* positions,
                                int float_positions, int axes, const float* frequencies, const int* axis, int pairs,
                                int adjacent, musc_b200_stream stream) {
  using namespace rotary;
  if (dtype != MUSC_B200_F32 && dtype != MUSC_B200_F16 && dtype != MUSC_B200_BF16)
    return fail(MUSC_B200_ERR_INVALID, "rotary: dtype must be f32, f16 or bf16");
  if (tokens < 0 || heads <= 0 || kv_heads < 0 || head_dim <= 0 || axes <= 0 || heads > 65536 || kv_heads > 65536)
    return fail(MUSC_B200_ERR_INVALID, "rotary: tokens >= 0, heads > 0, kv_heads >= 0, head_dim > 0 and axes > 0");
  if (head_dim > 512 || pairs <= 0 || 2 * pairs > head_dim)
    return fail(MUSC_B200_ERR_INVALID, "rotary: head_dim at most 512 and 1 <= pairs <= head_dim / 2");
  if (tokens == 0) return MUSC_B200_OK;
  if (!q || !q_out || !positions || !frequencies || !axis || (kv_heads > 0 && (!k || !k_out)))
    return fail(MUSC_B200_ERR_INVALID, "rotary: null pointer");
  for (const void* ptr : {positions, (const void*)frequencies, (const void*)axis})
    if (reinterpret_cast<uintptr_t>(ptr) % 4 != 0)
      return fail(MUSC_B200_ERR_INVALID, "rotary: positions, frequencies and axis must be aligned to 4 bytes");
  const long long widths[2] = {(long long)heads * head_dim, (long long)kv_heads * head_dim};
  const int size = dtype == MUSC_B200_F32 ? 4 : 2;
  Params p;
  p.in[0] = q, p.in[1] = k, p.out[0] = q_out, p.out[1] = k_out;
  p.in_stride[0] = q_stride, p.in_stride[1] = k_stride, p.out_stride[0] = q_out_stride, p.out_stride[1] = k_out_stride;
  p.heads[0] = heads, p.heads[1] = kv_heads;
  const int parts = kv_heads > 0 ? 2 : 1;
  bool vec = (size * head_dim) % 16 == 0 && (size * pairs) % 16 == 0;
  Block in[2], out[2];
  for (int i = 0; i < parts; ++i) {
    if (tokens > 1 && (p.in_stride[i] < widths[i] || p.out_stride[i] < widths[i]))
      return fail(MUSC_B200_ERR_INVALID, "rotary: row strides must hold all heads of a token");
    in[i] = {static_cast<const char*>(p.in[i]), p.in_stride[i] * size, widths[i] * size,
             ((tokens - 1) * p.in_stride[i] + widths[i]) * size};
    out[i] = {static_cast<const char*>(p.out[i]), p.out_stride[i] * size, widths[i] * size,
              ((tokens - 1) * p.out_stride[i] + widths[i]) * size};
    for (const Block* b : {&in[i], &out[i]}) {
      if (reinterpret_cast<uintptr_t>(b->base) % size != 0)
        return fail(MUSC_B200_ERR_INVALID, "rotary: pointers must be aligned to their element");
      vec = vec && reinterpret_cast<uintptr_t>(b->base) % 16 == 0 && (tokens == 1 || b->stride % 16 == 0);
    }
  }
  for (int i = 0; i < parts; ++i)
    for (int j = 0; j < parts; ++j) {
      const bool in_place = i == j && in[i].base == out[j].base && (tokens == 1 || in[i].stride == out[j].stride);
      if ((!in_place && overlap(in[i], out[j])) || (i != j && overlap(out[i], out[j])))
        return fail(MUSC_B200_ERR_INVALID, "rotary: an output may be its own input, and overlap nothing else");
    }
  MUSC_TRY(require_sm100());
  p.positions = positions, p.float_positions = float_positions, p.axes = axes;
  p.frequencies = frequencies, p.axis = axis, p.pairs = pairs, p.head_dim = head_dim;
  p.tokens = tokens;
  const int v = vec ? 16 / size : 1;
  const int per_head = pairs / v + (head_dim - 2 * pairs + 2 * v - 1) / (2 * v);
  const long long per_token = (long long)per_head * (heads + kv_heads);
  // More tokens in a CTA while one has few items, but not fewer than two CTAs per SM.
  long long n = ITEMS_PER_CTA / per_token;
  n = std::min<long long>(n, std::max<long long>(1, tokens / (2 * sm_count())));
  p.tokens_per_cta = (int)std::max<long long>(1, std::min<long long>(n, MAX_TOKENS));
  const long long grid = (tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
  if (grid > 0x7FFFFFFFLL || per_token * p.tokens_per_cta > 0x3FFFFFFFLL)
    return fail(MUSC_B200_ERR_INVALID, "rotary: too many tokens or heads");
  const long long most = std::max<long long>(per_token * p.tokens_per_cta, per_token) * per_token;
  p.token_magic = most < (1LL << 32) && per_token > 1 ? (uint32_t)(((1ULL << 32) + per_token - 1) / per_token) : 0;
  p.head_magic = most < (1LL << 32) && per_head > 1 ? (uint32_t)(((1ULL << 32) + per_head - 1) / per_head) : 0;
  const size_t smem = (size_t)p.tokens_per_cta * pairs * sizeof(float2);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == MUSC_B200_F32) return launch<float>(p, adjacent != 0, vec, (unsigned)grid, smem, s);
  if (dtype == MUSC_B200_F16) return launch<__half>(p, adjacent != 0, vec, (unsigned)grid, smem, s);
  return launch<__nv_bfloat16>(p, adjacent != 0, vec, (unsigned)grid, smem, s);
}
