// Entry point of masked attention (masked.cuh has the operator): checks, the choice of the
// kernel and of the splits, and the kernel that joins the splits' partial sums.
#include "masked.cuh"

#include <algorithm>
#include <cmath>
#include <string>

namespace musc {
namespace masked {
namespace {

// Joins the splits: out = sum_s w_s O_s / sum_s w_s l_s with w_s = 2^(m_s - max m).  One
// warp per (row, head); the lanes hold the splits' weights, and the partial outputs, which were
// just written and come out of L2, are loaded eight splits ahead.
template <int D, bool FP16>
__global__ void __launch_bounds__(128) combine_kernel(const Params p) {
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= p.q_rows * p.heads) return;
  const int lane = threadIdx.x & 31;
  const long long row = unit / p.heads;
  if (p.q_offsets && (row < __ldg(p.q_offsets) || row >= __ldg(p.q_offsets + p.documents))) return;  // of no document
  const long long per_split = p.q_rows * p.heads;
  float m[2], l[2], w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // splits lane and lane + 32
    const int s = lane + 32 * i;
    const float2 ml = s < p.splits ? p.part_ml[s * per_split + unit] : make_float2(-INFINITY, 0.f);
    m[i] = ml.x, l[i] = ml.y;
  }
  const float common = warp_max(fmaxf(m[0], m[1]));
  float total = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] = split_weight(m[i], common);
    total = fmaf(w[i], l[i], total);
    if (l[i] == 0.f) w[i] = 0.f;  // nothing was written for it
  }
  total = warp_sum(total);
  float acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  const float* part = p.part + unit * D + lane * (D / 32);
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) {
    const float weight = __shfl_sync(0xffffffffu, s < 32 ? w[0] : w[1], s & 31);
    float o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = weight != 0.f ? part[s * per_split * D + i] : 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(weight, o[i], acc[i]);
  }
  const float inv = inverse_sum(total, common != -INFINITY);
  const int head = (int)(unit - row * p.heads);
  uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.out_stride + (long long)head * D + lane * (D / 32);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const float v = acc[i] * inv;
    out[i] = FP16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
  }
}

}  // namespace

int combine_launch(const Params& p, int head_dim, bool fp16, cudaStream_t s) {
  const unsigned grid = (unsigned)((p.q_rows * p.heads + 3) / 4);
  if (head_dim == 64)
    fp16 ? combine_kernel<64, true><<<grid, 128, 0, s>>>(p) : combine_kernel<64, false><<<grid, 128, 0, s>>>(p);
  else
    fp16 ? combine_kernel<128, true><<<grid, 128, 0, s>>>(p) : combine_kernel<128, false><<<grid, 128, 0, s>>>(p);
  return check_launch("masked combine_kernel");
}

namespace {

struct Plan {
  bool tiles = false;
  int splits = 1, block_rows = 1;
  size_t ml_offset = 0, bytes = 0;
};

// Keys of a document, as far as the host knows: of packed ones the mean.
long long mean_keys(const musc_b200_masked_attention_args& a) {
  return a.q_offsets ? (a.kv_rows + a.documents - 1) / a.documents : a.kv_len;
}

// Whether the tile kernel is the faster one, by estimates in microseconds for mean documents that were
// fitted to 110 shapes (1 to 490 documents of 2 to 1865 rows over 2 to 14000 keys).  Over the faster of both:
// 0.5 % in the mean, at most 1.42 times; on 110 others 0.6 % and 1.45 times.  A CTA of the row kernel takes up
// to 16 rows x heads of one document and key head; one of the tile kernel takes 256 rows of one head over the
// keys of all documents in them, and starts slowly.
//   43 documents of 3 rows over 366 keys, 16/2 heads x 64: rows 8.6 us, tiles 211
//   129 documents of 1020 rows, 1 head x 64: rows 268 us, tiles 101
//   403 documents of 12 rows, 16 heads x 128: rows 116 us, tiles 58
//   2 documents of 4 rows over 20000 keys, 8/1 heads x 128: rows 25 us, tiles 52
// Means: a call of one long document and many short ones takes one kernel for both.  One of 4096 rows with 63 of
// 1 row over 4096 keys each, 32/8 heads x 128, takes tiles, whose 63 single rows share a row tile that walks all
// their keys: 4.5 ms, 0.35 in two calls.
// A row tile of a head has at most MAX_TILE_SPLITS CTAs, so fewer than five of them leave SMs idle.  On 103 shapes
// of 1 to 300 rows, 1 to 8 heads and 8000 to 1000000 keys: 5 % over the faster of both in the mean, at most
// 1.46 times (without that bound 15 % and 2.45 times).
//   1 row over 300000 keys, 1 head x 64: rows 48 us, tiles 106
//   256 rows over 300000 keys, 2 heads x 64: rows 272 us, tiles 146
bool tiles_faster(const musc_b200_masked_attention_args& a, long long units) {
  const double keys = (double)mean_keys(a), rows = std::max(1.0, (double)a.q_rows / a.documents);
  const double fill = units / (a.head_dim == 64 ? 592.0 : 444.0);
  // a lone unit's keys in eight splits, or in as many as pay (40 keys' times each, and the second launch)
  const double lone = std::min(0.12 * keys, 450 + 2 * std::sqrt(40 * keys));
  const double rows_time = 2 + 3 * std::max(1.0, fill) + (fill * keys + lone) * (a.head_dim == 64 ? 0.0075 : 0.0106);
  const double tiles = rows < 256 ? std::ceil(a.q_rows / 256.0) : a.documents * std::ceil(rows / 256);
  const double tile_keys = rows < 256 ? keys * std::min((double)a.documents, std::ceil(256 / rows)) : keys;
  const double sms = std::min(148.0, MAX_TILE_SPLITS * tiles * a.heads);
  return 10 + (2 + 0.7 * tile_keys / 64) * tiles * a.heads / sms < rows_time;
}

Plan make_plan(const musc_b200_masked_attention_args& a) {
  Plan plan;
  const long long rows = a.q_rows * a.heads;
  const int group = a.heads / a.kv_heads;
  plan.block_rows = rows_together(group, a.q_rows > a.documents);
  const long long mean_rows = (a.q_rows + a.documents - 1) / a.documents;
  const long long used = std::min<long long>(plan.block_rows, mean_rows);
  // documents that have rows: at most as many as there are rows
  const long long units = std::min<long long>(a.documents, a.q_rows) * ((mean_rows + used - 1) / used) * a.kv_heads * ((group + 15) / 16);
  plan.tiles = a.kv_rows > 0 && tiles_faster(a, units);
  if (plan.tiles)
    plan.splits = tiles_splits((a.q_rows + 255) / 256 * a.heads, mean_keys(a), a.causal != 0);
  else
    plan.splits = rows_splits(units, mean_keys(a), (int)used * std::min(group, 16), a.head_dim);
  if (plan.splits > (plan.tiles ? 1 : MAX_CLUSTER)) {
    plan.ml_offset = ((size_t)plan.splits * rows * a.head_dim * sizeof(float) + 255) / 256 * 256;
    plan.bytes = plan.ml_offset + (size_t)plan.splits * rows * sizeof(float2);
  }
  return plan;
}

int invalid(const char* what) { return fail(MUSC_B200_ERR_INVALID, std::string("masked_attention: ") + what); }

int check_args(const musc_b200_masked_attention_args& a) {
  if (a.dtype != MUSC_B200_F16 && a.dtype != MUSC_B200_BF16) return invalid("dtype must be f16 or bf16");
  if (a.head_dim != 64 && a.head_dim != 128) return invalid("head_dim must be 64 or 128");
  if (a.heads <= 0 || a.kv_heads <= 0 || a.heads % a.kv_heads != 0 || a.heads > 4096)
    return invalid("heads must be a multiple of kv_heads, both positive, at most 4096");
  if (a.q_rows < 0 || a.kv_rows < 0 || a.q_rows > 0x7FFFFFFF - 256 || a.kv_rows > 0x7FFFFFFF - 256)
    return invalid("q_rows and kv_rows must be below 2^31 - 256");
  if (a.documents < 0) return invalid("documents must not be negative");
  if (!(a.scale >= 1e-20f && a.scale <= 1e20f)) return invalid("scale must be from 1e-20 to 1e20");
  if (a.softcap != 0.f && !(a.softcap >= 1e-15f && a.softcap <= 1e15f))
    return invalid("softcap must be 0 (none) or from 1e-15 to 1e15");
  if (a.prefix && !a.causal) return invalid("a prefix needs causal");
  if (a.q_offsets) {
    if (!a.kv_offsets) return invalid("q_offsets and kv_offsets go together");
  } else {
    if (a.kv_offsets) return invalid("q_offsets and kv_offsets go together");
    // (an empty batch has no rows, whatever its items' length)
    if (a.q_len < 0 || a.kv_len < 0 || a.kv_pitch < a.kv_len || (a.documents > 0 && a.q_len > a.q_rows) || a.kv_pitch > 0x7FFFFFFF)
      return invalid("0 <= q_len <= q_rows and 0 <= kv_len <= kv_pitch < 2^31");
    if (a.q_len * a.documents != a.q_rows) return invalid("documents of q_len rows must make q_rows");
    if (a.documents > 0 && (a.documents - 1) * a.kv_pitch + a.kv_len > a.kv_rows)
      return invalid("the documents' key slots must lie within kv_rows");
  }
  return MUSC_B200_OK;
}

int check_tensors(const musc_b200_masked_attention_args& a) {
  const long long qw = (long long)a.heads * a.head_dim, kw = (long long)a.kv_heads * a.head_dim;
  if (!a.q || !a.out || (a.kv_rows > 0 && (!a.k || !a.v))) return invalid("null pointer");
  if ((a.q_rows > 1 && (a.q_stride < qw || a.out_stride < qw)) || (a.kv_rows > 1 && (a.k_stride < kw || a.v_stride < kw)))
    return invalid("row strides must hold all heads of a row");
  for (long long s : {a.q_rows > 1 ? a.q_stride : 0, a.q_rows > 1 ? a.out_stride : 0, a.kv_rows > 1 ? a.k_stride : 0,
                      a.kv_rows > 1 ? a.v_stride : 0})
    if (s % 8 != 0 || s >= (1LL << 36)) return invalid("row strides must be multiples of 8 below 2^36");
  for (const void* ptr : {a.q, a.k, a.v, (const void*)a.out})
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0) return invalid("q, k, v and out must be 16-byte aligned");
  // Byte ranges that a matrix spans: the output may share none of them.
  const auto begin = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr); };
  const auto end = [](const void* ptr, long long rows, long long stride, long long width) {
    return reinterpret_cast<uintptr_t>(ptr) + (rows > 0 ? ((rows - 1) * stride + width) * 2 : 0);
  };
  const uintptr_t o0 = begin(a.out), o1 = end(a.out, a.q_rows, a.out_stride, qw);
  if ((o0 < end(a.q, a.q_rows, a.q_stride, qw) && begin(a.q) < o1) ||
      (o0 < end(a.k, a.kv_rows, a.k_stride, kw) && begin(a.k) < o1) ||
      (o0 < end(a.v, a.kv_rows, a.v_stride, kw) && begin(a.v) < o1))
    return invalid("out must not overlap q, k or v");
  for (const void* ptr : {(const void*)a.q_offsets, (const void*)a.kv_offsets, (const void*)a.kv_lengths,
                          (const void*)a.prefix, (const void*)a.slopes})
    if (reinterpret_cast<uintptr_t>(ptr) % 4 != 0) return invalid("offsets, lengths and slopes must be 4-byte aligned");
  return MUSC_B200_OK;
}

}  // namespace
}  // namespace masked
}  // namespace musc

using namespace musc;

extern "C" size_t musc_b200_masked_attention_bytes(const musc_b200_masked_attention_args* args) {
  if (!args || masked::check_args(*args) != MUSC_B200_OK || args->q_rows == 0 || args->documents == 0) return 0;
  return masked::make_plan(*args).bytes;
}

extern "C" int musc_b200_masked_attention_plan(const musc_b200_masked_attention_args* args, int* tile_kernel, int* splits) {
  using namespace masked;
  if (!args || !tile_kernel || !splits) return invalid("null arguments");
  *tile_kernel = *splits = 0;
  MUSC_TRY(check_args(*args));
  if (args->q_rows == 0 || args->documents == 0) return MUSC_B200_OK;
  const Plan plan = make_plan(*args);
  *tile_kernel = plan.tiles, *splits = plan.splits;
  return MUSC_B200_OK;
}

extern "C" int musc_b200_masked_attention(const musc_b200_masked_attention_args* args, musc_b200_stream stream) {
  using namespace masked;
  if (!args) return invalid("null arguments");
  const musc_b200_masked_attention_args& a = *args;
  MUSC_TRY(check_args(a));
  if (a.q_rows == 0 || a.documents == 0) return MUSC_B200_OK;  // no row belongs to a document
  MUSC_TRY(check_tensors(a));
  const Plan plan = make_plan(a);
  if (plan.bytes > 0) {
    if (!a.workspace || a.workspace_bytes < plan.bytes)
      return fail(MUSC_B200_ERR_WORKSPACE, "masked_attention: workspace smaller than musc_b200_masked_attention_bytes");
    if (reinterpret_cast<uintptr_t>(a.workspace) % 256 != 0) return invalid("workspace must be 256-byte aligned");
  }
  MUSC_TRY(require_sm100());
  Params p;
  p.q = a.q, p.k = a.k, p.v = a.v, p.out = a.out;
  p.q_stride = a.q_stride, p.k_stride = a.k_stride, p.v_stride = a.v_stride, p.out_stride = a.out_stride;
  p.q_rows = a.q_rows, p.kv_rows = a.kv_rows;
  p.q_offsets = a.q_offsets, p.kv_offsets = a.kv_offsets, p.kv_lengths = a.kv_lengths, p.prefix = a.prefix;
  p.documents = a.documents;
  p.q_len = a.q_len, p.kv_len = a.kv_len, p.kv_pitch = a.kv_pitch;
  p.slopes = a.slopes;
  p.heads = a.heads, p.kv_heads = a.kv_heads, p.group = a.heads / a.kv_heads;
  p.causal = a.causal, p.scale = a.scale, p.cap = a.softcap;
  p.splits = plan.splits;
  // A document's blocks of rows begin at its first row.  Packed, document d's are counted from
  // q_offsets[d] / block_rows + d on, which leaves room for the last one of every document.
  p.block_rows = plan.block_rows;
  p.row_blocks = p.block_rows == 1 ? a.q_rows
                 : a.q_offsets     ? a.q_rows / p.block_rows + a.documents
                                   : a.documents * ((a.q_len + p.block_rows - 1) / p.block_rows);
  p.part = static_cast<float*>(a.workspace);
  p.part_ml = plan.bytes ? reinterpret_cast<float2*>(static_cast<char*>(a.workspace) + plan.ml_offset) : nullptr;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool fp16 = a.dtype == MUSC_B200_F16;
  p.aligned = tiles_aligned(p), p.row_tiles = 0;
  const long long row_tiles = tiles_of_rows(p);
  if (row_tiles > 0x7FFFFFFF) return invalid("too many rows");
  p.row_tiles = (int)row_tiles;
  MUSC_TRY(plan.tiles ? tiles_launch(p, a.head_dim, fp16, s) : rows_launch(p, a.head_dim, fp16, s));
  if (plan.bytes > 0) MUSC_TRY(combine_launch(p, a.head_dim, fp16, s));
  return MUSC_B200_OK;
}
