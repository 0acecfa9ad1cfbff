// Attention of a batch's newest tokens over the paged cache (glm_paged_attention).
//
// Row (b, t, h) sees the positions j < len_b - (q_len - 1 - t) of request b:
//   s_j = scale q . k_j,  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m = max_j s_j.
// The cache is read once, so the positions are cut into items that fill the
// chip whatever the lengths are: every workgroup reads the lengths and cuts
// them alike (attn_item), keeps a running maximum and sum over its item's
// positions, and a request cut into several items is joined by a second
// launch (attn_join_kernel) from their partial results (m, l, acc).
#include <climits>
#include <cmath>

#include "glm_common.h"

namespace glm {

constexpr int kAttnTile = 64;  // positions; items are whole tiles
constexpr float kLog2e = 1.44269504088896341f;

struct AttnArgs {
  const uint16_t *q;
  long long q_stride;  // elements from token to token
  const void *kc, *vc;  // caches [page][kv head][page size][dim]; vc null: values are kc's first channels
  const uint8_t *ks, *vs;
  const int32_t *tables, *lens;
  uint16_t *out;
  int2 *plan;        // [B] {splits, first partial}, for the join
  float *part, *ml;  // partial results [item][rows][dv], [item][rows][2]
  int B, q_len, heads, kv_heads, dk, dv, num_pages, page, max_blocks;
  int rows;     // rows of an item: one kv head's row block
  int hblocks;  // kv_heads x row blocks
  int target, min_c;  // items wanted over all, fewest tiles of an item
  float scale_log2;
};

// The rows of a kv head: row = token * group + head of the group.
__device__ __forceinline__ int attn_rows(const AttnArgs &a) { return a.q_len * (a.heads / a.kv_heads); }

__device__ __forceinline__ int attn_len(const AttnArgs &a, int b) {
  return max(0, min(a.lens[b], a.max_blocks * a.page));
}

struct AttnItem {
  int b, hb, len, t0, t1;      // request, head block, its length, tile range
  int splits, split, partial;  // of the request; this item's, and the request's first partial
};

// This workgroup's item: c tiles of one request and head block, c the least
// that gives at most `target` items beyond one a request.  Every wave finds it
// by itself from the lengths (no barrier, no plan from the host).  False for a
// workgroup past the last item.
__device__ __forceinline__ bool attn_item(const AttnArgs &a, int block, AttnItem &it) {
  const int lane = threadIdx.x & 63;
  int total = 0;
  for (int b = lane; b < a.B; b += kWave) total += (attn_len(a, b) + kAttnTile - 1) / kAttnTile;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, kWave);
  const int c =
      max(a.min_c, (int)(((long long)total * a.hblocks + a.target - 1) / a.target));
  const int s = block / a.hblocks;
  it.hb = block - s * a.hblocks;
  int upto_s = 0, upto_p = 0;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const int b = b0 + lane;
    const int len = b < a.B ? attn_len(a, b) : 0;
    const int nt = (len + kAttnTile - 1) / kAttnTile;
    const int mine = b < a.B ? max(1, (nt + c - 1) / c) : 0;
    int sum_s = mine, sum_p = mine > 1 ? mine : 0;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int vs = __shfl_up(sum_s, off, kWave), vp = __shfl_up(sum_p, off, kWave);
      if (lane >= off) {
        sum_s += vs;
        sum_p += vp;
      }
    }
    const int first = upto_s + sum_s - mine;
    const unsigned long long hit = __ballot(s >= first && s < first + mine);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      it.b = b0 + l;
      it.len = __builtin_amdgcn_readlane(len, l);
      it.splits = __builtin_amdgcn_readlane(mine, l);
      it.split = s - __builtin_amdgcn_readlane(first, l);
      it.partial = upto_p + __builtin_amdgcn_readlane(sum_p, l) - (it.splits > 1 ? it.splits : 0);
      it.t0 = it.split * c;
      it.t1 = min((it.len + kAttnTile - 1) / kAttnTile, it.t0 + c);
      return true;
    }
    upto_s += __builtin_amdgcn_readlane(sum_s, kWave - 1);
    upto_p += __builtin_amdgcn_readlane(sum_p, kWave - 1);
  }
  return false;
}

__device__ __forceinline__ void attn_plan(const AttnArgs &a, const AttnItem &it) {
  if (it.split == 0 && it.hb == 0 && threadIdx.x == 0) a.plan[it.b] = int2{it.splits, it.partial};
}
__device__ __forceinline__ long long attn_partial(const AttnArgs &a, const AttnItem &it) {
  return (long long)(it.partial + it.split) * a.hblocks + it.hb;
}

// The cache row (of dk or dv elements) of a request's position, -1 where its
// page is not one of the cache's.
__device__ __forceinline__ long long cache_row(const AttnArgs &a, const int32_t *table, int head,
                                               int pos) {
  const int id = table[pos / a.page];
  if ((uint32_t)id >= (uint32_t)a.num_pages) return -1;
  return ((long long)id * a.kv_heads + head) * a.page + pos % a.page;
}

__device__ __forceinline__ float cache_value(const void *cache, const uint8_t *scales, int fmt,
                                             long long row, int dim, int ch) {
  if (fmt == GLM_FMT_BF16) return bf16_to_f32(((const uint16_t *)cache)[row * dim + ch]);
  const float sc = e8m0_to_f32(scales[row * (dim / 32) + ch / 32]);
  const uint32_t code = ((const uint8_t *)cache)[row * dim + ch];
  return (float)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code, sc, false)[0];
}

// ---------------------------------------------------------------------------
// Any widths: one row a workgroup, 256 positions at a time.  A thread forms
// one position's score, then the threads share the channels of the values.
// ---------------------------------------------------------------------------
constexpr int kAnyDim = 1024;

template <int FMT>
__global__ __launch_bounds__(256) void attn_any_kernel(AttnArgs a) {
  __shared__ float s_q[kAnyDim], s_p[256], s_red[4];
  __shared__ long long s_row[256];
  AttnItem it;
  if (!attn_item(a, blockIdx.x, it)) return;
  attn_plan(a, it);
  const int tid = threadIdx.x, R = attn_rows(a), group = a.heads / a.kv_heads;
  const int head = it.hb / R, r = it.hb - head * R, t = r / group;
  const uint16_t *q = a.q + ((long long)it.b * a.q_len + t) * a.q_stride +
                      (head * group + r % group) * a.dk;
  for (int ch = tid; ch < a.dk; ch += 256) s_q[ch] = bf16_to_f32(q[ch]);
  const int32_t *table = a.tables + (long long)it.b * a.max_blocks;
  const int end = min(it.t1 * kAttnTile, it.len - (a.q_len - 1 - t));
  const void *vc = a.vc ? a.vc : a.kc;
  const uint8_t *vs = a.vc ? a.vs : a.ks;
  const int vdim = a.vc ? a.dv : a.dk;
  float m = -INFINITY, l = 0.0f, acc[kAnyDim / 256] = {};
  __syncthreads();
  for (int p0 = it.t0 * kAttnTile; p0 < end; p0 += 256) {
    const int pos = p0 + tid;
    const long long row = pos < end ? cache_row(a, table, head, pos) : -1;
    float s = -INFINITY;
    if (row >= 0) {
      s = 0.0f;
      for (int ch = 0; ch < a.dk; ++ch)
        s += s_q[ch] * cache_value(a.kc, a.ks, FMT, row, a.dk, ch);
      s *= a.scale_log2;
    }
    float top = s;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
    if ((tid & 63) == 0) s_red[tid >> 6] = top;
    __syncthreads();
    const float next = fmaxf(m, fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3])));
    const float from = next == -INFINITY ? 0.0f : next;
    const float keep = exp2f(m - from);
    m = next;
    const float p = row >= 0 ? exp2f(s - from) : 0.0f;
    s_p[tid] = p;
    s_row[tid] = row;
    __syncthreads();
    l *= keep;
#pragma unroll
    for (int i = 0; i < kAnyDim / 256; ++i) acc[i] *= keep;
    const int n = min(256, end - p0);
    for (int j = 0; j < n; ++j) {
      const float pj = s_p[j];
      l += pj;
      const long long rj = s_row[j];
      if (rj < 0) continue;
#pragma unroll
      for (int i = 0; i < kAnyDim / 256; ++i)
        if (tid + 256 * i < a.dv) acc[i] += pj * cache_value(vc, vs, FMT, rj, vdim, tid + 256 * i);
    }
    __syncthreads();
  }
  if (it.splits == 1) {
    uint16_t *out = a.out + (((long long)it.b * a.q_len + t) * a.heads + head * group + r % group) * a.dv;
#pragma unroll
    for (int i = 0; i < kAnyDim / 256; ++i)
      if (tid + 256 * i < a.dv) out[tid + 256 * i] = (uint16_t)f32_to_bf16(l == 0.0f ? 0.0f : acc[i] / l);
  } else {
    const long long at = attn_partial(a, it);
#pragma unroll
    for (int i = 0; i < kAnyDim / 256; ++i)
      if (tid + 256 * i < a.dv) a.part[at * a.dv + tid + 256 * i] = acc[i];
    if (tid == 0) *reinterpret_cast<float2 *>(a.ml + 2 * at) = float2{m, l};
  }
}

// ---------------------------------------------------------------------------
// The requests that were cut into several items: out = sum_i 2^(m_i - m) acc_i
// / sum_i 2^(m_i - m) l_i over the items in order.  A thread has four channels
// of a row.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  const int b = blockIdx.y;
  const int2 plan = a.plan[b];
  if (plan.x <= 1) return;
  const int R = attn_rows(a), group = a.heads / a.kv_heads, rb = a.hblocks / a.kv_heads;
  const int i = blockIdx.x * 256 + threadIdx.x, quads = a.dv / 4;
  const int row = i / quads, ch = 4 * (i - row * quads);
  if (row >= a.kv_heads * R) return;
  const int head = row / R, r = row - head * R;
  const int hb = head * rb + r / a.rows;
  const long long first = (long long)plan.y * a.hblocks + hb;
  float m = -INFINITY;
  for (int s = 0; s < plan.x; ++s)
    m = fmaxf(m, a.ml[2 * ((first + (long long)s * a.hblocks) * a.rows + r % a.rows)]);
  const float from = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  glm_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < plan.x; ++s) {
    const long long at = (first + (long long)s * a.hblocks) * a.rows + r % a.rows;
    const float2 ml = *reinterpret_cast<const float2 *>(a.ml + 2 * at);
    const float w = exp2f(ml.x - from);
    l += w * ml.y;
    acc += w * *reinterpret_cast<const glm_f32x4 *>(a.part + at * a.dv + ch);
  }
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = f32_to_bf16(l == 0.0f ? 0.0f : acc[j] / l);
  const int t = r / group;
  uint16_t *out = a.out + (((long long)b * a.q_len + t) * a.heads + head * group + r % group) * a.dv + ch;
  *reinterpret_cast<uint2 *>(out) = uint2{o[0] | (o[1] << 16), o[2] | (o[3] << 16)};
}

}  // namespace glm

namespace {

struct AttnSizes {
  int rows, hblocks, target, min_c;
  long long grid, partials;  // workgroups; partial results
  size_t plan_bytes, part_bytes, ml_bytes;
};

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// Sizes that follow from a call's shape; false for shapes that are refused.
bool attn_sizes(int B, int q_len, int heads, int kv_heads, int key_dim, int value_dim, int page_size,
                int max_blocks, AttnSizes &z) {
  if (B < 0 || q_len < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || key_dim < 1 ||
      value_dim < 1 || page_size < 1 || max_blocks < 1)
    return false;
  if (B > 65535 || q_len > 16 || heads > 1024 || (long long)max_blocks * page_size > INT_MAX - glm::kAttnTile)
    return false;
  const int R = q_len * (heads / kv_heads);
  z.rows = 1;
  z.hblocks = kv_heads * R;
  z.target = 2048;
  z.min_c = 4;
  const long long tiles = ((long long)max_blocks * page_size + glm::kAttnTile - 1) / glm::kAttnTile;
  if (tiles * B > INT_MAX / 2 || (long long)B * z.hblocks > INT_MAX / 2) return false;
  const long long splits = (tiles + z.min_c - 1) / z.min_c;
  z.grid = z.hblocks * B * splits;
  if (z.grid > z.target + (long long)z.hblocks * B) z.grid = z.target + (long long)z.hblocks * B;
  // a request of nt > c tiles has at most 2 nt / c items, so at most 2 target / hblocks over all
  long long p = B * splits;
  if (p > 2LL * z.target / z.hblocks) p = 2LL * z.target / z.hblocks;
  if (splits == 1) p = 0;
  z.partials = p * z.hblocks;
  z.plan_bytes = up256((size_t)B * sizeof(int2));
  z.part_bytes = up256((size_t)z.partials * z.rows * value_dim * sizeof(float));
  z.ml_bytes = up256((size_t)z.partials * z.rows * 2 * sizeof(float));
  return true;
}

}  // namespace

extern "C" size_t glm_paged_attention_workspace_bytes(int B, int q_len, int heads, int kv_heads,
                                                      int key_dim, int value_dim, int page_size,
                                                      int max_blocks) {
  AttnSizes z;
  if (!attn_sizes(B, q_len, heads, kv_heads, key_dim, value_dim, page_size, max_blocks, z)) return 0;
  return z.plan_bytes + z.part_bytes + z.ml_bytes + 256;
}

extern "C" int glm_paged_attention(void *stream, const uint16_t *q, int64_t q_stride, int B,
                                   int q_len, int heads, int kv_heads, int key_dim, int value_dim,
                                   const void *key_cache, const uint8_t *key_scales,
                                   const void *value_cache, const uint8_t *value_scales, int fmt,
                                   int num_pages, int page_size, const int32_t *tables,
                                   const int32_t *lens, int max_blocks, float scale,
                                   void *workspace, size_t workspace_bytes, uint16_t *out) {
  glm::clear_error();
  const bool mx = fmt == GLM_FMT_MXFP8, shared = value_cache == nullptr;
  GLM_REQUIRE(fmt == GLM_FMT_BF16 || mx, GLM_ERR_INVALID_ARGUMENT,
              "paged_attention: unsupported format %d", fmt);
  GLM_REQUIRE(q && key_cache && tables && lens && workspace && out && (!mx || key_scales) &&
                  (!mx || shared || value_scales),
              GLM_ERR_INVALID_ARGUMENT, "paged_attention: null pointer");
  GLM_REQUIRE(B >= 0 && q_len >= 1 && heads >= 1 && kv_heads >= 1 && key_dim >= 1 &&
                  value_dim >= 1 && num_pages >= 1 && page_size >= 1 && max_blocks >= 1,
              GLM_ERR_INVALID_ARGUMENT, "paged_attention: invalid sizes");
  GLM_REQUIRE(heads % kv_heads == 0, GLM_ERR_UNSUPPORTED_SHAPE,
              "paged_attention: %d heads over %d kv heads", heads, kv_heads);
  const int unit = mx ? 32 : 8;
  GLM_REQUIRE(key_dim % unit == 0 && value_dim % unit == 0 && key_dim <= glm::kAnyDim &&
                  value_dim <= glm::kAnyDim,
              GLM_ERR_UNSUPPORTED_SHAPE,
              "paged_attention: widths %d and %d must be multiples of %d up to %d", key_dim,
              value_dim, unit, glm::kAnyDim);
  GLM_REQUIRE(!shared || value_dim <= key_dim, GLM_ERR_UNSUPPORTED_SHAPE,
              "paged_attention: values of %d channels in rows of %d", value_dim, key_dim);
  GLM_REQUIRE((long long)num_pages * page_size * kv_heads <= INT_MAX, GLM_ERR_UNSUPPORTED_SHAPE,
              "paged_attention: %d pages of %d x %d rows pass 32 bits", num_pages, kv_heads,
              page_size);
  AttnSizes z;
  GLM_REQUIRE(attn_sizes(B, q_len, heads, kv_heads, key_dim, value_dim, page_size, max_blocks, z),
              GLM_ERR_UNSUPPORTED_SHAPE,
              "paged_attention: batch %d, %d tokens, %d heads or %d blocks of %d are too many", B,
              q_len, heads, max_blocks, page_size);
  GLM_REQUIRE(q_stride >= (int64_t)heads * key_dim && q_stride % 8 == 0, GLM_ERR_INVALID_ARGUMENT,
              "paged_attention: the query's token stride must cover the heads and be a multiple of 8");
  GLM_REQUIRE(std::isfinite(scale * glm::kLog2e), GLM_ERR_INVALID_ARGUMENT, "paged_attention: scale is not finite");
  GLM_REQUIRE(glm_aligned16({q, key_cache, key_scales, value_cache, value_scales, workspace, out}),
              GLM_ERR_INVALID_ARGUMENT, "paged_attention: buffers must be 16-byte aligned");
  const uintptr_t ws = ((uintptr_t)workspace + 255) & ~(uintptr_t)255;
  const size_t need = z.plan_bytes + z.part_bytes + z.ml_bytes;
  GLM_REQUIRE(workspace_bytes >= need + (ws - (uintptr_t)workspace), GLM_ERR_WORKSPACE,
              "paged_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need + 256);
  if (B == 0) return GLM_OK;
  glm::AttnArgs a{};
  a.q = q;
  a.q_stride = q_stride;
  a.kc = key_cache;
  a.vc = value_cache;
  a.ks = key_scales;
  a.vs = value_scales;
  a.tables = tables;
  a.lens = lens;
  a.out = out;
  a.plan = (int2 *)ws;
  a.part = (float *)(ws + z.plan_bytes);
  a.ml = (float *)(ws + z.plan_bytes + z.part_bytes);
  a.B = B;
  a.q_len = q_len;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dk = key_dim;
  a.dv = value_dim;
  a.num_pages = num_pages;
  a.page = page_size;
  a.max_blocks = max_blocks;
  a.rows = z.rows;
  a.hblocks = z.hblocks;
  a.target = z.target;
  a.min_c = z.min_c;
  a.scale_log2 = scale * glm::kLog2e;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)z.grid);
  if (mx)
    hipLaunchKernelGGL(glm::attn_any_kernel<GLM_FMT_MXFP8>, grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(glm::attn_any_kernel<GLM_FMT_BF16>, grid, dim3(256), 0, s, a);
  GLM_LAUNCH_CHECK("attn_any_kernel");
  if (z.partials > 0) {
    const long long quads = (long long)q_len * heads * value_dim / 4;
    hipLaunchKernelGGL(glm::attn_join_kernel, dim3((unsigned)((quads + 255) / 256), B), dim3(256), 0,
                       s, a);
    GLM_LAUNCH_CHECK("attn_join_kernel");
  }
  return GLM_OK;
}
