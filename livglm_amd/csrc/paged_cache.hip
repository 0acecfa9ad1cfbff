// The paged attention cache: pages taken and given back from request lengths
// (glm_cache_step), and new rows written into their slots (glm_cache_write).
#include <climits>

#include "glm_common.h"

namespace glm {

// ---------------------------------------------------------------------------
// One step of the cache's bookkeeping, for B requests:
//   gone_b = new_b < 0, n_b = gone_b ? -1 - new_b : new_b,
//   base_b = gone_b ? 0 : len_b, have_b = gone_b ? 0 : blocks_b,
//   need_b = max(0, ceil((base_b + n_b) / page) - have_b).
// The pages of requests that are gone go on top of the free stack in request
// order; the i-th new page (requests in order, blocks in order) is the i-th
// from the top.  Three exclusive sums over the requests (pages given back,
// pages needed, tokens) say where each of them lies, so every page and token
// is then a thread's own work: it finds its request by bisection in LDS.
// One workgroup, since a page given back may be taken in the same call and
// only a workgroup can wait for its own writes; bound by latency: the
// requests' loads, the pages', the tables': 6 us for 64 requests of one token,
// of a call's 9.5.  The tokens' slots ride in this launch up to kStepTokens and
// take a launch over all CUs beyond: 12.7 us for 13.9 at 6748 tokens, 18.4 for
// 13.5 at 14010.
// ---------------------------------------------------------------------------
constexpr int kStepThreads = 1024;
constexpr int kStepRequests = 4096;  // three sums per request in LDS
constexpr int kStepTokens = 8192;

struct StepSums {
  long long given, need, tokens;
};
__device__ __forceinline__ StepSums operator+(const StepSums &a, const StepSums &b) {
  return {a.given + b.given, a.need + b.need, a.tokens + b.tokens};
}
__device__ __forceinline__ StepSums shfl_up(const StepSums &a, int by) {
  return {__shfl_up(a.given, by, kWave), __shfl_up(a.need, by, kWave),
          __shfl_up(a.tokens, by, kWave)};
}

// The last request r in [0, B) with first[r] <= i, for ascending first[0] = 0.
__device__ __forceinline__ int owner_of(const int *first, int B, int i) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Token t of a step: its slot and position, from the sums of the requests'
// tokens and their new lengths.  tables as this step left them; an entry that
// is no page of the cache gives no slot (times page, it might name another's).
__device__ __forceinline__ void token_slot(int t, int B, const int *cu, const int32_t *kv_lens,
                                           const int32_t *tables, int max_blocks,
                                           int num_pages, int page, int32_t *slots,
                                           int32_t *positions) {
  int slot = -1, pos = 0;
  if (t < cu[B]) {
    const int r = owner_of(cu, B, t);
    pos = kv_lens[r] - cu[r + 1] + t;
    const int id = tables[(long long)r * max_blocks + pos / page];
    if ((uint32_t)id < (uint32_t)num_pages) slot = id * page + pos % page;
  }
  slots[t] = slot;
  positions[t] = pos;
}

__global__ __launch_bounds__(kStepThreads) void cache_step_kernel(
    const int32_t *new_lens, int B, int num_pages, int page, int max_blocks, int max_tokens,
    const int32_t *lens, int32_t *blocks, int32_t *tables, int32_t *free_pages, int32_t *num_free,
    int32_t *kv_lens, int32_t *cu_new, int32_t *slots, int32_t *positions, int32_t *status,
    bool own_slots) {
  __shared__ int s_given[kStepRequests + 1], s_need[kStepRequests + 1], s_cu[kStepRequests + 1];
  __shared__ StepSums s_wave[kStepThreads / kWave];
  __shared__ int s_flags;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nt = blockDim.x;
  const int per = (B + nt - 1) / nt;  // consecutive requests of a thread
  const int b0 = min(B, tid * per), b1 = min(B, b0 + per);
  const int top = *num_free;
  if (tid == 0) s_flags = 0;

  int flags = 0;
  StepSums mine{0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    const int nb = new_lens[b], len = lens[b], held = blocks[b];
    const bool gone = nb < 0;
    const long long n = gone ? -1 - nb : nb;
    const long long base = gone ? 0 : len, have = gone ? 0 : held, total = base + n;
    long long need = (total + page - 1) / page - have;
    need = need > 0 ? need : 0;
    if (total > (long long)max_blocks * page) flags |= GLM_CACHE_TABLE_FULL;
    if (len < 0 || held < 0 || held > max_blocks || base > have * page)
      flags |= GLM_CACHE_BAD_STATE;
    mine = mine + StepSums{gone ? held : 0, need, n};
  }
  // exclusive sums over the threads
  StepSums upto = mine;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const StepSums before = shfl_up(upto, off);
    if (lane >= off) upto = upto + before;
  }
  if (lane == kWave - 1) s_wave[wave] = upto;
  __syncthreads();
  if (flags) atomicOr(&s_flags, flags);
  StepSums at{0, 0, 0}, all{0, 0, 0};
  for (int w = 0; w < nt / kWave; ++w) {
    const StepSums v = s_wave[w];
    if (w < wave) at = at + v;
    all = all + v;
  }
  at = {at.given + upto.given - mine.given, at.need + upto.need - mine.need,
        at.tokens + upto.tokens - mine.tokens};
  __syncthreads();
  flags = s_flags;
  const long long left = (long long)top + all.given - all.need;
  if (left < 0) flags |= GLM_CACHE_OUT_OF_PAGES;
  if (all.tokens > max_tokens) flags |= GLM_CACHE_TOO_MANY_TOKENS;
  if (top < 0 || top + all.given > num_pages) flags |= GLM_CACHE_BAD_STATE;
  if (tid == 0) *status = flags;
  if (flags) {  // (uniform) nothing changes
    for (int b = b0; b < b1; ++b) {
      kv_lens[b] = lens[b];
      cu_new[b] = 0;
    }
    if (tid == 0) cu_new[B] = 0;
    if (own_slots)
      for (int t = tid; t < max_tokens; t += nt) {
        slots[t] = -1;
        positions[t] = 0;
      }
    return;
  }
  for (int b = b0; b < b1; ++b) {
    const int nb = new_lens[b];
    const bool gone = nb < 0;
    const int n = gone ? -1 - nb : nb, have = gone ? 0 : blocks[b];
    const int total = (gone ? 0 : lens[b]) + n;
    const int need = max(0, total / page + (total % page != 0) - have);  // (total + page may pass 32 bits)
    s_given[b] = (int)at.given;
    s_need[b] = (int)at.need;
    s_cu[b] = (int)at.tokens;
    cu_new[b] = (int)at.tokens;
    at = at + StepSums{gone ? blocks[b] : 0, need, n};
  }
  if (tid == 0) {
    s_given[B] = (int)all.given;
    s_need[B] = (int)all.need;
    s_cu[B] = (int)all.tokens;
    cu_new[B] = (int)all.tokens;
    *num_free = (int)left;
  }
  __syncthreads();
  const int given = s_given[B], needed = s_need[B];
  if (given > 0) {
    for (int i = tid; i < given; i += nt) {
      const int r = owner_of(s_given, B, i);
      int32_t *entry = tables + (long long)r * max_blocks + (i - s_given[r]);
      free_pages[top + i] = *entry;
      *entry = -1;
    }
    __syncthreads();
  }
  for (int i = tid; i < needed; i += nt) {
    const int r = owner_of(s_need, B, i);
    const int have = new_lens[r] < 0 ? 0 : blocks[r];
    tables[(long long)r * max_blocks + have + (i - s_need[r])] = free_pages[top + given - 1 - i];
  }
  __syncthreads();
  for (int b = b0; b < b1; ++b) {
    const bool gone = new_lens[b] < 0;
    const int len = lens[b];  // (kv_lens may be lens itself)
    blocks[b] = (gone ? 0 : blocks[b]) + s_need[b + 1] - s_need[b];
    kv_lens[b] = (gone ? 0 : len) + s_cu[b + 1] - s_cu[b];
  }
  if (!own_slots) return;
  __syncthreads();
  for (int t = tid; t < max_tokens; t += nt)
    token_slot(t, B, s_cu, kv_lens, tables, max_blocks, num_pages, page, slots, positions);
}

// The tokens' slots of a large step, over all CUs.
__global__ __launch_bounds__(256) void cache_slots_kernel(
    const int32_t *cu_new, const int32_t *kv_lens, const int32_t *tables, int B, int num_pages,
    int page, int max_blocks, int max_tokens, int32_t *slots, int32_t *positions) {
  __shared__ int s_cu[kStepRequests + 1];
  for (int b = threadIdx.x; b <= B; b += blockDim.x) s_cu[b] = cu_new[b];
  __syncthreads();
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t < max_tokens)
    token_slot(t, B, s_cu, kv_lens, tables, max_blocks, num_pages, page, slots, positions);
}

// ---------------------------------------------------------------------------
// New rows into their slots.  Cache layout [page][kv head][page size][dim]:
// a head's rows of one page lie together, so the attention streams them.
// A thread moves eight channels (16 bytes of bf16) of every so many tokens:
// what follows from the channel is formed once, and four tokens are in flight.
// Consecutive threads take consecutive channels of a token's keys, then of its
// values.  bf16 rows are copied; MXFP8 groups of 32 channels lie in four lanes,
// which find the group's largest magnitude by DPP and its exponent
//   e = the smallest >= -124 with amax <= 448 2^e
// from the bf16 bits alone (448 = 1.75 2^8), so no code saturates -- the
// rounding rules of glm_mx_quantize may cut a group's largest element by up
// to 29 %, which a softmax would see; -124, because 2^-9 2^-124 is bf16's own
// smallest step.  An infinity or a NaN is stored as E4M3's NaN and does not
// enter amax.  A slot outside the cache is skipped.
// Bound by the bytes: 13.4 us for 7777 tokens of 8 heads of 128 + 128 channels
// into MXFP8 (48 MB, 3.6 TB/s with the launch), 101 us for 60000 into bf16
// (491 MB, 4.9 TB/s); 2.9 us for 64 tokens, which is latency.
// ---------------------------------------------------------------------------
struct CacheWrite {
  const uint16_t *rows[2];  // keys, values
  long long stride[2];      // elements from token to token
  void *cache[2];
  uint8_t *scales[2];
  int dim[2];
  const int32_t *slots;
  int N, heads, page, num_slots;
  uint32_t page_magic;  // floor(2^32 / page), at most 2^32 - 1
};

// Eight bf16 channels as MXFP8, four lanes a group.
__device__ __forceinline__ uint2 mxfp8_codes(const glm_u32x4 &x, uint32_t &scale) {
  float f[8];
  int m = 0;  // largest finite magnitude's bf16 bits
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t bits = j % 2 ? x[j / 2] >> 16 : x[j / 2] & 0xffffu;
    const int mag = bits & 0x7fffu;
    m = mag < 0x7f80 ? max(m, mag) : m;
    f[j] = mag < 0x7f80 ? __uint_as_float(bits << 16) : __uint_as_float(0x7fc00000u);
  }
  m = max(m, __builtin_amdgcn_mov_dpp(m, 0xB1, 0xf, 0xf, true));
  m = max(m, __builtin_amdgcn_mov_dpp(m, 0x4E, 0xf, 0xf, true));
  const int e = max((m >> 7) - 127 - 8 + ((m & 0x7f) > 0x60 ? 1 : 0), -124);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);  // 2^-e, exact
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] *= inv;  // exact, within 448
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  uint32_t code[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    s16x2 o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(s16x2{0, 0}, f[4 * j], f[4 * j + 1], 1.0f, false);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, f[4 * j + 2], f[4 * j + 3], 1.0f, true);
    code[j] = __builtin_bit_cast(uint32_t, o);
  }
  scale = (uint32_t)(e + 127);
  return uint2{code[0], code[1]};
}

template <int FMT>
__global__ __launch_bounds__(256) void cache_write_kernel(CacheWrite a) {
  constexpr int kFlight = 4;
  const int keys = a.heads * a.dim[0] / 8, pieces = keys + a.heads * a.dim[1] / 8;
  const int tokens = pieces < 256 ? 256 / pieces : 1;  // of a workgroup at once
  const int tl = pieces < 256 ? threadIdx.x / pieces : 0;
  const int step = gridDim.x * tokens;
  for (int c0 = pieces < 256 ? threadIdx.x - tl * pieces : threadIdx.x; c0 < pieces && tl < tokens; c0 += 256) {
    const int v = c0 >= keys, c = c0 - (v ? keys : 0);
    const int dim = a.dim[v], head = c / (dim / 8), ch = 8 * (c - head * (dim / 8));
    const uint16_t *rows = a.rows[v] + 8 * c;
    for (int t0 = blockIdx.x * tokens + tl; t0 < a.N; t0 += kFlight * step) {
      int slot[kFlight];
      glm_u32x4 x[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        const int token = t0 + j * step;
        slot[j] = token < a.N ? a.slots[token] : -1;
        x[j] = *reinterpret_cast<const glm_u32x4 *>(rows + (long long)min(token, a.N - 1) * a.stride[v]);
      }
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        if ((uint32_t)slot[j] >= (uint32_t)a.num_slots) continue;  // (a token's lanes leave together)
        int page = (int)__umulhi((uint32_t)slot[j], a.page_magic), off = slot[j] - page * a.page;
        if (off >= a.page) {  // the quotient is one short at most
          ++page;
          off -= a.page;
        }
        const long long row = ((long long)page * a.heads + head) * a.page + off;
        if constexpr (FMT == GLM_FMT_BF16) {
          *reinterpret_cast<glm_u32x4 *>((uint16_t *)a.cache[v] + row * dim + ch) = x[j];
        } else {
          uint32_t scale;
          *reinterpret_cast<uint2 *>((uint8_t *)a.cache[v] + row * dim + ch) = mxfp8_codes(x[j], scale);
          if ((c & 3) == 0) a.scales[v][row * (dim / 32) + ch / 32] = (uint8_t)scale;
        }
      }
    }
  }
}

}  // namespace glm

extern "C" int glm_cache_step(void *stream, const int32_t *new_lens, int B, int num_pages,
                              int page_size, int max_blocks, int max_tokens, const int32_t *lens,
                              int32_t *blocks, int32_t *tables, int32_t *free_pages,
                              int32_t *num_free, int32_t *kv_lens, int32_t *cu_new,
                              int32_t *slots, int32_t *positions, int32_t *status) {
  glm::clear_error();
  GLM_REQUIRE(B >= 1 && num_pages >= 1 && page_size >= 1 && max_blocks >= 1 && max_tokens >= 0,
              GLM_ERR_INVALID_ARGUMENT, "cache_step: invalid sizes");
  GLM_REQUIRE(B <= glm::kStepRequests, GLM_ERR_UNSUPPORTED_SHAPE,
              "cache_step: %d requests, at most %d", B, glm::kStepRequests);
  GLM_REQUIRE(max_tokens <= 1 << 30, GLM_ERR_UNSUPPORTED_SHAPE,
              "cache_step: %d tokens, at most 2^30", max_tokens);
  GLM_REQUIRE((long long)num_pages * page_size <= INT_MAX &&
                  (long long)max_blocks * page_size <= INT_MAX,
              GLM_ERR_UNSUPPORTED_SHAPE,
              "cache_step: %d pages (%d a request) of %d tokens pass 32 bits", num_pages,
              max_blocks, page_size);
  GLM_REQUIRE(new_lens && lens && blocks && tables && free_pages && num_free && kv_lens && cu_new &&
                  status && (max_tokens == 0 || (slots && positions)),
              GLM_ERR_INVALID_ARGUMENT, "cache_step: null pointer");
  hipStream_t s = (hipStream_t)stream;
  const bool own = max_tokens <= glm::kStepTokens;
  hipLaunchKernelGGL(glm::cache_step_kernel, dim3(1), dim3(glm::kStepThreads), 0, s, new_lens, B,
                     num_pages, page_size, max_blocks, max_tokens, lens, blocks, tables, free_pages,
                     num_free, kv_lens, cu_new, slots, positions, status, own);
  GLM_LAUNCH_CHECK("cache_step_kernel");
  if (!own) {
    hipLaunchKernelGGL(glm::cache_slots_kernel, dim3((max_tokens + 255) / 256), dim3(256), 0, s,
                       cu_new, kv_lens, tables, B, num_pages, page_size, max_blocks, max_tokens,
                       slots, positions);
    GLM_LAUNCH_CHECK("cache_slots_kernel");
  }
  return GLM_OK;
}

extern "C" int glm_cache_write(void *stream, const uint16_t *keys, int64_t key_stride,
                               const uint16_t *values, int64_t value_stride, const int32_t *slots,
                               int N, int num_pages, int page_size, int kv_heads, int key_dim,
                               int value_dim, int fmt, void *key_cache, uint8_t *key_scales,
                               void *value_cache, uint8_t *value_scales) {
  glm::clear_error();
  const bool mx = fmt == GLM_FMT_MXFP8;
  GLM_REQUIRE(fmt == GLM_FMT_BF16 || mx, GLM_ERR_INVALID_ARGUMENT,
              "cache_write: unsupported format %d", fmt);
  GLM_REQUIRE(N >= 0 && num_pages >= 1 && page_size >= 1 && kv_heads >= 1 && key_dim >= 1 &&
                  value_dim >= 0,
              GLM_ERR_INVALID_ARGUMENT, "cache_write: invalid sizes");
  GLM_REQUIRE(keys && slots && key_cache && (!mx || key_scales) &&
                  (value_dim == 0 || (values && value_cache && (!mx || value_scales))),
              GLM_ERR_INVALID_ARGUMENT, "cache_write: null pointer");
  const int unit = mx ? 32 : 8;
  GLM_REQUIRE(key_dim % unit == 0 && value_dim % unit == 0 && key_dim <= 1024 && value_dim <= 1024,
              GLM_ERR_UNSUPPORTED_SHAPE,
              "cache_write: widths %d and %d must be multiples of %d up to 1024", key_dim,
              value_dim, unit);
  GLM_REQUIRE(N <= 1 << 30, GLM_ERR_UNSUPPORTED_SHAPE, "cache_write: %d tokens, at most 2^30", N);
  GLM_REQUIRE((long long)num_pages * page_size * kv_heads <= INT_MAX && kv_heads <= 65536,
              GLM_ERR_UNSUPPORTED_SHAPE, "cache_write: %d pages of %d x %d rows pass 32 bits",
              num_pages, kv_heads, page_size);
  GLM_REQUIRE(key_stride >= (int64_t)kv_heads * key_dim && key_stride % 8 == 0 &&
                  (value_dim == 0 ||
                   (value_stride >= (int64_t)kv_heads * value_dim && value_stride % 8 == 0)),
              GLM_ERR_INVALID_ARGUMENT,
              "cache_write: token strides must cover the heads and be multiples of 8");
  GLM_REQUIRE(glm_aligned16({keys, key_cache, key_scales}) &&
                  (value_dim == 0 || glm_aligned16({values, value_cache, value_scales})),
              GLM_ERR_INVALID_ARGUMENT, "cache_write: buffers must be 16-byte aligned");
  if (N == 0) return GLM_OK;
  glm::CacheWrite a{{keys, values}, {key_stride, value_stride}, {key_cache, value_cache},
                    {key_scales, value_scales}, {key_dim, value_dim}, slots, N, kv_heads,
                    page_size, num_pages * page_size,
                    page_size == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / page_size)};
  // as many workgroups as the chip holds, a thread's channels serve all its tokens: 7777 tokens with at most
  // 1024, 2048, no limit: 13.6, 14.0, 15.4 us, 60000 tokens 101.5, 101.4, 112.5
  const int pieces = kv_heads * (key_dim + value_dim) / 8, tokens = pieces < 256 ? 256 / pieces : 1;
  const int blocks = (N - 1) / tokens + 1;
  const dim3 grid(blocks < 2048 ? blocks : 2048);
  if (mx)
    hipLaunchKernelGGL(glm::cache_write_kernel<GLM_FMT_MXFP8>, grid, dim3(256), 0,
                       (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(glm::cache_write_kernel<GLM_FMT_BF16>, grid, dim3(256), 0,
                       (hipStream_t)stream, a);
  GLM_LAUNCH_CHECK("cache_write_kernel");
  return GLM_OK;
}
