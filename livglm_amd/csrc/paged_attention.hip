// Attention of a batch's newest tokens over the paged cache (glm_paged_attention).
//
// Row (b, t, h) sees the positions j < len_b - (q_len - 1 - t) of request b:
//   s_j = scale q . k_j,  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m = max_j s_j.
// The cache is read once, and the chip is filled whatever the lengths are: the
// tiles of all requests and kv heads, one after the other, are cut into as
// many equal parts as workgroups fit the chip (AttnWalk: every wave finds its
// part from the lengths), and a workgroup walks through its part, request by
// request, keeping a running maximum and sum.  What a cut leaves of a request
// on either side goes to the workspace as (m, l, acc), and a second launch
// (attn_join_kernel) joins it.
//
// Three forms, by the widths alone: the grouped one for heads of 64, 128, 256
// or 192 / 128 channels, the latent one for rows of 576 channels whose first
// 512 are the values, and one for all other widths.  The last form on the
// others' cases: 3513 us for 90 (32 ragged requests, 32 heads over 8 of 128),
// 387 for 26 (45 requests, 16 heads of 64), 49 for 13 (one request of 517),
// 15.9 ms for 57 us (64 latent requests).
#include <climits>
#include <cmath>

#include "glm_common.h"
#include "lds_stage.h"

namespace glm {

constexpr int kAttnTile = 64;  // positions; parts are cut between tiles
constexpr float kLog2e = 1.44269504088896341f;
// Weights are 2^(s - top): where a score passes top it is raised to that score and this many powers of two more,
// so that the sums are seldom rescaled.  None passes 1, and neither bf16 nor the sums in 32 bits lose a digit.  (With
// top the score itself and weights up to 2^8 one value near the type's largest made its sum infinite; now it takes
// 2^8 equal ones.)  A row's pieces are joined by their tops, whatever they lie above.
constexpr float kAttnSlack = 8.0f;

// Sums over the wave by DPP: row_shr 1, 2, 4, 8, then a row's last lane to the next rows.
__device__ __forceinline__ int wave_scan(int v) {  // inclusive
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

struct AttnArgs {
  const uint16_t *q;
  long long q_stride;  // elements from token to token
  const void *kc, *vc;  // caches [page][kv head][page size][dim]; vc null: values are kc's first channels
  const uint8_t *ks, *vs;
  const int32_t *tables, *lens;
  uint16_t *out;
  int4 *plan;        // [parts] the pair that ends in a part and was cut: {b, head, its first part, 0}, b -1 for none
  float *part, *ml;  // partial results [2 part + end][row block][rows][dv], [..][2]
  int B, q_len, heads, kv_heads, dk, dv, num_pages, page, max_blocks;
  uint32_t page_magic;   // floor(2^32 / page), at most 2^32 - 1
  int rows, rblocks;    // query rows a workgroup takes, blocks of them in a kv head
  int parts, min_part;  // most parts, fewest units of a part
  int over;  // what a request costs beside its tiles (rows, the first loads' latency, the result), in tiles
  float scale_log2;
};

// The rows of a kv head: row = token * group + head of the group.
__device__ __forceinline__ int attn_rows(const AttnArgs &a) { return a.q_len * (a.heads / a.kv_heads); }

__device__ __forceinline__ int attn_len(const AttnArgs &a, int b) {
  return max(0, min(a.lens[b], a.max_blocks * a.page));
}

// Tiles [t0, t1) of one request, kv head and row block.
struct AttnItem {
  int b, head, rb, len, t0, t1;
  bool whole;     // all of the request's
  int partial;    // else where its partial result goes
};

// A workgroup's part of the work.  Requests in order, kv heads in order, a
// pair of them takes a.over units and one for each of its tiles; part i has
// the units [i u, (i + 1) u), u the least that makes do with `parts` parts.
// At most one pair began before the part and one ends after it: partial
// results 2 i and 2 i + 1.
struct AttnWalk {
  int x, x1, u, part, rb, over;  // units left [x, x1)
  int b, head, before, len, w;  // the pair: the request's units before it (of one kv head), its units

  __device__ __forceinline__ int units(int len_b) const {
    return over + (len_b + kAttnTile - 1) / kAttnTile;
  }

  // False where the part is empty.  Every wave does this by itself, without a barrier.
  __device__ __forceinline__ bool start(const AttnArgs &a, int block) {
    const int lane = threadIdx.x & 63;
    part = block;
    rb = 0;
    over = a.over;
    if (a.rblocks > 1) {
      // a head's row blocks read the same positions: consecutive workgroups go to the eight XCDs
      // in turn, so the row blocks of a part are dealt out eight apart and share an XCD's cache
      part = block / (8 * a.rblocks) * 8 + block % 8;
      rb = block / 8 % a.rblocks;
    }
    // the first 256 requests' lengths stay in registers
    constexpr int kHold = 4;
    int held[kHold], total = 0;
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      const int i = lane + kWave * j;
      held[j] = i < a.B ? attn_len(a, i) : -1;
    }
#pragma unroll
    for (int j = 0; j < kHold; ++j) total += held[j] >= 0 ? units(held[j]) : 0;
    for (int i = lane + kWave * kHold; i < a.B; i += kWave) total += units(attn_len(a, i));
    total = __builtin_amdgcn_readlane(wave_scan(total), kWave - 1) * a.kv_heads;
    u = max(a.min_part, (total + a.parts - 1) / a.parts);
    const bool writes = rb == 0 && threadIdx.x == 0 && part < a.parts;
    if (part > (total - 1) / u) {
      if (writes) a.plan[part] = int4{-1, 0, 0, 0};
      return false;
    }
    x = part * u;
    x1 = min(total, x + u);
    before = 0;
    for (int b0 = 0;; b0 += kWave) {
      const int i = b0 + lane;
      int len_i = -1;
#pragma unroll
      for (int j = 0; j < kHold; ++j) len_i = b0 == kWave * j ? held[j] : len_i;
      if (b0 >= kWave * kHold) len_i = i < a.B ? attn_len(a, i) : -1;
      const int w_i = len_i >= 0 ? units(len_i) : 0;
      const int upto = wave_scan(w_i);
      const int first = before + upto - w_i;
      const unsigned long long hit = __ballot(x >= first * a.kv_heads && x < (first + w_i) * a.kv_heads);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        b = b0 + l;
        len = __builtin_amdgcn_readlane(len_i, l);
        before = __builtin_amdgcn_readlane(first, l);
        w = __builtin_amdgcn_readlane(w_i, l);
        head = (x - before * a.kv_heads) / w;
        // for the join: a pair that has tiles before the part and ends in it
        const int begin = before * a.kv_heads + head * w;
        if (writes)
          a.plan[part] = x - begin > over && begin + w <= x1 ? int4{b, head, (begin + over) / u, 0}
                                                             : int4{-1, 0, 0, 0};
        return true;
      }
      before += __builtin_amdgcn_readlane(upto, kWave - 1);
    }
  }

  // The part's next item.
  __device__ __forceinline__ bool next(const AttnArgs &a, AttnItem &it) {
    while (x < x1) {
      const int first = before * a.kv_heads + head * w, from = x - first, to = min(x1 - first, w);
      it.b = b;
      it.head = head;
      it.rb = rb;
      it.len = len;
      it.t0 = max(0, from - over);
      it.t1 = to - over;
      it.whole = w == over || (it.t0 == 0 && it.t1 == w - over);  // (an empty request: wherever it begins)
      it.partial = (2 * part + (it.t0 == 0)) * a.rblocks + rb;
      const bool some = it.t1 > it.t0 || (w == over && from == 0);
      x = first + w;
      if (++head == a.kv_heads) {
        head = 0;
        before += w;
        if (++b < a.B) {
          // (a scalar load: a vector one would wait for the rows in flight)
          const auto lens = (const __attribute__((address_space(4))) int32_t *)(uintptr_t)a.lens;
          len = max(0, min(lens[b], a.max_blocks * a.page));
          w = units(len);
        }
      }
      if (some) return true;
    }
    return false;
  }
};

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
// Bound by latency and by the scalar products (no matrix instructions): 250 us
// for 32 requests of 100 .. 4000 positions, 8 heads over 2 of 96 channels.
// ---------------------------------------------------------------------------
constexpr int kAnyDim = 1024;

template <int FMT>
__global__ __launch_bounds__(256) void attn_any_kernel(AttnArgs a) {
  __shared__ float s_q[kAnyDim], s_p[256], s_red[4];
  __shared__ long long s_row[256];
  AttnWalk walk;
  if (!walk.start(a, blockIdx.x)) return;
  const int tid = threadIdx.x, group = a.heads / a.kv_heads;
  for (AttnItem it; walk.next(a, it);) {
    const int head = it.head, r = it.rb, t = r / group;
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
    if (it.whole) {
      uint16_t *out = a.out + (((long long)it.b * a.q_len + t) * a.heads + head * group + r % group) * a.dv;
#pragma unroll
      for (int i = 0; i < kAnyDim / 256; ++i)
        if (tid + 256 * i < a.dv) out[tid + 256 * i] = (uint16_t)f32_to_bf16(l == 0.0f ? 0.0f : acc[i] / l);
    } else {
      const long long at = it.partial;
#pragma unroll
      for (int i = 0; i < kAnyDim / 256; ++i)
        if (tid + 256 * i < a.dv) a.part[at * a.dv + tid + 256 * i] = acc[i];
      if (tid == 0) *reinterpret_cast<float2 *>(a.ml + 2 * at) = float2{m, l};
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Grouped heads on the matrix cores.  A workgroup takes 16 MT query rows
// of one kv head (its group's heads, times the new tokens) over a range of
// positions; its four waves take 32 positions in turn, each by itself, and
// are joined in LDS at the range's end.  A wave forms
//   S^T = K Q^T   (A: 16 positions x 32 channels straight from the cache,
//                  B: the rows, in registers for good),
//   O^T += V^T P^T (A: V^T by transposing LDS reads, B: P^T)
// with v_mfma_f32_16x16x32_bf16.  S^T leaves lane (n, quad) with row n's
// scores of positions 4 quad .. + 3 of two 16-position tiles: exactly the
// eight k-slots of the B operand P^T, if V^T's slots are given the same
// order, so the probabilities never leave their lane, and a row's maximum,
// sum and rescaling are one lane column's own.  Only V goes through LDS (a
// wave's own part: no barrier in the loop).  The next tile's keys are loaded
// as soon as the products with this one's are formed, its values as soon as
// these are in LDS, its page numbers a tile earlier.
// Bound by the cache's bytes; a wave holds 32 positions of keys and values in
// flight.  Measured, 128 channels in bf16: 90 us for 461 MB of 32 ragged
// requests (5.1 TB/s), 195 us for 1.07 GB of two requests of 131000 positions
// (5.5 TB/s; a large copy moves 4.9 TB/s, counting both ways).  96 requests of
// two tokens on an MXFP8 cache, 164 MB: 48 us, where conversion and rescaling
// show; 45 requests of 16 heads of 64 channels, 102 MB: 26 us.
// Masks: rows of a tile see the same positions but where it ends, so only
// tiles with a position that some row does not see take the masked form.
// ---------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;

// One cache row's channels as lane (n, quad) holds them: pieces of 16 bytes,
// 64 bytes of four quads in turn, and the scales of its pieces.  Plain loads: a
// non-temporal hint kept a head's row blocks from sharing their tiles in an
// XCD's cache (40 requests of 64 rows: 38.4 us for 32.7 with 128 channels, 44.2
// for 39.8 with 192) and gained little or lost where there is one block (32
// ragged requests 91.2 for 89.5, 64-wide heads 30.8 for 26.5, 40 requests of 256
// channels 58.8 for 55.2; 96 MXFP8 requests 47.4 for 48.0).
template <int FMT, int D>
struct CacheRow {
  static constexpr int kPieces = FMT == GLM_FMT_BF16 ? D / 32 : D / 64;
  glm_u32x4 v[kPieces];
  uint32_t sc[FMT == GLM_FMT_BF16 ? 1 : (D + 127) / 128];

  __device__ __forceinline__ void load(const void *cache, const uint8_t *scales, long long row,
                                       int dim, int quad) {
    const uint8_t *p = (const uint8_t *)cache + row * (FMT == GLM_FMT_BF16 ? 2 * dim : dim) + 16 * quad;
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      v[i] = *reinterpret_cast<const glm_u32x4 *>(p + 64 * i);
    if constexpr (FMT != GLM_FMT_BF16) {
      const uint8_t *s = scales + row * (dim / 32);
#pragma unroll
      for (int i = 0; i < (D + 127) / 128; ++i) {  // (a row's scales need not be 4-byte aligned)
        if (128 * (i + 1) <= D) {
          __builtin_memcpy(&sc[i], s + 4 * i, 4);
        } else {
          uint16_t two;
          __builtin_memcpy(&two, s + 4 * i, 2);
          sc[i] = two;
        }
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) v[i] = glm_u32x4{0, 0, 0, 0};
  }
  // channels of MFMA step s: bf16 32 s + 8 quad .. + 7; MXFP8 64 (s / 2) + 16 quad + 8 (s % 2) .. + 7
  __device__ __forceinline__ glm_bf16x8 step(int s, int quad) const {
    if constexpr (FMT == GLM_FMT_BF16) {
      return __builtin_bit_cast(glm_bf16x8, v[s]);
    } else {
      const int j = s / 2, h = s % 2;
      const uint32_t byte = (sc[j / 2] >> (16 * (j % 2) + 8 * (quad >> 1))) & 0xffu;
      return mxfp8_words_to_bf16x8(v[j][2 * h], v[j][2 * h + 1], e8m0_to_f32(byte));
    }
  }
  static __device__ __forceinline__ int channel(int s, int quad) {
    return FMT == GLM_FMT_BF16 ? 32 * s + 8 * quad : 64 * (s / 2) + 16 * quad + 8 * (s % 2);
  }
};

__device__ __forceinline__ bf16x4 lds_read_tr(const uint16_t *p) {
  typedef __attribute__((ext_vector_type(4))) short s16x4;
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_bit_cast(
      bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(__attribute__((address_space(3))) void *)p));
}

// Over the four lanes n, n + 16, n + 32, n + 48, for all of them.
__device__ __forceinline__ float max_over_quads(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_quads(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Cache rows of the positions of two 16-position tiles, lane (n, .) position
// p + 16 u + n; a position past `end` or on a page that is not one of the
// cache's gets row 0 and a cleared bit.
struct TileRows {
  int row[2];
  uint32_t seen;  // bit 16 u + n
};
// pos / page and the rest, by a product: the quotient is one short at most.
__device__ __forceinline__ void page_of(const AttnArgs &a, int pos, int &block, int &off) {
  block = (int)__umulhi((uint32_t)pos, a.page_magic);
  off = pos - block * a.page;
  if (off >= a.page) {
    ++block;
    off -= a.page;
  }
}
struct TileIds {
  int id[2], off[2];
};
__device__ __forceinline__ TileIds tile_ids(const AttnArgs &a, const int32_t *table, int p, int end, int n) {
  TileIds t;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    int block;
    page_of(a, min(p + 16 * u + n, end - 1), block, t.off[u]);
    t.id[u] = table[block];
  }
  return t;
}
__device__ __forceinline__ TileRows tile_rows(const AttnArgs &a, const TileIds &t, int head, int p, int end,
                                              int n) {
  TileRows r;
  uint32_t seen[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const bool fine = (uint32_t)t.id[u] < (uint32_t)a.num_pages;
    r.row[u] = fine ? (t.id[u] * a.kv_heads + head) * a.page + t.off[u] : 0;
    seen[u] = (uint32_t)__ballot(fine && p + 16 * u + n < end) & 0xffffu;
  }
  r.seen = seen[0] | (seen[1] << 16);
  return r;
}

template <int DK, int DV, int MT, int FMT, int OCC>
__global__ __launch_bounds__(256, OCC) void attn_group_kernel(AttnArgs a) {
  constexpr int kStride = DV + 16;      // of a position's values in LDS, elements
  constexpr int kAccStride = DV + 4;    // of a row's sums in LDS, floats
  constexpr int kLds = 4 * (32 * kStride * 2 > 16 * kAccStride * 4 ? 32 * kStride * 2 : 16 * kAccStride * 4);
  __shared__ __align__(16) uint8_t s_buf[kLds];
  __shared__ float s_m[4][16 * MT], s_l[4][16 * MT];
  AttnWalk walk;
  if (!walk.start(a, blockIdx.x)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, quad = lane >> 4;
  const int R = attn_rows(a), group = a.heads / a.kv_heads;
  const void *vc = a.vc ? a.vc : a.kc;
  const uint8_t *vs = a.vc ? a.vs : a.ks;
  const int vdim = a.vc ? DV : DK;
  typedef CacheRow<FMT, DK> KRow;
  typedef CacheRow<FMT, DV> VRow;

  uint16_t *lv = reinterpret_cast<uint16_t *>(s_buf) + wave * 32 * kStride;
  const uint16_t *lt = lv + (4 * quad + (n >> 2)) * kStride + 4 * (n & 3);  // transposing reads
  for (AttnItem it; walk.next(a, it);) {
    const int head = it.head, r0 = it.rb * 16 * MT;
    const int32_t *table = a.tables + (long long)it.b * a.max_blocks;
    const int end = min(it.t1 * kAttnTile, it.len);
    const int all_see = it.len - (a.q_len - 1);  // positions below it are seen by every token
    int p = it.t0 * kAttnTile + 32 * wave;
    // (ahead of the query rows: loads return in order, and the first keys wait for these)
    const TileIds ids = tile_ids(a, table, max(0, min(p, end - 1)), max(1, end), n);
    glm_bf16x8 q[MT][DK / 32];
    int tok[MT];  // this lane's rows' new token
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = min(r0 + 16 * m + n, R - 1);
      tok[m] = r / group;
      const uint16_t *p = a.q + ((long long)it.b * a.q_len + tok[m]) * a.q_stride +
                          (head * group + r - tok[m] * group) * DK;
#pragma unroll
      for (int s = 0; s < DK / 32; ++s)
        q[m][s] = *reinterpret_cast<const glm_bf16x8 *>(p + KRow::channel(s, quad));
    }
    glm_f32x4 acc[DV / 16][MT];
    float top[MT], sum[MT];  // what weights are formed below; this lane's part of the running sum
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      top[m] = -INFINITY;
      sum[m] = 0.0f;
#pragma unroll
      for (int d = 0; d < DV / 16; ++d) acc[d][m] = glm_f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (p < end) {
      TileRows cur = tile_rows(a, ids, head, p, end, n), nxt = cur;
      KRow k[2];
      VRow v[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) k[u].load(a.kc, a.ks, cur.row[u], DK, quad);
#pragma unroll
      for (int u = 0; u < 2; ++u) v[u].load(vc, vs, cur.row[u], vdim, quad);
      if (p + 128 < end) nxt = tile_rows(a, tile_ids(a, table, p + 128, end, n), head, p + 128, end, n);
      while (true) {
        const bool more = p + 128 < end;
        glm_f32x4 s[2][MT];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int m = 0; m < MT; ++m) s[u][m] = glm_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < DK / 32; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const glm_bf16x8 kf = k[u].step(i, quad);
#pragma unroll
            for (int m = 0; m < MT; ++m)
              s[u][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[m][i], s[u][m], 0, 0, 0);
          }
        if (more) {
#pragma unroll
          for (int u = 0; u < 2; ++u) k[u].load(a.kc, a.ks, nxt.row[u], DK, quad);
        }
        const bool whole = cur.seen == 0xffffffffu && p + 32 <= all_see;  // (uniform)
        glm_bf16x8 prob[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = s[i / 4][m][i % 4] * a.scale_log2;
          if (!whole) {
            const uint32_t bits = cur.seen >> (4 * quad);
            const int left = all_see + tok[m] - p - 4 * quad;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int at = 16 * (i / 4) + i % 4;
              if (!((bits >> at) & 1u) || at >= left) x[i] = -INFINITY;
            }
          }
          float mx = x[0];
#pragma unroll
          for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[i]);
          mx = max_over_quads(mx);
          if (__any(mx > top[m])) {
            const float next = mx > top[m] ? mx + kAttnSlack : top[m];  // (no row depends on another)
            const float keep = __builtin_amdgcn_exp2f(top[m] - (next == -INFINITY ? 0.0f : next));
            top[m] = next;
            sum[m] *= keep;
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) acc[d][m] *= keep;
          }
          const float from = top[m] == -INFINITY ? 0.0f : top[m];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float e = __builtin_amdgcn_exp2f(x[i] - from);
            sum[m] += e;
            // bf16 for the matrix product: off by 2^-8 of each weight at most, as the output's own rounding
            // is of the output; together 1.7e-3 to 2.4e-3 from 64 bits, 1.65e-3 of it the output's (2-norm)
            prob[m][i] = (__bf16)e;
          }
        }
        if (whole) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < DV / 32; ++i)
              *reinterpret_cast<glm_bf16x8 *>(lv + (16 * u + n) * kStride + VRow::channel(i, quad)) =
                  v[u].step(i, quad);
          if (more) {
#pragma unroll
            for (int u = 0; u < 2; ++u) v[u].load(vc, vs, nxt.row[u], vdim, quad);
          }
#pragma unroll
          for (int d = 0; d < DV / 16; ++d) {
            const bf16x4 lo = lds_read_tr(lt + 16 * d), hi = lds_read_tr(lt + 16 * kStride + 16 * d);
            const glm_bf16x8 vt = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int m = 0; m < MT; ++m)
              acc[d][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, prob[m], acc[d][m], 0, 0, 0);
          }
        } else {
          // a value that a row does not see must not meet its zero weight (it may be an infinity or
          // a NaN): one turn for each new token, with the values that it does not see as zeros, whose
          // sums only that token's rows take
          for (int t = p + 32 > all_see ? 0 : a.q_len - 1; t < a.q_len; ++t) {
            const int below = all_see + t;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int at = 16 * u + n;
              const bool fine = ((cur.seen >> at) & 1u) && p + at < below;
#pragma unroll
              for (int i = 0; i < DV / 32; ++i)
                *reinterpret_cast<glm_u32x4 *>(lv + at * kStride + VRow::channel(i, quad)) =
                    fine ? __builtin_bit_cast(glm_u32x4, v[u].step(i, quad)) : glm_u32x4{0, 0, 0, 0};
            }
            const bool every = p + 32 <= all_see;  // one turn for all rows
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) {
              const bf16x4 lo = lds_read_tr(lt + 16 * d), hi = lds_read_tr(lt + 16 * kStride + 16 * d);
              const glm_bf16x8 vt = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                const glm_f32x4 with =
                    __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, prob[m], acc[d][m], 0, 0, 0);
                if (every || tok[m] == t) acc[d][m] = with;
              }
            }
          }
          if (more) {
#pragma unroll
            for (int u = 0; u < 2; ++u) v[u].load(vc, vs, nxt.row[u], vdim, quad);
          }
        }
        if (!more) break;
        p += 128;
        cur = nxt;
        if (p + 128 < end) nxt = tile_rows(a, tile_ids(a, table, p + 128, end, n), head, p + 128, end, n);
      }
    }

    // the four waves joined, row tile by row tile
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      sum[m] = sum_over_quads(sum[m]);
      if (quad == 0) {
        s_m[wave][16 * m + n] = top[m];
        s_l[wave][16 * m + n] = sum[m];
      }
    }
    __syncthreads();
    float *la = reinterpret_cast<float *>(s_buf);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float mt = fmaxf(fmaxf(s_m[0][16 * m + n], s_m[1][16 * m + n]),
                             fmaxf(s_m[2][16 * m + n], s_m[3][16 * m + n]));
      const float w = __builtin_amdgcn_exp2f(top[m] - (mt == -INFINITY ? 0.0f : mt));
      if (m) __syncthreads();
#pragma unroll
      for (int d = 0; d < DV / 16; ++d)
        *reinterpret_cast<glm_f32x4 *>(la + (wave * 16 + n) * kAccStride + 16 * d + 4 * quad) =
            acc[d][m] * w;
      __syncthreads();
      for (int i = threadIdx.x; i < 16 * DV / 4; i += 256) {
        const int row = i / (DV / 4), ch = 4 * (i % (DV / 4)), r = r0 + 16 * m + row;
        float mr = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w4 = 0; w4 < 4; ++w4) mr = fmaxf(mr, s_m[w4][16 * m + row]);
        const float from = mr == -INFINITY ? 0.0f : mr;
        glm_f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w4 = 0; w4 < 4; ++w4) {
          l += s_l[w4][16 * m + row] * __builtin_amdgcn_exp2f(s_m[w4][16 * m + row] - from);
          o += *reinterpret_cast<const glm_f32x4 *>(la + (w4 * 16 + row) * kAccStride + ch);
        }
        if (r >= R) continue;
        if (it.whole) {
          const int t = r / group;
          uint32_t b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = f32_to_bf16(l == 0.0f ? 0.0f : o[j] / l);
          *reinterpret_cast<uint2 *>(
              a.out + (((long long)it.b * a.q_len + t) * a.heads + head * group + r - t * group) * DV + ch) =
              uint2{b[0] | (b[1] << 16), b[2] | (b[3] << 16)};
        } else {
          const long long at = (long long)it.partial * a.rows + 16 * m + row;
          *reinterpret_cast<glm_f32x4 *>(a.part + at * DV + ch) = o;
          if (ch == 0) *reinterpret_cast<float2 *>(a.ml + 2 * at) = float2{mr, l};
        }
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// The latent cache on the matrix cores: values are the first DV channels of
// the key rows, so a tile is read once and serves both products, and many
// heads share one row, so a workgroup takes 64 query rows and its eight waves
// share each tile of 32 positions through LDS.  Two waves have 16 rows: each
// forms the scores of 16 of the positions, they exchange them through LDS
// (lane for lane, so both know all 32 and hold the same maximum, sum and
// probabilities), and each adds half of the channels to the sums.  A wave
// alone with its rows would need 128 registers for the sums beside 72 for the
// rows, which left none to read ahead with; a pair's 64 do.  Products and
// operand layouts are those of attn_group_kernel, but a value that only later
// tokens see is added by itself and cleared in LDS before the matrix product.
// LDS holds a tile as blocks of 1 KB, 8 positions x 64 channels, the 16-byte
// piece c of position t at 128 t + 16 (c ^ t): a wave's load of one block
// reads eight whole 128-byte lines, and neither the products' reads (16
// positions x 4 pieces) nor the transposing ones (8 positions x 2 pieces a
// half wave) meet on a bank.  Rows go from the cache to LDS directly: bf16
// into a ring of four such tiles, by swizzled source addresses; MXFP8 codes
// and scales into a ring of two, from where the wave that loaded them converts
// them (exact) into a ring of three.  Three tiles (two) are in flight, across the requests of a workgroup's part too; positions that are
// not seen read a row of zeros.
// Measured: 64 bf16 requests of 100 .. 8100 positions, 64 heads, 127 MB: 56 us:
// a part's 14 tiles at 1.74 us are 24, its start and end 17 with one request (11
// with 16 heads), and the join 14 (54 requests are cut into 282 pieces, whose 37
// MB are written and read beside the cache's bytes).
// Five MXFP8 requests of 20000 .. 50000 positions, two tokens, 59 GFLOP: 135 us
// (0.44 PFLOP/s).  There no unit is full: of a tile's 2.2 us a SIMD has matrix
// instructions for a fifth and vector ones for less than half, and LDS reads
// (34 KB a wave) take as much.  Without products and conversion the launches
// take 94 us, without loads too 83, the join's 12 among them: softmax, exchange,
// addresses and the meeting at a tile's end are the larger part.  Half of the
// waves with the next tile's scores behind the values: 139 us for 135; with the
// conversion first: 157 for 154; waits for two operands at once: 136 for 134.
// ---------------------------------------------------------------------------
__device__ uint8_t attn_zero_row[2048];

// N bytes a lane (2, 4 or 16) from global memory to LDS: lane l's to lds + l * max(N, 4).
template <int N>
__device__ __forceinline__ void load_to_lds(const void *src, void *lds) {
  const auto from = (__attribute__((address_space(1))) void *)(const_cast<void *>(src));
  const auto to = (__attribute__((address_space(3))) void *)lds;
  static_assert(N == 2 || N == 4 || N == 16, "sizes used here");
  if constexpr (N == 2)
    __builtin_amdgcn_global_load_lds(from, to, 2, 0, 0);
  else if constexpr (N == 4)
    __builtin_amdgcn_global_load_lds(from, to, 4, 0, 0);
  else
    __builtin_amdgcn_global_load_lds(from, to, 16, 0, 0);
}

// A wave's scores of 16 positions: 18 steps of 32 channels, even ones from `km` and odd ones from `km1` (1 KB
// on every second step), the last two from `kr` and `kr1`.  Eight operands, in v224 .. v255, are on their way
// ahead of the products.  One statement with its waits: the compiler waits for all eight where it needs the
// first.  (The no-ops at the end: a vector instruction has to stay that far behind a product it reads.)
__device__ __forceinline__ glm_f32x4 latent_scores(const glm_bf16x8 (&q)[18], uint32_t km, uint32_t km1,
                                                   uint32_t kr, uint32_t kr1) {
  glm_f32x4 even, odd;
  asm volatile(
      "ds_read_b128 v[224:227], %2 offset:0\n\t"
      "ds_read_b128 v[228:231], %3 offset:0\n\t"
      "ds_read_b128 v[232:235], %2 offset:1024\n\t"
      "ds_read_b128 v[236:239], %3 offset:1024\n\t"
      "ds_read_b128 v[240:243], %2 offset:2048\n\t"
      "ds_read_b128 v[244:247], %3 offset:2048\n\t"
      "ds_read_b128 v[248:251], %2 offset:3072\n\t"
      "ds_read_b128 v[252:255], %3 offset:3072\n\t"
      "s_waitcnt lgkmcnt(7)\n\t"
      "v_mfma_f32_16x16x32_bf16 %0, v[224:227], %6, 0\n\t"
      "ds_read_b128 v[224:227], %2 offset:4096\n\t"
      "s_waitcnt lgkmcnt(7)\n\t"
      "v_mfma_f32_16x16x32_bf16 %1, v[228:231], %7, 0\n\t"
      "ds_read_b128 v[228:231], %3 offset:4096\n\t"
      "s_waitcnt lgkmcnt(7)\n\t"
      "v_mfma_f32_16x16x32_bf16 %0, v[232:235], %8, %0\n\t"
      "ds_read_b128 v[232:235], %2 offset:5120\n\t"
      "s_waitcnt lgkmcnt(7)\n\t"
      "v_mfma_f32_16x16x32_bf16 %1, v[236:239], %9, %1\n\t"
      "ds_read_b128 v[236:239], %3 offset:5120\n\t"
      "s_waitcnt lgkmcnt(7)\n\t"
      "v_mfma_f32_16x16x32_bf16 %0, v[240:243], %10, %0\n\t"
      "ds_read_b128 v[240:243], %2 offset:6144\n\t"
      "s_waitcnt lgkmcnt(7)\n\t"
      "v_mfma_f32_16x16x32_bf16 %1, v[244:247], %11, %1\n\t"
      "ds_read_b128 v[244:247], %3 offset:6144\n\t"
      "s_waitcnt lgkmcnt(7)\n\t"
      "v_mfma_f32_16x16x32_bf16 %0, v[248:251], %12, %0\n\t"
      "ds_read_b128 v[248:251], %2 offset:7168\n\t"
      "s_waitcnt lgkmcnt(7)\n\t"
      "v_mfma_f32_16x16x32_bf16 %1, v[252:255], %13, %1\n\t"
      "ds_read_b128 v[252:255], %3 offset:7168\n\t"
      "s_waitcnt lgkmcnt(7)\n\t"
      "v_mfma_f32_16x16x32_bf16 %0, v[224:227], %14, %0\n\t"
      "ds_read_b128 v[224:227], %4\n\t"
      "s_waitcnt lgkmcnt(7)\n\t"
      "v_mfma_f32_16x16x32_bf16 %1, v[228:231], %15, %1\n\t"
      "ds_read_b128 v[228:231], %5\n\t"
      "s_waitcnt lgkmcnt(7)\n\t"
      "v_mfma_f32_16x16x32_bf16 %0, v[232:235], %16, %0\n\t"
      "s_waitcnt lgkmcnt(6)\n\t"
      "v_mfma_f32_16x16x32_bf16 %1, v[236:239], %17, %1\n\t"
      "s_waitcnt lgkmcnt(5)\n\t"
      "v_mfma_f32_16x16x32_bf16 %0, v[240:243], %18, %0\n\t"
      "s_waitcnt lgkmcnt(4)\n\t"
      "v_mfma_f32_16x16x32_bf16 %1, v[244:247], %19, %1\n\t"
      "s_waitcnt lgkmcnt(3)\n\t"
      "v_mfma_f32_16x16x32_bf16 %0, v[248:251], %20, %0\n\t"
      "s_waitcnt lgkmcnt(2)\n\t"
      "v_mfma_f32_16x16x32_bf16 %1, v[252:255], %21, %1\n\t"
      "s_waitcnt lgkmcnt(1)\n\t"
      "v_mfma_f32_16x16x32_bf16 %0, v[224:227], %22, %0\n\t"
      "s_waitcnt lgkmcnt(0)\n\t"
      "v_mfma_f32_16x16x32_bf16 %1, v[228:231], %23, %1\n\t"
      "s_nop 7\n\t"
      "s_nop 7\n\t"
      : "=&v"(even), "=&v"(odd)
      : "v"(km), "v"(km1), "v"(kr), "v"(kr1), "v"(q[0]), "v"(q[1]), "v"(q[2]), "v"(q[3]), "v"(q[4]),
        "v"(q[5]), "v"(q[6]), "v"(q[7]), "v"(q[8]), "v"(q[9]), "v"(q[10]), "v"(q[11]), "v"(q[12]),
        "v"(q[13]), "v"(q[14]), "v"(q[15]), "v"(q[16]), "v"(q[17])
      : "memory", "v224", "v225", "v226", "v227", "v228", "v229", "v230", "v231", "v232", "v233",
        "v234", "v235", "v236", "v237", "v238", "v239", "v240", "v241", "v242", "v243", "v244",
        "v245", "v246", "v247", "v248", "v249", "v250", "v251", "v252", "v253", "v254", "v255");
  return even + odd;
}

// The products with a wave's 16 channel tiles of the values: tile d's transposed operand comes from at[d % 4]
// + 1024 (d / 4), and positions 16 .. 31 from 16 KB on.  Seven tiles are on their way, in one statement as above;
// the compiler would also wait for every load on its way to LDS, not knowing the place of a transposing read.
__device__ __forceinline__ void latent_values(glm_f32x4 (&acc)[16], const glm_bf16x8 &prob,
                                              const uint32_t (&at)[4]) {
  asm volatile(
      "ds_read_b64_tr_b16 v[224:225], %17 offset:0\n\t"
      "ds_read_b64_tr_b16 v[226:227], %17 offset:16384\n\t"
      "ds_read_b64_tr_b16 v[228:229], %18 offset:0\n\t"
      "ds_read_b64_tr_b16 v[230:231], %18 offset:16384\n\t"
      "ds_read_b64_tr_b16 v[232:233], %19 offset:0\n\t"
      "ds_read_b64_tr_b16 v[234:235], %19 offset:16384\n\t"
      "ds_read_b64_tr_b16 v[236:237], %20 offset:0\n\t"
      "ds_read_b64_tr_b16 v[238:239], %20 offset:16384\n\t"
      "ds_read_b64_tr_b16 v[240:241], %17 offset:1024\n\t"
      "ds_read_b64_tr_b16 v[242:243], %17 offset:17408\n\t"
      "ds_read_b64_tr_b16 v[244:245], %18 offset:1024\n\t"
      "ds_read_b64_tr_b16 v[246:247], %18 offset:17408\n\t"
      "ds_read_b64_tr_b16 v[248:249], %19 offset:1024\n\t"
      "ds_read_b64_tr_b16 v[250:251], %19 offset:17408\n\t"
      "s_waitcnt lgkmcnt(12)\n\t"
      "v_mfma_f32_16x16x32_bf16 %0, v[224:227], %16, %0\n\t"
      "ds_read_b64_tr_b16 v[224:225], %20 offset:1024\n\t"
      "ds_read_b64_tr_b16 v[226:227], %20 offset:17408\n\t"
      "s_waitcnt lgkmcnt(12)\n\t"
      "v_mfma_f32_16x16x32_bf16 %1, v[228:231], %16, %1\n\t"
      "ds_read_b64_tr_b16 v[228:229], %17 offset:2048\n\t"
      "ds_read_b64_tr_b16 v[230:231], %17 offset:18432\n\t"
      "s_waitcnt lgkmcnt(12)\n\t"
      "v_mfma_f32_16x16x32_bf16 %2, v[232:235], %16, %2\n\t"
      "ds_read_b64_tr_b16 v[232:233], %18 offset:2048\n\t"
      "ds_read_b64_tr_b16 v[234:235], %18 offset:18432\n\t"
      "s_waitcnt lgkmcnt(12)\n\t"
      "v_mfma_f32_16x16x32_bf16 %3, v[236:239], %16, %3\n\t"
      "ds_read_b64_tr_b16 v[236:237], %19 offset:2048\n\t"
      "ds_read_b64_tr_b16 v[238:239], %19 offset:18432\n\t"
      "s_waitcnt lgkmcnt(12)\n\t"
      "v_mfma_f32_16x16x32_bf16 %4, v[240:243], %16, %4\n\t"
      "ds_read_b64_tr_b16 v[240:241], %20 offset:2048\n\t"
      "ds_read_b64_tr_b16 v[242:243], %20 offset:18432\n\t"
      "s_waitcnt lgkmcnt(12)\n\t"
      "v_mfma_f32_16x16x32_bf16 %5, v[244:247], %16, %5\n\t"
      "ds_read_b64_tr_b16 v[244:245], %17 offset:3072\n\t"
      "ds_read_b64_tr_b16 v[246:247], %17 offset:19456\n\t"
      "s_waitcnt lgkmcnt(12)\n\t"
      "v_mfma_f32_16x16x32_bf16 %6, v[248:251], %16, %6\n\t"
      "ds_read_b64_tr_b16 v[248:249], %18 offset:3072\n\t"
      "ds_read_b64_tr_b16 v[250:251], %18 offset:19456\n\t"
      "s_waitcnt lgkmcnt(12)\n\t"
      "v_mfma_f32_16x16x32_bf16 %7, v[224:227], %16, %7\n\t"
      "ds_read_b64_tr_b16 v[224:225], %19 offset:3072\n\t"
      "ds_read_b64_tr_b16 v[226:227], %19 offset:19456\n\t"
      "s_waitcnt lgkmcnt(12)\n\t"
      "v_mfma_f32_16x16x32_bf16 %8, v[228:231], %16, %8\n\t"
      "ds_read_b64_tr_b16 v[228:229], %20 offset:3072\n\t"
      "ds_read_b64_tr_b16 v[230:231], %20 offset:19456\n\t"
      "s_waitcnt lgkmcnt(12)\n\t"
      "v_mfma_f32_16x16x32_bf16 %9, v[232:235], %16, %9\n\t"
      "s_waitcnt lgkmcnt(10)\n\t"
      "v_mfma_f32_16x16x32_bf16 %10, v[236:239], %16, %10\n\t"
      "s_waitcnt lgkmcnt(8)\n\t"
      "v_mfma_f32_16x16x32_bf16 %11, v[240:243], %16, %11\n\t"
      "s_waitcnt lgkmcnt(6)\n\t"
      "v_mfma_f32_16x16x32_bf16 %12, v[244:247], %16, %12\n\t"
      "s_waitcnt lgkmcnt(4)\n\t"
      "v_mfma_f32_16x16x32_bf16 %13, v[248:251], %16, %13\n\t"
      "s_waitcnt lgkmcnt(2)\n\t"
      "v_mfma_f32_16x16x32_bf16 %14, v[224:227], %16, %14\n\t"
      "s_waitcnt lgkmcnt(0)\n\t"
      "v_mfma_f32_16x16x32_bf16 %15, v[228:231], %16, %15\n\t"
      "s_nop 7\n\t"
      "s_nop 7\n\t"
      : "+&v"(acc[0]), "+&v"(acc[1]), "+&v"(acc[2]), "+&v"(acc[3]), "+&v"(acc[4]), "+&v"(acc[5]),
        "+&v"(acc[6]), "+&v"(acc[7]), "+&v"(acc[8]), "+&v"(acc[9]), "+&v"(acc[10]), "+&v"(acc[11]),
        "+&v"(acc[12]), "+&v"(acc[13]), "+&v"(acc[14]), "+&v"(acc[15])
      : "v"(prob), "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
      : "memory", "v224", "v225", "v226", "v227", "v228", "v229", "v230", "v231", "v232", "v233",
        "v234", "v235", "v236", "v237", "v238", "v239", "v240", "v241", "v242", "v243", "v244",
        "v245", "v246", "v247", "v248", "v249", "v250", "v251");
}

// At most LEFT of the wave's loads are outstanding, and nothing is moved across.
template <int LEFT>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(LEFT));
  __builtin_amdgcn_sched_barrier(0);
}

template <int DK, int DV, int FMT>
struct LatentLds {
  static constexpr bool kMx = FMT != GLM_FMT_BF16;
  static constexpr int kG = DV / 64, kGR = (DK - DV) / 64;  // 64-channel blocks: values and keys, keys alone
  static constexpr int kMain = 4 * kG * 1024, kRest = 4 * kGR * 1024;  // bytes of 32 positions
  static constexpr int kMains = kMx ? 3 : 4, kRests = kMx ? 2 : 3;     // tiles
  static constexpr int kRaw = kMx ? 4 * DK + 144 : 0;  // MXFP8: a wave's four rows and their scales
  static constexpr int kRestAt = kMains * kMain;
  static constexpr int kX = kRestAt + kRests * kRest;  // the exchanged scores of two tiles
  static constexpr int kId = kX + 2 * 4 * 2 * 64 * 16;  // page numbers of four tiles
  static constexpr int kRow = kId + 4 * 32 * 4;         // cache rows of two times four tiles
  static constexpr int kSeen = kRow + 2 * 4 * 32 * 4;   // which of them are seen
  static constexpr int kRawAt = kSeen + 2 * 4 * 4;
  static constexpr int kBytes = kRawAt + 2 * 8 * kRaw;
  static_assert(kBytes <= 160 * 1024, "one workgroup a CU");
};

template <int DK, int DV, int FMT>
__global__ __launch_bounds__(512, 1) void attn_latent_kernel(AttnArgs a) {
  typedef LatentLds<DK, DV, FMT> L;
  constexpr bool kMx = L::kMx;
  constexpr int kG = L::kG;
  constexpr int kD = DV / 32;  // 16-channel tiles of a wave's half
  constexpr int kLoads = kMx ? 4 : 5;  // of a wave and tile (bf16: a pair's middle block is both's)
  // (nine blocks of 64 channels; MXFP8: 36 pieces of 16 codes and 18 scales a row)
  static_assert(DK == 576 && DV == 512, "widths that the lanes' shares are made for");
  // (one dynamic array: for reads of a static one the compiler waits for every load on its way to it)
  extern __shared__ __align__(16) uint8_t smem[];
  glm_f32x4(*const s_x)[4][2][64] = reinterpret_cast<glm_f32x4(*)[4][2][64]>(smem + L::kX);
  int *const s_id = reinterpret_cast<int *>(smem + L::kId);
  int(*const s_row)[4][32] = reinterpret_cast<int(*)[4][32]>(smem + L::kRow);
  uint32_t(*const s_seen)[4] = reinterpret_cast<uint32_t(*)[4]>(smem + L::kSeen);
  AttnWalk walk;
  if (!walk.start(a, blockIdx.x)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4, rg = wave >> 1, half = wave & 1;
  const int R = attn_rows(a), group = a.heads / a.kv_heads;
  // (what follows from the lane alone is formed anew for every tile: held over the loop, it would not
  // leave the products their registers)
  const auto this_lane = [&]() {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  };

  // ---- the tiles of the part, one after the other, and past the last one zeros, so that every tile's
  // turn issues the same.  Four tiles' cache rows are found at once, by two waves.
  struct Place {
    int b, head, p, end;  // a tile's request, kv head, first position, end of the item
  };
  AttnWalk ahead = walk;
  AttnItem it, next_it;
  bool more = walk.next(a, it);
  Place place = {0, 0, 0, 0};
  const auto next_place = [&]() {
    while (place.p >= place.end) {
      if (!ahead.next(a, next_it)) return Place{0, 0, 0, 0};
      place = {next_it.b, next_it.head, next_it.t0 * kAttnTile, min(next_it.t1 * kAttnTile, next_it.len)};
    }
    const Place now = place;
    place.p += 32;
    return now;
  };
  // wave w < 2, lane l: position l % 32 of tile 2 w + l / 32 of the next four: its entry of the block
  // table, and its row within the page (-1: not seen)
  int within = -1;
  const auto entry = [&]() {
    Place t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = next_place();
    const Place t0 = wave & 1 ? t[2] : t[0], t1 = wave & 1 ? t[3] : t[1];
    const bool up = lane >= 32;
    const int pos = (up ? t1.p : t0.p) + (lane & 31), end = up ? t1.end : t0.end;
    int block, off;
    page_of(a, max(0, min(pos, end - 1)), block, off);
    within = pos < end ? (up ? t1.head : t0.head) * a.page + off : -1;
    return a.tables + (long long)(up ? t1.b : t0.b) * a.max_blocks + block;
  };
  const auto put_rows = [&](int id, int slot) {
    const bool fine = (uint32_t)id < (uint32_t)a.num_pages && within >= 0;
    (&s_row[slot][0][0])[64 * (wave & 1) + lane] = fine ? id * a.kv_heads * a.page + within : -1;
    const unsigned long long seen = __ballot(fine);
    if ((lane & 31) == 0) s_seen[slot][2 * (wave & 1) + (lane >> 5)] = (uint32_t)(seen >> (lane & 32));
  };
  // The cache rows that this lane loads a part of.  bf16: eight rows a wave, eight lanes a row; MXFP8: four
  // rows of 36 pieces of 16 codes: 16 lanes a row twice, then four lanes a row, and 9 a row for the scales.
  struct Rows {
    int a, b, c;
  };
  const auto rows_of = [&](int tile) {
    const int l = this_lane();
    const int *rows = s_row[(tile >> 2) & 1][tile & 3];
    if constexpr (!kMx)
      return Rows{rows[8 * rg + (l >> 3)], 0, 0};
    else
      return Rows{rows[4 * wave + (l >> 4)], rows[4 * wave + ((l & 15) >> 2)], rows[4 * wave + min(l / 9, 3)]};
  };
  // bf16: into the tile's places `main` and `rest`; MXFP8: into the place `main` of codes
  const auto load_rows = [&](const Rows &rows, int main, int rest) {
    const int l = this_lane();
    if constexpr (!kMx) {
      const int g0 = 4 * half;
      const uint8_t *src = (rows.a < 0 ? attn_zero_row : (const uint8_t *)a.kc + (long long)rows.a * (2 * DK)) +
                           (((l & 7) ^ (l >> 3)) << 4) + 128 * g0;
      uint8_t *to = smem + main * L::kMain + (rg * kG + g0) * 1024;
#pragma unroll
      for (int i = 0; i < 4; ++i) load_to_lds<16>(src + 128 * i, to + 1024 * i);
      load_to_lds<16>(src + 512, half ? smem + L::kRestAt + rest * L::kRest + rg * 1024 : to + 4096);
    } else {
      uint8_t *raw = smem + L::kRawAt + (main * 8 + wave) * L::kRaw;
      const auto code = [&](int row, int c) {
        return (row < 0 ? attn_zero_row : (const uint8_t *)a.kc + (long long)row * DK) + 16 * c;
      };
      const uint8_t *src = code(rows.a, l & 15);
      load_to_lds<16>(src, raw);
      load_to_lds<16>(src + 256, raw + 1024);
      const uint8_t *last = code(rows.b, 32 + (l & 3));
      const uint8_t *sc = (rows.c < 0 ? attn_zero_row : a.ks + (long long)rows.c * (DK / 32)) +
                          2 * (l - 9 * min(l / 9, 3));
      if (l < 16) load_to_lds<16>(last, raw + 2048);
      if (l < 36) load_to_lds<2>(sc, raw + 4 * DK);
    }
  };
  // MXFP8: this wave's rows of a tile: lane (t, c) = (l / 16, l % 16) has pieces c and 16 + c of row t, and
  // four codes of its last 64
  struct Codes {
    glm_u32x4 v0, v1;
    uint32_t last, s0, s1, s2;
  };
  const auto codes_of = [&](int from) {
    const int l = this_lane();
    const uint8_t *raw = smem + L::kRawAt + (from * 8 + wave) * L::kRaw;
    const uint8_t *sc = raw + 4 * DK + 36 * (l >> 4);
    const int at = 4 * ((l >> 2) & 3);
    return Codes{*reinterpret_cast<const glm_u32x4 *>(raw + 16 * l),
                 *reinterpret_cast<const glm_u32x4 *>(raw + 1024 + 16 * l),
                 *reinterpret_cast<const uint32_t *>(raw + 2048 + 4 * l),
                 *reinterpret_cast<const uint32_t *>(sc + at), *reinterpret_cast<const uint32_t *>(sc + at + 16),
                 *reinterpret_cast<const uint32_t *>(sc + 32)};
  };
  // .. to bf16 (exact): piece c to the tile's pieces 2 c, 2 c + 1 (the swizzle keeps them neighbours)
  const auto convert = [&](const Codes &codes, int main, int rest) {
    const int l = this_lane(), c = l & 15, pos = (4 * wave + (l >> 4)) & 7;
    const auto scale = [](uint32_t two, int second) { return e8m0_to_f32((two >> (8 * (second & 1))) & 0xffu); };
    const auto put = [&](uint8_t *to, const glm_u32x4 &v, float sc) {
      const int at = pos * 128 + (((2 * (c & 3)) ^ pos) << 4);
      *reinterpret_cast<glm_bf16x8 *>(to + at) = mxfp8_words_to_bf16x8(v[0], v[1], sc);
      *reinterpret_cast<glm_bf16x8 *>(to + (at ^ 16)) = mxfp8_words_to_bf16x8(v[2], v[3], sc);
    };
    // (a wave's four positions lie in one block of eight)
    uint8_t *tile = smem + main * L::kMain + ((wave >> 1) * kG + (c >> 2)) * 1024;
    put(tile, codes.v0, scale(codes.s0, l >> 1));
    put(tile + 4096, codes.v1, scale(codes.s1, l >> 1));
    const float sc = scale(codes.s2, c >> 3);
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes.last, sc, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes.last, sc, true);
    // (a vector of bf16: for a uint2 the compiler waits for every load on its way to LDS)
    *reinterpret_cast<bf16x4 *>(smem + L::kRestAt + rest * L::kRest + (wave >> 1) * 1024 + pos * 128 +
                                (((c >> 1) ^ pos) << 4) + 8 * (c & 1)) = bf16x4{lo[0], lo[1], hi[0], hi[1]};
  };
  // this wave's LDS writes are done, and every wave has come here
  const auto meet = [&]() {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(63) & ~(15 << 8));
    ring_barrier();
  };
  // Tile k's turn multiplies its values, and tile k + 1's keys for the next.
  //   bf16   turn k loads tile k + 3, into the place of tile k - 1, and ends when tile k + 2 has landed
  //   MXFP8  turn k converts tile k + 2 and loads the codes of tile k + 4 into its place
  // Turn 4 c asks for the page numbers of tiles 4 c + 8 .. + 11, turn 4 c + 3 finds their rows.
  constexpr int kAhead = kMx ? 4 : 3;
  int k = 0;
  int main_k = 0, rest_k = 1 % L::kRests;  // tile k's place among the mains, tile k + 1's among the rests
  const auto plus = [](int at, int by, int ring) { return at + by >= ring ? at + by - ring : at + by; };
  uint32_t seen[kAhead];  // of tiles k, k + 1, ..
  const auto seen_of = [&](int tile) {
    return (uint32_t)__builtin_amdgcn_readfirstlane(s_seen[(tile >> 2) & 1][tile & 3]);
  };
  // the query rows of an item, in registers for its tiles
  glm_bf16x8 q[DK / 32];
  const auto load_q = [&]() {
    const int r = min(it.rb * 64 + 16 * rg + n, R - 1), tok = r / group;
    const uint16_t *p = a.q + ((long long)it.b * a.q_len + tok) * a.q_stride +
                        (it.head * group + r - tok * group) * DK + 8 * quad;
#pragma unroll
    for (int s = 0; s < DK / 32; ++s) q[s] = *reinterpret_cast<const glm_bf16x8 *>(p + 32 * s);
  };
  int id0 = -1, id1 = -1, within0 = -1;
  if (wave < 2) {
    id0 = *entry();
    within0 = within;
    id1 = *entry();
  }
  __builtin_amdgcn_sched_barrier(0);
  if (more) load_q();  // (behind the page numbers: loads return in order)
  __builtin_amdgcn_sched_barrier(0);
  if (wave < 2) {
    const int within1 = within;
    within = within0;
    put_rows(id0, 0);
    within = within1;
    put_rows(id1, 1);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kAhead; ++i) seen[i] = seen_of(i);
  load_rows(rows_of(0), 0, 0);
  load_rows(rows_of(1), 1, 1);
  Rows rows{};  // bf16: of tile k + 3
  if constexpr (kMx) {
    wait_loads<kLoads>();
    convert(codes_of(0), 0, 0);
    load_rows(rows_of(2), 0, 0);
    wait_loads<kLoads>();
    convert(codes_of(1), 1, 1);
    load_rows(rows_of(3), 1, 0);
  } else {
    load_rows(rows_of(2), 2, 2);
    rows = rows_of(3);
    wait_loads<kLoads>();
  }
  meet();
  const auto load_ids = [&]() {
    if ((k & 3) == 0 && wave < 2) load_to_lds<4>(entry(), s_id + 64 * wave);
  };

  while (more) {
    const int head = it.head, r0 = it.rb * 64 + 16 * rg;
    const bool active = r0 < R;  // (uniform in a wave)
    const int begin = it.t0 * kAttnTile, end = min(it.t1 * kAttnTile, it.len);
    const int all_see = it.len - (a.q_len - 1);  // positions below it are seen by every token
    const int r = min(r0 + n, R - 1), tok = r / group;
    // (the rows' loads are waited for here once, or the compiler waits for them, and with them for all
    // rows in flight, in every turn)
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    constexpr glm_f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    glm_f32x4 acc[kD], own = zero;  // own: this wave's scores, of 16 positions of the tile to come
#pragma unroll
    for (int d = 0; d < kD; ++d) acc[d] = zero;
    float top = -INFINITY, sum = 0.0f;

    // this wave's scores of tile k + 1 (its places: main, rest)
    const auto scores = [&](int main, int rest) {
      // position 16 half + n, piece 4 (i % 2) + quad of 64 channels i / 2
      const int l = this_lane(), pos = 2 * half + ((l >> 3) & 1);
      const int at = (l & 7) * 128 + (((l >> 4) ^ (l & 7)) << 4);
      const uint8_t *km = smem + main * L::kMain + pos * kG * 1024 + at;
      const uint8_t *km1 = smem + main * L::kMain + pos * kG * 1024 + (at ^ 64);
      const uint8_t *kr = smem + L::kRestAt + rest * L::kRest + pos * 1024;
      const auto lds = [](const uint8_t *p) {
        return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
      };
      return latent_scores(q, lds(km), lds(km1), lds(kr + at), lds(kr + (at ^ 64)));
    };

    if (begin < end) {  // the first tile's scores
      if (active) {
        own = scores(main_k, plus(rest_k, L::kRests - 1, L::kRests));
        s_x[k & 1][rg][half][lane] = own;
      }
      meet();
    }
    for (int p = begin; p < end; p += 32, ++k) {
      const uint32_t last_seen = seen_of(k + kAhead);
      if constexpr (!kMx) {
        load_rows(rows, plus(main_k, 3, 4), plus(rest_k, 2, 3));
        __builtin_amdgcn_sched_barrier(0);
      }
      if ((k & 3) == 3 && wave < 2) put_rows(s_id[64 * wave + this_lane()], ((k >> 2) + 2) & 1);
      // positions that only later tokens see: a value there must not meet an earlier token's zero weight (it
      // may be an infinity or a NaN), so they stay out of the matrix product
      const bool fringe = p + 32 > all_see && a.q_len > 1;  // (uniform)
      uint8_t *kv = smem + main_k * L::kMain;
      glm_bf16x8 prob;
      if (active) {
        const int l0 = this_lane();
        const glm_f32x4 other = s_x[k & 1][rg][half ^ 1][l0];
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = (half ? other[i] : own[i]) * a.scale_log2;
          x[4 + i] = (half ? own[i] : other[i]) * a.scale_log2;
        }
        if (seen[0] != 0xffffffffu || p + 32 > all_see) {  // (uniform)
          const uint32_t bits = seen[0] >> (4 * quad);
          const int left = all_see + tok - p - 4 * quad;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = 16 * (i / 4) + i % 4;
            if (!((bits >> at) & 1u) || at >= left) x[i] = -INFINITY;
          }
        }
        // the next tile's scores beside this one's probabilities (past the item's end: of whatever
        // tile follows, and not used)
        const glm_f32x4 next_own = scores(plus(main_k, 1, L::kMains), rest_k);
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[i]);
        mx = max_over_quads(mx);
        if (__any(mx > top)) {
          const float next = mx > top ? mx + kAttnSlack : top;  // (no row depends on another)
          const float keep = __builtin_amdgcn_exp2f(top - (next == -INFINITY ? 0.0f : next));
          top = next;
          sum *= keep;
#pragma unroll
          for (int d = 0; d < kD; ++d) acc[d] *= keep;
        }
        const float from = top == -INFINITY ? 0.0f : top;
        const int l = this_lane(), common = all_see - p - 4 * (l >> 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = __builtin_amdgcn_exp2f(x[i] - from);
          sum += x[i];
          prob[i] = (__bf16)x[i];  // (see attn_group_kernel)
        }
        if (fringe) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (16 * (i / 4) + i % 4 >= common) prob[i] = (__bf16)0.0f;
        }
        own = next_own;
        s_x[(k + 1) & 1][rg][half][l] = own;
        if (fringe) {
          // one position after the other: the rows of the tokens that see it add its weight's share
          for (int j = max(0, all_see - p); j < min(32, it.len - p); ++j) {
            float w = 0.0f;  // of this lane's row: quad j / 4 % 4 has it
#pragma unroll
            for (int i = 0; i < 8; ++i) w = 16 * (i / 4) + i % 4 == (j & 19) ? x[i] : w;
            w = __shfl(w, n + 16 * ((j >> 2) & 3), kWave);
            const bool sees = p + j < all_see + tok && ((seen[0] >> j) & 1u);
#pragma unroll
            for (int d = 0; d < kD; ++d) {
              // channels 16 d + 4 quad .. + 3 of the wave's half: half of a piece
              const int c = half * kD + d, piece = 2 * c + (quad >> 1);
              const uint2 v = *reinterpret_cast<const uint2 *>(
                  kv + ((j >> 3) * kG + (piece >> 3)) * 1024 + (j & 7) * 128 +
                  (((piece & 7) ^ (j & 7)) << 4) + 8 * (quad & 1));
              if (sees) {
                acc[d][0] += w * bf16_to_f32(v.x & 0xffffu);
                acc[d][1] += w * __uint_as_float(v.x & 0xffff0000u);
                acc[d][2] += w * bf16_to_f32(v.y & 0xffffu);
                acc[d][3] += w * __uint_as_float(v.y & 0xffff0000u);
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
      }
      if (fringe) {  // zeros in their place, once every wave has added them
        meet();
        const int l = this_lane();
        for (int j = max(0, all_see - p) + wave; j < 32; j += 8)
          *reinterpret_cast<glm_u32x4 *>(kv + ((j >> 3) * kG + (l >> 3)) * 1024 + (j & 7) * 128 + 16 * (l & 7)) =
              glm_u32x4{0, 0, 0, 0};
        meet();
      }
      // MXFP8: tile k + 2's codes and tile k + 4's rows, asked for before the products with the values
      Codes codes;
      if constexpr (kMx) {
        wait_loads<kLoads>();
        codes = codes_of(k & 1);
      }
      rows = rows_of(k + 4);
      if (active) {
        // transposing reads: position 4 quad + n / 4, channels 4 (n % 4) of 16 d
        const int l = this_lane(), vt = 4 * (l >> 4) + ((l >> 2) & 3);
        const int vread = ((vt >> 3) * kG + half * kD / 4) * 1024 + (vt & 7) * 128 +
                          ((((l & 3) >> 1) ^ (vt & 7)) << 4) + 8 * (l & 1);
        const uint32_t kv0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)kv;
        const uint32_t at[4] = {kv0 + vread, kv0 + (vread ^ 32), kv0 + (vread ^ 64), kv0 + (vread ^ 96)};
        latent_values(acc, prob, at);
      }
      if constexpr (kMx) {
        convert(codes, plus(main_k, 2, 3), rest_k ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        load_ids();
        load_rows(rows, k & 1, 0);
      } else {
        wait_loads<kLoads>();  // tile k + 2
        load_ids();
      }
      meet();
      main_k = plus(main_k, 1, L::kMains);
      rest_k = plus(rest_k, 1, L::kRests);
#pragma unroll
      for (int i = 0; i + 1 < kAhead; ++i) seen[i] = seen[i + 1];
      seen[kAhead - 1] = last_seen;
    }

    const AttnItem done = it;
    more = walk.next(a, it);
    if (more) load_q();  // the next item's, while this one's results are written
    __builtin_amdgcn_sched_barrier(0);
    sum = sum_over_quads(sum);
    if (!active || r0 + n >= R) {
      // (a row past the last, or a wave of them)
    } else if (done.whole) {
      uint16_t *out = a.out + (((long long)done.b * a.q_len + tok) * a.heads + head * group + r - tok * group) * DV +
                      half * (DV / 2) + 4 * quad;
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int d = 0; d < kD; ++d) {
        uint32_t b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = f32_to_bf16(acc[d][j] * inv);
        *reinterpret_cast<uint2 *>(out + 16 * d) = uint2{b[0] | (b[1] << 16), b[2] | (b[3] << 16)};
      }
    } else {
      const long long at = (long long)done.partial * a.rows + 16 * rg + n;
#pragma unroll
      for (int d = 0; d < kD; ++d)
        *reinterpret_cast<glm_f32x4 *>(a.part + at * DV + half * (DV / 2) + 16 * d + 4 * quad) = acc[d];
      if (half == 0 && quad == 0) *reinterpret_cast<float2 *>(a.ml + 2 * at) = float2{top, sum};
    }
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // nothing may land in LDS that is left
}

// ---------------------------------------------------------------------------
// The pairs of request and kv head that were cut: out = sum_i 2^(m_i - m) acc_i
// / sum_i 2^(m_i - m) l_i over their pieces, with a running maximum, so that a
// piece's weight and sums are asked for together.  A part has the end of at
// most one of them, so the launch goes by parts and not by requests.  A thread
// has four channels of a row; a workgroup's four waves take every fourth piece
// of the same 64 such quads, two in flight each, and are joined in LDS in
// their order.  Bound by latency for few requests and by the pieces' bytes for
// many (39 MB in 12 us).  Four waves a quad and not one, with eight pieces in
// flight: 35 us for 51 (one request of 32000 positions, 63 pieces a head); two
// in flight for four or eight: 57.8, 59.9, 64.9 us (64 latent requests, some
// four pieces each), against 35.8, 34.1, 33.5 (the request of 32000).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  constexpr int kFlight = 2, kWaves = 4;
  __shared__ glm_f32x4 s_acc[kWaves][kWave];
  __shared__ float2 s_ml[kWaves][kWave];
  const int4 pair = a.plan[blockIdx.y];
  if (pair.x < 0) return;
  const int b = pair.x, head = pair.y, g0 = pair.z, g1 = blockIdx.y;  // (g0: the pair's beginning)
  const int R = attn_rows(a), group = a.heads / a.kv_heads, quads = a.dv / 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int i0 = blockIdx.x * kWave; i0 < R * quads; i0 += gridDim.x * kWave) {
    const int i = min(i0 + lane, R * quads - 1), r = i / quads, ch = 4 * (i - r * quads);
    const int block = r / a.rows, row = r - block * a.rows;
    float m = -INFINITY, l = 0.0f;
    glm_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int g = g0 + wave; g <= g1; g += kWaves * kFlight) {
      float2 ml[kFlight];
      glm_f32x4 part[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        const int from = g + kWaves * j;
        ml[j] = float2{-INFINITY, 0.0f};
        part[j] = glm_f32x4{0.f, 0.f, 0.f, 0.f};
        if (from > g1) continue;  // (uniform)
        const long long at = ((long long)(2 * from + (from == g0)) * a.rblocks + block) * a.rows + row;
        ml[j] = *reinterpret_cast<const float2 *>(a.ml + 2 * at);
        part[j] = *reinterpret_cast<const glm_f32x4 *>(a.part + at * a.dv + ch);
      }
      float next = m;
#pragma unroll
      for (int j = 0; j < kFlight; ++j) next = fmaxf(next, ml[j].x);
      const float from = next == -INFINITY ? 0.0f : next, keep = exp2f(m - from);
      m = next;
      l *= keep;
      acc *= keep;
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        const float scale = exp2f(ml[j].x - from);
        l += scale * ml[j].y;
        acc += scale * part[j];
      }
    }
    s_ml[wave][lane] = float2{m, l};
    s_acc[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && i0 + lane < R * quads) {
      float2 ml[kWaves];
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        ml[w] = s_ml[w][lane];
        top = fmaxf(top, ml[w].x);
      }
      const float from = top == -INFINITY ? 0.0f : top;
      l = 0.0f;
      acc = glm_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float scale = exp2f(ml[w].x - from);
        l += scale * ml[w].y;
        acc += scale * s_acc[w][lane];
      }
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = f32_to_bf16(l == 0.0f ? 0.0f : acc[j] / l);
      const int t = r / group;
      uint16_t *out =
          a.out + (((long long)b * a.q_len + t) * a.heads + head * group + r - t * group) * a.dv + ch;
      *reinterpret_cast<uint2 *>(out) = uint2{o[0] | (o[1] << 16), o[2] | (o[3] << 16)};
    }
    __syncthreads();
  }
}

}  // namespace glm

namespace {

enum AttnForm { kAttnAny, kAttnGroup, kAttnLatent };

struct AttnSizes {
  AttnForm form;
  int rows, rblocks, parts, min_part, over;
  unsigned grid;
  size_t plan_bytes, part_bytes, ml_bytes;
};

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// The widths that attn_group_kernel is built for.
bool group_widths(int key_dim, int value_dim) {
  return (key_dim == value_dim && (key_dim == 64 || key_dim == 128 || key_dim == 256)) ||
         (key_dim == 192 && value_dim == 128);
}

template <int DK, int DV, int FMT>
void launch_group(hipStream_t s, dim3 grid, const glm::AttnArgs &a) {
  // workgroups a CU: what the registers allow (and attn_sizes counts on)
  if (a.rows == 16)
    hipLaunchKernelGGL((glm::attn_group_kernel<DK, DV, 1, FMT, (DV > 128 ? 1 : DK == 64 ? 3 : 2)>), grid,
                       dim3(256), 0, s, a);
  else if constexpr (DK <= 192)
    hipLaunchKernelGGL((glm::attn_group_kernel<DK, DV, 2, FMT, (DK > 128 ? 1 : 2)>), grid, dim3(256), 0, s, a);
}

template <int FMT>
void launch_attention(hipStream_t s, dim3 grid, AttnForm form, const glm::AttnArgs &a) {
  if (form == kAttnAny)
    hipLaunchKernelGGL(glm::attn_any_kernel<FMT>, grid, dim3(256), 0, s, a);
  else if (form == kAttnLatent)
    hipLaunchKernelGGL((glm::attn_latent_kernel<576, 512, FMT>), grid, dim3(512),
                       (glm::LatentLds<576, 512, FMT>::kBytes), s, a);
  else if (a.dk == 64)
    launch_group<64, 64, FMT>(s, grid, a);
  else if (a.dk == 128)
    launch_group<128, 128, FMT>(s, grid, a);
  else if (a.dk == 192)
    launch_group<192, 128, FMT>(s, grid, a);
  else
    launch_group<256, 256, FMT>(s, grid, a);
}

// Sizes that follow from a call's shape; for shapes that are refused in either format, why.
const char *attn_sizes(int B, int q_len, int heads, int kv_heads, int key_dim, int value_dim, bool latent,
                       int page_size, int max_blocks, AttnSizes &z) {
  if (B < 0 || q_len < 1 || heads < 1 || kv_heads < 1 || key_dim < 1 || value_dim < 1 || page_size < 1 ||
      max_blocks < 1)
    return "invalid sizes";
  if (heads % kv_heads) return "the heads are no multiple of the kv heads";
  if (key_dim % 8 || value_dim % 8 || key_dim > glm::kAnyDim || value_dim > glm::kAnyDim)
    return "widths must be multiples of 8 up to 1024";
  if (latent && value_dim > key_dim) return "more value channels than a latent row has";
  if (B > 65535) return "at most 65535 requests";
  if (q_len > 16) return "at most 16 new tokens";
  if (heads > 1024) return "at most 1024 heads";
  // (positions a turn ahead of the last, 256 at most, are formed in 32 bits)
  if ((long long)max_blocks * page_size > INT_MAX - 1024) return "the tables' positions pass 32 bits";
  const int R = q_len * (heads / kv_heads);
  int slots;  // workgroups that the chip holds at once
  if (latent && key_dim == 576 && value_dim == 512) {
    z.form = kAttnLatent;
    z.rows = 64;
    slots = 256;  // (its LDS lets one workgroup on a CU)
    // 64 requests of 100 .. 8100 positions with 1, 2, 4 units: 65.4, 58.9, 59.5 us
    z.over = 2;
    z.min_part = 3;  // one request of 8000 with 3, 5: 32.4, 36.3 us
  } else if (group_widths(key_dim, value_dim)) {
    z.form = kAttnGroup;
    // 32 rows share a tile's operands where there are more than 16 and the registers hold them (256 channels:
    // not).  40 requests with 16, 32 rows a workgroup: 24 rows of 128 channels 26.8, 24.0 us, 64 rows 41.3,
    // 32.7; 48 rows of 64 channels 32.8, 28.1; 64 rows of 192 channels 49.8, 40.0
    z.rows = R <= 16 || key_dim > 192 ? 16 : 32;
    // workgroups a CU, as many as its registers hold: 45 requests of 64 channels with 2, 3, 4: 27.9, 26.7, 27.1
    // us, in MXFP8 23.6, 20.4, 19.4, but 60 longer ones 129, 133, 135; 32 ragged ones of 128 channels with 2, 3: 90,
    // 110 (spills); 32 rows of 192 channels with 2, 1: 35.1, 28.7 (one is resident)
    slots = 256 * (key_dim > 192 || (key_dim > 128 && z.rows == 32) ? 1 : key_dim == 64 && z.rows == 16 ? 3 : 2);
    // units 1, 2, 3 beside the tiles: 55.0, 48.0, 46.7 us (96 requests, MXFP8), 26.3, 26.5, 27.1 (45 requests
    // of 64 channels), 90.3, 90.2, 89.9 (32 ragged ones)
    z.over = 2;
    // one request with parts of 3, 6 or more units: 12.5, 13.2 us (517 positions), 12.4, 13.9 (2000), 16.9,
    // 15.9 (8000)
    z.min_part = 3;
  } else {
    z.form = kAttnAny;
    z.rows = 1;
    slots = 2048;  // (1024: the same)
    z.over = 1;
    // parts of 2, 5 units: 43, 82 us (one request of 517 positions), 251, 244 (32 of 100 .. 4000)
    z.min_part = 2;
  }
  z.rblocks = (R + z.rows - 1) / z.rows;
  z.parts = slots / z.rblocks > 1 ? slots / z.rblocks : 1;
  const long long tiles = ((long long)max_blocks * page_size + glm::kAttnTile - 1) / glm::kAttnTile;
  const long long units = (tiles + z.over) * B * kv_heads;
  if (units > INT_MAX / 2) return "the tables' tiles of all requests and kv heads pass 2^30";
  const long long most_parts = (units + z.min_part - 1) / z.min_part;
  if (z.parts > most_parts) z.parts = most_parts > 1 ? (int)most_parts : 1;
  z.grid = z.rblocks > 1 ? (unsigned)((z.parts + 7) / 8 * 8 * z.rblocks) : (unsigned)z.parts;
  const size_t results = (size_t)2 * z.parts * z.rblocks * z.rows;
  z.plan_bytes = up256((size_t)z.parts * sizeof(int4));
  z.part_bytes = up256(results * value_dim * sizeof(float));
  z.ml_bytes = up256(results * 2 * sizeof(float));
  return nullptr;
}

}  // namespace

extern "C" size_t glm_paged_attention_workspace_bytes(int B, int q_len, int heads, int kv_heads,
                                                      int key_dim, int value_dim, int latent,
                                                      int page_size, int max_blocks) {
  AttnSizes z;
  if (attn_sizes(B, q_len, heads, kv_heads, key_dim, value_dim, latent != 0, page_size, max_blocks, z))
    return 0;
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
  GLM_REQUIRE(B >= 0 && q_len >= 1 && heads >= 1 && kv_heads >= 1 && key_dim >= 1 &&
                  value_dim >= 1 && num_pages >= 1 && page_size >= 1 && max_blocks >= 1,
              GLM_ERR_INVALID_ARGUMENT, "paged_attention: invalid sizes");
  // (sizes first: a refused size has no workspace, whose pointer may then be null)
  AttnSizes z;
  const char *why = attn_sizes(B, q_len, heads, kv_heads, key_dim, value_dim, shared, page_size, max_blocks, z);
  GLM_REQUIRE(!why, GLM_ERR_UNSUPPORTED_SHAPE,
              "paged_attention: %s (%d requests, %d tokens, %d heads over %d, widths %d and %d, %d blocks of %d)",
              why, B, q_len, heads, kv_heads, key_dim, value_dim, max_blocks, page_size);
  GLM_REQUIRE(!mx || (key_dim % 32 == 0 && value_dim % 32 == 0), GLM_ERR_UNSUPPORTED_SHAPE,
              "paged_attention: MXFP8 widths %d and %d must be multiples of 32", key_dim, value_dim);
  GLM_REQUIRE((long long)num_pages * page_size * kv_heads <= INT_MAX, GLM_ERR_UNSUPPORTED_SHAPE,
              "paged_attention: %d pages of %d x %d rows pass 32 bits", num_pages, kv_heads,
              page_size);
  GLM_REQUIRE(q && key_cache && tables && lens && workspace && out && (!mx || key_scales) &&
                  (!mx || shared || value_scales),
              GLM_ERR_INVALID_ARGUMENT, "paged_attention: null pointer");
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
  a.plan = (int4 *)ws;
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
  a.page_magic = page_size == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / page_size);
  a.rows = z.rows;
  a.rblocks = z.rblocks;
  a.parts = z.parts;
  a.min_part = z.min_part;
  a.over = z.over;
  a.scale_log2 = scale * glm::kLog2e;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)z.grid);
  if (mx)
    launch_attention<GLM_FMT_MXFP8>(s, grid, z.form, a);
  else
    launch_attention<GLM_FMT_BF16>(s, grid, z.form, a);
  GLM_LAUNCH_CHECK("paged_attention");
  if (z.parts > 1) {
    // as many workgroups as have work for few cut pairs, and for many no more than fill the chip twice: 64
    // latent requests with 2048, 4096, 8192 in all: 61.0, 59.9, 62.3 us
    const int quads = q_len * (heads / kv_heads) * value_dim / 4;
    const int pairs = z.parts < (long long)B * kv_heads ? z.parts : B * kv_heads;
    int ways = (quads + 63) / 64;
    if (ways > 4096 / pairs) ways = 4096 / pairs > 1 ? 4096 / pairs : 1;
    hipLaunchKernelGGL(glm::attn_join_kernel, dim3(ways, z.parts), dim3(256), 0, s, a);
    GLM_LAUNCH_CHECK("attn_join_kernel");
  }
  return GLM_OK;
}
