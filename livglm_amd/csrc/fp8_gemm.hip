// Products of E4M3 rows and E4M3 weights with f32 scales (fp8_rows.h):
//   y[t][n] = sum_g sx[t][g] sw[n / 128][g] sum_{k in group g} x[t][k] w[n][k]
// in bf16, and the gated pair of them with its limited SwiGLU.  A group's inner
// sum is formed by the matrix cores from zero; its scales are applied to the
// f32 result, which no instruction of theirs does for scales that are no powers
// of two.
//
// MFMA lane (r, q), r = lane & 15, q = lane >> 4, holds 32 bytes of weight row
// r (A) and of token r (B): both operands take their bytes from the same
// channels, whichever they are, so the order within a group is free.  Output
// lane (r, q) holds weight rows 4q .. 4q + 3 for token r.
//
// Two forms of the inner sum.  As bf16 (every code is one, exactly) in four
// v_mfma_f32_16x16x32_bf16: exact products, f32 sums.  As it is in one
// v_mfma_f32_16x16x128_f8f6f4, at twice the rate: the core aligns eight products
// at a time to the largest of them and drops what lies 2^-13 of it below, which is
// 1.5e-5 of the sum on normal values, without a bias.  The latter serves products
// whose result is rounded to bf16 (1.7e-3) and whose time the matrix cores set.
#include "fp8_rows.h"
#include "fp8_span.h"
#include "lds_stage.h"
#include "mfma_tile.h"

#include <algorithm>

namespace glm {

typedef int fp8_frag __attribute__((ext_vector_type(8)));

constexpr int kExactTokens = 64;  // rows whose products are summed exactly in any case
// Rows that the product quantises itself: up to so many, and so many codes, for so
// many features.  (Each workgroup does it for itself: at K and N 4096 1, 4 and 8 rows
// so take 6.6, 7.1 and 8.5 us, quantised before 8.0, 8.1 and 8.2 and a launch more for
// the host; 16 rows of K 2048 5.8 and 5.9; 8 rows of K 8192 12.1 and 10.6; the gated
// pair of 16 rows, K 2048, 2 x 768 features 7.2 and 8.4.  At K 2048 1 and 8 rows into
// 8192 features 6.0 and 6.7, before 7.1 and 7.3; into 16384 11.5 and 12.1, before 10.8
// and 11.2; into 65536 32.3 and 34.8, before 25.0 and 25.3.)
constexpr int kFusedTokens = 16, kFusedCodes = 1 << 15, kFusedFeatures = 8192;

struct Fp8Args {
  const void *x;          // codes, or bf16 / f32 rows
  const float *xs;        // [T][groups], with codes
  const uint8_t *w[2];    // [N][K]
  const float *ws[2];     // [ceil(N / 128)][groups]
  int T, K, N, groups;
  float limit;
  int ahead;              // fp8_stream_kernel: groups that a wave has in flight
  uint32_t per_token;     // and 2^32 / T upwards, T from 2 to kFusedTokens, for quotients below 2^16
  uint16_t *out;          // NPROJ 1: bf16 [T][N]
  float *h;               // NPROJ 2, streamed: the sums, f32 [split][2][T][N]
  uint8_t *codes;         // gated and quantised
  float *scales;
};

__device__ __forceinline__ fp8_frag join16(const glm_u32x4 &a, const glm_u32x4 &b) {
  return fp8_frag{(int)a[0], (int)a[1], (int)a[2], (int)a[3],
                  (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// A lane's 32 codes of a group as an operand: as bf16, or (FAST) as they are.
template <bool FAST>
struct Fp8Operand;
template <>
struct Fp8Operand<false> {
  static constexpr int kSteps = 4;
  glm_bf16x8 v[4];
  __device__ __forceinline__ explicit Fp8Operand(const fp8_frag &f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) part(f, i);
  }
  __device__ __forceinline__ void part(const fp8_frag &f, int i) {
    v[i] = mxfp8_words_to_bf16x8((uint32_t)f[2 * i], (uint32_t)f[2 * i + 1], 1.0f);
  }
  Fp8Operand() = default;
};
template <>
struct Fp8Operand<true> {
  static constexpr int kSteps = 1;
  fp8_frag v;
  __device__ __forceinline__ explicit Fp8Operand(const fp8_frag &f) : v(f) {}
  Fp8Operand() = default;
};

// Step i of a b over the group's 128 channels, from zero in the first.
__device__ __forceinline__ glm_f32x4 step_sum(const Fp8Operand<false> &a,
                                              const Fp8Operand<false> &b, int i, glm_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      a.v[i], b.v[i], i == 0 ? glm_f32x4{0.f, 0.f, 0.f, 0.f} : c, 0, 0, 0);
}
__device__ __forceinline__ glm_f32x4 step_sum(const Fp8Operand<true> &a, const Fp8Operand<true> &b,
                                              int, glm_f32x4) {
  // (scale operands of zero: the unscaled instruction)
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      a.v, b.v, glm_f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// silu(min(g, limit)) * clip(u, limit) in f32; NaN passes through the clamps.
__device__ __forceinline__ float gated(float g, float u, float limit) {
  if (limit > 0.f) {
    g = __builtin_elementwise_minimum(g, limit);
    u = __builtin_elementwise_maximum(__builtin_elementwise_minimum(u, limit), -limit);
  }
  return g / (1.0f + expf(-g)) * u;
}

constexpr uint32_t kOutOfRange = 0x40000000u;  // past any tile's operand (256 rows of 2^20 codes)

// Waits until at most `ahead` (0 .. MAX, uniform) groups of LOADS loads are
// outstanding.
template <int MAX, int LOADS>
__device__ __forceinline__ void wait_groups_ahead(int ahead) {
  static_assert(MAX * LOADS < 64, "the wait counter's range");
  if (ahead >= MAX) {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(MAX * LOADS));
  } else if constexpr (MAX > 0) {
    wait_groups_ahead<MAX - 1, LOADS>(ahead);
  }
}

// ---------------------------------------------------------------------------
// Up to some hundred tokens: the weights are streamed once for 16 TB tokens.  A
// workgroup has 16 RB weight rows (of each projection); its four to eight waves take
// the groups of K in turn, each through LDS of its own, and add up their f32
// results at the end: no wave waits for another before that.  Gated pairs of
// few row tiles and at most 16 tokens a workgroup are split along K too (blockIdx.z);
// what reads their sums joins them.
//
// Operands come by direct loads, 16 bytes a lane, whose lanes walk along a
// row: an operand's own lanes lie in 16 rows, and loads into registers took 64
// address cycles instead of 16 (64 tokens of the pair, K 4096, 2 x 2048
// features: 20 us, now 8.7).  The group behind is asked for as soon as a group's
// operands are in registers.  ROWS says what x holds: bf16 and f32 rows are
// quantised by the workgroup into LDS while the first weights are on their way,
// four lanes a group (by each wave for its own groups, 16 columns whatever the
// tokens are, one token at K 4096 took 2 us more).
//
// One coded row, K and N 4096: 5.8 us, 16.8 MB at 4.4 TB/s behind a launch's 1.9; K
// 8192 8.3, 5.2 TB/s.  333 rows 15.2 us: 655 KB of operands into each CU's LDS at 80 to
// 100 B/ns are 6.5 to 8 of them, the rest the launch, the first trip to memory, a group a
// wave in flight, and the join.
// ---------------------------------------------------------------------------
constexpr int kStreamKB = 152;  // LDS of a workgroup where the CUs have one each
constexpr int kStreamPairKB = 78;  // else

// WAVES waves, RB blocks of 16 weight rows of each projection, TB of 16 tokens;
// FEW: up to 8 tokens, one load's; FAST: which of the two forms of the sum.
template <int WAVES, int NPROJ_, int RB_, int TB_, int ROWS_, bool FEW = false, bool FAST_ = false>
struct Fp8Stream {
  static constexpr int NPROJ = NPROJ_, RB = RB_, TB = TB_, ROWS = ROWS_;
  static constexpr bool FAST = FAST_;
  static constexpr int kWaves = WAVES, kThreads = 64 * WAVES;
  static constexpr int kRowBlocks = NPROJ * RB;
  static constexpr bool kCoded = ROWS == GLM_ROWS_FP8;
  static constexpr int kTok = !kCoded ? kFusedTokens : FEW ? 8 : 16 * TB;
  static constexpr int kW = kRowBlocks * 16 * kFp8Group;     // one group in LDS: the weight rows,
  static constexpr int kX = kCoded ? kTok * kFp8Group : 0;   // the tokens' codes
  static constexpr int kSLoads = kCoded ? (kTok + 63) / 64 : 0;
  static constexpr int kS = 256 * kSLoads;                   // and scales, a lane each
  static constexpr int kSlot = kW + kX + kS;
  static constexpr int kLoads = (kW + kX) / 1024 + kSLoads;
  static constexpr int kMost = kLoads <= 12 ? 4 : 2;         // groups a wave has in flight at most
  static constexpr int kPart = WAVES * kRowBlocks * TB * kWave * 16;
  static_assert(kLoads * (kMost - 1) < 64, "the wait counter's range");
  // piece p of row R lies at p ^ swz(R)
  __host__ __device__ static int swz(int row) { return (row >> 1) & 7; }
  // rows that the workgroup quantises: codes [group][token][128] and scales [group][token] behind
  // the ring, of so many groups
  __host__ __device__ static int coded_groups(int groups, int splits) {
    return kCoded ? 0 : WAVES * ((groups + WAVES * splits - 1) / (WAVES * splits));
  }
  static int coded_bytes(int groups, int splits, int T) {
    return coded_groups(groups, splits) * T * (kFp8Group + 4);
  }
};

template <class L>
__global__ __launch_bounds__(L::kThreads) void fp8_stream_kernel(Fp8Args a) {
  constexpr int NPROJ = L::NPROJ, RB = L::RB, TB = L::TB, ROWS = L::ROWS, kWaves = L::kWaves;
  constexpr bool FAST = L::FAST;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int n0 = 16 * RB * blockIdx.x, t0 = 16 * TB * blockIdx.y;
  const int K = a.K, groups = a.groups, ahead = a.ahead;
  const int first = wave + kWaves * blockIdx.z, step = kWaves * gridDim.z;
  const int mine = first < groups ? (groups - first + step - 1) / step : 0;  // groups of this wave
  uint8_t *ring = smem + wave * (ahead * L::kSlot);
  uint8_t *coded = smem + kWaves * ahead * L::kSlot;  // the workgroup's own codes and scales
  const int ncoded = L::coded_groups(groups, gridDim.z);
  const uint32_t feats = (uint32_t)min(a.N - n0, 16 * RB), toks = (uint32_t)min(a.T - t0, L::kTok);
  float *coded_scales = reinterpret_cast<float *>(coded + ncoded * (int)toks * kFp8Group);
  const __amdgpu_buffer_rsrc_t xres =
      make_rsrc((const uint8_t *)a.x + (long long)t0 * K, toks * (uint32_t)K);
  const __amdgpu_buffer_rsrc_t sres =
      make_rsrc(L::kCoded ? a.xs + (long long)t0 * groups : a.ws[0], toks * (uint32_t)groups * 4u);
  __amdgpu_buffer_rsrc_t wres[NPROJ];
#pragma unroll
  for (int p = 0; p < NPROJ; ++p)
    wres[p] = make_rsrc(a.w[p] + (long long)n0 * K, feats * (uint32_t)K);
  // rows past the last and channels past K are out of the buffers' range, which gives zeros
  auto issue = [&](int i, int slot) {  // the wave's i-th group
    const int g = first + i * step;
    uint8_t *to = ring + slot * L::kSlot;
    const int left = K - g * kFp8Group;
#pragma unroll
    for (int j = 0; j < (L::kW + L::kX) / 1024; ++j) {
      const bool isw = j < L::kW / 1024;
      const int row = (isw ? j % (2 * RB) : j - L::kW / 1024) * 8 + lane / 8;
      const int piece = (lane % 8) ^ L::swz(row);
      buf16_to_lds(isw ? wres[isw ? j / (2 * RB) : 0] : xres, to + j * 1024,
                   16 * piece < left ? (uint32_t)row * (uint32_t)K + 16 * piece : kOutOfRange,
                   (uint32_t)g * kFp8Group);
    }
#pragma unroll
    for (int j = 0; j < L::kSLoads; ++j)
      buf4_to_lds(sres, to + L::kW + L::kX + j * 256,
                  64 * j + lane < L::kTok ? (uint32_t)(64 * j + lane) * (uint32_t)groups * 4u : kOutOfRange,
                  (uint32_t)g * 4);
  };
  // lane l holds the block scales of the wave's l-th group of each 64
  float held[NPROJ];
  auto hold = [&](int i) {
#pragma unroll
    for (int p = 0; p < NPROJ; ++p)
      held[p] = a.ws[p][(long long)(n0 / kFp8Group) * groups + min(first + (i + lane) * step, groups - 1)];
  };
  hold(0);
  if constexpr (L::kCoded) {
    for (int i = 0; i < ahead; ++i)
      if (i < mine) issue(i, i);
  } else {
    // item: token item % toks of the workgroup's group item / toks; four lanes, of which each
    // has every fourth eight channels
    constexpr bool F32 = ROWS == GLM_ROWS_F32;
    constexpr int kPer = L::kThreads / 4, kBytes = F32 ? 4 : 2, kRaw = 2 * kBytes;
    const __amdgpu_buffer_rsrc_t rows = make_rsrc(a.x, toks * (uint32_t)K * kBytes);
    const int items = ncoded * (int)toks, l4 = threadIdx.x & 3;
    auto place = [&](int item, int &li, int &t) {
      li = toks == 1 ? item : (int)__umulhi((uint32_t)item, a.per_token);
      t = item - li * (int)toks;
    };
    glm_u32x4 raw[kRaw];
    auto load = [&](int item, glm_u32x4 (&to)[kRaw]) {
      int li, t;
      place(item, li, t);
      const int g = (li / kWaves) * step + kWaves * blockIdx.z + li % kWaves;
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // (no branches between the loads)
        const int k = g * kFp8Group + 8 * (4 * j + l4);
        const uint32_t off = item < items && k < K ? (uint32_t)(t * K + k) * kBytes : kOutOfRange;
#pragma unroll
        for (int i = 0; i < kRaw / 4; ++i)
          to[j * (kRaw / 4) + i] = __builtin_amdgcn_raw_buffer_load_b128(rows, off + 16 * i, 0, 0);
      }
    };
    load(threadIdx.x >> 2, raw);
    for (int i = 0; i < ahead; ++i)
      if (i < mine) issue(i, i);
    auto code = [&](int item) {
      float v[32];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float (&e)[8] = *reinterpret_cast<float (*)[8]>(v + 8 * j);
        if constexpr (F32) {
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = __uint_as_float(raw[2 * j + i / 4][i % 4]);
        } else {
          unpack8(raw[j], e);
        }
      }
      int li, t;
      place(item, li, t);
      auto over_lanes = [](float m) {
        m = fmaxf(m, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(m), 0xB1, 0xf, 0xf, true)));
        return fmaxf(m, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(m), 0x4E, 0xf, 0xf, true)));
      };
      float m = over_lanes(abs_max(v));
      if (__builtin_expect(isinf(m), 0)) m = over_lanes(finite_abs_max(v));  // (one answer in the four)
      m = fmaxf(m, kFp8Tiny);
      const float up = kFp8Max / m;
      uint8_t *row = coded + (li * (int)toks + t) * kFp8Group + 8 * (l4 & 1);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint2 *>(row + 16 * ((2 * j + (l4 >> 1)) ^ L::swz(t))) =
            uint2{fp8_codes4(v[8 * j], v[8 * j + 1], v[8 * j + 2], v[8 * j + 3], up),
                  fp8_codes4(v[8 * j + 4], v[8 * j + 5], v[8 * j + 6], v[8 * j + 7], up)};
      if (l4 == 0) coded_scales[li * (int)toks + t] = m / kFp8Max;
    };
    int item = threadIdx.x >> 2;
    if (items <= kPer) {  // (no loads behind the weights')
      if (item < items) code(item);
    } else {
      for (; item < items; item += kPer) {
        glm_u32x4 next[kRaw];
        load(item + kPer, next);
        code(item);
#pragma unroll
        for (int j = 0; j < kRaw; ++j) raw[j] = next[j];
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // this wave's codes are in LDS
    ring_barrier();
  }

  glm_f32x4 acc[L::kRowBlocks][TB];
#pragma unroll
  for (int b = 0; b < L::kRowBlocks; ++b)
#pragma unroll
    for (int t = 0; t < TB; ++t) acc[b][t] = glm_f32x4{0.f, 0.f, 0.f, 0.f};
  // the lane's pieces of a row of codes, p0 and p0 + 1 (fp8_tile_kernel): channels 16 p0 .. + 31
  const int p0 = 4 * (q & 1) + 2 * (q >> 1);
  auto frag = [&](const uint8_t *rows, int row) {
    const glm_u32x4 *p = reinterpret_cast<const glm_u32x4 *>(rows + row * kFp8Group);
    return join16(p[p0 ^ L::swz(row)], p[(p0 + 1) ^ L::swz(row)]);
  };
  int slot = 0;
  auto group = [&](int i) {
    wait_groups_ahead<L::kMost - 1, L::kLoads>(min(ahead - 1, mine - 1 - i));
    asm volatile("" ::: "memory");
    const uint8_t *from = ring + slot * L::kSlot;
    fp8_frag w[L::kRowBlocks];
#pragma unroll
    for (int b = 0; b < L::kRowBlocks; ++b) w[b] = frag(from + b * 16 * kFp8Group, r);
    // (columns past the tokens repeat one)
    const int li = i * kWaves + wave;
    const uint8_t *xrows = L::kCoded ? from + L::kW : coded + li * (int)toks * kFp8Group;
    const float *xscales = L::kCoded ? reinterpret_cast<const float *>(from + L::kW + L::kX)
                                     : coded_scales + li * (int)toks;
    fp8_frag xf[TB];
    float sx[TB];
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      const int t = min(b * 16 + r, L::kCoded ? L::kTok - 1 : (int)toks - 1);
      xf[b] = frag(xrows, t);
      sx[b] = xscales[t];
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // the slot's reads are done
    asm volatile("" ::: "memory");
    if (i + ahead < mine) issue(i + ahead, slot);
    slot = slot + 1 == ahead ? 0 : slot + 1;
    float s[NPROJ][TB];
#pragma unroll
    for (int p = 0; p < NPROJ; ++p) {
      const float sw = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(held[p]), i & 63));
#pragma unroll
      for (int t = 0; t < TB; ++t) s[p][t] = sx[t] * sw;
    }
    Fp8Operand<FAST> x[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t) x[t] = Fp8Operand<FAST>(xf[t]);
    // a block's sums are scaled beside the next block's products
    glm_f32x4 c[2][TB];
#pragma unroll
    for (int b = 0; b <= L::kRowBlocks; ++b) {
      if (b < L::kRowBlocks) {
        const Fp8Operand<FAST> now(w[b]);
#pragma unroll
        for (int j = 0; j < Fp8Operand<FAST>::kSteps; ++j)
#pragma unroll
          for (int t = 0; t < TB; ++t) c[b & 1][t] = step_sum(now, x[t], j, c[b & 1][t]);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (b > 0) {
#pragma unroll
        for (int t = 0; t < TB; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[b - 1][t][j] += c[(b - 1) & 1][t][j] * s[(b - 1) / RB][t];
      }
    }
  };
  for (int i = 0; i < mine;) {
    const int end = min(i + 64, mine);
    if (i != 0) hold(i);
#pragma unroll
    for (int p = 0; p < NPROJ; ++p) asm volatile("" ::"v"(held[p]));  // (waited for here, not within the loop)
#pragma clang loop unroll(disable)
    for (; i < end; ++i) group(i);
  }

  __syncthreads();  // (the ring is done with)
  glm_f32x4 *part = reinterpret_cast<glm_f32x4 *>(smem);  // [wave][row block][token block][lane]
  constexpr int kBlocks = L::kRowBlocks * TB;
#pragma unroll
  for (int b = 0; b < L::kRowBlocks; ++b)
#pragma unroll
    for (int t = 0; t < TB; ++t) part[(wave * kBlocks + b * TB + t) * kWave + lane] = acc[b][t];
  __syncthreads();
  // eight features of a token a thread, so that a row leaves in whole pieces
  constexpr int kPieces = 2 * RB;
  for (int i = threadIdx.x; i < kPieces * NPROJ * 16 * TB; i += L::kThreads) {
    const int piece = i % kPieces, p = i / kPieces % NPROJ, tok = i / (kPieces * NPROJ);
    const int t = t0 + tok, n = n0 + 8 * piece;
    if (t >= a.T || n >= a.N) continue;
    const glm_f32x4 *from = part + ((p * RB + piece / 2) * TB + tok / 16) * kWave + tok % 16 + 32 * (piece & 1);
    float v[8] = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const glm_f32x4 lo = from[w * kBlocks * kWave], hi = from[w * kBlocks * kWave + 16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] += lo[j];
        v[4 + j] += hi[j];
      }
    }
    if constexpr (NPROJ == 2) {  // (N % 16 == 0)
      glm_f32x4 *o = reinterpret_cast<glm_f32x4 *>(
          a.h + (((long long)blockIdx.z * 2 + p) * a.T + t) * a.N + n);
      o[0] = glm_f32x4{v[0], v[1], v[2], v[3]};
      o[1] = glm_f32x4{v[4], v[5], v[6], v[7]};
    } else {
      uint16_t *out = a.out + (long long)t * a.N + n;
      if (a.N % 8 == 0) {
        glm_u32x4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = f32_to_bf16(v[2 * j]) | (f32_to_bf16(v[2 * j + 1]) << 16);
        *reinterpret_cast<glm_u32x4 *>(out) = o;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (n + j < a.N) out[j] = (uint16_t)f32_to_bf16(v[j]);
      }
    }
  }
}

// The gated pair's sums [split][projection][T][N] joined, gated and quantised:
// sixteen lanes a group of features.  Its own launch, since a group's maximum
// spans eight workgroups' features (a workgroup for all 128 leaves most CUs idle:
// 2 rows, K 2048, 2 x 768 features 14.3 us, the two launches 7.1); 2.4 us for 2
// rows of 768, 3.9 for 64 of 2048, most of it the launch.
__global__ __launch_bounds__(256) void fp8_gate_kernel(const float *h, int splits, int T, int N,
                                                       float limit, uint8_t *codes, float *scales) {
  const int groups = fp8_groups(N), lane = threadIdx.x & 15;
  const long long item = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (item >= (long long)T * groups) return;
  const int t = (int)(item / groups), n = (int)(item - (long long)t * groups) * kFp8Group + 8 * lane;
  float v[8] = {};
  if (n < N) {
    float sum[2][8];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      load8<true>(h, ((long long)p * T + t) * N + n, sum[p]);
      for (int z = 1; z < splits; ++z) {
        float o[8];
        load8<true>(h, ((long long)(2 * z + p) * T + t) * N + n, o);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[p][j] += o[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = gated(sum[0][j], sum[1][j], limit);
  }
  const float amax = group_amax(v);
  const float up = kFp8Max / amax;
  if (n < N)
    *reinterpret_cast<uint2 *>(codes + (long long)t * N + n) =
        uint2{fp8_codes4(v[0], v[1], v[2], v[3], up), fp8_codes4(v[4], v[5], v[6], v[7], up)};
  if (lane == 0) scales[item] = amax / kFp8Max;
}

// ---------------------------------------------------------------------------
// Many tokens: a workgroup computes weight rows (NPROJ 2: half of them
// from each projection) x tokens with WN x WT waves of BN x BT blocks of 16 x 16.  Both
// operands come into LDS a group of K at a time by direct loads of 16-byte
// pieces, a ring of groups deep.  Piece p of
// row R lies at p ^ ((R >> 1) & 7): the 16 rows that a quarter of a wave reads
// are then on 16 different pieces of 256 bytes.  Pieces past K are out of the
// buffers' range, which gives zeros; rows past the last are that or the tile's
// first once more (fp8_span.h), and their sums are not stored.
//
// The largest tile is 256 x 256 (the pair: 2 x 128 x 256): 64 KB a group of K, two
// groups in LDS, 128 of 256 registers hold sums.  4096 rows, K and N 4096: 58 to 63
// us, 2.2 to 2.35 PFLOP/s where a library's product of plain 8-bit matrices has
// 2.8; 8192 rows, K and N 8192: 463 us, 2.37; the pair, 4001 rows, K 4096, 2 x 2048
// features: 104 to 111 us, 1.25 where a bf16 one has 1.45.  Matrix cores are busy for
// 55 to 59 % of the cycles, at a clock that power limits: without the loads 68.6 us
// are 62.6, and without the conversions the pair takes longer.
// ---------------------------------------------------------------------------
constexpr int kTileXcds = 8;

struct Fp8TileArgs {
  Fp8Args p;
  int row_tiles, tok_tiles;
  int strip;        // row tiles of a strip: consecutive items walk across it, then along the tokens
};

// WN x WT waves of BN x BT blocks; KB of LDS for a workgroup.
template <int WN_, int WT_, int BN_, int BT_, int KB = 156>
struct Fp8Tile {
  static constexpr int WN = WN_, WT = WT_, BN = BN_, BT = BT_;
  static constexpr int kWaves = WN * WT, kThreads = 64 * kWaves;
  static constexpr int kRows = 16 * BN * WN, kTok = 16 * BT * WT;
  static constexpr int kX = kTok * kFp8Group, kW = kRows * kFp8Group;
  static constexpr int kStage = kX + kW;
  static constexpr int kS = 2 * kTok * 16;  // the rows' scales, four groups at a time, twice
  static constexpr int kXLoads = kX / (1024 * kWaves), kWLoads = kW / (1024 * kWaves);
  static constexpr int kLoads = kXLoads + kWLoads;
  static constexpr int kFit = (KB * 1024 - kS) / kStage;
  static constexpr int kStages = kFit < 6 ? kFit : 6;
  static constexpr int kBytes = kStages * kStage + kS;
  static_assert(kX % (1024 * kWaves) == 0 && kW % (1024 * kWaves) == 0, "whole loads");
  static_assert(kTok <= kThreads && kTok % 64 == 0, "a lane has one token's scales");
  static_assert(kStages >= 2 && BN >= 2, "a ring, blocks in turn");
  __device__ static int swz(int row) { return (row >> 1) & 7; }
};

__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// NPROJ 1: bf16 products by the 8-bit instruction; 2: the gated pair, quantised, exact products.
template <int NPROJ, class L>
__global__ __launch_bounds__(L::kThreads) void fp8_tile_kernel(Fp8TileArgs a) {
  constexpr int BN = L::BN, BT = L::BT, kWaves = L::kWaves;
  constexpr int kS = L::kStages;
  constexpr int kFeat = L::kRows / NPROJ;  // features of a workgroup
  constexpr int HB = BN / NPROJ;           // 16-row blocks of a wave and projection
  constexpr bool FAST = NPROJ == 1;
  static_assert(NPROJ == 1 || kFeat == kFp8Group, "a group of features");
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  // workgroups are dealt to the XCDs in turn: each takes a contiguous share of the items
  const int items = a.row_tiles * a.tok_tiles;
  const int per_xcd = (items + kTileXcds - 1) / kTileXcds;
  const int on_xcd = (int)blockIdx.x / kTileXcds;
  const int item = ((int)blockIdx.x % kTileXcds) * per_xcd + on_xcd;
  if (on_xcd >= per_xcd || item >= items) return;
  const int above = item / (a.strip * a.tok_tiles) * a.strip;  // row tiles of the strips before
  const int wide = min(a.strip, a.row_tiles - above), in_strip = item - above * a.tok_tiles;
  const int rt = above + in_strip % wide, tt = in_strip / wide;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int wn = wave % L::WN, wt = wave / L::WN;
  const int K = a.p.K, N = a.p.N, T = a.p.T, groups = a.p.groups;
  const int f0 = rt * kFeat, t0 = tt * L::kTok;
  const int toks = min(T - t0, L::kTok), feats = min(N - f0, kFeat);

  // Load j fills the (kWaves j + wave)-th 1 KB of the tokens, then of the weight rows.
  // Every load has a descriptor of its own that begins at its first row, so that one
  // register holds the lane's offset in all of them (one each: 8 registers spilled at
  // 128 x 256 gated, and a reload in every group).
  constexpr int kStep = 8 * kWaves;  // rows of a load
  static_assert(kStep % 16 == 0 && kFeat % kStep == 0, "the same order of pieces, one projection");
  auto rows_from = [&](const uint8_t *rows, int first, int there) {
    const Fp8Span span = fp8_span(first, there);
    return make_rsrc(rows + (long long)span.first * K, (uint32_t)span.rows * (uint32_t)K);
  };
  __amdgpu_buffer_rsrc_t res[L::kLoads];
#pragma unroll
  for (int j = 0; j < L::kXLoads; ++j)
    res[j] = rows_from((const uint8_t *)a.p.x + (long long)t0 * K, j * kStep, toks);
#pragma unroll
  for (int j = 0; j < L::kWLoads; ++j)
    res[L::kXLoads + j] =
        rows_from(a.p.w[j * kStep / kFeat] + (long long)f0 * K, j * kStep % kFeat, feats);
  const int piece = 16 * ((lane % 8) ^ L::swz(wave * 8 + lane / 8));
  uint32_t off = (uint32_t)(wave * 8 + lane / 8) * (uint32_t)K + piece;
  const int tail = K % kFp8Group;  // codes of a last group that is not whole
  // Load j of group c into its stage; the x loads come first.
  auto issue = [&](int c, int stage, int j) {
    if (j == 0 && tail != 0 && c == groups - 1 && piece >= tail)
      off = kOutOfRange;  // (the last use of the offset)
    buf16_to_lds(res[j], smem + stage * L::kStage + (j * kWaves + wave) * 1024, off,
                 (uint32_t)c * kFp8Group);
  };
  // The rows' scales come the same way, four groups at a time and up to eight
  // ahead, the first waves' lanes a token each: 16 bytes a token where the rows
  // of scales lie on 16 bytes ([token][4 groups] in LDS), else a group at a time
  // ([4 groups][token]).
  const bool quads = groups % 4 == 0;
  float *slds = reinterpret_cast<float *>(smem + kS * L::kStage);
  const __amdgpu_buffer_rsrc_t sres =
      make_rsrc(a.p.xs + (long long)t0 * groups, (uint32_t)toks * (uint32_t)groups * 4u);
  auto issue_scales = [&](int g) {  // of groups g .. g + 3, g a multiple of 4
    if (wave * 64 >= L::kTok) return;
    float *to = slds + ((g >> 2) & 1) * (4 * L::kTok);
    const uint32_t off = (uint32_t)tid * (uint32_t)groups * 4u;
    if (quads) {
      buf16_to_lds(sres, to + wave * 256, off, (uint32_t)g * 4);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        buf4_to_lds(sres, to + j * L::kTok + wave * 64, off, (uint32_t)fp8_scale_group(g, j, groups) * 4);
    }
  };

  // The block scales of the wave's features (its rows lie in one block of 128):
  // lane l has the l-th group's of each 64.  No load into a register is within
  // the loop over these: it would share its counter with the direct loads, and
  // the compiler would wait for all of them in every group.
  const float *sw[NPROJ];
#pragma unroll
  for (int p = 0; p < NPROJ; ++p) {
    sw[p] = a.p.ws[p] + (long long)min((f0 + wn * HB * 16) / kFp8Group, (N - 1) / kFp8Group) * groups;
  }

  glm_f32x4 acc[BN][BT];
#pragma unroll
  for (int b = 0; b < BN; ++b)
#pragma unroll
    for (int t = 0; t < BT; ++t) acc[b][t] = glm_f32x4{0.f, 0.f, 0.f, 0.f};

  const int p0 = 4 * (q & 1) + 2 * (q >> 1);  // the lane's pieces of a row: p0, p0 + 1
  auto frag = [&](const uint8_t *row0, int row) {
    const uint8_t *p = row0 + row * kFp8Group;
    return join16(*reinterpret_cast<const glm_u32x4 *>(p + 16 * (p0 ^ L::swz(row))),
                  *reinterpret_cast<const glm_u32x4 *>(p + 16 * ((p0 + 1) ^ L::swz(row))));
  };
  // Row block b's products run beside the scaling of block b - 1's and the
  // reads (and the conversion) of block b + 1.  The order is written out: left
  // to itself the compiler scales a result right behind its product and waits
  // for it there.
  // side() is done beside block 0's products.
  auto compute = [&](int stage, int g, const float (&wsc)[2], auto side) {
    const uint8_t *base = smem + stage * L::kStage;
    const int tstep = quads ? 4 : 1, gstep = quads ? 1 : L::kTok;
    const float *sx = slds + ((g >> 2) & 1) * (4 * L::kTok) + (wt * BT * 16 + r) * tstep + (g & 3) * gstep;
    constexpr int kSteps = Fp8Operand<FAST>::kSteps;
    auto wfrag = [&](int b) {
      return frag(base + L::kX, (b / HB) * kFeat + wn * HB * 16 + (b % HB) * 16 + r);
    };
    // two blocks' reads ahead of the products (all of them ahead: 8 % more time at BT 1)
    constexpr int kAhead = 2;
    fp8_frag w[BN], xf[BT];
    w[0] = wfrag(0);
#pragma unroll
    for (int t = 0; t < BT; ++t) xf[t] = frag(base, (wt * BT + t) * 16 + r);
    float s[NPROJ][BT];
#pragma unroll
    for (int t = 0; t < BT; ++t) s[0][t] = sx[16 * t * tstep];
    // One result a token block, scaled before the next block's first step
    // overwrites it, or two in turn where too few blocks lie between.
    constexpr int kBuf = BT >= 4 ? 1 : 2;
    glm_f32x4 c[kBuf][BT];
    auto scale = [&](int b, int t) {
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[b][t][j] += c[b % kBuf][t][j] * s[b / HB][t];
    };
#pragma unroll
    for (int b = 1; b < kAhead; ++b) w[b] = wfrag(b);
    Fp8Operand<FAST> x[BT], now(w[0]);
    // block 0: token blocks in turn, so that the first products do not wait for the last's operands
#pragma unroll
    for (int t = 0; t < BT; ++t) {
      x[t] = Fp8Operand<FAST>(xf[t]);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) c[0][t] = step_sum(now, x[t], i, c[0][t]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int t = 0; t < BT; ++t)
#pragma unroll
      for (int p = NPROJ - 1; p >= 0; --p) s[p][t] = s[0][t] * wsc[p];
    side();
    now = Fp8Operand<FAST>(w[1]);
    if constexpr (kAhead < BN) w[kAhead] = wfrag(kAhead);
#pragma unroll
    for (int b = 1; b <= BN; ++b) {
      Fp8Operand<FAST> next = now;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if constexpr (!FAST) {
          if (i > 0 && b + 1 < BN) next.part(w[b + 1], i - 1);
        }
#pragma unroll
        for (int t = 0; t < BT; ++t) {
          if (i == 0 && (kBuf == 1 || b == BN)) scale(b - 1, t);
          if (b < BN) c[b % kBuf][t] = step_sum(now, x[t], i, c[b % kBuf][t]);
          if (i == 0 && kBuf == 2 && b < BN) {
            __builtin_amdgcn_sched_barrier(0);
            scale(b - 1, t);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (b == BN) break;
      }
      if constexpr (FAST) {
        if (b + 1 < BN) now = Fp8Operand<FAST>(w[b + 1]);
      } else {
        if (b + 1 < BN) next.part(w[b + 1], kSteps - 1);
        now = next;
      }
      if (b + kAhead < BN) w[b + kAhead] = wfrag(b + kAhead);
    }
  };
  issue_scales(0);
#pragma unroll
  for (int g = 0; g < kS - 1; ++g)
    if (g < groups)
#pragma unroll
      for (int j = 0; j < L::kLoads; ++j) issue(g, g, j);
  // The loads are asked for behind the first products: the address unit takes 16
  // cycles for one, and a wave stands still meanwhile.  Scales asked for in group
  // c are there in group c + 4: as many groups' loads as may be outstanding then
  // (kS - 2) were asked for behind them.
  static_assert(kS <= 6, "the scales' loads are older than those that may be outstanding");
  int stage = 0;
  auto group = [&](int c, bool more, const float (&held)[NPROJ]) {
    float ws[2];
    ws[0] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(held[0]), c & 63));
    ws[1] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(held[NPROJ - 1]), c & 63));
    if (more) {
      __builtin_amdgcn_s_waitcnt(vmcnt_imm((kS - 2) * L::kLoads));
    } else {
      wait_groups_ahead<kS - 2, L::kLoads>(min(kS - 2, groups - 1 - c));
    }
    ring_barrier();
    const int into = stage == 0 ? kS - 1 : stage - 1;
    compute(stage, c, ws, [&] {
      if ((c & 3) == 0 && c + 4 < groups) issue_scales(c + 4);
      if (more) {
#pragma unroll
        for (int j = 0; j < L::kLoads; ++j) issue(c + kS - 1, into, j);
      }
    });
    stage = stage + 1 == kS ? 0 : stage + 1;
  };
  for (int c = 0; c < groups;) {
    const int end = min(c + 64, groups), whole = min(end, groups - (kS - 1));
    float held[NPROJ];
#pragma unroll
    for (int p = 0; p < NPROJ; ++p) {
      held[p] = sw[p][min(c + lane, groups - 1)];
      asm volatile("" ::"v"(held[p]));  // (waited for here, not within the loops)
    }
#pragma clang loop unroll(disable)
    for (; c < whole; ++c) group(c, true, held);
#pragma clang loop unroll(disable)
    for (; c < end; ++c) group(c, false, held);
  }

  const int fw = f0 + wn * HB * 16, tw = t0 + wt * BT * 16;  // the wave's first feature and token
  if constexpr (NPROJ == 1) {
    // rows of no 16-byte pieces: element by element (K 4096, N 4095 for 4096: 333 rows 16.5 us for
    // 16.1, 1024 31.4 for 26.9, 4096 84.8 for 66.2)
    if (N % 8 != 0) {
#pragma unroll
      for (int b = 0; b < BN; ++b)
#pragma unroll
        for (int t = 0; t < BT; ++t) {
          const int tok = tw + 16 * t + r;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int n = fw + 16 * b + 4 * q + j;
            if (tok < T && n < N)
              a.p.out[(long long)tok * N + n] = (uint16_t)f32_to_bf16(acc[b][t][j]);
          }
        }
      return;
    }
    // each 16-token block through the wave's own LDS: a token's features leave in whole pieces
    ring_barrier();
    constexpr int kSegs = 2 * BN, kStride = 16 * kSegs + 16;
    static_assert(kWaves * 16 * kStride <= L::kBytes, "output staging");
    uint8_t *st = smem + wave * 16 * kStride;
#pragma unroll
    for (int t = 0; t < BT; ++t) {
#pragma unroll
      for (int b = 0; b < BN; ++b) {
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = f32_to_bf16(acc[b][t][j]);
        *reinterpret_cast<uint2 *>(st + r * kStride + (b * 16 + 4 * q) * 2) =
            uint2{o[0] | (o[1] << 16), o[2] | (o[3] << 16)};
      }
      wave_lds_fence();
#pragma unroll
      for (int p = 0; p < 16 * kSegs; p += 64) {
        const int tok = (p + lane) / kSegs, seg = (p + lane) % kSegs;
        if (tok < 16 && tw + 16 * t + tok < T && fw + 8 * seg < N)
          *reinterpret_cast<glm_u32x4 *>(a.p.out + (long long)(tw + 16 * t + tok) * N + fw +
                                         8 * seg) =
              *reinterpret_cast<const glm_u32x4 *>(st + tok * kStride + 16 * seg);
      }
      wave_lds_fence();
    }
  } else {
    // h in the gate's accumulators
#pragma unroll
    for (int b = 0; b < HB; ++b)
#pragma unroll
      for (int t = 0; t < BT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[b][t][j] = gated(acc[b][t][j], acc[HB + b][t][j], a.p.limit);
    // a token's largest finite magnitude over the 128 features: the lane's 4 HB, the four lanes of
    // the token, the waves along the features
    ring_barrier();
    float *red = reinterpret_cast<float *>(smem);  // [L::WN][kTok]
    uint8_t *st = smem + L::WN * L::kTok * 4;    // [kTok][128 codes, 16 bytes of padding]
    constexpr int kStride = kFp8Group + 16;
    static_assert(L::WN * L::kTok * 4 + L::kTok * kStride <= L::kBytes, "output staging");
#pragma unroll
    for (int t = 0; t < BT; ++t) {
      float m = 0.f;
#pragma unroll
      for (int b = 0; b < HB; ++b) {
        float (&v)[4] = reinterpret_cast<float (&)[4]>(acc[b][t]);
        if (fw + 16 * b + 4 * q < N) m = fmaxf(m, finite_abs_max(v));
      }
      m = fmaxf(m, __shfl_xor(m, 16, kWave));
      m = fmaxf(m, __shfl_xor(m, 32, kWave));
      if (q == 0) red[wn * L::kTok + (wt * BT + t) * 16 + r] = m;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < BT; ++t) {
      const int tok = (wt * BT + t) * 16 + r;
      float m = kFp8Tiny;
#pragma unroll
      for (int w = 0; w < L::WN; ++w) m = fmaxf(m, red[w * L::kTok + tok]);
      const float up = kFp8Max / m;
#pragma unroll
      for (int b = 0; b < HB; ++b)
        *reinterpret_cast<uint32_t *>(st + tok * kStride + wn * HB * 16 + 16 * b + 4 * q) =
            fp8_codes4(acc[b][t][0], acc[b][t][1], acc[b][t][2], acc[b][t][3], up);
      if (wn == 0 && q == 0 && t0 + tok < T)
        a.p.scales[(long long)(t0 + tok) * fp8_groups(N) + f0 / kFp8Group] = m / kFp8Max;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < L::kTok * 8 / L::kThreads; ++i) {
      const int slot = i * L::kThreads + tid, tok = slot / 8, n = f0 + 16 * (slot % 8);
      if (t0 + tok < T && n < N)
        *reinterpret_cast<glm_u32x4 *>(a.p.codes + (long long)(t0 + tok) * N + n) =
            *reinterpret_cast<const glm_u32x4 *>(st + tok * kStride + 16 * (slot % 8));
    }
  }
}

}  // namespace glm

using namespace glm;

static size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// splits: the workgroups along K.
template <class L>
static int launch_stream(hipStream_t stream, Fp8Args a, int splits = 1) {
  const dim3 grid((unsigned)((a.N + 16 * L::RB - 1) / (16 * L::RB)),
                  (unsigned)((a.T + 16 * L::TB - 1) / (16 * L::TB)), (unsigned)splits);
  // a workgroup a CU takes all the LDS for its groups in flight, else two share it
  const int coded = L::coded_bytes(a.groups, splits, a.T);
  const long long wgs = (long long)grid.x * grid.y * grid.z;
  const int room = (wgs <= 256 ? kStreamKB : kStreamPairKB) * 1024 - coded;
  int ahead = room / (L::kWaves * L::kSlot);
  const int per_wave = (a.groups + L::kWaves * splits - 1) / (L::kWaves * splits);
  ahead = ahead < L::kMost ? ahead : L::kMost;
  ahead = ahead < per_wave ? ahead : per_wave;
  a.ahead = ahead < 1 ? 1 : ahead;
  a.per_token = a.T > 1 && a.T <= kFusedTokens ? (uint32_t)(((1ull << 32) + a.T - 1) / a.T) : 0;
  const int bytes = L::kWaves * a.ahead * L::kSlot + coded;
  hipLaunchKernelGGL((fp8_stream_kernel<L>), grid, dim3(L::kThreads),
                     (size_t)(bytes > L::kPart ? bytes : L::kPart), stream, a);
  GLM_LAUNCH_CHECK("fp8_stream_kernel");
  return GLM_OK;
}

// Workspace of rows that the product does not take as they are.
static size_t rows_bytes(int T, int K, int N, int type) {
  const long long codes = (long long)T * fp8_groups(K) * kFp8Group;
  if (type == GLM_ROWS_FP8 || (T <= kFusedTokens && codes <= kFusedCodes && N <= kFusedFeatures)) return 0;
  return round256((size_t)T * K) + round256((size_t)T * fp8_groups(K) * 4);
}

// Rows as the kernels take them: few as they are, more of them quantised into
// the workspace first.
static int rows_for(hipStream_t stream, Fp8Args &a, int &type, uint8_t *&ws) {
  if (!rows_bytes(a.T, a.K, a.N, type)) return GLM_OK;
  uint8_t *codes = ws;
  ws += round256((size_t)a.T * a.K);
  float *scales = reinterpret_cast<float *>(ws);
  ws += round256((size_t)a.T * a.groups * 4);
  const int rc = glm_fp8_quantize_rows(stream, a.x, type, a.T, a.K, codes, scales);
  a.x = codes;
  a.xs = scales;
  type = GLM_ROWS_FP8;
  return rc;
}

template <int NPROJ, class L>
static int launch_tile(hipStream_t stream, const Fp8Args &p) {
  constexpr int feat = L::kRows / NPROJ;
  Fp8TileArgs a{p, (p.N + feat - 1) / feat, (p.T + L::kTok - 1) / L::kTok, 1};
  const int items = a.row_tiles * a.tok_tiles;
  // What an XCD's 32 CUs work on at once as square as it goes: the fewest rows and
  // tokens for its L2 to fetch.  (8192 rows, K and N 8192: 511 us along the tokens, 463
  // in strips; 4096, 256 x 128 tiles: 84 and 79.5.)
  const int square = std::min((items + kTileXcds - 1) / kTileXcds, 32);
  while (a.strip * a.strip * L::kRows < square * L::kTok) ++a.strip;
  a.strip = std::min(a.strip, a.row_tiles);
  hipLaunchKernelGGL((fp8_tile_kernel<NPROJ, L>),
                     dim3((unsigned)((items + kTileXcds - 1) / kTileXcds * kTileXcds)),
                     dim3(L::kThreads), (size_t)L::kBytes, stream, a);
  GLM_LAUNCH_CHECK("fp8_tile_kernel");
  return GLM_OK;
}

// A way to cut a product: features and tokens of a workgroup, and its time in
// tenths of a us at K 4096, base + each for every 256 workgroups begun (one a CU);
// `groups` where the second part alone goes by K.  Over 9 pairs of K from 1024 to
// 16384 and N from 1024 to 8192, 12 to 6000 rows, each cut timed by a build that took
// it as an argument, what the costs choose took 0.5 % more than the fastest on
// average, 26 % at most (72 rows, K 16384, N 4096: above 64 rows the choice leaves K
// out); of the gated pair's 5 % at most.
struct Fp8Cut {
  int feat, tok, base, each;
  long long workgroups(int T, int N) const {
    return (long long)((N + feat - 1) / feat) * ((T + tok - 1) / tok);
  }
  long long cost(int T, int N, int groups = 32) const {
    return base + each * ((workgroups(T, N) + 255) / 256) * groups / 32;
  }
};
template <int M>
static int cheapest(const Fp8Cut (&cuts)[M], int T, int N, int groups) {
  int best = 0;
  for (int i = 1; i < M; ++i)
    if (cuts[i].cost(T, N, groups) < cuts[best].cost(T, N, groups)) best = i;
  return best;
}

template <int WAVES, int NPROJ, int RB, int TB, bool FAST = false>
using CodedStream = Fp8Stream<WAVES, NPROJ, RB, TB, GLM_ROWS_FP8, false, FAST>;

// Rows that come as bf16 or f32, and up to 8 coded ones: 16 features a workgroup.
template <int NPROJ>
static int stream_few(hipStream_t stream, const Fp8Args &a, int type, int splits) {
  if (type == GLM_ROWS_BF16)
    return launch_stream<Fp8Stream<8, NPROJ, 1, 1, GLM_ROWS_BF16, true>>(stream, a, splits);
  if (type == GLM_ROWS_F32)
    return launch_stream<Fp8Stream<8, NPROJ, 1, 1, GLM_ROWS_F32, true>>(stream, a, splits);
  return launch_stream<Fp8Stream<8, NPROJ, 1, 1, GLM_ROWS_FP8, true>>(stream, a, splits);
}
static bool few(int T, int type) { return type != GLM_ROWS_FP8 || T <= 8; }

// Products: up to 64 rows by the exact sum, whose time the weights' bytes set, more
// by the 8-bit instruction; by the streaming kernel, whose waves do not wait for
// each other but read all operands of their tile, or in larger tiles.  At N 4096,
// K 4096, us by tile: 64 rows 16 x 32 9.6, 32 x 32 8.5, 16 x 64 9.0; 80 rows 32 x 48
// 8.1, 64 x 32 8.8, 256 x 256 46.8; 600 rows 64 x 48 26.7, tiles of 64 x 64 22.9;
// 1024 rows 128 x 128 24.5, 64 x 64 34.0; 1600 rows 64 x 48 54.2, 64 x 64 52.8, 256 x
// 128 36.1, 256 x 256 49.5; 4096 rows 124.6, 151.3, 79.5, 61.9.  A workgroup a CU has all its LDS: five or six waves there, each with a group
// in flight: 150 rows 64 x 48 of four waves 11.3, six 9.8; 256 rows 64 x 64 of six 11.9,
// eight 11.9, the tile 15.1; 333 rows 64 x 96 of four 15.8, five 15.0, six 15.5, 64 x 48 of
// four 16.2; but 512 rows 64 x 64 of six 20.8, the tile 18.5.
static int linear_product(hipStream_t stream, const Fp8Args &a, int type) {
  if (few(a.T, type)) return stream_few<1>(stream, a, type, 1);
  if (a.T <= kExactTokens) {
    static const Fp8Cut cuts[] = {{16, 16, 42, 23}, {16, 32, 46, 34}, {32, 32, 32, 78}, {16, 64, 154, 37}};
    switch (cheapest(cuts, a.T, a.N, a.groups)) {
      case 0: return launch_stream<CodedStream<8, 1, 1, 1>>(stream, a);
      case 1: return launch_stream<CodedStream<8, 1, 1, 2>>(stream, a);
      case 2: return launch_stream<CodedStream<8, 1, 2, 2>>(stream, a);
      default: return launch_stream<CodedStream<8, 1, 1, 4>>(stream, a);
    }
  }
  static const Fp8Cut cuts[] = {{32, 48, 30, 52},  {64, 32, 40, 46},   {64, 48, 45, 62}, {64, 64, 90, 54},
                                {128, 128, 25, 227}, {256, 128, 10, 331}, {256, 256, 0, 500},
                                {64, 48, 28, 70}, {64, 64, 30, 87}, {64, 96, 36, 113}};
  switch (cheapest(cuts, a.T, a.N, 32)) {
    case 0: return launch_stream<CodedStream<8, 1, 2, 3, true>>(stream, a);
    case 1: return launch_stream<CodedStream<4, 1, 4, 2, true>>(stream, a);
    case 2: return launch_stream<CodedStream<4, 1, 4, 3, true>>(stream, a);
    case 3: return launch_tile<1, Fp8Tile<2, 2, 2, 2, 52>>(stream, a);
    case 4: return launch_tile<1, Fp8Tile<2, 4, 4, 2>>(stream, a);
    case 5: return launch_tile<1, Fp8Tile<2, 4, 8, 2>>(stream, a);
    case 6: return launch_tile<1, Fp8Tile<2, 4, 8, 4>>(stream, a);
    case 7: return launch_stream<CodedStream<6, 1, 4, 3, true>>(stream, a);
    case 8: return launch_stream<CodedStream<6, 1, 4, 4, true>>(stream, a);
    default: return launch_stream<CodedStream<5, 1, 4, 6, true>>(stream, a);
  }
}

// Gated pairs: streamed, their sums gated by a second launch, or in tiles that gate
// and quantise by themselves.  At 2 x 2048 features, K 4096, us by tile (streamed
// ones without the second launch's 2.5 us and more): 64 rows 16 x 16 9.7, 16 x 32 8.7,
// 16 x 48 9.2; 333 rows 32 x 32 21.7, 32 x 48 19.0, 32 x 64 21.4, 128 x 64 38.9, 128 x 128
// 60.9; 1000 rows 32 x 48 51.4, 32 x 64 46.7, 128 x 64 44.4, 128 x 128 64.5, 128 x 256 101;
// 1500 rows 71.5, 65.8, 75.8, 64.7, 101; 3000 rows 128 x 128 121, 128 x 256 104.  256 rows
// of K 2048 into 2 x 7168: 32 x 64 and its second launch take 1.4 times 128 x 64.
constexpr Fp8Cut kGatedCuts[] = {{16, 16, 44, 26}, {16, 32, 50, 35}, {16, 48, 30, 62},   {32, 32, 55, 52},
                                 {32, 48, 60, 71}, {32, 64, 60, 84}, {128, 64, 30, 380}, {128, 128, 0, 520},
                                 {128, 256, 0, 865}};
constexpr int kGatedStreams = 6, kGatedWays = 9;
struct GatedPlan {
  // splits of K, of the first cut where its workgroups are at most half the CUs: as many as leave
  // every wave a group
  int cut, splits;
};
static GatedPlan gated_plan(int T, int K, int N, int type) {
  GatedPlan plan{0, 1};
  double best = 0;
  for (int i = 0; i < (few(T, type) ? 1 : kGatedWays); ++i) {
    double c = (double)kGatedCuts[i].cost(T, N) * fp8_groups(K) / 32;
    if (i < kGatedStreams) c += 25 + (double)T * N * 2e-5;  // the second launch: 8 bytes a feature
    if (i == 0 || c < best) {
      plan.cut = i;
      best = c;
    }
  }
  // (a larger cut costs less only where the one before it takes two rounds of 256 workgroups,
  // and so has more than 128 itself: none of them has CUs to spare for splits)
  if (plan.cut != 0) return plan;
  const int most = fp8_groups(K) / 8;  // eight waves
  long long s = 256 / kGatedCuts[0].workgroups(T, N);
  s = s < most ? s : most;
  plan.splits = s < 1 ? 1 : s < 8 ? (int)s : 8;
  return plan;
}

static int gated_product(hipStream_t stream, const Fp8Args &a, int type) {
  const GatedPlan plan = gated_plan(a.T, a.K, a.N, type);
  const int splits = plan.splits;
  int rc;
  if (few(a.T, type)) {
    rc = stream_few<2>(stream, a, type, splits);
  } else {
    switch (plan.cut) {
      case 0: rc = launch_stream<CodedStream<8, 2, 1, 1>>(stream, a, splits); break;
      case 1: rc = launch_stream<CodedStream<8, 2, 1, 2>>(stream, a); break;
      case 2: rc = launch_stream<CodedStream<8, 2, 1, 3>>(stream, a); break;
      case 3: rc = launch_stream<CodedStream<4, 2, 2, 2>>(stream, a); break;
      case 4: rc = launch_stream<CodedStream<4, 2, 2, 3>>(stream, a); break;
      case 5: rc = launch_stream<CodedStream<4, 2, 2, 4>>(stream, a); break;
      case 6: return launch_tile<2, Fp8Tile<4, 2, 4, 2>>(stream, a);
      case 7: return launch_tile<2, Fp8Tile<2, 4, 8, 2>>(stream, a);
      default: return launch_tile<2, Fp8Tile<2, 4, 8, 4>>(stream, a);
    }
  }
  if (rc) return rc;
  const long long items = (long long)a.T * fp8_groups(a.N);
  hipLaunchKernelGGL(fp8_gate_kernel, dim3((unsigned)((items + 15) / 16)), dim3(256), 0, stream,
                     a.h, splits, a.T, a.N, a.limit, a.codes, a.scales);
  GLM_LAUNCH_CHECK("fp8_gate_kernel");
  return GLM_OK;
}

// The pair's f32 sums, where a second launch gates them.  Rows that the workspace
// holds as codes are coded for the plan.
static size_t gated_bytes(int T, int K, int N, int type) {
  const GatedPlan plan = gated_plan(T, K, N, rows_bytes(T, K, N, type) ? GLM_ROWS_FP8 : type);
  return plan.cut < kGatedStreams ? round256((size_t)plan.splits * 2 * T * N * 4) : 0;
}

static bool sizes_fit(int T, int K, int N) {
  return T >= 0 && K >= 16 && N >= 1 && K % 16 == 0 && K <= 1 << 20 && N <= 1 << 20 && T <= 1 << 20;
}

static int check_product(const char *name, const void *x, int x_type, const float *x_scales, int T,
                         int K, int N, const void *workspace, size_t need, size_t bytes) {
  GLM_REQUIRE(T >= 0 && K >= 1 && N >= 1 && x_type >= GLM_ROWS_BF16 && x_type <= GLM_ROWS_FP8,
              GLM_ERR_INVALID_ARGUMENT, "%s: invalid sizes or row type", name);
  GLM_REQUIRE(sizes_fit(T, K, N), GLM_ERR_UNSUPPORTED_SHAPE,
              "%s: %d rows of %d channels (a multiple of 16) into %d: up to 2^20 rows and 2^20 "
              "channels", name, T, K, N);
  GLM_REQUIRE(x && (x_type != GLM_ROWS_FP8 || x_scales), GLM_ERR_INVALID_ARGUMENT,
              "%s: null pointer", name);
  GLM_REQUIRE(bytes >= need && (need == 0 || workspace), GLM_ERR_WORKSPACE,
              "%s: workspace of %zu bytes, %zu needed", name, bytes, need);
  GLM_REQUIRE(glm_aligned16({x, x_scales, workspace}), GLM_ERR_INVALID_ARGUMENT,
              "%s: buffers must be 16-byte aligned", name);
  return GLM_OK;
}

extern "C" size_t glm_fp8_workspace_bytes(int x_type, int T, int K, int N, int gated) {
  if (!sizes_fit(T, K, N) || x_type < GLM_ROWS_BF16 || x_type > GLM_ROWS_FP8) return 0;
  return rows_bytes(T, K, N, x_type) + (gated && T > 0 ? gated_bytes(T, K, N, x_type) : 0);
}

extern "C" int glm_fp8_linear(void *stream, const void *x, int x_type, const float *x_scales, int T,
                              int K, const uint8_t *weight, const float *scales, int N,
                              void *workspace, size_t workspace_bytes, uint16_t *out) {
  glm::clear_error();
  const int bad = check_product("fp8_linear", x, x_type, x_scales, T, K, N, workspace,
                                glm_fp8_workspace_bytes(x_type, T, K, N, 0), workspace_bytes);
  if (bad) return bad;
  GLM_REQUIRE(weight && scales && out, GLM_ERR_INVALID_ARGUMENT, "fp8_linear: null pointer");
  GLM_REQUIRE(glm_aligned16({weight, scales, out}), GLM_ERR_INVALID_ARGUMENT,
              "fp8_linear: buffers must be 16-byte aligned");
  if (T == 0) return GLM_OK;
  Fp8Args a{x, x_scales, {weight, nullptr}, {scales, nullptr}, T, K, N, fp8_groups(K), 0.f, 0,
            0, out, nullptr, nullptr, nullptr};
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  hipStream_t s = (hipStream_t)stream;
  const int rc = rows_for(s, a, x_type, ws);
  return rc ? rc : linear_product(s, a, x_type);
}

extern "C" int glm_fp8_gate_up(void *stream, const void *x, int x_type, const float *x_scales,
                               int T, int K, const uint8_t *gate, const float *gate_scales,
                               const uint8_t *up, const float *up_scales, int N, float limit,
                               void *workspace, size_t workspace_bytes, uint8_t *codes,
                               float *scales) {
  glm::clear_error();
  const int bad = check_product("fp8_gate_up", x, x_type, x_scales, T, K, N, workspace,
                                glm_fp8_workspace_bytes(x_type, T, K, N, 1), workspace_bytes);
  if (bad) return bad;
  GLM_REQUIRE(N % 16 == 0, GLM_ERR_UNSUPPORTED_SHAPE, "fp8_gate_up: %d features, a multiple of 16",
              N);
  GLM_REQUIRE(gate && gate_scales && up && up_scales && codes && scales, GLM_ERR_INVALID_ARGUMENT,
              "fp8_gate_up: null pointer");
  GLM_REQUIRE(glm_aligned16({gate, gate_scales, up, up_scales, codes, scales}),
              GLM_ERR_INVALID_ARGUMENT, "fp8_gate_up: buffers must be 16-byte aligned");
  if (T == 0) return GLM_OK;
  Fp8Args a{x, x_scales, {gate, up}, {gate_scales, up_scales}, T, K, N, fp8_groups(K), limit,
            0, 0, nullptr, nullptr, codes, scales};
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  hipStream_t s = (hipStream_t)stream;
  int rc = rows_for(s, a, x_type, ws);
  if (rc) return rc;
  a.h = reinterpret_cast<float *>(ws);
  return gated_product(s, a, x_type);
}
