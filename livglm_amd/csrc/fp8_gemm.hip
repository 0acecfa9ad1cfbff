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
// v_mfma_f32_16x16x32_bf16: exact products, f32 sums (1e-8 relative error on
// normal values).  As it is in one v_mfma_f32_16x16x128_f8f6f4, at twice the
// rate: the core aligns eight products at a time to the largest of them and
// drops what lies 2^-14 of it below, which is 1.5e-5 of the sum on normal
// values, without a bias.  The latter serves products whose result is rounded
// to bf16 (1.7e-3) and whose time the matrix cores set.
#include "fp8_rows.h"
#include "lds_stage.h"

#include <climits>

namespace glm {

typedef int fp8_frag __attribute__((ext_vector_type(8)));

constexpr int kStreamWaves = 8;
constexpr int kStreamThreads = 64 * kStreamWaves;
constexpr int kStreamAhead = 4;  // groups whose weights a wave has in flight
constexpr int kFusedTokens = 16; // rows that the product quantises itself, up to so many

struct Fp8Args {
  const void *x;          // codes, or bf16 / f32 rows
  const float *xs;        // [T][groups], with codes
  const uint8_t *w[2];    // [N][K]
  const float *ws[2];     // [ceil(N / 128)][groups]
  int T, K, N, groups;
  float limit;
  uint16_t *out;          // NPROJ 1: bf16 [T][N]
  float *h;               // NPROJ 2: f32 [T][N]
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
  glm_bf16x8 v[4];
  __device__ __forceinline__ explicit Fp8Operand(const fp8_frag &f) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = mxfp8_words_to_bf16x8((uint32_t)f[2 * i], (uint32_t)f[2 * i + 1], 1.0f);
  }
  Fp8Operand() = default;
};
template <>
struct Fp8Operand<true> {
  fp8_frag v;
  __device__ __forceinline__ explicit Fp8Operand(const fp8_frag &f) : v(f) {}
  Fp8Operand() = default;
};

// c[t] = a b[t] over the group's 128 channels
template <int TB>
__device__ __forceinline__ void group_sums(const Fp8Operand<false> &a,
                                           const Fp8Operand<false> (&b)[TB], glm_f32x4 (&c)[TB]) {
#pragma unroll
  for (int t = 0; t < TB; ++t) c[t] = glm_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < TB; ++t)
      c[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b[t].v[i], c[t], 0, 0, 0);
}
template <int TB>
__device__ __forceinline__ void group_sums(const Fp8Operand<true> &a,
                                           const Fp8Operand<true> (&b)[TB], glm_f32x4 (&c)[TB]) {
#pragma unroll
  for (int t = 0; t < TB; ++t)  // (scale operands of zero: the unscaled instruction)
    c[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
        a.v, b[t].v, glm_f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// 16 codes at k of a row, zeros behind its end (K % 16 == 0).
__device__ __forceinline__ glm_u32x4 codes16(const uint8_t *row, int k, int K) {
  return k < K ? *reinterpret_cast<const glm_u32x4 *>(row + k) : glm_u32x4{0, 0, 0, 0};
}

// silu(min(g, limit)) * clip(u, limit) in f32; NaN passes through the clamps.
__device__ __forceinline__ float gated(float g, float u, float limit) {
  if (limit > 0.f) {
    g = __builtin_elementwise_minimum(g, limit);
    u = __builtin_elementwise_maximum(__builtin_elementwise_minimum(u, limit), -limit);
  }
  return g / (1.0f + expf(-g)) * u;
}

// ---------------------------------------------------------------------------
// Few tokens: the weights are streamed once for up to 16 TB tokens.  A
// workgroup has 16 weight rows (of each projection); its eight waves take the
// groups of K in turn and add up their f32 results in LDS.  ROWS says what x
// holds: bf16 and f32 rows are quantised in registers, where the four lanes of
// a token hold its group.
// ---------------------------------------------------------------------------
template <int ROWS>
struct StreamRow {
  fp8_frag b;
  float scale;
  __device__ __forceinline__ void load(const Fp8Args &a, int t, int g, int q) {
    const int k = g * kFp8Group + 32 * q;
    if constexpr (ROWS == GLM_ROWS_FP8) {
      const uint8_t *row = (const uint8_t *)a.x + (long long)t * a.K;
      b = join16(codes16(row, k, a.K), codes16(row, k + 16, a.K));
      scale = a.xs[(long long)t * a.groups + g];
    } else {
      float v[32];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float (&p)[8] = *reinterpret_cast<float (*)[8]>(v + 8 * i);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = 0.f;
        if (k + 8 * i < a.K) load8<ROWS == GLM_ROWS_F32>(a.x, (long long)t * a.K + k + 8 * i, p);
      }
      float m = abs_max(v);
      m = fmaxf(m, __shfl_xor(m, 16, kWave));
      m = fmaxf(m, __shfl_xor(m, 32, kWave));
      if (__builtin_expect(__any(isinf(m)), 0)) {
        m = finite_abs_max(v);
        m = fmaxf(m, __shfl_xor(m, 16, kWave));
        m = fmaxf(m, __shfl_xor(m, 32, kWave));
      }
      m = fmaxf(m, kFp8Tiny);
      const float up = kFp8Max / m;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        b[j] = (int)fp8_codes4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], up);
      scale = m / kFp8Max;
    }
  }
};

template <int NPROJ, int TB, int ROWS>
__global__ __launch_bounds__(kStreamThreads) void fp8_stream_kernel(Fp8Args a) {
  __shared__ glm_f32x4 part[kStreamWaves][NPROJ * TB][kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int n0 = 16 * blockIdx.x, t0 = 16 * TB * blockIdx.y;
  const uint8_t *wrow[NPROJ];
  const float *wscale[NPROJ];
#pragma unroll
  for (int p = 0; p < NPROJ; ++p) {
    wrow[p] = a.w[p] + (long long)min(n0 + r, a.N - 1) * a.K;
    wscale[p] = a.ws[p] + (long long)(n0 / kFp8Group) * a.groups;
  }
  glm_f32x4 acc[NPROJ][TB];
#pragma unroll
  for (int p = 0; p < NPROJ; ++p)
#pragma unroll
    for (int b = 0; b < TB; ++b) acc[p][b] = glm_f32x4{0.f, 0.f, 0.f, 0.f};

  for (int g0 = wave; g0 < a.groups; g0 += kStreamWaves * kStreamAhead) {
    glm_u32x4 wv[kStreamAhead][NPROJ][2];
    float sw[kStreamAhead][NPROJ];
#pragma unroll
    for (int i = 0; i < kStreamAhead; ++i) {
      const int g = min(g0 + i * kStreamWaves, a.groups - 1), k = g * kFp8Group + 32 * q;
#pragma unroll
      for (int p = 0; p < NPROJ; ++p) {
        wv[i][p][0] = codes16(wrow[p], k, a.K);
        wv[i][p][1] = codes16(wrow[p], k + 16, a.K);
        sw[i][p] = wscale[p][g];
      }
    }
#pragma unroll
    for (int i = 0; i < kStreamAhead; ++i) {
      const int g = g0 + i * kStreamWaves;
      if (g >= a.groups) break;
      Fp8Operand<false> x[TB];
      float sx[TB];
#pragma unroll
      for (int b = 0; b < TB; ++b) {
        StreamRow<ROWS> row;
        row.load(a, min(t0 + 16 * b + r, a.T - 1), g, q);
        x[b] = Fp8Operand<false>(row.b);
        sx[b] = row.scale;
      }
#pragma unroll
      for (int p = 0; p < NPROJ; ++p) {
        glm_f32x4 c[TB];
        group_sums(Fp8Operand<false>(join16(wv[i][p][0], wv[i][p][1])), x, c);
#pragma unroll
        for (int b = 0; b < TB; ++b) {
          const float s = sx[b] * sw[i][p];
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[p][b][j] += c[b][j] * s;
        }
      }
    }
  }
#pragma unroll
  for (int p = 0; p < NPROJ; ++p)
#pragma unroll
    for (int b = 0; b < TB; ++b) part[wave][p * TB + b][lane] = acc[p][b];
  __syncthreads();
  if (wave >= TB) return;
  const int t = t0 + 16 * wave + r, n = n0 + 4 * q;
  glm_f32x4 sum[NPROJ];
#pragma unroll
  for (int p = 0; p < NPROJ; ++p) {
    sum[p] = part[0][p * TB + wave][lane];
#pragma unroll
    for (int w = 1; w < kStreamWaves; ++w) {
      const glm_f32x4 o = part[w][p * TB + wave][lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[p][j] += o[j];
    }
  }
  if (t >= a.T || n >= a.N) return;
  if constexpr (NPROJ == 2) {
    glm_f32x4 h;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = gated(sum[0][j], sum[1][j], a.limit);
    *reinterpret_cast<glm_f32x4 *>(a.h + (long long)t * a.N + n) = h;  // (N % 16 == 0)
  } else {
    uint16_t *out = a.out + (long long)t * a.N + n;
    if (a.N % 4 == 0) {
      *reinterpret_cast<uint2 *>(out) =
          uint2{f32_to_bf16(sum[0][0]) | (f32_to_bf16(sum[0][1]) << 16),
                f32_to_bf16(sum[0][2]) | (f32_to_bf16(sum[0][3]) << 16)};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < a.N) out[j] = (uint16_t)f32_to_bf16(sum[0][j]);
    }
  }
}

// ---------------------------------------------------------------------------
// Many tokens: a workgroup computes 32 BN weight rows (NPROJ 2: half of them
// from each projection) x 64 BT tokens.  Eight waves, two along the weight rows
// x four along the tokens; a wave holds BN x BT blocks of 16 x 16.  Both
// operands come into LDS a group of K at a time by direct loads of 16-byte
// pieces, a ring of groups deep, with the rows' scales behind them.  Piece p of
// row R lies at p ^ ((R >> 1) & 7): the 16 rows that a quarter of a wave reads
// are then on 16 different pieces of 256 bytes.  Rows past the last and pieces
// past K are out of the buffers' range, which gives zeros.
// ---------------------------------------------------------------------------
constexpr int kTileWN = 2, kTileWT = 4, kTileWaves = kTileWN * kTileWT;
constexpr int kTileThreads = 64 * kTileWaves;
constexpr int kTileXcds = 8;
constexpr int kTileKB = 156;  // LDS of a workgroup
constexpr uint32_t kOutOfRange = 0x40000000u;  // past any tile's operand (256 rows of 2^20 bytes)

struct Fp8TileArgs {
  Fp8Args p;
  uint8_t *codes;   // gated and quantised
  float *scales;
  int row_tiles, tok_tiles;
  int rows_outer;   // consecutive items walk the tokens of one row tile, else the reverse
};

template <int BN, int BT>
struct Fp8Tile {
  static constexpr int kRows = 16 * BN * kTileWN, kTok = 16 * BT * kTileWT;
  static constexpr int kX = kTok * kFp8Group, kW = kRows * kFp8Group, kS = kTileThreads * 4;
  static constexpr int kStage = kX + kW + kS;
  static constexpr int kXLoads = kX / (1024 * kTileWaves), kWLoads = kW / (1024 * kTileWaves);
  static constexpr int kLoads = kXLoads + kWLoads + 1;
  static constexpr int kFit = kTileKB * 1024 / kStage;
  static constexpr int kStages = kFit < 6 ? kFit : 6;
  static constexpr int kBytes = kStages * kStage;
  static_assert(kX % (1024 * kTileWaves) == 0 && kW % (1024 * kTileWaves) == 0, "whole loads");
  static_assert(kTok <= kTileThreads, "one load of scales");
  static_assert(kStages >= 2, "a ring");
  __device__ static int swz(int row) { return (row >> 1) & 7; }
};

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

__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

enum { kOutBf16, kOutF32, kOutCodes };

template <int NPROJ, bool FAST, int BN, int BT, int OUT>
__global__ __launch_bounds__(kTileThreads) void fp8_tile_kernel(Fp8TileArgs a) {
  using L = Fp8Tile<BN, BT>;
  constexpr int kS = L::kStages;
  constexpr int kFeat = L::kRows / NPROJ;  // features of a workgroup
  constexpr int HB = BN / NPROJ;           // 16-row blocks of a wave and projection
  static_assert(OUT != kOutCodes || kFeat == kFp8Group, "a group of features");
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  // workgroups are dealt to the XCDs in turn: each takes a contiguous share of the items
  const int items = a.row_tiles * a.tok_tiles;
  const int per_xcd = (items + kTileXcds - 1) / kTileXcds;
  const int on_xcd = (int)blockIdx.x / kTileXcds;
  const int item = ((int)blockIdx.x % kTileXcds) * per_xcd + on_xcd;
  if (on_xcd >= per_xcd || item >= items) return;
  const int rt = a.rows_outer ? item / a.tok_tiles : item % a.row_tiles;
  const int tt = a.rows_outer ? item % a.tok_tiles : item / a.row_tiles;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int wn = wave % kTileWN, wt = wave / kTileWN;
  const int K = a.p.K, N = a.p.N, T = a.p.T, groups = a.p.groups;
  const int f0 = rt * kFeat, t0 = tt * L::kTok;
  const int toks = min(T - t0, L::kTok), feats = min(N - f0, kFeat);

  const __amdgpu_buffer_rsrc_t xres =
      make_rsrc((const uint8_t *)a.p.x + (long long)t0 * K, (uint32_t)toks * (uint32_t)K);
  const __amdgpu_buffer_rsrc_t sres =
      make_rsrc(a.p.xs + (long long)t0 * groups, (uint32_t)toks * (uint32_t)groups * 4u);
  __amdgpu_buffer_rsrc_t wres[NPROJ];
#pragma unroll
  for (int p = 0; p < NPROJ; ++p)
    wres[p] = make_rsrc(a.p.w[p] + (long long)f0 * K, (uint32_t)feats * (uint32_t)K);
  // load j of wave w fills the (kTileWaves j + w)-th 1 KB of the tokens, then of the weight rows
  uint32_t xoff[L::kXLoads], woff[L::kWLoads];
#pragma unroll
  for (int j = 0; j < L::kXLoads; ++j) {
    const int slot = (j * kTileWaves + wave) * 64 + lane, row = slot / 8;
    xoff[j] = (uint32_t)row * (uint32_t)K + 16 * ((slot % 8) ^ L::swz(row));
  }
#pragma unroll
  for (int j = 0; j < L::kWLoads; ++j) {
    const int slot = (j * kTileWaves + wave) * 64 + lane, row = slot / 8;
    woff[j] = (uint32_t)(row % kFeat) * (uint32_t)K + 16 * ((slot % 8) ^ L::swz(row));
  }
  const uint32_t soff = (uint32_t)((wave * 64 + lane) % L::kTok) * (uint32_t)groups * 4u;
  const int tail = K % kFp8Group;  // codes of a last group that is not whole
  auto issue = [&](int c, int stage) {
    uint8_t *base = smem + stage * L::kStage;
    const bool cut = tail != 0 && c == groups - 1;
#pragma unroll
    for (int j = 0; j < L::kXLoads; ++j) {
      const int slot = (j * kTileWaves + wave) * 64 + lane;
      const bool in = !cut || 16 * ((slot % 8) ^ L::swz(slot / 8)) < tail;
      buf16_to_lds(xres, base + (j * kTileWaves + wave) * 1024, in ? xoff[j] : kOutOfRange,
                   (uint32_t)c * kFp8Group);
    }
#pragma unroll
    for (int j = 0; j < L::kWLoads; ++j) {
      const int slot = (j * kTileWaves + wave) * 64 + lane;
      const bool in = !cut || 16 * ((slot % 8) ^ L::swz(slot / 8)) < tail;
      // (a 1 KB block of rows lies in one projection)
      const int p = NPROJ == 2 && (j * kTileWaves + wave) * 8 >= kFeat;
      buf16_to_lds(NPROJ == 2 && p ? wres[NPROJ - 1] : wres[0],
                   base + L::kX + (j * kTileWaves + wave) * 1024, in ? woff[j] : kOutOfRange,
                   (uint32_t)c * kFp8Group);
    }
    buf4_to_lds(sres, base + L::kX + L::kW + wave * 256, soff, (uint32_t)c * 4);
  };

  // the block scales of the wave's features (its rows lie in one block of 128)
  const float *sw[NPROJ];
#pragma unroll
  for (int p = 0; p < NPROJ; ++p)
    sw[p] = a.p.ws[p] + (long long)min((f0 + wn * HB * 16) / kFp8Group, (N - 1) / kFp8Group) * groups;

  glm_f32x4 acc[BN][BT];
#pragma unroll
  for (int b = 0; b < BN; ++b)
#pragma unroll
    for (int t = 0; t < BT; ++t) acc[b][t] = glm_f32x4{0.f, 0.f, 0.f, 0.f};

  auto frag = [&](const uint8_t *row0, int row) {
    const uint8_t *p = row0 + row * kFp8Group;
    return join16(*reinterpret_cast<const glm_u32x4 *>(p + 16 * ((2 * q) ^ L::swz(row))),
                  *reinterpret_cast<const glm_u32x4 *>(p + 16 * ((2 * q + 1) ^ L::swz(row))));
  };
  auto compute = [&](int stage, const float (&ws)[NPROJ]) {
    const uint8_t *base = smem + stage * L::kStage;
    const float *sx = reinterpret_cast<const float *>(base + L::kX + L::kW) + wt * BT * 16 + r;
    Fp8Operand<FAST> x[BT];
    float s[NPROJ][BT];
#pragma unroll
    for (int t = 0; t < BT; ++t) {
      x[t] = Fp8Operand<FAST>(frag(base, (wt * BT + t) * 16 + r));
#pragma unroll
      for (int p = 0; p < NPROJ; ++p) s[p][t] = sx[16 * t] * ws[p];
    }
#pragma unroll
    for (int b = 0; b < BN; ++b) {
      const int row = (b / HB) * kFeat + wn * HB * 16 + (b % HB) * 16 + r;
      glm_f32x4 c[BT];
      group_sums(Fp8Operand<FAST>(frag(base + L::kX, row)), x, c);
#pragma unroll
      for (int t = 0; t < BT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[b][t][j] += c[t][j] * s[b / HB][t];
    }
  };
  // The loads of the next kS - 1 groups are in flight while one is multiplied.
  // The barrier of group c also says that every wave is done with group c - 1,
  // whose stage the loads of group c + kS - 1 overwrite.
#pragma unroll
  for (int c = 0; c < kS - 1; ++c)
    if (c < groups) issue(c, c);
  int stage = 0;
  for (int c = 0; c < groups; ++c) {
    float ws[NPROJ];
#pragma unroll
    for (int p = 0; p < NPROJ; ++p) ws[p] = sw[p][c];
    wait_groups_ahead<kS - 2, L::kLoads>(min(kS - 2, groups - 1 - c));
    ring_barrier();
    if (c + kS - 1 < groups) issue(c + kS - 1, stage == 0 ? kS - 1 : stage - 1);
    compute(stage, ws);
    stage = stage + 1 == kS ? 0 : stage + 1;
  }

  const int fw = f0 + wn * HB * 16, tw = t0 + wt * BT * 16;  // the wave's first feature and token
  if constexpr (OUT == kOutBf16) {
    if (N % 8 != 0) {  // rows of no 16-byte pieces: element by element
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
    static_assert(kTileWaves * 16 * kStride <= L::kBytes, "output staging");
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
    if constexpr (OUT == kOutF32) {
#pragma unroll
      for (int b = 0; b < HB; ++b)
#pragma unroll
        for (int t = 0; t < BT; ++t) {
          const int tok = tw + 16 * t + r, n = fw + 16 * b + 4 * q;
          if (tok < T && n < N)  // (N % 16 == 0)
            *reinterpret_cast<glm_f32x4 *>(a.p.h + (long long)tok * N + n) = acc[b][t];
        }
    } else {
      // a token's largest finite magnitude over the 128 features: the lane's 4 HB, the four lanes of
      // the token, the waves along the features
      ring_barrier();
      float *red = reinterpret_cast<float *>(smem);  // [kTileWN][kTok]
      uint8_t *st = smem + kTileWN * L::kTok * 4;    // [kTok][128 codes, 16 bytes of padding]
      constexpr int kStride = kFp8Group + 16;
      static_assert(kTileWN * L::kTok * 4 + L::kTok * kStride <= L::kBytes, "output staging");
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
        for (int w = 0; w < kTileWN; ++w) m = fmaxf(m, red[w * L::kTok + tok]);
        const float up = kFp8Max / m;
#pragma unroll
        for (int b = 0; b < HB; ++b)
          *reinterpret_cast<uint32_t *>(st + tok * kStride + wn * HB * 16 + 16 * b + 4 * q) =
              fp8_codes4(acc[b][t][0], acc[b][t][1], acc[b][t][2], acc[b][t][3], up);
        if (wn == 0 && q == 0 && t0 + tok < T)
          a.scales[(long long)(t0 + tok) * fp8_groups(N) + f0 / kFp8Group] = m / kFp8Max;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < L::kTok * 8 / kTileThreads; ++i) {
        const int slot = i * kTileThreads + tid, tok = slot / 8, n = f0 + 16 * (slot % 8);
        if (t0 + tok < T && n < N)
          *reinterpret_cast<glm_u32x4 *>(a.codes + (long long)(t0 + tok) * N + n) =
              *reinterpret_cast<const glm_u32x4 *>(st + tok * kStride + 16 * (slot % 8));
      }
    }
  }
}

}  // namespace glm

using namespace glm;

static size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

template <int NPROJ, int ROWS>
static int launch_stream(hipStream_t stream, const Fp8Args &a) {
  const unsigned n = (unsigned)((a.N + 15) / 16);
  if (a.T <= 16) {
    hipLaunchKernelGGL((fp8_stream_kernel<NPROJ, 1, ROWS>), dim3(n), dim3(kStreamThreads), 0, stream, a);
  } else if constexpr (ROWS == GLM_ROWS_FP8) {
    if (a.T <= 32)
      hipLaunchKernelGGL((fp8_stream_kernel<NPROJ, 2, ROWS>), dim3(n), dim3(kStreamThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((fp8_stream_kernel<NPROJ, 4, ROWS>), dim3(n, (unsigned)((a.T + 63) / 64)),
                         dim3(kStreamThreads), 0, stream, a);
  }
  GLM_LAUNCH_CHECK("fp8_stream_kernel");
  return GLM_OK;
}

// Rows as the kernels take them: up to kFusedTokens as they are, more of them
// quantised into the workspace first.
static int rows_for(hipStream_t stream, Fp8Args &a, int &type, uint8_t *&ws) {
  if (type == GLM_ROWS_FP8 || a.T <= kFusedTokens) return GLM_OK;
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
static size_t rows_bytes(int T, int K, int type) {
  if (type == GLM_ROWS_FP8 || T <= kFusedTokens) return 0;
  return round256((size_t)T * K) + round256((size_t)T * fp8_groups(K) * 4);
}

template <int NPROJ, bool FAST, int BN, int BT, int OUT>
static int launch_tile(hipStream_t stream, Fp8TileArgs a) {
  using L = Fp8Tile<BN, BT>;
  constexpr int feat = L::kRows / NPROJ;
  a.row_tiles = (a.p.N + feat - 1) / feat;
  a.tok_tiles = (a.p.T + L::kTok - 1) / L::kTok;
  a.rows_outer = NPROJ * a.p.N >= a.p.T;
  const int items = a.row_tiles * a.tok_tiles;
  hipLaunchKernelGGL((fp8_tile_kernel<NPROJ, FAST, BN, BT, OUT>),
                     dim3((unsigned)((items + kTileXcds - 1) / kTileXcds * kTileXcds)),
                     dim3(kTileThreads), (size_t)L::kBytes, stream, a);
  GLM_LAUNCH_CHECK("fp8_tile_kernel");
  return GLM_OK;
}

constexpr int kStreamTokens = 64;  // up to so many the weights are streamed

static int linear_product(hipStream_t stream, const Fp8Args &a, int type) {
  if (type == GLM_ROWS_BF16) return launch_stream<1, GLM_ROWS_BF16>(stream, a);
  if (type == GLM_ROWS_F32) return launch_stream<1, GLM_ROWS_F32>(stream, a);
  if (a.T <= kStreamTokens) return launch_stream<1, GLM_ROWS_FP8>(stream, a);
  const Fp8TileArgs t{a, nullptr, nullptr, 0, 0, 0};
  if (a.T <= 512) return launch_tile<1, true, 4, 1, kOutBf16>(stream, t);
  return launch_tile<1, true, 8, 4, kOutBf16>(stream, t);
}

static int gated_product(hipStream_t stream, const Fp8Args &a, int type, uint8_t *codes,
                         float *scales) {
  if (a.T > kStreamTokens) {
    const Fp8TileArgs t{a, codes, scales, 0, 0, 0};
    if (a.T <= 1024) return launch_tile<2, false, 8, 1, kOutCodes>(stream, t);
    return launch_tile<2, false, 8, 4, kOutCodes>(stream, t);
  }
  const int rc = type == GLM_ROWS_BF16  ? launch_stream<2, GLM_ROWS_BF16>(stream, a)
                 : type == GLM_ROWS_F32 ? launch_stream<2, GLM_ROWS_F32>(stream, a)
                                        : launch_stream<2, GLM_ROWS_FP8>(stream, a);
  return rc ? rc : glm_fp8_quantize_rows(stream, a.h, GLM_ROWS_F32, a.T, a.N, codes, scales);
}

static bool sizes_fit(int T, int K, int N) {
  return T >= 0 && K >= 16 && N >= 1 && K % 16 == 0 && K <= 1 << 20 && N <= 1 << 20 && T <= 1 << 21;
}

static int check_product(const char *name, const void *x, int x_type, const float *x_scales, int T,
                         int K, int N, const void *workspace, size_t need, size_t bytes) {
  GLM_REQUIRE(T >= 0 && K >= 1 && N >= 1 && x_type >= GLM_ROWS_BF16 && x_type <= GLM_ROWS_FP8,
              GLM_ERR_INVALID_ARGUMENT, "%s: invalid sizes or row type", name);
  GLM_REQUIRE(sizes_fit(T, K, N), GLM_ERR_UNSUPPORTED_SHAPE,
              "%s: %d rows of %d channels (a multiple of 16) into %d: up to 2^21 rows and 2^20 "
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
  return rows_bytes(T, K, x_type) + (gated && T <= kStreamTokens ? round256((size_t)T * N * 4) : 0);
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
  Fp8Args a{x, x_scales, {weight, nullptr}, {scales, nullptr}, T, K, N, fp8_groups(K), 0.f, out,
            nullptr};
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
            nullptr, nullptr};
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  hipStream_t s = (hipStream_t)stream;
  int rc = rows_for(s, a, x_type, ws);
  if (rc) return rc;
  a.h = reinterpret_cast<float *>(ws);
  return gated_product(s, a, x_type, codes, scales);
}
