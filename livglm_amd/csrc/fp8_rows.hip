// The quantisers of the block-scaled 8-bit format (fp8_rows.h): rows, weights,
// and the residual's addition with the RMS norm in front of the rows'.  The
// reference keeps its resident weights in group-32 MXFP8 (layers.py:72-99) and
// multiplies bf16 rows; here both sides of a product are E4M3.
#include "fp8_rows.h"
#include "lds_stage.h"

namespace glm {

constexpr int kRowsThreads = 256;

// ---------------------------------------------------------------------------
// Rows: one pass over the bytes, sixteen lanes a group with eight channels each,
// so that a lane loads 16 bytes of bf16 and the maximum is four steps over lanes.
// Bound by bytes: 7777 bf16 rows of 4096 (96.6 MB) 16.4 us, 5.9 TB/s (a large copy
// has 4.9; the rest is the memory-side cache's); 64 rows 2.5, a launch.
// ---------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(kRowsThreads) void fp8_quantize_rows_kernel(
    const void *x, int K, int groups, long long total, uint8_t *codes, float *scales) {
  const int lane = threadIdx.x & 15;
  const long long step = (long long)gridDim.x * (kRowsThreads / 16);
  for (long long i = (long long)blockIdx.x * (kRowsThreads / 16) + (threadIdx.x >> 4); i < total;
       i += step) {
    const long long t = i / groups;
    const int k = (int)(i - t * groups) * kFp8Group + 8 * lane;
    float v[8] = {};
    if (k < K) load8<F32>(x, t * K + k, v);
    const float amax = group_amax(v);
    const float up = kFp8Max / amax;
    if (k < K)
      *reinterpret_cast<uint2 *>(codes + t * K + k) =
          uint2{fp8_codes4(v[0], v[1], v[2], v[3], up), fp8_codes4(v[4], v[5], v[6], v[7], up)};
    if (lane == 0) scales[i] = amax / kFp8Max;
  }
}

// ---------------------------------------------------------------------------
// Weights: a workgroup holds one 128 x 128 block, 64 values a thread, so that the
// block is read once.  Done once, when a weight is loaded.  Bound by bytes: 8192 x
// 8192 (201 MB) 43.0 us, 4.7 TB/s; 4096 x 4096 11.9, 4.2; 768 x 2048, 96 workgroups, 4.8.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kRowsThreads) void fp8_quantize_weight_kernel(
    const uint16_t *w, int N, int K, uint8_t *codes, float *scales) {
  __shared__ float red[kRowsThreads / 64];
  const int k = blockIdx.x * kFp8Group + 8 * (threadIdx.x & 15);
  const int n0 = blockIdx.y * kFp8Group + (threadIdx.x >> 4);
  float v[64];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float (&r)[8] = *reinterpret_cast<float (*)[8]>(v + 8 * i);
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = 0.f;
    if (k < K && n0 + 16 * i < N) load8<false>(w, (long long)(n0 + 16 * i) * K + k, r);
  }
  float m = finite_abs_max(v);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = kFp8Tiny;
#pragma unroll
  for (int i = 0; i < kRowsThreads / 64; ++i) m = fmaxf(m, red[i]);
  const float up = kFp8Max / m;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k < K && n0 + 16 * i < N)
      *reinterpret_cast<uint2 *>(codes + (long long)(n0 + 16 * i) * K + k) =
          uint2{fp8_codes4(v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3], up),
                fp8_codes4(v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7], up)};
  if (threadIdx.x == 0) scales[(long long)blockIdx.y * gridDim.x + blockIdx.x] = m / kFp8Max;
}

template <bool F32>
__device__ __forceinline__ void values8(const glm_u32x4 *raw, float v[8]) {
  if constexpr (F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(raw[j / 4][j % 4]);
  } else {
    unpack8(raw[0], v);
  }
}

// ---------------------------------------------------------------------------
// h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, y quantised.  A
// workgroup holds its row in registers, 8 STEPS channels a thread, so that x and
// the residual are read once; h is not rounded before the norm.  As many threads
// as a row needs with one step each, as far as a workgroup goes.  Bound by bytes:
// 8191 bf16 rows of 4096 (236 MB) 41 us, 5.8 TB/s; 1500 f32 rows of 2048 (40 MB) 8.7,
// 4.6 TB/s; one row of 4096 3.4, a launch, a trip to memory and the sum.
// ---------------------------------------------------------------------------
struct NormArgs {
  const void *x, *residual;
  const float *weight;
  void *residual_out;
  uint8_t *codes;
  float *scales;
  int d, groups;
  float eps;
};

template <int THREADS, int STEPS, bool XF32, bool RF32>
__global__ __launch_bounds__(THREADS) void add_rms_norm_fp8_kernel(NormArgs a) {
  __shared__ float red[THREADS / 64];
  const long long row = (long long)blockIdx.x * a.d;
  constexpr int kX = XF32 ? 4 : 2, kR = RF32 ? 4 : 2;  // bytes
  // What a row needs is asked for at once and without branches, past d and of absent
  // operands zeros from outside the buffers' range: a wait behind each load, and the
  // weight's behind the sum, cost one row of 4096 0.2 us and 8191 of them 1.
  const auto of = [&](const void *p, int bytes) {
    return make_rsrc((const uint8_t *)p + (p ? row * bytes : 0), p ? (uint32_t)(a.d * bytes) : 0u);
  };
  const __amdgpu_buffer_rsrc_t xres = of(a.x, kX), rres = of(a.residual, kR),
                               wres = make_rsrc(a.weight, a.weight ? (uint32_t)a.d * 4 : 0u);
  const auto get = [](__amdgpu_buffer_rsrc_t res, int byte) {
    return __builtin_amdgcn_raw_buffer_load_b128(res, byte, 0, 0);
  };
  glm_u32x4 x[STEPS][kX / 2], r[STEPS][kR / 2], w[STEPS][2];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int c = 8 * (i * THREADS + threadIdx.x);
#pragma unroll
    for (int j = 0; j < kX / 2; ++j) x[i][j] = get(xres, c * kX + 16 * j);
#pragma unroll
    for (int j = 0; j < kR / 2; ++j) r[i][j] = get(rres, c * kR + 16 * j);
#pragma unroll
    for (int j = 0; j < 2; ++j) w[i][j] = get(wres, c * 4 + 16 * j);
  }
  float h[STEPS][8];
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int c = 8 * (i * THREADS + threadIdx.x);
    float add[8];
    values8<XF32>(x[i], h[i]);
    values8<RF32>(r[i], add);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[i][j] = a.residual ? h[i][j] + add[j] : h[i][j];
    if (a.residual_out && c < a.d) {
      if constexpr (RF32) {
        glm_f32x4 *o = reinterpret_cast<glm_f32x4 *>((float *)a.residual_out + row + c);
        o[0] = glm_f32x4{h[i][0], h[i][1], h[i][2], h[i][3]};
        o[1] = glm_f32x4{h[i][4], h[i][5], h[i][6], h[i][7]};
      } else {
        glm_u32x4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[j] = f32_to_bf16(h[i][2 * j]) | (f32_to_bf16(h[i][2 * j + 1]) << 16);
        *reinterpret_cast<glm_u32x4 *>((uint16_t *)a.residual_out + row + c) = o;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sq += h[i][j] * h[i][j];
  }
  sq = wave_sum(sq);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sq;
  __syncthreads();
  sq = 0.f;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) sq += red[i];
  const float inv = 1.0f / sqrtf(sq / (float)a.d + a.eps);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int c = 8 * (i * THREADS + threadIdx.x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[i][j] *= inv;
      if (a.weight) h[i][j] *= __uint_as_float(w[i][j / 4][j % 4]);
    }
    const float amax = group_amax(h[i]);  // (all lanes of the group are here)
    const float up = kFp8Max / amax;
    if (c < a.d)
      *reinterpret_cast<uint2 *>(a.codes + row + c) =
          uint2{fp8_codes4(h[i][0], h[i][1], h[i][2], h[i][3], up),
                fp8_codes4(h[i][4], h[i][5], h[i][6], h[i][7], up)};
    if ((threadIdx.x & 15) == 0 && c < a.d)
      a.scales[(long long)blockIdx.x * a.groups + c / kFp8Group] = amax / kFp8Max;
  }
}

}  // namespace glm

using namespace glm;

static bool row_type(int type) { return type == GLM_ROWS_BF16 || type == GLM_ROWS_F32; }

extern "C" int glm_fp8_quantize_rows(void *stream, const void *x, int x_type, int T, int K,
                                     uint8_t *codes, float *scales) {
  glm::clear_error();
  GLM_REQUIRE(T >= 0 && K >= 1 && row_type(x_type), GLM_ERR_INVALID_ARGUMENT,
              "fp8_quantize_rows: invalid sizes or row type");
  GLM_REQUIRE(K % 8 == 0 && K <= INT32_MAX - (kFp8Group - 1), GLM_ERR_UNSUPPORTED_SHAPE,
              "fp8_quantize_rows: K = %d (a multiple of 8, whole groups of 128 below 2^31)", K);
  GLM_REQUIRE(x && codes && scales, GLM_ERR_INVALID_ARGUMENT, "fp8_quantize_rows: null pointer");
  GLM_REQUIRE(glm_aligned16({x, codes, scales}), GLM_ERR_INVALID_ARGUMENT,
              "fp8_quantize_rows: buffers must be 16-byte aligned");
  if (T == 0) return GLM_OK;
  const int groups = fp8_groups(K);
  const long long total = (long long)T * groups;
  const long long blocks = (total + kRowsThreads / 16 - 1) / (kRowsThreads / 16);
  const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
  if (x_type == GLM_ROWS_F32)
    hipLaunchKernelGGL(fp8_quantize_rows_kernel<true>, grid, dim3(kRowsThreads), 0,
                       (hipStream_t)stream, x, K, groups, total, codes, scales);
  else
    hipLaunchKernelGGL(fp8_quantize_rows_kernel<false>, grid, dim3(kRowsThreads), 0,
                       (hipStream_t)stream, x, K, groups, total, codes, scales);
  GLM_LAUNCH_CHECK("fp8_quantize_rows_kernel");
  return GLM_OK;
}

extern "C" int glm_fp8_quantize_weight(void *stream, const uint16_t *w, int N, int K,
                                       uint8_t *codes, float *scales) {
  glm::clear_error();
  GLM_REQUIRE(N >= 1 && K >= 1, GLM_ERR_INVALID_ARGUMENT, "fp8_quantize_weight: invalid sizes");
  GLM_REQUIRE(K % 8 == 0 && N <= 1 << 20 && K <= 1 << 20, GLM_ERR_UNSUPPORTED_SHAPE,
              "fp8_quantize_weight: a %d x %d weight (the columns in eights, at most 2^20 of "
              "either)", N, K);
  GLM_REQUIRE(w && codes && scales, GLM_ERR_INVALID_ARGUMENT, "fp8_quantize_weight: null pointer");
  GLM_REQUIRE(glm_aligned16({w, codes, scales}), GLM_ERR_INVALID_ARGUMENT,
              "fp8_quantize_weight: buffers must be 16-byte aligned");
  hipLaunchKernelGGL(fp8_quantize_weight_kernel, dim3(fp8_groups(K), fp8_groups(N)),
                     dim3(kRowsThreads), 0, (hipStream_t)stream, w, N, K, codes, scales);
  GLM_LAUNCH_CHECK("fp8_quantize_weight_kernel");
  return GLM_OK;
}

template <int THREADS, int STEPS>
static void launch_norm(hipStream_t stream, int T, bool xf32, bool rf32, const NormArgs &a) {
  auto kernel = xf32 ? (rf32 ? add_rms_norm_fp8_kernel<THREADS, STEPS, true, true>
                             : add_rms_norm_fp8_kernel<THREADS, STEPS, true, false>)
                     : (rf32 ? add_rms_norm_fp8_kernel<THREADS, STEPS, false, true>
                             : add_rms_norm_fp8_kernel<THREADS, STEPS, false, false>);
  hipLaunchKernelGGL(kernel, dim3(T), dim3(THREADS), 0, stream, a);
}

extern "C" int glm_add_rms_norm_fp8(void *stream, const void *x, int x_type, const void *residual,
                                    int residual_type, int T, int d, const float *weight,
                                    float eps, void *residual_out, uint8_t *codes, float *scales) {
  glm::clear_error();
  GLM_REQUIRE(T >= 0 && d >= 1 && row_type(x_type) && row_type(residual_type) && eps >= 0.f,
              GLM_ERR_INVALID_ARGUMENT, "add_rms_norm_fp8: invalid sizes, row type or eps");
  GLM_REQUIRE(d % 8 == 0 && d <= 32768 && T < 1 << 22, GLM_ERR_UNSUPPORTED_SHAPE,
              "add_rms_norm_fp8: %d rows of d = %d, fewer than 2^22 (a grid has 2^32 threads at "
              "most) of a multiple of 8 up to 32768", T, d);
  GLM_REQUIRE(x && codes && scales, GLM_ERR_INVALID_ARGUMENT, "add_rms_norm_fp8: null pointer");
  GLM_REQUIRE(!residual == !residual_out, GLM_ERR_INVALID_ARGUMENT,
              "add_rms_norm_fp8: residual and residual_out come together");
  GLM_REQUIRE(glm_aligned16({x, residual, weight, residual_out, codes, scales}),
              GLM_ERR_INVALID_ARGUMENT, "add_rms_norm_fp8: buffers must be 16-byte aligned");
  if (T == 0) return GLM_OK;
  const NormArgs a{x, residual, weight, residual_out, codes, scales, d, fp8_groups(d), eps};
  const bool xf = x_type == GLM_ROWS_F32, rf = residual_type == GLM_ROWS_F32;
  hipStream_t s = (hipStream_t)stream;
  // One step a thread where a workgroup can.  bf16 without a weight, us: one row of 2048 by 256 x 1
  // threads and steps 2.9 to 3.1, 128 x 2 3.4; 4096 by 512 x 1 3.1, 256 x 2 3.5; 8192
  // by 1024 x 1 3.5, 256 x 4 5.0; many rows of 2048 23.5 and 24.9; 4096 43.8 and 46.0,
  // 1024 x 1 54.0; 8192 42.8 and 47.9; 16384 by 1024 x 2 44.4, 1024 x 4 45.2.
  if (d <= 2048) launch_norm<256, 1>(s, T, xf, rf, a);
  else if (d <= 4096) launch_norm<512, 1>(s, T, xf, rf, a);
  else if (d <= 8192) launch_norm<1024, 1>(s, T, xf, rf, a);
  else if (d <= 16384) launch_norm<1024, 2>(s, T, xf, rf, a);
  else launch_norm<1024, 4>(s, T, xf, rf, a);
  GLM_LAUNCH_CHECK("add_rms_norm_fp8_kernel");
  return GLM_OK;
}
