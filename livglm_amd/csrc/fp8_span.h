// Which rows and groups the block-scaled tiles' loads may touch, apart from the
// kernel so that a host program can check it.  A buffer load past its
// descriptor's size gives zeros by the lane's offset; how the scalar offset
// enters that check is not relied on: every descriptor has a row at least, which
// is more than any scalar offset here, and no scalar offset passes its row.
#pragma once

#ifdef __HIPCC__
#define GLM_SPAN __host__ __device__ __forceinline__ constexpr
#else
#define GLM_SPAN constexpr
#endif

namespace glm {

// Of a tile's `there` rows (1 or more) those of a load that begins at row `first`.
// One behind them all gets the tile's first row, whose values nothing reads.
struct Fp8Span {
  int first, rows;
};
GLM_SPAN Fp8Span fp8_span(int first, int there) {
  return first < there ? Fp8Span{first, there - first} : Fp8Span{0, 1};
}

// The group of a token's scales that load j of four from group g on brings: past
// the last the last once more.
GLM_SPAN int fp8_scale_group(int g, int j, int groups) {
  return g + j < groups ? g + j : groups - 1;
}

}  // namespace glm
