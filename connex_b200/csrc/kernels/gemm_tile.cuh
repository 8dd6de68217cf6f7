// What the dense GEMM kernels share: the order of their output tiles and the
// gate's activation.
#pragma once

namespace cx {

// Grouped raster: bands of `group` tile-rows, each band walked column by
// column, so the CTAs of one wave share A rows and B columns through L2.
__device__ __forceinline__ void tile_coords(int t, int num_m, int num_n, int group, int& tm, int& tn) {
  const int per_group = group * num_n;
  const int g = t / per_group;
  const int first_m = g * group;
  const int gm = min(num_m - first_m, group);
  const int r = t - g * per_group;
  tm = first_m + r % gm;
  tn = r / gm;
}

__device__ __forceinline__ float silu(float x) { return x / (1.0f + __expf(-x)); }

}  // namespace cx
