// Which bin of sampling's weights a logit falls into (plain C++: the kernels and the CPU's tests share it).
#pragma once

#include <cmath>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define FG_BINS_BOTH __host__ __device__ __forceinline__
#else
#define FG_BINS_BOTH inline
#endif

namespace fg {

constexpr int kBins = 1024;
constexpr float kPerUnit = 32.0f;  // bins a unit of z

// -z in bins of a logit: 32 (largest - logit) / temperature, at least 0. All kernels go by `bins_of` and
// `weight_of`, so a token's bin and weight are the same in each. (A largest logit of +inf is taken as
// 1e300: the infinite ones are above it, and all others weigh nothing.) It may be infinite, or past an int's
// range: the last bin's end it, before it is a whole number.
FG_BINS_BOTH double bins_of(float x, double top, double scale) { return fmax((top - double(x)) * scale, 0.0); }
FG_BINS_BOTH int bin_of(double t) { return int(fmin(t, double(kBins - 1))); }
FG_BINS_BOTH double top_of(float x) { return x == INFINITY ? 1e300 : double(x); }

}  // namespace fg
