// Rotary positions (fg_rotary): a step's rows turned by their positions. cache.hip turns keys on their way into the cache.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>
#include <vector>

#include "rotary.h"

namespace fg {
namespace {

// Bounded by memory: 8192 rows of 16 heads of 128, 134 MB, 22.6 us, 5.9 TB/s (four heads' loads on their way at once); by its
// launch and the chain of the row's sequence, its span and the angles for one token, 2.9 us. Pairs that do not come in quads go value by
// value: 8192 rows of 16 heads of 80, 84 MB, 20 values in halves 42 us, 2.0 TB/s, 24 of them 22.
template <bool QUADS>
__global__ __launch_bounds__(256) void rotate_kernel(RotateParams p)
{
    const unsigned units = unsigned(p.b.rows) * unsigned(p.units);
    for (unsigned unit = blockIdx.x * 4 + (threadIdx.x >> 6); unit < units; unit += gridDim.x * 4) rotate_unit<QUADS>(p, unit);
}

}  // namespace

RotateParams rotate_params(const fg_rotary *r, const fg_batch *b, const float *x, size_t x_stride, size_t heads, size_t head_dim,
                           float *out, size_t out_stride)
{
    RotateParams p{};
    p.b = batch_params(b);
    p.r = rotary_params(r);
    p.x = x;
    p.x_stride = x_stride;
    p.out = out;
    p.out_stride = out_stride;
    p.heads = int(heads);
    p.head_dim = int(head_dim);
    p.keep = out == x && out_stride == x_stride;
    // the heads of one pass of a wave, and as many passes as leave every SIMD a wave, up to four
    const int half = r->dims / 2, turning = whole_quads(r) ? (r->halves ? half / 4 : r->dims / 4) : half;
    const int rest = (p.head_dim - r->dims) / (whole_quads(r) ? 4 : 1), items = p.keep ? turning : turning + rest;
    int team = 1;
    while (team < items && team < 64) team *= 2;
    const size_t per = size_t(64 / team), passes = (heads + per - 1) / per;
    const size_t many = std::min<size_t>(std::max<size_t>(b->rows * passes / 1024, 1), kAhead);
    p.unit_heads = int(per * many);
    p.units = int((heads + p.unit_heads - 1) / p.unit_heads);
    return p;
}

int launch_rotate(const RotateParams &p, bool quads, hipStream_t s)
{
    const size_t units = size_t(p.b.rows) * p.units;
    if (units > 0xf0000000) return set_error(FG_ERR_SHAPE, "rotary positions: more rows times heads than a launch takes");
    const unsigned grid = unsigned(std::min((units + 3) / 4, kMaxGrid));
    if (quads) rotate_kernel<true><<<grid, 256, 0, s>>>(p);
    else rotate_kernel<false><<<grid, 256, 0, s>>>(p);
    FG_HIP(hipGetLastError());
    return FG_OK;
}

int check_rotary(const fg_rotary *r, int device, size_t head_dim, const std::string &who)
{
    if (!r) return set_error(FG_ERR_ARG, who + ": null rotary positions");
    if (r->device != device)
        return set_error(FG_ERR_ARG, who + ": the rotary positions are on device " + std::to_string(r->device) + ", the current one is " +
                                         std::to_string(device));
    if (size_t(r->dims) > head_dim)
        return set_error(FG_ERR_SHAPE, who + ": " + std::to_string(r->dims) + " values are turned, a head has " + std::to_string(head_dim));
    return FG_OK;
}

bool rows_meet(const float *a, size_t a_stride, size_t a_width, const float *b, size_t b_stride, size_t b_width, size_t rows)
{
    if (!rows || !a || !b) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    if (y >= x + ((rows - 1) * a_stride + a_width) * sizeof(float) || x >= y + ((rows - 1) * b_stride + b_width) * sizeof(float)) return false;
    if (rows == 1) return true;
    if (a_stride != b_stride || !a_stride) return false;
    // b's rows begin so far behind a's (as each begins before the other's end, the rows that meet are there)
    const size_t stride = a_stride * sizeof(float), behind = y >= x ? (y - x) % stride : (stride - (x - y) % stride) % stride;
    return behind < a_width * sizeof(float) || stride - behind < b_width * sizeof(float);
}

int check_rotated(const fg_batch *b, const float *x, size_t x_stride, size_t heads, size_t head_dim, const float *out, size_t out_stride,
                  const std::string &who)
{
    if (!heads || heads > 65536) return set_error(FG_ERR_SHAPE, who + ": 1 to 65536 heads");
    if (b->rows && b->sequences && (!x || !out)) return set_error(FG_ERR_ARG, who + ": null rows or outputs");
    if (b->rows > 1 && out_stride < heads * head_dim) return set_error(FG_ERR_SHAPE, who + ": a row's heads run past the row stride");
    if (out == x && out_stride != x_stride && b->rows > 1)
        return set_error(FG_ERR_SHAPE, who + ": outputs over the rows have the rows' stride");
    if (out != x && rows_meet(out, out_stride, heads * head_dim, x, x_stride, heads * head_dim, b->rows))
        return set_error(FG_ERR_SHAPE, who + ": outputs lie over a part of the rows");
    return FG_OK;
}

}  // namespace fg

using namespace fg;

extern "C" {

int fg_rotary_create(const double *frequencies, size_t dims, int layout, double magnitude, void *stream, fg_rotary **out)
{
    if (!out) return set_error(FG_ERR_ARG, "fg_rotary_create: a null output handle");
    *out = nullptr;
    if (!dims || dims % 2 || dims > 256) return set_error(FG_ERR_SHAPE, "fg_rotary_create: an even number of values, 2 to 256");
    if (layout != FG_ROTARY_HALVES && layout != FG_ROTARY_PAIRS)
        return set_error(FG_ERR_ARG, "fg_rotary_create: the layout must be FG_ROTARY_HALVES or FG_ROTARY_PAIRS");
    if (!frequencies) return set_error(FG_ERR_ARG, "fg_rotary_create: null frequencies");
    if (!(std::fabs(magnitude) <= 1e30)) return set_error(FG_ERR_ARG, "fg_rotary_create: the magnitude must be a number of at most 1e30");
    RotaryPair pairs[128];
    for (size_t i = 0; i < dims / 2; i++) {
        if (!(std::fabs(frequencies[i]) <= 1024.0))
            return set_error(FG_ERR_ARG, "fg_rotary_create: frequencies must be numbers of at most 1024 radians a token");
        pairs[i] = rotary_pair(frequencies[i]);
    }
    int device = 0;
    FG_HIP(hipGetDevice(&device));
    RotaryPair *memory = nullptr;
    hipError_t e = hipMalloc(reinterpret_cast<void **>(&memory), dims / 2 * sizeof(RotaryPair));
    if (e != hipSuccess) return check_hip(e, "fg_rotary_create: hipMalloc");
    const hipStream_t s = as_stream(stream);
    e = hipMemcpyAsync(memory, pairs, dims / 2 * sizeof(RotaryPair), hipMemcpyHostToDevice, s);
    const hipError_t waited = hipStreamSynchronize(s);
    if (e == hipSuccess) e = waited;
    if (e != hipSuccess) {
        (void)hipFree(memory);
        return check_hip(e, "fg_rotary_create");
    }
    fg_rotary *r = new (std::nothrow) fg_rotary{device, int(dims), layout == FG_ROTARY_HALVES, magnitude, memory};
    if (!r) {
        (void)hipFree(memory);
        return set_error(FG_ERR_NOMEM, "fg_rotary_create: host memory");
    }
    *out = r;
    return FG_OK;
}

int fg_rotary_free(fg_rotary *r)
{
    if (!r) return FG_OK;
    (void)hipFree(r->pairs);
    delete r;
    return FG_OK;
}

int fg_rotary_rotate(const fg_rotary *r, const fg_batch *b, const float *x, size_t x_stride, size_t heads, size_t head_dim, float *out,
                     size_t out_stride, void *stream)
{
    const std::string who = "fg_rotary_rotate";
    if (!r) return set_error(FG_ERR_ARG, who + ": null rotary positions");
    int rc = check_batch_arrays(b, false, who.c_str());
    if (rc) return rc;
    int device = 0;
    FG_HIP(hipGetDevice(&device));
    if ((rc = check_rotary(r, device, head_dim, who))) return rc;
    if (!head_dim || head_dim % 4 || head_dim > 256) return set_error(FG_ERR_SHAPE, who + ": heads of whole quads, at most 256 values");
    if ((rc = check_rotated(b, x, x_stride, heads, head_dim, out, out_stride, who))) return rc;
    if (!b->rows || !b->sequences) return FG_OK;
    return launch_rotate(rotate_params(r, b, x, x_stride, heads, head_dim, out, out_stride), whole_quads(r), as_stream(stream));
}

}  // extern "C"
