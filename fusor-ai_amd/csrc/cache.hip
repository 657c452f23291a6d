// The paged 8-bit cache (fg_cache): its pages, the new tokens' keys and values quantized into them, and
// read back. cache_layout.h says where a level lies; cache_attend.hip reads the pages.
#include <algorithm>
#include <new>

#include "cache.h"

namespace fg {
namespace {

typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));  // four floats at any float's address

struct StoreParams {
    BatchParams b;
    uint8_t *records;
    int pages, kv_heads, head_dim, padded;
    const float *in[2];  // keys, values
    float *out[2];
    size_t stride[2];
};

// The scale of a head whose largest magnitude is amax (`none` where all its levels are 0), and four of its levels as
// stored (level + 128).
__device__ __forceinline__ float head_levels(float amax, const v4f &x, float none, unsigned &packed)
{
    int l0, l1, l2, l3;
    float d;
    if (amax >= 0x1p-52f && amax <= 0x1p66f) {
        d = scale_and_levels(amax, x.x, x.y, x.z, x.w, l0, l1, l2, l3);
    } else {
        d = amax / 127.0f;
        const float by = d == 0.0f ? 1.0f : d;
        l0 = quantize_level(x.x, by);
        l1 = quantize_level(x.y, by);
        l2 = quantize_level(x.z, by);
        l3 = quantize_level(x.w, by);
        d = d == 0.0f ? none : d;
    }
    packed = unsigned(pack4(l0, l1, l2, l3)) ^ 0x80808080u;
    return d;
}

// The largest magnitude of four values, NaN ignored.
__device__ __forceinline__ float amax4(const v4f &x)
{
    return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
}

// ... over 32 aligned lanes, or over all 64
__device__ __forceinline__ float team_max(float v, bool wide)
{
    v = fmaxf(v, __int_as_float(xor1(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(xor2(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(mirror8(__float_as_int(v))));
    v = fmaxf(v, xor8(v));
    const float2 r = row_pair(v);
    v = fmaxf(r.x, r.y);
    if (wide) {
        const float2 h = half_pair(v);
        v = fmaxf(h.x, h.y);
    }
    return v;
}

__device__ __forceinline__ v4f levels_to_values(unsigned packed, float d)
{
    v4f x;
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = float(int((packed >> (8 * j)) & 255u) - 128) * d;
    return x;
}

// Pages of zero levels, with the scales of such.
__global__ __launch_bounds__(256) void cache_clear_kernel(uint8_t *records, size_t dwords, unsigned levels, unsigned record)
{
    for (size_t i = size_t(blockIdx.x) * 256 + threadIdx.x; i < dwords; i += size_t(gridDim.x) * 256) {
        const unsigned at = unsigned(i % record);
        reinterpret_cast<unsigned *>(records)[i] = at < levels ? 0x80808080u : __float_as_uint(at < levels + kPage ? 1.0f : kNoValueScale);
    }
}

// A wave per new row and head, for few new tokens a sequence. Four dimensions a lane; heads of up to 128
// take half a wave for the key and half for the value. A value's levels go to single bytes, 16 apart, of a kilobyte
// that 64 tokens share (cache_layout.h): 64 stores of a byte a token, which is what bounds long runs of tokens,
// and why they take the kernels below. A step's single tokens are bounded by the launch and three loads one
// after the other (the row's sequence, its page, then its values, though their address needs neither): 8 tokens of
// 2 heads of 64 written in 3.3 us, read back in 3.0; 512 of 8 heads of 128 in 7.8 and 5.0.
template <bool WRITE>
__device__ __forceinline__ void store_row(const StoreParams &p, unsigned unit)
{
    const int lane = threadIdx.x & 63;
    const int row = int(unit / unsigned(p.kv_heads)), head = int(unit % unsigned(p.kv_heads));
    const int s = sequence_of_row(p.b, row);
    if (s < 0) return;
    const Span span = sequence_span(p.b, s);
    const int at = row - span.begin;
    if (at < 0 || at >= span.rows) return;
    const int position = span.first + at;
    const int page = position < 0 ? -1 : page_at(p.b.pages + size_t(s) * p.b.max_pages, position / kPage, p.b.max_pages, p.pages);
    if (WRITE && page < 0) return;
    const bool wide = p.padded > 128;
    const int token = position & (kPage - 1), dim = (wide ? lane : lane & 31) * 4;
    uint8_t *record = p.records + (size_t(page < 0 ? 0 : page) * p.kv_heads + head) * record_bytes(p.padded);
    const bool live = dim < p.head_dim;
    for (int i = 0; i < (wide ? 2 : 1); i++) {
        const bool value = wide ? i != 0 : lane >= 32;
        const size_t place = size_t(row) * p.stride[value] + size_t(head) * p.head_dim + dim;
        float *scale = reinterpret_cast<float *>(record + (value ? value_scale_byte(p.padded, token) : key_scale_byte(p.padded, token)));
        if (WRITE) {
            v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
            if (live) x = *reinterpret_cast<const v4f_any *>((value ? p.in[1] : p.in[0]) + place);
            unsigned packed;
            const float d = head_levels(team_max(amax4(x), wide), x, value ? kNoValueScale : 1.0f, packed);
            if (live && !value) *reinterpret_cast<unsigned *>(record + key_byte(p.padded, token, dim)) = packed;
            if (live && value) {
#pragma unroll
                for (int j = 0; j < 4; j++) record[value_byte(p.padded, token, dim + j)] = uint8_t(packed >> (8 * j));
            }
            if (dim == 0) *scale = d;
        } else if (live) {
            v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
            if (page >= 0) {
                unsigned packed = 0;
                if (value) {
#pragma unroll
                    for (int j = 0; j < 4; j++) packed |= unsigned(record[value_byte(p.padded, token, dim + j)]) << (8 * j);
                } else {
                    packed = *reinterpret_cast<const unsigned *>(record + key_byte(p.padded, token, dim));
                }
                x = levels_to_values(packed, *scale);
            }
            *reinterpret_cast<v4f_any *>((value ? p.out[1] : p.out[0]) + place) = x;
        }
    }
}

template <bool WRITE>
__global__ __launch_bounds__(256) void cache_rows_kernel(StoreParams p)
{
    const unsigned units = unsigned(p.b.rows) * unsigned(p.kv_heads);
    for (unsigned unit = blockIdx.x * 4 + (threadIdx.x >> 6); unit < units; unit += gridDim.x * 4) store_row<WRITE>(p, unit);
}

// A workgroup per page that new tokens lie in, head, and keys or values. A thread takes four tokens (an
// aligned run, so one dword of each dimension's values) of four dimensions, heads of up to 128 all of a page
// at once; the levels meet in LDS in the record's order, and whole 16-byte pieces go to the page or come from it.
// Pieces that also hold other tokens' values are written in part. Bounded by memory for long runs, and by one load's
// wait after another for short ones: 3618 tokens of 4 heads of 128 (14.8 MB of f32, 3.8 MB of levels and scales) written
// in 9.2 us, 2.0 TB/s, and read back in 7.5. Keys and values are each a workgroup's, for twice the loads in flight (both in
// one: 16.8 and 9.8).
constexpr int kPageThreads = 512;

template <bool WRITE>
__global__ __launch_bounds__(kPageThreads) void cache_pages_kernel(StoreParams p)
{
    extern __shared__ __align__(16) uint8_t levels[];
    __shared__ float scales[kPage];
    const int tid = threadIdx.x, head = int(blockIdx.y), value = int(blockIdx.z);
    int index;
    const int s = find_unit(p.b.sequences, int(blockIdx.x), &index, [&](int q) {
        const PageRange r = pages_of_new(sequence_span(p.b, q));
        return r.hi - r.lo;
    });
    if (s < 0) return;  // the whole workgroup
    const Span span = sequence_span(p.b, s);
    const int place = pages_of_new(span).lo + index;
    const int page = page_at(p.b.pages + size_t(s) * p.b.max_pages, place, p.b.max_pages, p.pages);
    if (WRITE && page < 0) return;
    // the page's tokens [t0, t1) are new
    const int t0 = max(span.first - place * kPage, 0), t1 = min(span.first + span.rows - place * kPage, kPage);
    // this half of the record, and the byte in it of a token's dimension
    uint8_t *record = p.records + (size_t(page < 0 ? 0 : page) * p.kv_heads + head) * record_bytes(p.padded);
    uint8_t *half = record + (value ? kPage * p.padded : 0);
    float *record_scales = reinterpret_cast<float *>(record + (value ? value_scale_byte(p.padded, 0) : key_scale_byte(p.padded, 0)));
    const bool wide = p.padded > 128;
    const int lanes = wide ? 64 : 32, quads = kPageThreads / lanes, dim = (tid & (lanes - 1)) * 4;
    const bool live = dim < p.head_dim;
    const size_t row0 = size_t(span.begin) + size_t(place * kPage - span.first);  // the row of the page's token 0 (may wrap below 0)
    const int pieces = kPage * p.padded / 16;
    const uint4 none = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
    if (WRITE) {
        if (p.head_dim != p.padded) {  // the padding's levels
            for (int i = tid; i < pieces; i += kPageThreads) reinterpret_cast<uint4 *>(levels)[i] = none;
            __syncthreads();
        }
    } else {
        for (int i = tid; i < pieces; i += kPageThreads) {
            uint4 w = none;  // (a choice between the two would be one of addresses, and `none` in scratch memory)
            if (page >= 0) w = reinterpret_cast<const uint4 *>(half)[i];
            reinterpret_cast<uint4 *>(levels)[i] = w;
        }
        if (tid < kPage) scales[tid] = page < 0 ? 1.0f : record_scales[tid];
        __syncthreads();
    }
    const size_t stride = p.stride[value];
    for (int unit = tid / lanes; unit < kPage / 4; unit += quads) {  // whole teams
        const int t = unit * 4;
        if (t + 4 <= t0 || t >= t1) continue;
        const size_t at = (row0 + t) * stride + size_t(head) * p.head_dim + dim;
        unsigned packed[4];
        if (WRITE) {
            v4f x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                if (live && t + i >= t0 && t + i < t1) x[i] = *reinterpret_cast<const v4f_any *>((value ? p.in[1] : p.in[0]) + at + i * stride);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float d = head_levels(team_max(amax4(x[i]), wide), x[i], value ? kNoValueScale : 1.0f, packed[i]);
                if (dim == 0) scales[t + i] = d;
            }
        }
        if (!value) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                unsigned *word = reinterpret_cast<unsigned *>(levels + key_byte(p.padded, t + i, dim));
                if (WRITE && live) *word = packed[i];
                if (!WRITE && live) packed[i] = *word;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {  // dimension dim + j of the four tokens
                unsigned *word = reinterpret_cast<unsigned *>(levels + value_byte(p.padded, t, dim + j) - kPage * p.padded);
                if (WRITE && live) {
                    unsigned w = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) w |= (packed[i] >> (8 * j) & 255u) << (8 * i);
                    *word = w;
                }
                if (!WRITE) {
                    const unsigned w = live ? *word : 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) packed[i] = (j ? packed[i] : 0) | (w >> (8 * i) & 255u) << (8 * j);
                }
            }
        }
        if (!WRITE && live) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (t + i >= t0 && t + i < t1)
                    *reinterpret_cast<v4f_any *>((value ? p.out[1] : p.out[0]) + at + i * stride) = levels_to_values(packed[i], scales[t + i]);
        }
    }
    if (!WRITE) return;
    __syncthreads();
    for (int i = tid; i < pieces; i += kPageThreads) {
        const int lane = i & 63, block = i >> 6;
        const uint4 w = reinterpret_cast<const uint4 *>(levels)[i];
        uint8_t *at = half + size_t(i) * 16;
        if (!value) {  // one token's
            const int t = block / (p.padded >> 5) * 32 + (lane & 31);
            if (t >= t0 && t < t1) *reinterpret_cast<uint4 *>(at) = w;
            continue;
        }
        const int t = (block & 1) * 32 + (lane >> 5) * 4;  // tokens t + 8 j + i
        if (t >= t0 && t + 28 <= t1) {
            *reinterpret_cast<uint4 *>(at) = w;
            continue;
        }
        const unsigned dword[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int q = t + 8 * j;
            if (q >= t0 && q + 4 <= t1) {
                reinterpret_cast<unsigned *>(at)[j] = dword[j];
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (q + k >= t0 && q + k < t1) at[4 * j + k] = uint8_t(dword[j] >> (8 * k));
            }
        }
    }
    if (tid < kPage && tid >= t0 && tid < t1) record_scales[tid] = scales[tid];
}

template <bool WRITE>
int launch_store(const StoreParams &p, hipStream_t s)
{
    if (p.b.rows == 0 || p.b.sequences == 0) return FG_OK;
    const size_t units = size_t(p.b.rows) * p.kv_heads;
    if (units > 0xf0000000) return set_error(FG_ERR_SHAPE, "the paged cache: more rows times heads than a launch takes");
    // A wave a row and head, or a workgroup a page: the first up to 16 new tokens a sequence or 2048 rows times heads.
    // Microseconds of a write, rows' and pages': 8 heads of 128, 64 sequences of 1 new token 3.8 and 9.5, 16 11.4 and
    // 11.3, 32 17.6 and 13.2, 128 51 and 23; one of 128 3.8 and 4.8; 8 of 32 4.9 and 5.9, of 128 10.5 and 6.5;
    // 512 (each workgroup of a page looks through all of them) of 1 7.8 and 80, 16 52 and 100, 64 190 and 148.
    if (p.b.rows <= 16 * p.b.sequences || units <= 2048) {
        cache_rows_kernel<WRITE><<<unsigned(std::min((units + 3) / 4, kMaxGrid)), 256, 0, s>>>(p);
    } else {
        // a run of n rows lies in at most (n + 62) / 64 + 1 pages
        const size_t runs = size_t(p.b.rows) / kPage + 2 * size_t(std::min(p.b.sequences, p.b.rows));
        cache_pages_kernel<WRITE><<<dim3(unsigned(runs), unsigned(p.kv_heads), 2), kPageThreads, size_t(kPage * p.padded), s>>>(p);
    }
    FG_HIP(hipGetLastError());
    return FG_OK;
}

}  // namespace

int check_batch(const fg_cache *c, const fg_batch *b, const char *who)
{
    const std::string name(who);
    if (!c || !b) return set_error(FG_ERR_ARG, name + ": a null cache or batch");
    if (b->sequences > 65536 || b->rows > (size_t(1) << 24) || b->max_pages > (size_t(1) << 24))
        return set_error(FG_ERR_SHAPE, name + ": at most 65536 sequences, 2^24 rows and 2^24 pages a sequence");
    if (b->sequences && (!b->row_starts || !b->lengths || (b->max_pages && !b->pages)))
        return set_error(FG_ERR_ARG, name + ": a null array of the batch");
    int device = 0;
    FG_HIP(hipGetDevice(&device));
    if (device != c->device)
        return set_error(FG_ERR_ARG, name + ": the cache is on device " + std::to_string(c->device) + ", the current one is " +
                                         std::to_string(device));
    return FG_OK;
}

namespace {

int check_store(const fg_cache *c, const fg_batch *b, const void *key, size_t key_stride, const void *value, size_t value_stride,
                bool writes_rows, const char *who)
{
    const int rc = check_batch(c, b, who);
    if (rc) return rc;
    if (b->rows && b->sequences && (!key || !value)) return set_error(FG_ERR_ARG, std::string(who) + ": null keys or values");
    const size_t width = size_t(c->kv_heads) * c->head_dim;
    // rows that are only read may overlap (one row for all of them, stride 0)
    if (writes_rows && b->rows > 1 && (key_stride < width || value_stride < width))
        return set_error(FG_ERR_SHAPE, std::string(who) + ": a row's heads run past the row stride");
    return FG_OK;
}

StoreParams store_params(const fg_cache *c, const fg_batch *b, size_t key_stride, size_t value_stride)
{
    StoreParams p{};
    p.b = batch_params(b);
    p.records = c->records;
    p.pages = c->pages;
    p.kv_heads = c->kv_heads;
    p.head_dim = c->head_dim;
    p.padded = c->padded;
    p.stride[0] = key_stride;
    p.stride[1] = value_stride;
    return p;
}

}  // namespace
}  // namespace fg

using namespace fg;

extern "C" {

int fg_cache_create(size_t pages, size_t kv_heads, size_t head_dim, void *stream, fg_cache **out)
{
    if (!out) return set_error(FG_ERR_ARG, "fg_cache_create: a null output handle");
    *out = nullptr;
    if (!kv_heads || !head_dim || head_dim % 4 || head_dim > 256)
        return set_error(FG_ERR_SHAPE, "fg_cache_create: heads of whole quads, at most 256 values, and at least one head");
    if (kv_heads > 4096 || pages > (size_t(1) << 24))
        return set_error(FG_ERR_SHAPE, "fg_cache_create: at most 4096 heads and 2^24 pages");
    const int padded = padded_head(int(head_dim));
    // (at least one page: attention's loads for a page that is not there read page 0)
    const size_t bytes = std::max<size_t>(pages, 1) * kv_heads * size_t(record_bytes(padded));
    int device = 0;
    FG_HIP(hipGetDevice(&device));
    uint8_t *records = nullptr;
    hipError_t e = hipMalloc(reinterpret_cast<void **>(&records), bytes);
    if (e != hipSuccess) return check_hip(e, "fg_cache_create: hipMalloc");
    const hipStream_t s = as_stream(stream);
    cache_clear_kernel<<<4096, 256, 0, s>>>(records, bytes / 4, unsigned(2 * kPage * padded / 4), unsigned(record_bytes(padded) / 4));
    e = hipGetLastError();
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    if (e != hipSuccess) {
        (void)hipFree(records);
        return check_hip(e, "fg_cache_create");
    }
    fg_cache *c = new (std::nothrow) fg_cache{device, int(pages), int(kv_heads), int(head_dim), padded, records};
    if (!c) {
        (void)hipFree(records);
        return set_error(FG_ERR_NOMEM, "fg_cache_create: host memory");
    }
    *out = c;
    return FG_OK;
}

int fg_cache_free(fg_cache *c)
{
    if (!c) return FG_OK;
    (void)hipFree(c->records);
    delete c;
    return FG_OK;
}

int fg_cache_write(fg_cache *c, const fg_batch *b, const float *key, size_t key_stride, const float *value, size_t value_stride,
                   void *stream)
{
    const int rc = check_store(c, b, key, key_stride, value, value_stride, false, "fg_cache_write");
    if (rc) return rc;
    StoreParams p = store_params(c, b, key_stride, value_stride);
    p.in[0] = key;
    p.in[1] = value;
    return launch_store<true>(p, as_stream(stream));
}

int fg_cache_read(const fg_cache *c, const fg_batch *b, float *key, size_t key_stride, float *value, size_t value_stride, void *stream)
{
    const int rc = check_store(c, b, key, key_stride, value, value_stride, true, "fg_cache_read");
    if (rc) return rc;
    StoreParams p = store_params(c, b, key_stride, value_stride);
    p.out[0] = key;
    p.out[1] = value;
    return launch_store<false>(p, as_stream(stream));
}

}  // extern "C"
