// The paged 8-bit cache (fg_cache): its pages, the new tokens' keys and values quantized into them, and
// read back. cache_layout.h says where a level lies; cache_attend.hip reads the pages.
#include <algorithm>
#include <new>

#include "rotary.h"

namespace fg {
namespace {

struct StoreParams {
    BatchParams b;
    uint8_t *records;
    int pages, kv_heads, head_dim, padded;
    const float *in[2];  // keys, values
    float *out[2];
    size_t stride[2];
};

// ... and with keys that are turned by their positions before they are kept (and, in the row kernel's launch, queries).
struct TurnParams : StoreParams {
    RotaryParams r;
    RotateParams queries;
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

// Four values of a key from dimension dim on, x, turned: `head` is where the head's values lie, `angle(pair, j)` the pair's
// factors (its j-th of this lane's). Values 2i and 2i + 1 are partners in the lane itself; the partners of halves are read a second time (the
// lane that has them may be anywhere in the wave, and they come from the cache).
template <class F>
__device__ __forceinline__ v4f turned_quad(const RotaryParams &r, const float *head, int dim, const v4f &x, F angle)
{
    if (dim >= r.dims) return x;
    v4f u = x;
    if (!r.halves) {
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            if (dim + j >= r.dims) continue;
            const Turn t = angle((dim + j) / 2, j / 2);
            u[j] = turned(x[j], x[j + 1], t, true);
            u[j + 1] = turned(x[j + 1], x[j], t, false);
        }
        return u;
    }
    const int half = r.dims / 2;
    v4f partner = {0.0f, 0.0f, 0.0f, 0.0f};
    if (half % 4 == 0) {
        partner = *reinterpret_cast<const v4f_any *>(head + (dim < half ? dim + half : dim - half));
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = dim + j;
            if (d < r.dims) partner[j] = head[d < half ? d + half : d - half];
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int d = dim + j;
        if (d < r.dims) u[j] = turned(x[j], partner[j], angle(d < half ? d : d - half, j), d < half);
    }
    return u;
}

// A wave per new row and head, for few new tokens a sequence. Four dimensions a lane; heads of up to 128
// take half a wave for the key and half for the value. A value's levels go to single bytes, 16 apart, of a kilobyte
// that 64 tokens share (cache_layout.h): 64 stores of a byte a token, which is what bounds long runs of tokens,
// and why they take the kernels below. A step's single tokens are bounded by the launch and three loads one
// after the other (the row's sequence, its page, then its values, though their address needs neither): 8 tokens of
// 2 heads of 64 written in 3.3 us, read back in 3.0; 512 of 8 heads of 128 in 7.8 and 5.0.
template <bool WRITE, bool TURN, class P>
__device__ __forceinline__ void store_row(const P &p, unsigned unit)
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
            if constexpr (TURN) {
                if (live && !value)
                    x = turned_quad(p.r, p.in[0] + place - dim, dim, x, [&](int pair, int) { return turn_at(p.r, pair, position); });
            }
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
    for (unsigned unit = blockIdx.x * 4 + (threadIdx.x >> 6); unit < units; unit += gridDim.x * 4) store_row<WRITE, false>(p, unit);
}

// The same for keys to be turned, and behind the rows' units those of the queries: one launch for a decode step. 8 tokens, 14
// heads of 64 over 2: 5.1 us, of which the angles are 1.5.
template <bool QUADS>
__global__ __launch_bounds__(256) void turn_rows_kernel(TurnParams p)
{
    RotateParams queries = p.queries;
    queries.b = p.b, queries.r = p.r;  // (the same scalar registers)
    const unsigned units = unsigned(p.b.rows) * unsigned(p.kv_heads), all = units + unsigned(p.b.rows) * unsigned(p.queries.units);
    for (unsigned unit = blockIdx.x * 4 + (threadIdx.x >> 6); unit < all; unit += gridDim.x * 4) {
        if (unit < units) store_row<true, true>(p, unit);
        else rotate_unit<QUADS>(queries, unit - units);
    }
}

// A workgroup per page that new tokens lie in, head, and keys or values. A thread takes four tokens (an
// aligned run, so one dword of each dimension's values) of four dimensions, heads of up to 128 all of a page
// at once; the levels meet in LDS in the record's order, and whole 16-byte pieces go to the page or come from it.
// Pieces that also hold other tokens' values are written in part. Bounded by memory for long runs, and by one load's
// wait after another for short ones: 3618 tokens of 4 heads of 128 (14.8 MB of f32, 3.8 MB of levels and scales) written
// in 9.2 us, 2.0 TB/s, and read back in 7.5. Keys and values are each a workgroup's, for twice the loads in flight (both in
// one: 16.8 and 9.8).
constexpr int kPageThreads = 512;

template <bool WRITE, bool TURN, class P>
__device__ __forceinline__ void store_page(const P &p, int run, int head, int value, uint8_t *levels, float *scales)
{
    const int tid = threadIdx.x;
    int index;
    const int s = find_unit(p.b.sequences, run, &index, [&](int q) {
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
            if constexpr (TURN) {
                if (live && !value) {
                    Angle four[4];  // of t, a whole four
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // (tokens that are not new have the first new one's partners, and their levels go nowhere)
                        const float *row = p.in[0] + (row0 + min(max(t + i, t0), t1 - 1)) * stride + size_t(head) * p.head_dim;
                        x[i] = turned_quad(p.r, row, dim, x[i], [&](int pair, int j) {
                            const RotaryPair &r = p.r.pairs[pair];
                            if (i == 0) four[j] = whole_four(r, place * kPage + t);
                            return turn_of(both(four[j], r.more[i]), p.r.magnitude);
                        });
                    }
                }
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
__global__ __launch_bounds__(kPageThreads) void cache_pages_kernel(StoreParams p)
{
    extern __shared__ __align__(16) uint8_t levels[];
    __shared__ float scales[kPage];
    store_page<WRITE, false>(p, int(blockIdx.x), int(blockIdx.y), int(blockIdx.z), levels, scales);
}

// The same for keys to be turned, and behind the pages' workgroups those of the queries' rows, which memory bounds while the
// pages wait for one load after another. (Bounded to two workgroups a CU: the angles' 64-bit arithmetic took 129 registers, and
// one fewer of them is two workgroups instead of one. 3618 tokens of 4 heads of 128, 64 values turned: 11.7 us, with one
// 15.9, with three, which spill, 21.5; with the queries' 16 heads in the same launch 20.9, where the two apart take 11.9 + 11.7.)
template <bool QUADS>
__global__ __launch_bounds__(kPageThreads, 4) void turn_pages_kernel(TurnParams p, unsigned runs)
{
    extern __shared__ __align__(16) uint8_t levels[];
    __shared__ float scales[kPage];
    const unsigned pages = runs * unsigned(p.kv_heads) * 2;
    if (blockIdx.x < pages) {
        const unsigned run = blockIdx.x / 2 / unsigned(p.kv_heads);
        store_page<true, true>(p, int(run), int(blockIdx.x / 2 - run * unsigned(p.kv_heads)), int(blockIdx.x & 1), levels, scales);
        return;
    }
    RotateParams queries = p.queries;
    queries.b = p.b, queries.r = p.r;
    const unsigned units = unsigned(p.b.rows) * unsigned(p.queries.units), step = (gridDim.x - pages) * (kPageThreads / 64);
    for (unsigned unit = (blockIdx.x - pages) * (kPageThreads / 64) + (threadIdx.x >> 6); unit < units; unit += step)
        rotate_unit<QUADS>(queries, unit);
}

// A workgroup a page: a run of n rows lies in at most (n + 62) / 64 + 1 pages.
dim3 page_grid(const StoreParams &p)
{
    const size_t runs = size_t(p.b.rows) / kPage + 2 * size_t(std::min(p.b.sequences, p.b.rows));
    return dim3(unsigned(runs), unsigned(p.kv_heads), 2);
}

// Whether a write takes the row kernels: up to 16 new tokens a sequence, or 2048 rows times heads (launch_store's figures).
bool by_rows(const StoreParams &p) { return p.b.rows <= 16 * p.b.sequences || size_t(p.b.rows) * p.kv_heads <= 2048; }

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
    if (by_rows(p)) {
        cache_rows_kernel<WRITE><<<unsigned(std::min((units + 3) / 4, kMaxGrid)), 256, 0, s>>>(p);
    } else {
        cache_pages_kernel<WRITE><<<page_grid(p), kPageThreads, size_t(kPage * p.padded), s>>>(p);
    }
    FG_HIP(hipGetLastError());
    return FG_OK;
}

int launch_turned(const TurnParams &p, bool quads, hipStream_t s)
{
    if (p.b.rows == 0 || p.b.sequences == 0) return FG_OK;
    const size_t units = size_t(p.b.rows) * p.kv_heads, all = units + size_t(p.b.rows) * p.queries.units;
    if (all > 0xf0000000) return set_error(FG_ERR_SHAPE, "the paged cache: more rows times heads than a launch takes");
    const size_t runs = page_grid(p).x, pages = runs * size_t(p.kv_heads) * 2, waves = kPageThreads / 64;
    // (a launch has fewer than 2^32 threads in one direction: batches whose pages times heads are more than 2^22 go by rows)
    if (!by_rows(p) && pages <= kMaxGrid / 4) {
        const size_t rows = std::min((size_t(p.b.rows) * p.queries.units + waves - 1) / waves, kMaxGrid / 4);
        const unsigned grid = unsigned(pages + rows);
        if (quads) turn_pages_kernel<true><<<grid, kPageThreads, size_t(kPage * p.padded), s>>>(p, unsigned(runs));
        else turn_pages_kernel<false><<<grid, kPageThreads, size_t(kPage * p.padded), s>>>(p, unsigned(runs));
        FG_HIP(hipGetLastError());
        return FG_OK;
    }
    const unsigned grid = unsigned(std::min((all + 3) / 4, kMaxGrid));
    if (quads) turn_rows_kernel<true><<<grid, 256, 0, s>>>(p);
    else turn_rows_kernel<false><<<grid, 256, 0, s>>>(p);
    FG_HIP(hipGetLastError());
    return FG_OK;
}

}  // namespace

int check_batch_arrays(const fg_batch *b, bool reads_pages, const char *who)
{
    const std::string name(who);
    if (!b) return set_error(FG_ERR_ARG, name + ": a null batch");
    if (b->sequences > 65536 || b->rows > (size_t(1) << 24) || b->max_pages > (size_t(1) << 24))
        return set_error(FG_ERR_SHAPE, name + ": at most 65536 sequences, 2^24 rows and 2^24 pages a sequence");
    if (b->sequences && (!b->row_starts || !b->lengths || (reads_pages && b->max_pages && !b->pages)))
        return set_error(FG_ERR_ARG, name + ": a null array of the batch");
    return FG_OK;
}

int check_batch(const fg_cache *c, const fg_batch *b, const char *who)
{
    const std::string name(who);
    if (!c || !b) return set_error(FG_ERR_ARG, name + ": a null cache or batch");
    const int rc = check_batch_arrays(b, true, who);
    if (rc) return rc;
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

template <class P>
P store_params(const fg_cache *c, const fg_batch *b, size_t key_stride, size_t value_stride)
{
    P p{};
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
    StoreParams p = store_params<StoreParams>(c, b, key_stride, value_stride);
    p.in[0] = key;
    p.in[1] = value;
    return launch_store<true>(p, as_stream(stream));
}

int fg_cache_write_rotated(fg_cache *c, const fg_batch *b, const fg_rotary *r, const float *key, size_t key_stride, const float *value,
                           size_t value_stride, const float *query, size_t query_stride, size_t heads, float *out, size_t out_stride,
                           void *stream)
{
    const char *who = "fg_cache_write_rotated";
    int rc = check_store(c, b, key, key_stride, value, value_stride, false, who);
    if (rc) return rc;
    if ((rc = check_rotary(r, c->device, size_t(c->head_dim), who))) return rc;
    if ((heads || query || out) && (rc = check_rotated(b, query, query_stride, heads, size_t(c->head_dim), out, out_stride, who))) return rc;
    const size_t width = size_t(c->kv_heads) * c->head_dim, turned = heads * c->head_dim;
    if (rows_meet(out, out_stride, turned, key, key_stride, width, b->rows) || rows_meet(out, out_stride, turned, value, value_stride, width, b->rows))
        return set_error(FG_ERR_SHAPE, std::string(who) + ": turned queries lie over the keys or values, which the same launch reads");
    TurnParams p = store_params<TurnParams>(c, b, key_stride, value_stride);
    p.in[0] = key;
    p.in[1] = value;
    p.r = rotary_params(r);
    if (heads) p.queries = rotate_params(r, b, query, query_stride, heads, size_t(c->head_dim), out, out_stride);
    return launch_turned(p, whole_quads(r), as_stream(stream));
}

int fg_cache_read(const fg_cache *c, const fg_batch *b, float *key, size_t key_stride, float *value, size_t value_stride, void *stream)
{
    const int rc = check_store(c, b, key, key_stride, value, value_stride, true, "fg_cache_read");
    if (rc) return rc;
    StoreParams p = store_params<StoreParams>(c, b, key_stride, value_stride);
    p.out[0] = key;
    p.out[1] = value;
    return launch_store<false>(p, as_stream(stream));
}

}  // extern "C"
