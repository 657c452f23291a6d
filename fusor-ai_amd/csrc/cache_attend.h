// What the kernels of attention over the paged cache share (cache_attend.hip, cache_attend_shared.hip): out = sum_j w_j v_j /
// sum_j w_j, w_j = exp(scale q.k_j - m), in one pass over the pages with a running reference in m's place.
#pragma once

#include <climits>
#include <cmath>
#include <utility>

#include "cache.h"

namespace fg {

// The arguments that calls of attention check.
int check_attend(const fg_cache *c, const fg_batch *b, const float *query, size_t heads, float scale, const float *out, size_t out_stride,
                 const char *who);

namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));

struct Note;

struct AttendParams {
    BatchParams b;
    const uint8_t *records;
    int pages, kv_heads, heads, group, head_dim;
    const float *query;
    size_t query_stride;
    float *out;
    size_t out_stride;
    float scale2;  // the scale times log2 e
    int window;
    int grid;      // tasks a head there is room for
    int target;    // tasks a head aims at; 0: no row tile is split
    float *partial;
    Note *notes;   // [grid]
};

template <class P>
P attend_params(const fg_cache *c, const fg_batch *b, const float *query, size_t query_stride, size_t heads, float scale, size_t window,
                float *out, size_t out_stride)
{
    P p{};
    p.b = batch_params(b);
    p.records = c->records;
    p.pages = c->pages;
    p.kv_heads = c->kv_heads;
    p.heads = int(heads);
    p.group = int(heads) / c->kv_heads;
    p.head_dim = c->head_dim;
    p.query = query;
    p.query_stride = query_stride;
    p.out = out;
    p.out_stride = out_stride;
    p.scale2 = scale * 1.44269504088896340736f;
    p.window = int(window < size_t(INT_MAX) ? window : size_t(INT_MAX));
    return p;
}

constexpr size_t kUnits = 256;  // CUs
constexpr int kMaxSplit = 64;   // parts of one row tile
constexpr int kMinPages = 4;    // pages of a part, a wave each

struct Task {
    int seq, tile, split, nsplit;
    int slot;  // the task's index
    Span span;
};

// A task in scalar registers (every wave finds it whole).
__device__ __forceinline__ Task uniform(Task t)
{
    auto same = [](int &x) { x = __builtin_amdgcn_readfirstlane(x); };
    same(t.seq), same(t.tile), same(t.split), same(t.nsplit), same(t.slot);
    same(t.span.begin), same(t.span.rows), same(t.span.first), same(t.span.length);
    return t;
}

// One pair of a tile: its operand row, query head and position.
struct Pair {
    int row, head, position;
    bool live;
};

// Where the rows of a task's span are, and the positions that a tile's rows lie between: those of one sequence follow each
// other.
struct InSequence {
    int first, low, high;
    __device__ __forceinline__ int of(int at) const { return first + at; }
    // the position of a lane's pair, once more
    __device__ __forceinline__ int again(const Pair &pair, int) const { return pair.position; }
};

template <class Places>
__device__ __forceinline__ Pair pair_of(const AttendParams &p, const Task &t, int kv, int m, const Places &places)
{
    const int pairs = t.span.rows * p.group;
    Pair r;
    r.live = m < pairs;
    m = min(m, pairs - 1);  // the last again past the pairs
    const int at = m / p.group;
    r.row = t.span.begin + at;
    r.head = kv * p.group + (m - at * p.group);
    r.position = places.of(at);
    return r;
}

// -------------------------------------------------------------------------- the numerics
//
// A level is exact in f16, so the products take f16 operands and f32 sums, and the f32 side of each is
// split into two f16 pieces, x = hi + lo to 2^-22 of x (and to 2^-35 of the row's largest, where lo falls
// under f16's normal range):
//   queries: a row is scaled by a power of two to a largest magnitude in [2^9, 2^10);
//   weights: 2^(t - r) times the value's scale, for t the score times log2 e and r a reference of the row,
//            a whole number. r is set when a weight passes 2^15, so that the largest is in (2^9, 2^11] (or,
//            where values are so small that none does, when 2^(t - r) passes 2^102), and the row's
//            sums are scaled by the power of two between; the total of 2^(t - r) is kept in f32, and r
//            cancels in the quotient.
// r rises with the largest of a weight times its value's scale, not with the largest weight alone: a
// value far larger than the others whose weight is next to nothing does not cost the others their bits. (Nor does a
// value of zeros: its scale is kNoValueScale.)

// Eight stored levels (level + 128, two dwords) as f16: 0x6400 + u is 1024 + u.
__device__ __forceinline__ v8h widen8(unsigned a, unsigned b)
{
    union {
        unsigned u[4];
        v2h h[4];
        v8h v;
    } w;
    w.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
    w.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
    w.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
    w.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
    const v2h bias = {_Float16(-1152.0f), _Float16(-1152.0f)};
#pragma unroll
    for (int i = 0; i < 4; i++) w.h[i] = w.h[i] + bias;
    return w.v;
}

__device__ __forceinline__ void split8(const float *x, v8h &hi, v8h &lo)
{
    typedef float v2f __attribute__((ext_vector_type(2)));
    union {
        unsigned u[4];
        v8h v;
    } h, l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const v2h top = __builtin_convertvector((v2f{x[2 * i], x[2 * i + 1]}), v2h);
        h.u[i] = __builtin_bit_cast(unsigned, top);
        // x - hi, exactly, straight from the packed pair
        v2f rest;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rest.x) : "v"(h.u[i]), "v"(x[2 * i]));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rest.y) : "v"(h.u[i]), "v"(x[2 * i + 1]));
        l.u[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(rest, v2h));
    }
    hi = h.v;
    lo = l.v;
}

// Eight query values from dimension d on (0 past the head's).
__device__ __forceinline__ void load8(const float *row, int d, int head_dim, float *x)
{
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
        v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (d + i < head_dim) v = *reinterpret_cast<const v4f_any *>(row + d + i);
#pragma unroll
        for (int j = 0; j < 4; j++) x[i + j] = v[j];
    }
}

// The power of two that brings a row's largest magnitude to [2^9, 2^10).
__device__ __forceinline__ int query_shift(float amax)
{
    return amax > 0.0f ? min(10 - __builtin_amdgcn_frexp_expf(amax), 126) : 0;
}

// The operand rows' queries, each split into its two pieces by the lanes that multiply them: `pair` is the pair's place among a
// key head's of all rows.
struct RawQueries {
    template <int DP>
    __device__ __forceinline__ void few(const AttendParams &p, const Pair &pair, int, int, int g, v8h (&qh)[(DP + 63) / 64][2],
                                        v8h (&ql)[(DP + 63) / 64][2], float &f) const
    {
        constexpr int J = (DP + 63) / 64;
        const float *row = p.query + size_t(pair.row) * p.query_stride + size_t(pair.head) * p.head_dim;
        float q[J][2][8];
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                load8(row, 64 * j + 16 * g + 8 * e, p.head_dim, q[j][e]);
#pragma unroll
                for (int k = 0; k < 8; k++) amax = fmaxf(amax, fabsf(q[j][e][k]));
            }
        float2 w = row_pair(amax);
        w = half_pair(fmaxf(w.x, w.y));
        const int shift = query_shift(fmaxf(w.x, w.y));
        f = ldexpf(p.scale2, -shift);
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int k = 0; k < 8; k++) q[j][e][k] = ldexpf(q[j][e][k], shift);
                split8(q[j][e], qh[j][e], ql[j][e]);
            }
    }
    template <int DP>
    __device__ __forceinline__ void many(const AttendParams &p, const Pair &pair, int, int, int h, v8h (&qh)[DP / 16], v8h (&ql)[DP / 16],
                                         float &f) const
    {
        constexpr int K = DP / 16;
        const float *row = p.query + size_t(pair.row) * p.query_stride + size_t(pair.head) * p.head_dim;
        float x[K][8];
        float amax = 0.0f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            load8(row, 32 * (k >> 1) + 16 * h + 8 * (k & 1), p.head_dim, x[k]);
#pragma unroll
            for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[k][e]));
        }
        const float2 w = half_pair(amax);
        const int shift = query_shift(fmaxf(w.x, w.y));
        f = ldexpf(p.scale2, -shift);
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[k][e] = ldexpf(x[k][e], shift);
            split8(x[k], qh[k], ql[k]);
        }
    }
};

constexpr float kWeightLimit = 32768.0f;
// Where a value's scale is under kSmallScale 2^(t - r) is looked at too: 2^25 of up to 2^102 stay in f32's range.
constexpr float kSmallScale = 0x1p-82f, kAloneLimit = 102.0f;
static_assert(kNoValueScale >= kSmallScale, "zeros are no reason to look");

// Lane n of each row of 16 lanes, to every lane of its row (DPP row_newbcast, which the multiplication that
// takes it reads by itself). A lane's scores are those of 16 keys that its row of lanes shares, so one register
// of 16 scales a row of lanes serves them all: read by every lane the scales took as much of LDS as half
// the levels did.
template <int N>
__device__ __forceinline__ float of_row_lane(float x)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x150 + N, 0xF, 0xF, true));
}
template <class F, size_t... N>
__device__ __forceinline__ void for_row_lanes(float x, F f, std::index_sequence<N...>)
{
    (f(int(N), of_row_lane<int(N)>(x)), ...);
}
// f(n, the row's scale n) for the 16 of them
template <class F>
__device__ __forceinline__ void for_scales(float x, F f)
{
    for_row_lanes(x, f, std::make_index_sequence<16>{});
}

// The running sums of a row: its reference r (-inf: no key yet, and then a total of 0) and the total of 2^(t - r) over the
// keys that this lane holds.
struct RowSums {
    float r, total;
};

// 16 scores of one row in this lane, t = s * f, to weights times the values' scales, into x; the row's other
// scores are in the lanes that `combine` joins. edge: keys outside [low, high] are masked (key(i) is score i's
// position). small: a value's scale is under kSmallScale. rescale(a) scales the row's sums of this lane by a.
// LEAN: in a kernel whose registers are full.
template <bool LEAN, class Key, class Combine, class Rescale>
__device__ __forceinline__ void weigh(const float (&s)[16], float (&x)[16], float vs, float f, bool small, bool edge,
                                      int low, int high, RowSums &sums, Key key, Combine combine, Rescale rescale)
{
    float top = 0.0f, total = 0.0f;
    auto weights = [&]() {
        top = total = 0.0f;
        for_scales(vs, [&](int i, float v) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], f, -sums.r));
            x[i] = v * e;
            total = total + e;
            top = fmaxf(top, x[i]);
        });
    };
    auto masked = [&]() {
        top = total = 0.0f;
        // (an f of its own: else the compiler may take the exponentials out of both branches, 16 registers more than there are)
        float g = f;
        if constexpr (LEAN) asm volatile("" : "+v"(g));
        for_scales(vs, [&](int i, float v) {
            const bool seen = key(i) >= low && key(i) <= high;
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], g, -sums.r));
            x[i] = seen ? v * e : 0.0f;
            total = total + (seen ? e : 0.0f);
            top = fmaxf(top, x[i]);
        });
    };
    if (edge) masked();
    else weights();
    if (__builtin_expect(small || __any(top > kWeightLimit), 0)) {
        top = combine(top);
        float u = -INFINITY, m = -INFINITY;
        float logs = vs;
        asm volatile("" : "+v"(logs));  // (keeps the logarithm in this branch)
        if constexpr (LEAN) asm volatile("" : "+v"(low), "+v"(high));  // (the masks once more: all of them kept do not fit the scalar registers)
        logs = __builtin_amdgcn_logf(logs);
        for_scales(logs, [&](int i, float v) {
            const float t = s[i] * f;
            const bool seen = !edge || (key(i) >= low && key(i) <= high);
            u = seen ? fmaxf(u, t + v) : u;
            m = seen ? fmaxf(m, t) : m;
        });
        u = combine(u);
        m = combine(m);
        if (top > kWeightLimit || m - sums.r > kAloneLimit) {
            // (a weight alone stays under 2^100, whatever the values' scales)
            const float r = fmaxf(ceilf(u) - 10.0f, ceilf(m) - 100.0f);
            const float a = __builtin_amdgcn_exp2f(sums.r - r);
            sums.r = r;
            sums.total = sums.total * a;
            rescale(a);
        }
        if (edge) masked();
        else weights();
    }
    sums.total = sums.total + total;
}

// The factor of a part's sums in the joined ones, whose reference is the largest of the parts'.
__device__ __forceinline__ float part_factor(float r, float joined) { return r == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(r - joined); }

// ---------------------------------------------------------------- few rows: decode steps
//
// A workgroup of four waves takes 16 pairs of one key head over its task's pages; each wave takes
// whole pages (the task's first, fifth ...), straight from memory to registers: nothing is shared
// between waves until their sums are joined at the end. The products are 16 x 16 x 32; lane l holds
// pair l % 16, and with g = l / 16 and 4 t + r the record's own order of values:
//   scores:  four products of 16 keys: row i of product t is key 32 (i / 8) + 8 t + i % 8, so lane l gets
//            the scores of keys 32 (g / 2) + 8 t + 4 (g % 2) + r, r = 0 .. 3;
//   values:  16 dimensions by 32 keys: the lane's 16 bytes of dimension l % 16 are those keys', in order.
// A decode step's pairs are the heads of a key head's group, 4 to 16 in most models: 16 rows leave the
// matrix cores idle lanes that cost nothing, for memory is what bounds long caches: 8 sequences of 34000 to 70000 tokens,
// 4 key heads of 128 (442 MB), 88 us, 5.0 TB/s, about the rate of a large copy. 64 sequences of 6 to 8001 tokens (87 MB)
// take 28.7 us, 3.0 TB/s, for parts of 16 pages or so that each start with a chain of waits (the plan, the table, the
// first page): half of the waves' cycles are waits, over long caches a third. One of 511 tokens, 2 key heads of
// 64, is that chain alone, 7.7 us.
// (Two tiles of rows a workgroup, which halves the reading of 17 to 32 pairs, left one workgroup a CU: 64 sequences
// of up to 3200 tokens, 28 pairs, 25.5 against 24.1 us, 32 pairs over one key head 36.9 against 24.2.)
// The tile's sums over the pages `range` of `table`, to `part`, or where that is null divided to the output: by WAVES waves
// together, 4, or by one for itself, which needs no `join`.
constexpr int few_floats(int DP) { return 16 * DP + 128; }  // of a part
template <int DP>
struct FewJoin {  // the waves' sums on their way to each other
    float sums[2][DP / 16 * 4 + 2][64];
};
template <int DP, int WAVES, class Places, class Queries>
__device__ __forceinline__ void attend_few(const AttendParams &p, const Task &task, const PageRange range, const int32_t *table, int kv,
                                           const Places &places, const Queries &queries, FewJoin<DP> *join, float *part)
{
    constexpr int TM = 16, J = (DP + 63) / 64, T = DP / 16, R = DP / 32;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = WAVES > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const Pair pair = pair_of(p, task, kv, task.tile * TM + i, places);
    v8h qh[J][2], ql[J][2];
    float f;
    queries.template few<DP>(p, pair, kv, task.span.begin * p.group + min(task.tile * TM + i, task.span.rows * p.group - 1), g, qh, ql, f);
    RowSums sums{-INFINITY, 0.0f};
    v4f o[T];
#pragma unroll
    for (int d = 0; d < T; d++) o[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int first = places.low, last = places.high;
    // A page's levels and scales stay in the same registers as the next one's: the keys' are asked for
    // when this page's scores are formed, the values' when it is done, the id a page
    // before, and it is looked at a page later: loads come back in order.
    uint4 k[4][J], v[T];
    float ks, vs;  // of key and value i of the lane's row of 16
    const int token = 32 * (g >> 1) + 8 * (i >> 2) + 4 * (g & 1) + (i & 3);
    auto entry_of = [&](int page) { return page < range.hi ? table[page] : -1; };
    auto id_of = [&](int entry) { return __builtin_amdgcn_readfirstlane(valid_page(entry, p.pages)); };
    auto record_of = [&](int id) { return p.records + (size_t(id) * p.kv_heads + kv) * record_bytes(DP); };
    auto load_keys = [&](int id) {
        const uint8_t *record = record_of(id);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int j = 0; j < J; j++) {
                const int block = min(2 * j + (g >> 1), R - 1);  // (the last dimensions of an odd count again: the queries' are 0)
                k[t][j] = *reinterpret_cast<const uint4 *>(record + ((i >> 3) * R + block) * 1024 + ((g & 1) * 32 + 8 * t + (i & 7)) * 16);
            }
        ks = *reinterpret_cast<const float *>(record + key_scale_byte(DP, token));
    };
    auto load_values = [&](int id) {
        const uint8_t *record = record_of(id);
        vs = *reinterpret_cast<const float *>(record + value_scale_byte(DP, token));
#pragma unroll
        for (int d = 0; d < T; d++)
            v[d] = *reinterpret_cast<const uint4 *>(record + kPage * DP + ((d >> 1) * 2 + (g >> 1)) * 1024 + ((g & 1) * 32 + (d & 1) * 16 + i) * 16);
    };
    int id = id_of(entry_of(range.lo + wave)), next = entry_of(range.lo + wave + WAVES), loaded = max(id, 0);
    load_keys(loaded);
    load_values(loaded);
    for (int page = range.lo + wave; page < range.hi; page += WAVES) {
        const bool held = id >= 0;
        id = id_of(next);
        loaded = id >= 0 ? id : loaded;  // (what is loaded already, again, where there is no next one)
        next = entry_of(page + 2 * WAVES);
        if (!held) {
            load_keys(loaded);
            load_values(loaded);
            continue;
        }
        v4f s[4];
#pragma unroll
        for (int t = 0; t < 4; t++) s[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const v8h a = e ? widen8(k[t][j].z, k[t][j].w) : widen8(k[t][j].x, k[t][j].y);
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[j][e], s[t], 0, 0, 0);
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[j][e], s[t], 0, 0, 0);
                }
        float scores[16], weights[16];
        for_scales(ks, [&](int n, float k) { scores[n] = k * s[n / 4][n % 4]; });
        load_keys(loaded);
        const int base = page * kPage + 32 * (g >> 1) + 4 * (g & 1);
        const bool edge = page * kPage + kPage - 1 > first || page * kPage < first_seen(last, p.window);
        const int high = pair.position, low = first_seen(high, p.window);
        weigh<true>(scores, weights, vs, f, __any(vs < kSmallScale), edge, low, high, sums, [&](int n) { return base + 8 * (n / 4) + n % 4; },
              [](float a) {
                  float2 w = row_pair(a);
                  w = half_pair(fmaxf(w.x, w.y));
                  return fmaxf(w.x, w.y);
              },
              [&](float a) {
#pragma unroll
                  for (int d = 0; d < T; d++)
#pragma unroll
                      for (int r = 0; r < 4; r++) o[d][r] = o[d][r] * a;
              });
        v8h wh[2], wl[2];
        split8(weights, wh[0], wl[0]);
        split8(weights + 8, wh[1], wl[1]);
#pragma unroll
        for (int d = 0; d < T; d++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const v8h a = e ? widen8(v[d].z, v[d].w) : widen8(v[d].x, v[d].y);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, wl[e], o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, wh[e], o[d], 0, 0, 0);
            }
        load_values(loaded);
    }
    {
        float2 w = row_pair(sums.total);
        w = half_pair(w.x + w.y);
        sums.total = w.x + w.y;
    }
    // the waves' sums joined, lane by lane: waves 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
    for (int step = WAVES / 2; step >= 1; step >>= 1) {
        float(*joined)[T * 4 + 2][64] = join->sums;
        float(*to)[64] = joined[wave & 1];
        if (wave >= step && wave < 2 * step) {
            to[0][lane] = sums.r;
            to[1][lane] = sums.total;
#pragma unroll
            for (int d = 0; d < T; d++)
#pragma unroll
                for (int r = 0; r < 4; r++) to[2 + d * 4 + r][lane] = o[d][r];
        }
        __syncthreads();
        if (wave < step) {
            float(*from)[64] = joined[(wave + step) & 1];
            const float other = from[0][lane], r = fmaxf(sums.r, other);
            const float a = part_factor(sums.r, r), b = part_factor(other, r);
            sums.r = r;
            sums.total = sums.total * a + from[1][lane] * b;
#pragma unroll
            for (int d = 0; d < T; d++)
#pragma unroll
                for (int c = 0; c < 4; c++) o[d][c] = o[d][c] * a + from[2 + d * 4 + c][lane] * b;
        }
        __syncthreads();
    }
    if (wave != 0 || !pair.live) return;
    if (part) {
        part[lane] = sums.r;
        part[64 + lane] = sums.total;
#pragma unroll
        for (int d = 0; d < T; d++) *reinterpret_cast<v4f *>(part + 128 + d * 256 + lane * 4) = o[d];
        return;
    }
    float *row = p.out + size_t(pair.row) * p.out_stride + size_t(pair.head) * p.head_dim;
#pragma unroll
    for (int d = 0; d < T; d++) {
        v4f x;
#pragma unroll
        for (int c = 0; c < 4; c++) x[c] = sums.total == 0.0f ? 0.0f : o[d][c] / sums.total;
        if (16 * d + 4 * g < p.head_dim) *reinterpret_cast<v4f_any *>(row + 16 * d + 4 * g) = x;
    }
}

// -------------------------------------------------------------------- many rows: prompts
//
// A workgroup of four waves takes 128 pairs of one key head, 32 a wave, and walks its task's pages
// together: a page's levels are widened to f16 once, by all four waves, into one of two LDS buffers in
// the products' operand order (16 bytes a lane, lane after lane: no bank conflicts), while the other is
// read. The products are 32 x 32 x 16; lane l holds pair l % 32 and, with h = l / 32, the scores of
// keys 8 j + 4 h + i in register 4 j + i: the order of the values' record.
// Bounded by the matrix cores, with the vector units close behind: of a page and head of 128 a wave has
// 64 products of 32 cycles and about 1600 cycles of vector work (per score a multiplication by the key's scale, an
// exponential, the value's scale, the total, the maximum and two f16 pieces), and two waves a SIMD overlap them in part.
// 8192 tokens of 16 heads of 128 over 4: 492 us, 1118 TFLOP/s in f16 products (two an operand, for the
// pieces), the matrix cores busy 61 % of the time and the vector units 57 %, at the 1.74 GHz that the card keeps under this
// load (2.35 in the others here); a large f16 product of the library's reaches 1339. Chunks of 2700 tokens, 16 heads of
// 72 over a window of 1000: 75 us, 336 TFLOP/s: its 350 tiles of 19 pages are 1400 waves for 1024 SIMDs, so some have
// two, and CUs are busy 69 % of the time. 17 chunks of 1 to 512 tokens, 14 heads of 64 over 2: 52.5 us; CUs are busy
// 72 % of the time, and then the vector units 51 %, the matrix cores 29, with 1.6 waves a SIMD. 32 pairs a wave: with 64, or with four waves a SIMD, the sums do not fit the registers.
template <int DP>
constexpr size_t many_lds() { return size_t(2) * (256 * DP + 2 * kPage * 4); }

// The tile's sums over the pages `range` of `table`, to `parts`, four of them, or where that is null divided to the output.
// `places` are those of the wave's pairs. LEAN: what a lane knows of its place is computed in every page from its index, not
// kept, for a kernel that has other things in registers too (heads of 128 leave it five); kept it is 4 % faster: a prompt of 8192
// tokens, 16 heads of 128 over 4, 496 and 519 us.
constexpr int many_floats(int DP) { return 32 * DP + 128; }  // of a wave's part
template <int DP, bool LEAN, class Places, class Queries>
__device__ __forceinline__ void attend_many(const AttendParams &p, const Task &task, const PageRange range, const int32_t *table, int kv,
                                            const Places &places, const Queries &queries, uint8_t *lds, float *parts)
{
    constexpr int TM = 128, K = DP / 16, T = DP / 32, L = DP / 32;  // steps, tiles of 32 dimensions, 16-byte loads a thread
    constexpr int kBuffer = 256 * DP + 2 * kPage * 4;
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    uint4 staged[L];
    float staged_scale = 0.0f;
    // (a table's entry is looked at an iteration after it was asked for: loads come back in order, and a
    // look would wait for the records asked for before it)
    auto entry_of = [&](int page) { return page < range.hi ? table[page] : -1; };
    auto id_of = [&](int entry) { return __builtin_amdgcn_readfirstlane(valid_page(entry, p.pages)); };
    auto load = [&](int id) {  // a page's record into registers
        if (id < 0) return;
        const uint8_t *record = p.records + (size_t(id) * p.kv_heads + kv) * record_bytes(DP);
        if constexpr (LEAN) {
            unsigned thread = threadIdx.x;
            asm volatile("" : "+v"(thread));  // (a 32-bit offset beside a scalar address, no 64-bit one kept in registers)
#pragma unroll
            for (int c = 0; c < L; c++) staged[c] = *reinterpret_cast<const uint4 *>(record + c * 4096 + thread * 16u);
            if (tid < 2 * kPage) staged_scale = *reinterpret_cast<const float *>(record + key_scale_byte(DP, 0) + thread * 4u);
        } else {
#pragma unroll
            for (int c = 0; c < L; c++) staged[c] = *reinterpret_cast<const uint4 *>(record + (c * 256 + tid) * 16);
            if (tid < 2 * kPage) staged_scale = *reinterpret_cast<const float *>(record + key_scale_byte(DP, tid));
        }
    };
    auto store = [&](uint8_t *to) {  // ... widened into a buffer: each kilobyte of 64 lanes as two
#pragma unroll
        for (int c = 0; c < L; c++) {
            const int piece = c * 256 + tid;
            uint8_t *at = to + (piece >> 6) * 2048 + (piece & 63) * 16;
            *reinterpret_cast<v8h *>(at) = widen8(staged[c].x, staged[c].y);
            *reinterpret_cast<v8h *>(at + 1024) = widen8(staged[c].z, staged[c].w);
        }
        if (tid < 2 * kPage) reinterpret_cast<float *>(to + 256 * DP)[tid] = staged_scale;
    };
#pragma unroll
    for (int c = 0; c < L; c++) staged[c] = make_uint4(0, 0, 0, 0);
    // the pages read (-1: nothing there), staged, and the entry of the one after
    int here = id_of(entry_of(range.lo)), next = id_of(entry_of(range.lo + 1)), after = entry_of(range.lo + 2);
    load(here);

    const Pair pair = pair_of(p, task, kv, task.tile * TM + wave * 32 + l31, places);
    v8h qh[K], ql[K];
    float f;
    queries.template many<DP>(p, pair, kv, task.span.begin * p.group + min(task.tile * TM + wave * 32 + l31, task.span.rows * p.group - 1), h, qh,
                              ql, f);
    RowSums sums{-INFINITY, 0.0f};
    v16f o[T];
#pragma unroll
    for (int d = 0; d < T; d++) o[d] = v16f{};
    const int first = places.low, last = places.high;
    const bool any = task.tile * TM + wave * 32 < task.span.rows * p.group;

    store(lds);
    load(next);
    __syncthreads();
    for (int page = range.lo; page < range.hi; page++) {
        const int b = (page - range.lo) & 1;
        const bool held = here >= 0;
        if (next >= 0) store(lds + (b ^ 1) * kBuffer);
        here = next;
        next = id_of(after);
        load(next);
        after = entry_of(page + 3);
        const uint8_t *buffer = lds + b * kBuffer;
        const float *key_scales = reinterpret_cast<const float *>(buffer + 256 * DP), *value_scales = key_scales + kPage;
        const bool seen = held && any && page * kPage <= last && page * kPage + kPage - 1 >= first_seen(first, p.window);
        if (seen) {
            const bool edge = page * kPage + kPage - 1 > first || page * kPage < first_seen(last, p.window);
            const uint8_t *values = buffer + 128 * DP;
            // The operands of a step are read while the step before multiplies: left to itself the compiler reads
            // each step's into the registers of the one before, and waits.
            v16f s[2] = {};
            v8h a[2][2];
            float ks[2], vs[2];
            int here_lane = lane, high = pair.position;
            if constexpr (LEAN) {
                here_lane = int(threadIdx.x);
                asm volatile("" : "+v"(here_lane));
                high = places.again(pair, (here_lane >> 6) * 32 + (here_lane & 31));
                asm volatile("" : "+v"(high));
                here_lane &= 63;
            }
            const int low = first_seen(high, p.window), here_half = here_lane >> 5;
            auto read_keys = [&](int k) {
#pragma unroll
                for (int kt = 0; kt < 2; kt++) a[k & 1][kt] = *reinterpret_cast<const v8h *>(buffer + (kt * K + k) * 1024 + here_lane * 16);
            };
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                const int token = 32 * kt + 8 * ((here_lane >> 2) & 3) + 4 * here_half + (here_lane & 3);
                ks[kt] = key_scales[token];
                vs[kt] = value_scales[token];
            }
            const bool small = __any(fminf(vs[0], vs[1]) < kSmallScale);
            read_keys(0);
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (k + 1 < K) read_keys(k + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int kt = 0; kt < 2; kt++) s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[k & 1][kt], ql[k], s[kt], 0, 0, 0);
#pragma unroll
                for (int kt = 0; kt < 2; kt++) s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[k & 1][kt], qh[k], s[kt], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            v8h wh[4], wl[4], b[2][T];
            auto read_values = [&](int c) {
#pragma unroll
                for (int d = 0; d < T; d++) b[c & 1][d] = *reinterpret_cast<const v8h *>(values + ((d * 2 + c / 2) * 2 + c % 2) * 1024 + here_lane * 16);
            };
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {  // 32 keys at a time: half the registers
                float scores[16], x[16];
                for_scales(ks[kt], [&](int i, float k) { scores[i] = k * s[kt][i]; });
                if (kt) read_values(0);
                __builtin_amdgcn_sched_barrier(0);
                weigh<LEAN>(scores, x, vs[kt], f, small, edge, low, high, sums,
                          [&](int i) { return page * kPage + 32 * kt + 2 * (i & ~3) + 4 * here_half + i % 4; },
                          [](float v) {
                              const float2 w = half_pair(v);
                              return fmaxf(w.x, w.y);
                          },
                          [&](float factor) {
#pragma unroll
                              for (int d = 0; d < T; d++)
#pragma unroll
                                  for (int r = 0; r < 16; r++) o[d][r] = o[d][r] * factor;
                              // the first 32 keys' weights are not in the sums yet; the factor, a power of two, in two
                              // steps, for f16's range
                              if (kt) {
                                  const float step = fmaxf(factor, 0x1p-14f);
                                  const _Float16 once = _Float16(step), rest = _Float16(factor / step);
#pragma unroll
                                  for (int c = 0; c < 2; c++) {
                                      wh[c] = wh[c] * once * rest;
                                      wl[c] = wl[c] * once * rest;
                                  }
                              }
                          });
                split8(x, wh[2 * kt], wl[2 * kt]);
                split8(x + 8, wh[2 * kt + 1], wl[2 * kt + 1]);
            }
#pragma unroll
            for (int c = 0; c < 4; c++) {  // 16 keys
                if (c < 3) read_values(c + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = 0; d < T; d++) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b[c & 1][d], wl[c], o[d], 0, 0, 0);
#pragma unroll
                for (int d = 0; d < T; d++) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b[c & 1][d], wh[c], o[d], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __syncthreads();
    }
    const float2 w = half_pair(sums.total);
    sums.total = w.x + w.y;
    if constexpr (LEAN) {
        int thread = int(threadIdx.x);
        asm volatile("" : "+v"(thread));
        if (task.tile * TM + (thread >> 6) * 32 + (thread & 31) >= task.span.rows * p.group) return;  // (a pair that is not live)
    } else if (!pair.live) {
        return;
    }
    if (parts) {
        float *part = parts + wave * many_floats(DP);
        part[lane] = sums.r;
        part[64 + lane] = sums.total;
#pragma unroll
        for (int d = 0; d < T; d++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                *reinterpret_cast<v4f *>(part + 128 + (d * 4 + c) * 256 + lane * 4) = v4f{o[d][4 * c], o[d][4 * c + 1], o[d][4 * c + 2], o[d][4 * c + 3]};
        return;
    }
    float *row = p.out + size_t(pair.row) * p.out_stride + size_t(pair.head) * p.head_dim;
#pragma unroll
    for (int d = 0; d < T; d++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            v4f x;
#pragma unroll
            for (int r = 0; r < 4; r++) x[r] = sums.total == 0.0f ? 0.0f : o[d][4 * c + r] / sums.total;
            const int dim = 32 * d + 8 * c + 4 * h;
            if (dim < p.head_dim) *reinterpret_cast<v4f_any *>(row + dim) = x;
        }
}

}  // namespace
}  // namespace fg
