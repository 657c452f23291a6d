// Next tokens drawn from logits (fg_sample).
//
// A row's tokens are ordered by (logit descending, index ascending); temperature, top-k, top-p and min-p
// each keep a first part of that order, so what is kept ends at one token, the cut. No sort is needed to find
// it: the weights' logarithms z = (logit - largest) / temperature are counted and summed in kBins bins of
// 1/32, the bin of a cut follows from the running sums, and only that bin's tokens are looked at one by one.
//   1 top      the largest logit of each chunk of the row, and its first index;
//   2 bins     the tokens and the weight of every bin;
//   3 collect  from the bins: which are kept whole, and which hold a cut. The kept weight of each segment
//              (a wave's run of the row), and a list of the tokens whose bins hold a cut (or of all
//              tokens up to the cut, where they are few);
//   4 draw     the cut among the list; the segment, or the listed token, on which the random number falls.
// Weights are 64-bit: exp in f64 (one ulp), rounded to a whole number of units of 2^-45 of the first token's
// (less for more than 2^18 tokens), so that every sum is exact and their order changes nothing. Tokens
// under half a unit (z < -31.9) weigh 0; the last bin holds only such.
// Bound: the row is read three times, the first from memory and the others mostly from the caches (rows are
// taken in batches that fit the Infinity Cache), and twice about 25 f64 operations for a weight.
#include <algorithm>
#include <atomic>

#include "cache.h"

namespace fg {
namespace {

typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned long long u64;

constexpr int kThreads = 256;
constexpr int kBins = 1024;
constexpr float kPerUnit = 32.0f;   // bins a unit of z
constexpr int kList = 3584;         // tokens a row's list holds
constexpr int kMaxChunks = 64;      // workgroups of a row; four segments each

struct SampleParams {
    const float *logits;
    size_t stride;
    int vocab, chunks, segment;  // segment: tokens of a wave
    const float *random, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    double unit;                 // units of the first token's weight, a power of two
    u64 *top;                    // [rows][chunks]: (ordered logit, ~index)
    u64 *mass;                   // [rows][kBins]
    unsigned *count;             // [rows][kBins]
    u64 *segments;               // [rows][chunks * 4]
    unsigned *listed;            // [rows]: tokens of the list (past kList: not all are in it)
    u64 *list;                   // [rows][kList]: (logit bits, index)
    int32_t *tokens;
    float *chances;
};

// A logit's place in the order of floats as an unsigned integer; NaN is -inf, and -0 is 0.
__device__ __forceinline__ float plain_logit(float x) { return x != x ? -INFINITY : x + 0.0f; }
__device__ __forceinline__ unsigned ordered(float x)
{
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }

// What a row asks for.
struct Row {
    double inverse;  // 1 / temperature
    float top_p, min_p;
    int top_k;
    bool greedy, has_k, has_p;
};
__device__ __forceinline__ Row row_of(const SampleParams &p, int row)
{
    Row r;
    const float t = p.temperature ? p.temperature[row] : 1.0f;
    const float tp = p.top_p ? p.top_p[row] : 1.0f, mp = p.min_p ? p.min_p[row] : 0.0f;
    r.top_k = p.top_k ? p.top_k[row] : 0;
    r.has_k = r.top_k > 0 && r.top_k < p.vocab;
    r.has_p = tp < 1.0f;
    r.top_p = tp;
    r.min_p = mp;
    r.greedy = !(t > 0.0f) || r.top_k == 1 || tp <= 0.0f || mp > 1.0f;
    r.inverse = 1.0 / double(t);
    return r;
}

// exp(z) for z in [-40, 0]: z = n ln 2 + r, the Taylor series of exp to r^12 (|r| <= 0.347: the next term is
// under 2^-52 of it), times 2^n.
__device__ __forceinline__ double weight_of(double z)
{
    const double n = __builtin_rint(z * 1.4426950408889634);
    double r = __builtin_fma(n, -0.6931471805599453, z);
    r = __builtin_fma(n, -2.3190468138462996e-17, r);
    double e = 1.0 / 479001600.0;
    e = __builtin_fma(e, r, 1.0 / 39916800.0);
    e = __builtin_fma(e, r, 1.0 / 3628800.0);
    e = __builtin_fma(e, r, 1.0 / 362880.0);
    e = __builtin_fma(e, r, 1.0 / 40320.0);
    e = __builtin_fma(e, r, 1.0 / 5040.0);
    e = __builtin_fma(e, r, 1.0 / 720.0);
    e = __builtin_fma(e, r, 1.0 / 120.0);
    e = __builtin_fma(e, r, 1.0 / 24.0);
    e = __builtin_fma(e, r, 1.0 / 6.0);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    return __builtin_ldexp(e, int(n));
}
// Whole units of a weight: below 2^52 a sum with 2^52 rounds to them.
__device__ __forceinline__ u64 units_of(double e, double unit)
{
    return u64(__double_as_longlong(__builtin_fma(e, unit, 4503599627370496.0))) & 0xFFFFFFFFFFFFFull;
}

// z of a logit, and its bin. The first token's z is 0 (its difference is, infinite or not).
__device__ __forceinline__ double z_of(float x, float top, double inverse)
{
    return x == top ? 0.0 : (double(x) - double(top)) * inverse;
}
__device__ __forceinline__ int bin_of(double z)
{
    const float b = float(z) * -kPerUnit;  // (monotone in z: a rounding and a multiplication)
    return b < float(kBins - 1) ? int(b) : kBins - 1;
}

__device__ __forceinline__ u64 wave_sum(u64 v)
{
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// The workgroup's sum of a value before this thread's, and of all. `part` is LDS of four; every thread calls.
__device__ __forceinline__ u64 block_before(u64 v, u64 *part, u64 *total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 up = __shfl_up(x, d, 64);
        if (lane >= d) x += up;
    }
    __syncthreads();
    if (lane == 63) part[wave] = x;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) {
        if (w < wave) before += part[w];
        all += part[w];
    }
    *total = all;
    return before + x - v;
}

// The row's largest logit from its chunks', (ordered logit, ~index); every wave of the workgroup by itself.
__device__ __forceinline__ u64 row_top(const SampleParams &p, int row)
{
    const int lane = threadIdx.x & 63;
    u64 t = lane < p.chunks ? p.top[size_t(row) * p.chunks + lane] : 0;
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const u64 o = __shfl_xor(t, d, 64);
        t = o > t ? o : t;
    }
    return t;
}

// Calls f(logit, index) for this wave's segment, in runs of 256 tokens, four a lane.
template <class F>
__device__ __forceinline__ void for_segment(const SampleParams &p, int row, int segment, F f)
{
    const float *x = p.logits + size_t(row) * p.stride;
    const int lane = threadIdx.x & 63;
    const int begin = segment * p.segment, end = min(begin + p.segment, p.vocab);  // (segments past the row: empty)
    int i = begin + lane * 4;
    constexpr int kAhead = 4;
    for (; i + (kAhead - 1) * 256 + 4 <= end; i += kAhead * 256) {
        v4f v[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; a++) v[a] = *reinterpret_cast<const v4f_any *>(x + i + a * 256);
#pragma unroll
        for (int a = 0; a < kAhead; a++)
#pragma unroll
            for (int j = 0; j < 4; j++) f(plain_logit(v[a][j]), i + a * 256 + j);
    }
    for (; i < end; i += 256)
        for (int j = 0; j < 4 && i + j < end; j++) f(plain_logit(x[i + j]), i + j);
}

__global__ __launch_bounds__(kThreads) void sample_top_kernel(SampleParams p)
{
    __shared__ u64 tops[kThreads / 64];
    const int row = int(blockIdx.x / unsigned(p.chunks)), chunk = int(blockIdx.x % unsigned(p.chunks));
    const int wave = threadIdx.x >> 6;
    // the row's bins start at nothing
    for (int i = chunk * kThreads + int(threadIdx.x); i < kBins; i += p.chunks * kThreads) {
        p.mass[size_t(row) * kBins + i] = 0;
        p.count[size_t(row) * kBins + i] = 0;
    }
    if (chunk == 0 && threadIdx.x == 0) p.listed[row] = 0;
    float best = -INFINITY;
    int at = p.vocab;
    for_segment(p, row, chunk * 4 + wave, [&](float x, int i) {
        if (x > best) {
            best = x;
            at = i;
        }
    });
    u64 t = u64(ordered(best)) << 32 | unsigned(~at);
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const u64 o = __shfl_xor(t, d, 64);
        t = o > t ? o : t;
    }
    if ((threadIdx.x & 63) == 0) tops[wave] = t;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 64; w++) t = tops[w] > t ? tops[w] : t;
        p.top[size_t(row) * p.chunks + chunk] = t;
    }
}

__global__ __launch_bounds__(kThreads) void sample_bins_kernel(SampleParams p)
{
    __shared__ u64 mass[kBins];
    __shared__ unsigned count[kBins];
    const int row = int(blockIdx.x / unsigned(p.chunks)), chunk = int(blockIdx.x % unsigned(p.chunks));
    const Row r = row_of(p, row);
    const float top = unordered(unsigned(row_top(p, row) >> 32));
    if (r.greedy || top == -INFINITY || !(r.has_k || r.has_p)) return;  // the whole workgroup
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        mass[i] = 0;
        count[i] = 0;
    }
    __syncthreads();
    for_segment(p, row, chunk * 4 + (threadIdx.x >> 6), [&](float x, int) {
        const double z = z_of(x, top, r.inverse);
        const int b = bin_of(z);
        if (b == kBins - 1) return;  // weighs 0
        atomicAdd(&count[b], 1u);
        if (r.has_p) atomicAdd(&mass[b], units_of(weight_of(z), p.unit));
    });
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        if (count[i] == 0) continue;
        atomicAdd(&p.count[size_t(row) * kBins + i], count[i]);
        if (r.has_p) atomicAdd(&p.mass[size_t(row) * kBins + i], mass[i]);
    }
}

// What the bins say. Tokens of bins under `low` are kept but for min-p; those of [low, high] and of `last`
// are listed; the others are not kept. last: the bin of top-k's cut (kBins: none, and then all tokens that
// weigh anything are in the first `kBins - 1` bins).
struct Cut {
    int low, high, last;
    unsigned before_last;      // tokens of the bins under `last`
    u64 mass_last, mass_low;   // weight of the bins under `last`, under `low`
};
struct CutShared {
    u64 part[4];
    int last, low, high;
    unsigned before_last, upto;
    u64 mass_last, mass_after, mass_low;
};

__device__ Cut cut_of(const SampleParams &p, int row, const Row &r, CutShared &sh)
{
    Cut c{kBins, kBins, kBins, 0, 0, 0};
    if (!(r.has_k || r.has_p)) {
        c.high = -1;
        return c;
    }
    const int tid = threadIdx.x;
    constexpr int kEach = kBins / kThreads;
    u64 n[kEach], m[kEach], here_n = 0, here_m = 0, all_n, all_m;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        n[i] = p.count[size_t(row) * kBins + tid * kEach + i];
        m[i] = p.mass[size_t(row) * kBins + tid * kEach + i];
        here_n += n[i];
        here_m += m[i];
    }
    const u64 before_n = block_before(here_n, sh.part, &all_n), before_m = block_before(here_m, sh.part, &all_m);
    __syncthreads();
    if (tid == 0) {
        sh.last = kBins;
        sh.low = sh.high = kBins - 1;
        sh.mass_last = sh.mass_after = all_m;
        sh.before_last = sh.upto = unsigned(all_n);
        sh.mass_low = 0;
    }
    __syncthreads();
    if (r.has_k && u64(r.top_k) < all_n) {  // (else every token that weighs anything is among the first top_k)
        u64 a = before_n, b = before_m;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            if (a < u64(r.top_k) && a + n[i] >= u64(r.top_k)) {
                sh.last = tid * kEach + i;
                sh.before_last = unsigned(a);
                sh.upto = unsigned(a + n[i]);
                sh.mass_last = b;
                sh.mass_after = b + m[i];
            }
            a += n[i];
            b += m[i];
        }
    }
    __syncthreads();
    c.last = sh.last;
    c.before_last = sh.before_last;
    c.mass_last = sh.mass_last;
    if (r.has_p) {
        // the cut's bin, for a total between the weight under `last` and that up to it
        const double least = double(r.top_p) * double(sh.mass_last) * (1.0 - 0x1p-50);
        const double most = double(r.top_p) * double(sh.mass_after) * (1.0 + 0x1p-50);
        u64 b = before_m;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            if (n[i]) {
                if (double(b) < least && double(b + m[i]) >= least) sh.low = tid * kEach + i;
                if (double(b) < most && double(b + m[i]) >= most) sh.high = tid * kEach + i;
                if (b == 0 && least <= 0.0) sh.low = 0;
            }
            b += m[i];
        }
        __syncthreads();
        c.low = sh.low;
        c.high = max(sh.high, sh.low);
        if (c.last < kBins) {
            c.high = min(c.high, c.last);
            c.low = min(c.low, c.high);
        }
    } else {
        c.low = c.high = c.last;
        if (c.last == kBins) c.high = -1;  // top_k of more tokens than weigh anything
    }
    // few tokens up to the last listed bin: all of them are listed
    const int end = c.last < kBins ? c.last : c.high;
    if (end >= 0 && end < kBins) {
        u64 a = before_n;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            a += n[i];
            if (tid * kEach + i == end) sh.upto = unsigned(a);
        }
        __syncthreads();
        if (sh.upto <= unsigned(kList)) {
            c.low = 0;
            c.high = end;
        }
        u64 b = before_m;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            if (tid * kEach + i == c.low) sh.mass_low = b;
            b += m[i];
        }
        __syncthreads();
        c.mass_low = sh.mass_low;
    }
    return c;
}

__device__ __forceinline__ bool is_listed(const Cut &c, int bin) { return (bin >= c.low && bin <= c.high) || bin == c.last; }

__global__ __launch_bounds__(kThreads) void sample_collect_kernel(SampleParams p)
{
    __shared__ CutShared sh;
    const int row = int(blockIdx.x / unsigned(p.chunks)), chunk = int(blockIdx.x % unsigned(p.chunks));
    const Row r = row_of(p, row);
    const float top = unordered(unsigned(row_top(p, row) >> 32));
    if (r.greedy || top == -INFINITY) return;  // the whole workgroup
    const Cut c = cut_of(p, row, r, sh);
    u64 sum = 0;
    const int segment = chunk * 4 + (threadIdx.x >> 6);
    for_segment(p, row, segment, [&](float x, int i) {
        const double z = z_of(x, top, r.inverse);
        const int b = bin_of(z);
        if (b == kBins - 1) return;
        if (b < c.low) {
            const double e = weight_of(z);
            if (!(e < double(r.min_p))) sum += units_of(e, p.unit);
        } else if (is_listed(c, b)) {
            const unsigned at = atomicAdd(&p.listed[row], 1u);
            if (at < unsigned(kList)) p.list[size_t(row) * kList + at] = u64(__float_as_uint(x)) << 32 | unsigned(i);
        }
    });
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) p.segments[size_t(row) * p.chunks * 4 + segment] = sum;
}

// One workgroup a row. The listed tokens are in LDS, or, if they are too many, found in the row again by
// every pass over them.
struct DrawShared {
    u64 key[kList];     // (~ordered logit, index): the order, ascending
    u64 weight[kList];
    u64 mass[256];
    unsigned count[256];
    u64 part[4];
    u64 chosen;         // the digit's results
    u64 mass_before;
    unsigned count_before, digit, inside;
    CutShared cut;
};

__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleParams p)
{
    extern __shared__ __align__(16) unsigned char memory[];
    DrawShared &sh = *reinterpret_cast<DrawShared *>(memory);
    const int row = int(blockIdx.x), tid = threadIdx.x;
    const Row r = row_of(p, row);
    const u64 t = row_top(p, row);
    const float top = unordered(unsigned(t >> 32));
    if (r.greedy || top == -INFINITY) {
        if (tid == 0) {
            p.tokens[row] = top == -INFINITY ? -1 : int(~unsigned(t));
            if (p.chances) p.chances[row] = top == -INFINITY ? 0.0f : 1.0f;
        }
        return;
    }
    if (tid == 0) {
        sh.chosen = sh.mass_before = 0;
        sh.count_before = sh.digit = sh.inside = 0;
    }
    const Cut c = cut_of(p, row, r, sh.cut);
    __syncthreads();
    const unsigned listed = c.high < 0 && c.last == kBins ? 0 : p.listed[row];
    const bool kept_here = listed <= unsigned(kList);
    const double least = double(r.min_p);
    // f(key, weight, bin) for the listed tokens
    auto for_listed = [&](auto f) {
        if (kept_here) {
            for (unsigned i = tid; i < listed; i += kThreads) {
                const float x = unordered(~unsigned(sh.key[i] >> 32));
                f(sh.key[i], sh.weight[i], bin_of(z_of(x, top, r.inverse)));
            }
            return;
        }
        const float *x = p.logits + size_t(row) * p.stride;
        for (int i = tid; i < p.vocab; i += kThreads) {
            const float v = plain_logit(x[i]);
            const double z = z_of(v, top, r.inverse);
            const int b = bin_of(z);
            if (b == kBins - 1 || !is_listed(c, b)) continue;
            f(u64(~ordered(v)) << 32 | unsigned(i), units_of(weight_of(z), p.unit), b);
        }
    };
    if (kept_here) {
        for (unsigned i = tid; i < listed; i += kThreads) {
            const u64 e = p.list[size_t(row) * kList + i];
            const float x = __uint_as_float(unsigned(e >> 32));
            sh.key[i] = u64(~ordered(x)) << 32 | unsigned(e);
            sh.weight[i] = units_of(weight_of(z_of(x, top, r.inverse)), p.unit);
        }
        __syncthreads();
    }
    // The key at which, in ascending order of key(token) among the tokens that `take` takes, the first
    // `count` tokens end (BY_COUNT), or the token on which the running weight first exceeds `mass`;
    // *mass_upto: the weight up to and with it. Eight bits of the key, of `bits`, at a time.
    auto select = [&](int bits, bool by_count, unsigned count, u64 mass, auto key, auto take, u64 *mass_upto) {
        u64 prefix = 0, mass_before = 0;
        unsigned count_before = 0;
        for (int shift = bits - 8; shift >= 0; shift -= 8) {
            sh.mass[tid] = 0;
            sh.count[tid] = 0;
            __syncthreads();
            for_listed([&](u64 k, u64 w, int b) {
                if (!take(k, w, b)) return;
                const u64 q = key(k);
                if (shift < bits - 8 && q >> (shift + 8) != prefix >> (shift + 8)) return;
                atomicAdd(&sh.count[(q >> shift) & 255], 1u);
                atomicAdd(&sh.mass[(q >> shift) & 255], w);
            });
            __syncthreads();
            const u64 m = sh.mass[tid];
            const unsigned n = sh.count[tid];
            u64 all;
            const u64 before = mass_before + block_before(m, sh.part, &all);
            const unsigned before_n = count_before + unsigned(block_before(n, sh.part, &all));
            if (by_count ? before_n < count && before_n + n >= count : before <= mass && before + m > mass) {
                sh.digit = tid;
                sh.inside = n;
                sh.mass_before = before;
                sh.count_before = before_n;
                sh.chosen = m;
            }
            __syncthreads();
            prefix |= u64(sh.digit) << shift;
            mass_before = sh.mass_before;
            count_before = sh.count_before;
            *mass_upto = mass_before + sh.chosen;
            const bool done = sh.inside == 1;
            __syncthreads();
            if (done) {  // one token: its key
                for_listed([&](u64 k, u64 w, int b) {
                    if (!take(k, w, b)) return;
                    const u64 q = key(k);
                    if (q >> shift == prefix >> shift) sh.chosen = q;
                });
                __syncthreads();
                const u64 q = sh.chosen;
                __syncthreads();
                return q;
            }
        }
        return prefix;
    };
    auto order = [](u64 k) { return k; };
    u64 cut = ~0ull, total = c.mass_last;
    if (c.last < kBins) {
        u64 upto;
        cut = select(64, true, unsigned(r.top_k) - c.before_last, 0, order, [&](u64, u64, int b) { return b == c.last; }, &upto);
        total = c.mass_last + upto;
    }
    if (r.has_p) {
        // the first token whose running weight reaches top_p of the total: exceeds the whole number before
        const double goal = double(r.top_p) * double(total);
        u64 over = u64(ceil(goal));
        over = over > 0 ? over - 1 : 0;
        over = over >= total ? total - 1 : over;
        over = over > c.mass_low ? over - c.mass_low : 0;
        u64 upto;
        const u64 k = select(64, false, 0, over, order, [&](u64 q, u64, int b) { return b >= c.low && b <= c.high && q <= cut; }, &upto);
        cut = k < cut ? k : cut;
    }
    // the kept weight: the segments', and the listed tokens up to the cut
    auto kept = [&](u64 k, double e) { return k <= cut && !(e < least); };
    auto keeps = [&](u64 k, u64, int) {
        return kept(k, weight_of(z_of(unordered(~unsigned(k >> 32)), top, r.inverse)));
    };
    const int segments = p.chunks * 4;
    const bool whole = c.low > 0;  // some bins are kept whole
    sh.mass[tid] = whole && tid < segments ? p.segments[size_t(row) * segments + tid] : 0;
    __syncthreads();
    for_listed([&](u64 k, u64 w, int b) {
        if (keeps(k, w, b)) atomicAdd(&sh.mass[whole ? unsigned(k) / unsigned(p.segment) : 0], w);
    });
    __syncthreads();
    u64 all;
    const u64 m = sh.mass[tid], before = block_before(m, sh.part, &all);
    float u = p.random[row];
    u = u > 0.0f ? u : 0.0f;  // (NaN too)
    u64 goal = u64(double(u) * double(all));
    goal = goal < all ? goal : all - 1;
    if (!whole) {
        u64 upto;
        const u64 k = select(24, false, 0, goal, [](u64 q) { return q & 0xFFFFFFFFull; }, keeps, &upto);
        // the token's weight
        for_listed([&](u64 q, u64 w, int) {
            if ((q & 0xFFFFFFFFull) == k) sh.mass_before = w;
        });
        __syncthreads();
        if (tid == 0) {
            p.tokens[row] = int(k);
            if (p.chances) p.chances[row] = float(double(sh.mass_before) / double(all));
        }
        return;
    }
    if (before <= goal && before + m > goal) {
        sh.digit = tid;
        sh.mass_before = before;
    }
    __syncthreads();
    // the segment again: a run of tokens a thread
    const int begin = int(sh.digit) * p.segment, end = min(begin + p.segment, p.vocab);
    goal -= sh.mass_before;
    const int run = (p.segment + kThreads - 1) / kThreads, first = begin + tid * run, last = min(first + run, end);
    const float *x = p.logits + size_t(row) * p.stride;
    auto units = [&](int i) {
        const float v = plain_logit(x[i]);
        const double z = z_of(v, top, r.inverse);
        const int b = bin_of(z);
        if (b == kBins - 1 || !(b < c.low || is_listed(c, b))) return u64(0);
        const double e = weight_of(z);
        if (e < least || (b >= c.low && !kept(u64(~ordered(v)) << 32 | unsigned(i), e))) return u64(0);
        return units_of(e, p.unit);
    };
    u64 mine = 0, sum;
    for (int i = first; i < last; i++) mine += units(i);
    u64 running = block_before(mine, sh.part, &sum);
    if (running <= goal && running + mine > goal) {
        for (int i = first; i < last; i++) {
            const u64 w = units(i);
            running += w;
            if (running > goal) {
                p.tokens[row] = i;
                if (p.chances) p.chances[row] = float(double(w) / double(all));
                break;
            }
        }
    }
}

}  // namespace
}  // namespace fg

using namespace fg;

extern "C" int fg_sample(const float *logits, size_t rows, size_t vocab, size_t stride, const fg_sampling *settings, int32_t *tokens,
                         float *chances, void *stream)
{
    if (rows > (size_t(1) << 20) || vocab > (size_t(1) << 22))
        return set_error(FG_ERR_SHAPE, "fg_sample: at most 2^20 rows and 2^22 logits a row");
    if (!vocab && rows) return set_error(FG_ERR_SHAPE, "fg_sample: rows of at least one logit");
    if (!settings) return set_error(FG_ERR_ARG, "fg_sample: null settings");
    if (!rows) return FG_OK;
    if (!logits || !tokens || !settings->random) return set_error(FG_ERR_ARG, "fg_sample: null logits, random numbers or tokens");
    const hipStream_t s = as_stream(stream);
    SampleParams p{};
    p.stride = stride;
    p.vocab = int(vocab);
    int bits = 0;
    while ((size_t(1) << bits) < vocab) bits++;
    p.unit = double(size_t(1) << std::min(45, 63 - bits));
    // rows of a batch: what the Infinity Cache (256 MB) holds beside the rest
    const size_t batch = std::max<size_t>(1, std::min(rows, (size_t(192) << 20) / (vocab * 4)));
    // workgroups enough to fill the chip, of at least 4096 logits
    p.chunks = int(std::min<size_t>({kMaxChunks, (2048 + batch - 1) / batch, (vocab + 4095) / 4096}));
    p.segment = int((vocab + size_t(p.chunks) * 4 - 1) / (size_t(p.chunks) * 4) + 255) / 256 * 256;
    const size_t sizes[6] = {batch * p.chunks * 8, batch * kBins * 8, batch * kBins * 4, batch * p.chunks * 32, batch * 4, batch * kList * 8};
    size_t at[7] = {0};
    for (int i = 0; i < 6; i++) at[i + 1] = at[i] + (sizes[i] + 255) / 256 * 256;
    static std::atomic<u64> raised{0};  // the devices where the draw's LDS limit is raised
    int device = 0;
    FG_HIP(hipGetDevice(&device));
    if (sizeof(DrawShared) > 64 * 1024 && (device > 63 || !(raised.load() >> device & 1))) {
        FG_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(sample_draw_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                   int(sizeof(DrawShared))));
        raised.fetch_or(u64(1) << (device & 63));
    }
    void *ws = nullptr;
    bool owned = false;
    FG_HIP(stream_scratch(at[6], s, &ws, &owned));
    char *base = static_cast<char *>(ws);
    p.top = reinterpret_cast<u64 *>(base + at[0]);
    p.mass = reinterpret_cast<u64 *>(base + at[1]);
    p.count = reinterpret_cast<unsigned *>(base + at[2]);
    p.segments = reinterpret_cast<u64 *>(base + at[3]);
    p.listed = reinterpret_cast<unsigned *>(base + at[4]);
    p.list = reinterpret_cast<u64 *>(base + at[5]);
    int rc = FG_OK;
    for (size_t r = 0; r < rows && rc == FG_OK; r += batch) {
        const unsigned n = unsigned(std::min(batch, rows - r)), grid = n * unsigned(p.chunks);
        p.logits = logits + r * stride;
        p.random = settings->random + r;
        p.temperature = settings->temperature ? settings->temperature + r : nullptr;
        p.top_k = settings->top_k ? settings->top_k + r : nullptr;
        p.top_p = settings->top_p ? settings->top_p + r : nullptr;
        p.min_p = settings->min_p ? settings->min_p + r : nullptr;
        p.tokens = tokens + r;
        p.chances = chances ? chances + r : nullptr;
        sample_top_kernel<<<grid, kThreads, 0, s>>>(p);
        if (p.top_k || p.top_p) sample_bins_kernel<<<grid, kThreads, 0, s>>>(p);
        sample_collect_kernel<<<grid, kThreads, 0, s>>>(p);
        sample_draw_kernel<<<n, kThreads, sizeof(DrawShared), s>>>(p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) rc = check_hip(e, "fg_sample");
    }
    if (owned) {
        const hipError_t e = hipFreeAsync(ws, s);
        if (rc == FG_OK && e != hipSuccess) rc = check_hip(e, "hipFreeAsync");
    }
    return rc;
}
