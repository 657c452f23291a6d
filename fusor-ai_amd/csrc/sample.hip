// Next tokens drawn from logits (fg_sample).
//
// A row's tokens are ordered by (logit descending, index ascending); temperature, top-k, top-p and min-p
// each keep a first part of that order, so what is kept ends at one token, the cut. No sort is needed to find
// it: the weights' logarithms z = (logit - largest) / temperature are counted and summed in kBins bins of
// 1/32, the bin of a cut follows from the running sums, and only that bin's tokens are looked at one by one.
//   1 top      the largest logit of each chunk of the row, and its first index;
//   2 bins     the tokens and the weight of every bin, chunk by chunk;
//   3 cut      from the bins, which are kept whole and which hold a cut, and the logits between them;
//   4 collect  a list of the tokens whose bins hold a cut (or of all tokens up to it, where they are few);
//   5 draw     the cut among the list; the chunk, or the listed token, on which the random number falls.
// Few rows take a launch for each, their chunks over the chip; many rows all five in one workgroup a row
// (sample_route.h).
// Weights are 64-bit: exp in f64 (off by |z| 2^-52 and a few 2^-53 of it, for z is rounded and two series are
// multiplied), rounded to a whole number of units of 2^-45 of the first token's (less for more than 2^18 tokens), so
// that every sum is exact and their order changes nothing. Tokens under half a unit (z < -31.9) weigh 0; the last
// bin holds only such. Equal logits have equal weights; which side of min-p a token within that error of it falls on
// is not decided.
//
// What it costs: a logit is read three times, by top, bins and collect (the draw reads one chunk more), mostly from
// the Infinity Cache after the first, and takes about 35 vector instructions in f64 and one 64-bit LDS addition in
// the bins. 64 rows of 151936 (39 MB): top 10.5 us, 3.7 TB/s; bins 17, the arithmetic (the vector units are busy
// 76 % of the time); cut 8.4; collect 9.4, 4.1 TB/s; draw 9.4. One row: 3.6, 6.0, 7.0, 3.8, 4.5: each launch is a
// chain of dependent steps on 1 to 16 CUs. In one workgroup a row, 512 rows 200 us: two rounds of 256, of cycles about
// 48 thousand top (memory's first reading), 100 bins (arithmetic), 50 collect and 30 the rest; 200 rows of 32003 35 us
// (8, 22, 10, 22). The vector units are busy half the time: one row's waits have no other row's work beside them.
//
// Where a cut's bin holds more tokens than a list (kList), the draw walks the row once for each pass over them,
// about ten a cut, by one workgroup: 151936 logits of spread s at temperature T, top-p 0.9, in microseconds,
// s / T = 0.7 and 0.5: one row 39 and 273, 64 rows 62 and 472, 512 rows 225 and 1052; with top-k 50000 too, s / T = 2 and 1:
// 42 and 463, 68 and 811, 233 and 1656. Of 262144 logits top-p alone does so at s / T = 1 (one row 39 and 453 for 2 and 1).
#include <algorithm>
#include <type_traits>

#include "cache.h"
#include "sample_bins.h"
#include "sample_route.h"

namespace fg {
namespace {

typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned long long u64;

constexpr int kThreads = 1024;      // of the kernels that walk a row, and of the draw
constexpr int kWaves = kThreads / 64;
constexpr int kList = 2560;         // tokens a row's list holds: what 64 KB of LDS hold beside the rest
constexpr int kRank = 128;          // up to so many listed tokens are compared with each other, all in one step
constexpr int kFew = 1024;          // up to so many tokens before the cut are all listed: no chunk is walked then
constexpr int kMaxChunks = kSampleChunks;
static_assert(kSampleRun == kThreads * 4, "a run is four tokens a thread");

// What the bins say of a row. Tokens of bins under `low` are kept whole; those of [low, high] and of
// `last` are listed; the others are not kept. last: the bin of top-k's cut (kBins: none).
struct Cut {
    int low, high, last;
    unsigned before_last;     // tokens of the bins under `last`
    u64 mass_last, mass_low;  // weight of the bins under `last`, under `low`
    // the smallest logits of the bins up to low - 1, high, last - 1 and last (NaN: of none)
    float whole, listed, before, tie;
    int lists, by_p;          // whether any bin is listed, and whether top-p's cut is in one
    int done;                 // whether the row's token is there already
    int top_k;
    float top_p;
    double top, scale, least;  // the largest logit, bins a logit, and the weight that min-p asks for
};

struct SampleParams {
    const float *logits;
    size_t stride;
    int vocab, chunks, chunk;    // chunk: tokens of a workgroup, whole runs of 256
    const float *random, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    double unit;                 // units of the first token's weight, a power of two
    u64 *top;                    // [rows][chunks]: (ordered logit, ~index)
    u64 *mass;                   // [rows][chunks][kBins]
    unsigned *count;             // [rows][chunks][kBins], where top_k asks
    u64 *whole;                  // [rows][chunks]: weight of a chunk's tokens kept whole
    Cut *cuts;                   // [rows]
    unsigned *listed;            // [rows]: tokens of the list (past kList: not all are in it)
    u64 *list;                   // [rows][kList]: (logit bits, index)
    int32_t *tokens;
    float *chances;
};

// A logit's place in the order of floats as an unsigned integer; NaN is -inf, and -0 is 0.
__device__ __forceinline__ float plain_logit(float x) { return fmaxf(x, -INFINITY) + 0.0f; }
__device__ __forceinline__ unsigned ordered(float x)
{
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }

// What a row asks for.
struct Row {
    double scale;    // bins a logit: 32 / temperature
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
    r.min_p = mp > 0.0f ? mp : 0.0f;
    r.greedy = !(t > 0.0f) || r.top_k == 1 || tp <= 0.0f || mp > 1.0f;
    r.scale = fmax(double(kPerUnit) / double(t), 1e-290);  // (an infinite temperature: every finite logit weighs 1)
    return r;
}

// exp(-(b + 1/2) / 32), a bin's middle: -(b + 1/2) / 32 = n ln 2 + r, the Taylor series of exp to r^12
// (|r| <= 0.347: the next term is under 2^-52 of it), times 2^n.
__device__ __forceinline__ double middle_of(int b)
{
    const double z = (double(b) + 0.5) * (-1.0 / kPerUnit);
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
// A weight exp(-t / 32), in the units of its bin's `middle`: that times exp(d / 32) for d = 1/2 less t's
// fraction, the Taylor series to d^6 (|d / 32| <= 2^-6: the next term is under 2^-54).
__device__ __forceinline__ double weight_of(double t, double middle)
{
    const double d = 0.5 - __builtin_amdgcn_fract(t);
    double e = 1.0 / 720.0 / 1073741824.0;
    e = __builtin_fma(e, d, 1.0 / 120.0 / 33554432.0);
    e = __builtin_fma(e, d, 1.0 / 24.0 / 1048576.0);
    e = __builtin_fma(e, d, 1.0 / 6.0 / 32768.0);
    e = __builtin_fma(e, d, 0.5 / 1024.0);
    e = __builtin_fma(e, d, 1.0 / 32.0);
    e = __builtin_fma(e, d, 1.0);
    return e * middle;
}
// Whole units: below 2^52 a sum with 2^52 rounds to them. (The first token's are exact: 2^45 and some
// 2^-7 of a unit.)
__device__ __forceinline__ u64 units_of(double weight)
{
    return u64(__double_as_longlong(weight + 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
}

// A value combined over the wave's lanes up to this one (DPP: rows of 16, then their last lanes); 0 changes
// nothing.
template <class F>
__device__ __forceinline__ u64 wave_combine(u64 v, F combine)
{
    auto step = [&](auto control, auto rows) {
        const unsigned lo = __builtin_amdgcn_update_dpp(0, int(unsigned(v)), decltype(control)::value, decltype(rows)::value, 0xF, false);
        const unsigned hi = __builtin_amdgcn_update_dpp(0, int(unsigned(v >> 32)), decltype(control)::value, decltype(rows)::value, 0xF, false);
        v = combine(v, u64(hi) << 32 | lo);
    };
    using All = std::integral_constant<int, 0xF>;
    step(std::integral_constant<int, 0x111>{}, All{});
    step(std::integral_constant<int, 0x112>{}, All{});
    step(std::integral_constant<int, 0x114>{}, All{});
    step(std::integral_constant<int, 0x118>{}, All{});
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
    return v;
}
__device__ __forceinline__ u64 wave_upto(u64 v)
{
    return wave_combine(v, [](u64 a, u64 b) { return a + b; });
}
__device__ __forceinline__ u64 wave_or(u64 v)
{
    return wave_combine(v, [](u64 a, u64 b) { return a | b; });
}
__device__ __forceinline__ u64 lane_of(u64 v, int lane)
{
    return u64(unsigned(__builtin_amdgcn_readlane(int(unsigned(v >> 32)), lane))) << 32 |
           unsigned(__builtin_amdgcn_readlane(int(unsigned(v)), lane));
}

// The workgroup's sum of a value before this thread's, and of all. `part` is LDS of a value a wave; every
// thread calls.
template <int WAVES>
__device__ __forceinline__ u64 block_before(u64 v, u64 *part, u64 *total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 x = wave_upto(v);
    __syncthreads();
    if (lane == 63) part[wave] = x;
    __syncthreads();
    const u64 sums = wave_upto(lane < WAVES ? part[lane] : 0);
    *total = lane_of(sums, WAVES - 1);
    return x - v + (wave ? lane_of(sums, __builtin_amdgcn_readfirstlane(wave) - 1) : 0);
}

// The row's largest logit from its chunks', (ordered logit, ~index); every wave by itself.
__device__ __forceinline__ u64 row_top(const SampleParams &p, int row)
{
    const int lane = threadIdx.x & 63;
    u64 t = p.top[size_t(row) * p.chunks + min(lane & 15, p.chunks - 1)];
#pragma unroll
    for (int d = 8; d; d >>= 1) {
        const u64 o = __shfl_xor(t, d, 64);
        t = o > t ? o : t;
    }
    return t;
}

// Calls f(logit, index) for the tokens [begin, end) of a row, four a thread of `threads`, the logits as they are
// there; the loads of several runs are asked for together.
template <class F>
__device__ __forceinline__ void for_tokens(const float *x, int begin, int end, int thread, int threads, F f)
{
    constexpr int kAhead = 4;
    int i = begin + thread * 4;
    for (; i + (kAhead - 1) * threads * 4 + 4 <= end; i += kAhead * threads * 4) {
        v4f v[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; a++) v[a] = *reinterpret_cast<const v4f_any *>(x + i + a * threads * 4);
#pragma unroll
        for (int a = 0; a < kAhead; a++)
#pragma unroll
            for (int j = 0; j < 4; j++) f(v[a][j], i + a * threads * 4 + j);
    }
    for (; i < end; i += threads * 4) {
        if (i + 4 <= end) {
            const v4f v = *reinterpret_cast<const v4f_any *>(x + i);
#pragma unroll
            for (int j = 0; j < 4; j++) f(v[j], i + j);
        } else {
            for (int j = 0; i + j < end; j++) f(x[i + j], i + j);
        }
    }
}

// The workgroup's row and chunk, and the chunk's tokens.
struct Place {
    int row, chunk, begin, end;
    const float *x;
};
__device__ __forceinline__ Place place_of(const SampleParams &p)
{
    Place a;
    a.row = int(blockIdx.x / unsigned(p.chunks));
    a.chunk = int(blockIdx.x % unsigned(p.chunks));
    a.begin = min(a.chunk * p.chunk, p.vocab);
    a.end = min(a.begin + p.chunk, p.vocab);
    a.x = p.logits + size_t(a.row) * p.stride;
    return a;
}

// The largest logit of the tokens [begin, end) and its first index, (ordered logit, ~index), to every thread of
// the workgroup. `part` is LDS of a value a wave.
__device__ __forceinline__ u64 top_of_tokens(const float *x, int begin, int end, int none, u64 *part)
{
    float best = -INFINITY;
    int at = none;
    for_tokens(x, begin, end, threadIdx.x, kThreads, [&](float v, int i) {
        if (v > best) {  // (not NaN; a zero of either sign is the first one's equal)
            best = v;
            at = i;
        }
    });
    u64 t = u64(ordered(plain_logit(best))) << 32 | unsigned(~at);
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const u64 o = __shfl_xor(t, d, 64);
        t = o > t ? o : t;
    }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = t;
    __syncthreads();
    t = part[threadIdx.x & (kWaves - 1)];
#pragma unroll
    for (int d = kWaves / 2; d; d >>= 1) {
        const u64 o = __shfl_xor(t, d, 64);
        t = o > t ? o : t;
    }
    return t;
}

// A token added to the bins' weights, and with top-k to their counts (LDS).
__device__ __forceinline__ void add_to_bins(float v, double top, double scale, bool counts, u64 *mass, unsigned *count,
                                            const double *middles)
{
    const double t = bins_of(fmaxf(v, -INFINITY), top, scale);
    const int b = bin_of(t);
    const u64 w = units_of(weight_of(t, middles[b]));
    if (b < kBins - 1) {  // (the last bin's weigh 0)
        if (counts) atomicAdd(&count[b], 1u);
        atomicAdd(&mass[b], w);
    }
}

// The token of a row that keeps its first alone, or has no logit above -inf.
__device__ __forceinline__ void write_first(const SampleParams &p, int row, u64 first)
{
    const bool none = unordered(unsigned(first >> 32)) == -INFINITY;
    p.tokens[row] = none ? -1 : int(~unsigned(first));
    if (p.chances) p.chances[row] = none ? 0.0f : 1.0f;
}

__global__ __launch_bounds__(kThreads) void sample_top_kernel(SampleParams p)
{
    __shared__ u64 part[kWaves];
    const Place a = place_of(p);
    if (a.chunk == 0 && threadIdx.x == 0) p.listed[a.row] = 0;
    const u64 t = top_of_tokens(a.x, a.begin, a.end, p.vocab, part);
    if (threadIdx.x == 0) p.top[size_t(a.row) * p.chunks + a.chunk] = t;
}

__global__ __launch_bounds__(kThreads) void sample_bins_kernel(SampleParams p)
{
    __shared__ u64 mass[kBins];
    __shared__ unsigned count[kBins];
    __shared__ double middles[kBins];
    const Place a = place_of(p);
    const Row r = row_of(p, a.row);
    const float first = unordered(unsigned(row_top(p, a.row) >> 32));
    if (r.greedy || first == -INFINITY) return;  // the whole workgroup
    const int tid = threadIdx.x;
    static_assert(kBins == kThreads, "a bin a thread");
    mass[tid] = 0;
    count[tid] = 0;
    middles[tid] = middle_of(tid) * p.unit;
    __syncthreads();
    const double top = top_of(first);
    for_tokens(a.x, a.begin, a.end, tid, kThreads, [&](float v, int) { add_to_bins(v, top, r.scale, r.has_k, mass, count, middles); });
    __syncthreads();
    const size_t at = (size_t(a.row) * p.chunks + a.chunk) * kBins + tid;
    p.mass[at] = mass[tid];
    if (r.has_k) p.count[at] = count[tid];
}

struct CutShared {
    u64 part[kWaves];
    int last, low, high;
    unsigned before_last, upto;
    u64 mass_last, mass_after, mass_low;
    u64 whole[kMaxChunks];
    float edge[4];
};

// The smallest logit whose bin is at most b: among the 64 floats around the bin's far end, or (rounding, next to 0,
// may have put it elsewhere) by dividing the order of floats 64 ways at a time.
__device__ __forceinline__ float smallest_of_bin(int b, float first, double scale)
{
    if (b >= kBins - 1) return -INFINITY;
    if (b < 0) return __builtin_nanf("");  // nothing is >= NaN
    const int lane = threadIdx.x & 63;
    const double top = top_of(first);
    auto within = [&](float x) { return bin_of(bins_of(x, top, scale)) <= b && x > -INFINITY; };
    unsigned lo = 0, n = ordered(first);  // the answer is in (lo, lo + n]; the first token has bin 0
    const unsigned near = ordered(plain_logit(float(top - double(b + 1) / scale)));
    if (near > 32 && near < n) {
        const unsigned at = min(near - 32 + unsigned(lane), n);
        const u64 yes = __ballot(within(plain_logit(unordered(at))));
        if (yes && !(yes & 1)) return unordered(near - 32 + unsigned(__builtin_ctzll(yes)));
    }
    while (n > 1) {
        const unsigned step = (n + 63) / 64, at = lo + (lane + 1) * step;
        const bool inside = u64(lane + 1) * step <= n;
        const float x = plain_logit(unordered(inside ? at : lo + n));
        const bool yes = within(x);
        const int k = __builtin_ctzll(__ballot(yes || !inside) | 1ull << 63);
        const unsigned from = lo + unsigned(k) * step, to = lo + n;
        lo = from;
        n = min(step, to - from);
    }
    return unordered(lo + n);
}

// The cuts of a row, from the weight m and the tokens n of this thread's bin. `mass` is its bins' weights in
// memory, [chunks][kBins], written before the workgroup's last barrier: of each chunk or (running) of each and those
// before it. Every thread of the workgroup calls and gets the result; sh.whole has the chunks' weight of whole bins.
__device__ __forceinline__ Cut cut_of(const SampleParams &p, const Row &r, float top, u64 m, u64 n, CutShared &sh, const u64 *mass,
                                      bool running)
{
    const int tid = threadIdx.x;
    u64 all_n = 0, all_m, before_n = 0;
    const u64 before_m = block_before<kWaves>(m, sh.part, &all_m);
    if (r.has_k) before_n = block_before<kWaves>(n, sh.part, &all_n);
    if (tid == 0) {
        sh.last = kBins;
        sh.low = sh.high = kBins - 1;
        sh.mass_last = sh.mass_after = all_m;
        sh.before_last = sh.upto = 0;
        sh.mass_low = all_m;
    }
    if (tid < kMaxChunks) sh.whole[tid] = 0;
    if (tid < 4) sh.edge[tid] = __builtin_nanf("");  // (of none, where nothing is listed)
    __syncthreads();
    // (top_k of all that weigh anything, or more: no cut)
    if (r.has_k && u64(r.top_k) < all_n && before_n < u64(r.top_k) && before_n + n >= u64(r.top_k)) {
        sh.last = tid;
        sh.before_last = unsigned(before_n);
        sh.upto = unsigned(before_n + n);
        sh.mass_last = before_m;
        sh.mass_after = before_m + m;
    }
    __syncthreads();
    Cut c{kBins, -1, sh.last, sh.before_last, sh.mass_last, 0, 0.0f, 0.0f, 0.0f, 0.0f, 0, r.has_p, 0, r.top_k, r.top_p,
          top_of(top), r.scale, double(r.min_p) * (1.0 - 0x1p-50) * p.unit};  // (a little less, for the first's equals at min_p = 1)
    if (r.has_p) {
        // the cut's bin, for a total between the weight under `last` and that up to it
        const double least = double(r.top_p) * double(sh.mass_last) * (1.0 - 0x1p-50);
        const double most = double(r.top_p) * double(sh.mass_after) * (1.0 + 0x1p-50);
        if (m) {
            if ((before_m == 0 || double(before_m) < least) && double(before_m + m) >= least) sh.low = tid;
            if ((before_m == 0 || double(before_m) < most) && double(before_m + m) >= most) sh.high = tid;
        }
        __syncthreads();
        c.high = min(max(sh.high, sh.low), c.last);
        c.low = min(sh.low, c.high);
    } else if (c.last < kBins) {
        c.low = c.high = c.last;
    }
    if (r.min_p > 0.0f) {
        // min-p's cut is in the bins of ln(min_p), to more than the rounding of weights
        const double t = log(double(r.min_p)) * -double(kPerUnit);
        const int first = bin_of(t > 1e-9 ? t - 1e-9 : 0.0), last = bin_of(t + 1e-9);
        if (last < c.low) {  // before any other cut: the others change nothing
            c.low = first;
            c.high = last;
            c.last = kBins;
            c.by_p = 0;
        } else if (first <= c.high) {
            c.low = min(c.low, first);
        }
    }
    const bool lists = c.high >= 0;
    if (lists) {
        c.high = min(c.high, kBins - 2);  // (the last bin's tokens weigh 0)
        c.low = min(c.low, c.high);
    }
    // few tokens up to top-k's bin, or (counted with top-k) up to the last cut's: all of them are listed
    if (lists && c.last < kBins && sh.upto <= unsigned(kFew)) {
        c.low = 0;
        c.high = c.last;
    }
    if (lists && c.last == kBins && r.has_k) {
        if (tid == c.high) sh.upto = unsigned(before_n + n);
        __syncthreads();
        if (sh.upto <= unsigned(kFew)) c.low = 0;
    }
    if (tid == c.low) sh.mass_low = before_m;
    const int wave = tid >> 6, lane = tid & 63;
    // the chunks' weight under `low`, a wave each
    static_assert(kMaxChunks == kWaves, "a wave a chunk");
    if (c.low > 0 && wave < p.chunks) {
        const ulonglong2 *of = reinterpret_cast<const ulonglong2 *>(mass + size_t(wave) * kBins);
        u64 w = 0;
#pragma unroll
        for (int i = 0; i < kBins; i += 128) {
            const ulonglong2 two = of[i / 2 + lane];
            w += (i + 2 * lane < c.low ? two.x : 0) + (i + 2 * lane + 1 < c.low ? two.y : 0);
        }
        w = wave_upto(w);
        if (lane == 63) sh.whole[wave] = w;
    }
    const int edge = wave == 0 ? c.low - 1 : wave == 1 ? c.high : wave == 2 ? c.last - 1 : c.last;
    if (lists && wave < 4) {
        const float x = smallest_of_bin(edge, top, r.scale);
        if (lane == 0) sh.edge[wave] = x;
    }
    __syncthreads();
    if (running) {
        const u64 before = tid > 0 && tid < p.chunks ? sh.whole[tid - 1] : 0;
        __syncthreads();
        if (tid < p.chunks) sh.whole[tid] -= before;
    }
    c.mass_low = sh.mass_low;
    c.lists = lists;
    c.whole = sh.edge[0];
    c.listed = sh.edge[1];
    c.before = sh.edge[2];
    c.tie = c.last < kBins ? sh.edge[3] : __builtin_nanf("");
    return c;
}

// One workgroup a row, a bin a thread.
__global__ __launch_bounds__(kThreads) void sample_cut_kernel(SampleParams p)
{
    __shared__ CutShared sh;
    const int row = int(blockIdx.x), tid = threadIdx.x;
    // everything is asked for at once (past the last chunk that one's again), and looked at then
    const u64 *mass = p.mass + size_t(row) * p.chunks * kBins + tid;
    const unsigned *count = p.count + size_t(row) * p.chunks * kBins + tid;
    u64 masses[kMaxChunks];
    unsigned counts[kMaxChunks] = {};
#pragma unroll
    for (int c = 0; c < kMaxChunks; c++) masses[c] = mass[min(c, p.chunks - 1) * kBins];
    if (p.top_k) {
#pragma unroll
        for (int c = 0; c < kMaxChunks; c++) counts[c] = count[min(c, p.chunks - 1) * kBins];
    }
    const Row r = row_of(p, row);
    u64 m = 0, n = 0;
#pragma unroll
    for (int c = 0; c < kMaxChunks; c++) {
        m += c < p.chunks ? masses[c] : 0;
        n += c < p.chunks ? counts[c] : 0;
    }
    const u64 first = row_top(p, row);
    const float top = unordered(unsigned(first >> 32));
    if (r.greedy || top == -INFINITY) {  // (its bins are not written: what was read is not used)
        if (tid == 0) {
            write_first(p, row, first);
            p.cuts[row].done = 1;
            p.cuts[row].lists = 0;
        }
        return;
    }
    const Cut c = cut_of(p, r, top, m, n, sh, p.mass + size_t(row) * p.chunks * kBins, false);
    if (tid < p.chunks) p.whole[size_t(row) * p.chunks + tid] = sh.whole[tid];
    if (tid == 0) p.cuts[row] = c;
}

__device__ __forceinline__ bool is_listed(const Cut &c, int bin) { return (bin >= c.low && bin <= c.high) || bin == c.last; }
// No token under it is listed, or of a bin that is kept whole: most of a row is passed over by one comparison.
__device__ __forceinline__ float floor_of(const Cut &c) { return c.lists ? fminf(c.listed, c.tie) : -INFINITY; }

// The listed ones of the tokens [begin, end) into `found` (LDS, kList of them), (logit bits, index); *count is
// how many there are.
__device__ __forceinline__ void list_tokens(const float *x, int begin, int end, const Cut &c, u64 *found, unsigned *count)
{
    const float whole = c.whole, listed = c.listed, before = c.before, tie = c.tie, floor = floor_of(c);
    for_tokens(x, begin, end, threadIdx.x, kThreads, [&](float v, int i) {
        if (!(v >= floor)) return;  // (NaN too)
        if (!((v >= listed && !(v >= whole)) || (v >= tie && !(v >= before)))) return;
        const unsigned at = atomicAdd(count, 1u);
        if (at < unsigned(kList)) found[at] = u64(__float_as_uint(plain_logit(v))) << 32 | unsigned(i);
    });
}

__global__ __launch_bounds__(kThreads) void sample_collect_kernel(SampleParams p)
{
    __shared__ u64 found[kList];
    __shared__ unsigned count, base;
    const Place a = place_of(p);
    const Cut &c = p.cuts[a.row];
    if (!c.lists) return;  // the whole workgroup
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    list_tokens(a.x, a.begin, a.end, c, found, &count);
    __syncthreads();
    const unsigned n = count;
    if (n == 0) return;
    if (threadIdx.x == 0) base = atomicAdd(&p.listed[a.row], n);
    __syncthreads();
    for (unsigned i = threadIdx.x; i < n && i < unsigned(kList); i += kThreads)
        if (base + i < unsigned(kList)) p.list[size_t(a.row) * kList + base + i] = found[i];
}

// The running weight that top-p's first token passes, of a total: the first whose sum reaches top_p of it exceeds the
// whole number before.
__device__ __forceinline__ u64 weight_over(const Cut &c, u64 total)
{
    u64 over = u64(ceil(double(c.top_p) * double(total)));
    over = over > 0 ? over - 1 : 0;
    return over >= total ? total - 1 : over;
}

// The running total that the drawn token passes, of the kept one.
__device__ __forceinline__ u64 goal_of(const SampleParams &p, int row, u64 all)
{
    float u = p.random[row];
    u = u > 0.0f ? u : 0.0f;  // (NaN too)
    const u64 goal = u64(double(u < 1.0f ? u : 1.0f) * double(all));
    return goal < all ? goal : all - 1;
}

struct DrawShared {
    u64 key[kList];     // (~ordered logit, index): the order, ascending
    u64 weight[kList];
    unsigned short bin[kList];
    u64 mass[256];
    unsigned count[256];
    u64 part[kWaves];
    ulonglong2 ranked[kRank];  // few tokens' keys and weights
    u64 before[kRank];         // the weight and the number of tokens before each
    unsigned tokens[kRank];
    u64 chosen;         // the digit's results
    u64 mass_before;
    unsigned count_before, digit, inside;
    double middles[kBins];
};

// A row's token from its cuts, where no bin is kept whole and the list is of at most kRank tokens, (logit bits, index)
// in sh.key: put in order by counting for each those before it, a wave then finds the cuts in the running
// sums, and each kept one's running total by index is the sum of the kept ones of lower index.
__device__ __forceinline__ void draw_few(const SampleParams &p, int row, const Cut &c, int listed, DrawShared &sh)
{
    const int tid = threadIdx.x, lane = tid & 63;
    const int width = listed <= 64 ? 64 : 128, rounds = kThreads / width, i = tid & (width - 1), part = tid / width;
    u64 key = ~0ull, w = 0;
    unsigned note = 0;  // the bin, and whether the weight is under min-p's
    if (tid < listed) {
        const u64 e = sh.key[tid];
        const float v = __uint_as_float(unsigned(e >> 32));
        const double t = bins_of(v, c.top, c.scale);
        const int b = bin_of(t);
        const double weight = weight_of(t, middle_of(b) * p.unit);
        key = u64(~ordered(v)) << 32 | unsigned(e);
        w = units_of(weight);
        note = unsigned(b) | (weight < c.least ? 0x10000u : 0u);
    }
    if (tid < width) {
        sh.ranked[tid] = ulonglong2{key, 0};
        sh.tokens[tid] = 0;
        sh.before[tid] = 0;
    }
    __syncthreads();
    {
        const u64 q = sh.ranked[i].x;
        unsigned n = 0;
#pragma unroll 4
        for (int j = part; j < listed; j += rounds) n += sh.ranked[j].x < q;
        if (i < listed) atomicAdd(&sh.tokens[i], n);
    }
    __syncthreads();
    if (tid < listed) {
        const unsigned at = sh.tokens[tid];
        sh.ranked[at] = ulonglong2{key, w};
        sh.count[at] = note;
    }
    __syncthreads();
    if (tid < 64) {  // two tokens a lane, in order
        const int at = 2 * lane;
        ulonglong2 a[2];
        int bin[2];
        bool light[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const bool there = at + k < listed;
            a[k] = there ? sh.ranked[at + k] : ulonglong2{~0ull, 0};
            bin[k] = there ? int(sh.count[at + k] & 0xFFFF) : kBins;
            light[k] = !there || (sh.count[at + k] & 0x10000u) != 0;
        }
        // the place and the running weight of the token of which hit(k) holds, in the sums of the tokens that take(k)
        // takes; hit is given the running weight before it
        auto find = [&](auto take, auto hit, u64 *upto) {
            const u64 w0 = take(0) ? a[0].y : 0, w1 = take(1) ? a[1].y : 0;
            const u64 sum = wave_upto(w0 + w1), before = sum - w0 - w1;
            const bool hit0 = take(0) && hit(0, before, w0), hit1 = take(1) && hit(1, before + w0, w1);
            const u64 lanes = __ballot(hit0 || hit1);
            const int from = lanes ? __builtin_ctzll(lanes) : 63;
            *upto = lane_of(hit0 ? before + w0 : sum, from);
            return __builtin_amdgcn_readlane(hit0 ? at : at + 1, from);
        };
        int cut = kRank;
        u64 total = c.mass_last;
        if (c.last < kBins) {
            const int n0 = bin[0] == c.last, n1 = bin[1] == c.last, need = c.top_k - int(c.before_last);
            int ignored;
            const int count = wave_scan(n0 + n1, &ignored);
            u64 upto;
            cut = find([&](int k) { return bin[k] == c.last; }, [&](int k, u64, u64) { return (k ? count : count - n1) == need; }, &upto);
            total = c.mass_last + upto;
        }
        if (c.by_p) {
            const u64 over = weight_over(c, total);
            u64 upto;
            const int k = find([&](int k) { return bin[k] <= c.high && at + k <= cut; },
                               [&](int, u64 before, u64 w) { return before <= over && before + w > over; }, &upto);
            cut = min(cut, k);
        }
        const bool keep0 = at <= cut && !light[0], keep1 = at + 1 <= cut && !light[1];
        const u64 w0 = keep0 ? a[0].y : 0, w1 = keep1 ? a[1].y : 0;
        const u64 all = lane_of(wave_upto(w0 + w1), 63);
        if (at < listed) sh.ranked[at] = ulonglong2{a[0].x & 0xFFFFFFFFull, w0};
        if (at + 1 < listed) sh.ranked[at + 1] = ulonglong2{a[1].x & 0xFFFFFFFFull, w1};
        if (lane == 0) sh.mass_before = all;
    }
    __syncthreads();
    const u64 all = sh.mass_before, goal = goal_of(p, row, all);
    if (i < listed) {
        const u64 q = sh.ranked[i].x;
        u64 m = 0;
#pragma unroll 4
        for (int j = part; j < listed; j += rounds) {
            const ulonglong2 other = sh.ranked[j];
            m += other.x < q ? other.y : 0;
        }
        atomicAdd(&sh.before[i], m);
    }
    __syncthreads();
    if (tid < listed) {
        const ulonglong2 mine = sh.ranked[tid];
        const u64 before = sh.before[tid];
        if (before <= goal && before + mine.y > goal) {
            p.tokens[row] = int(mine.x);
            if (p.chances) p.chances[row] = float(double(mine.y) / double(all));
        }
    }
}

// A row's token from its cuts, by one workgroup. The list's `listed` tokens are (logit bits, index) in sh.key, or,
// if they are too many, found in the row again by every pass over them. whole_of(k): the weight of chunk k's
// whole bins.
template <class F>
__device__ __forceinline__ void draw_token(const SampleParams &p, int row, const Cut &c, unsigned listed, DrawShared &sh, F whole_of)
{
    if (c.low == 0 && listed <= unsigned(kRank)) {
        __syncthreads();  // (the list is there)
        draw_few(p, row, c, int(listed), sh);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const double top = c.top, scale = c.scale, least = c.least;
    if (tid == 0) {
        sh.chosen = sh.mass_before = 0;
        sh.count_before = sh.digit = sh.inside = 0;
    }
    const float *x = p.logits + size_t(row) * p.stride;
    const bool kept_here = listed <= unsigned(kList);
    auto weight = [&](double t, int b) { return weight_of(t, middle_of(b) * p.unit); };
    // f(key, weight, bin) for the listed tokens
    auto for_listed = [&](auto f) {
        if (kept_here) {
            for (unsigned i = tid; i < listed; i += kThreads) {
                f(sh.key[i], sh.weight[i], int(sh.bin[i]));
            }
            return;
        }
        for (int i = tid; i < p.vocab; i += kThreads) {
            const float v = plain_logit(x[i]);
            const double t = bins_of(v, top, scale);
            const int b = bin_of(t);
            if (b == kBins - 1 || !is_listed(c, b)) continue;
            f(u64(~ordered(v)) << 32 | unsigned(i), units_of(weight(t, b)), b);
        }
    };
    if (kept_here) {
        for (unsigned i = tid; i < listed; i += kThreads) {
            const u64 e = sh.key[i];
            const float v = __uint_as_float(unsigned(e >> 32));
            sh.key[i] = u64(~ordered(v)) << 32 | unsigned(e);
            const double t = bins_of(v, top, scale);
            sh.weight[i] = units_of(weight(t, bin_of(t)));
            sh.bin[i] = (unsigned short)(bin_of(t));
        }
    }
    __syncthreads();
    // The key at which, in ascending order of key(token) among the tokens that `take` takes, the first
    // `count` tokens end (by_count), or the token on which the running weight first exceeds `mass`;
    // *mass_upto: the weight up to and with it. Few tokens: each against all others, by as many threads a
    // token as there are. Many: eight bits of the key, of `bits`, at a time.
    auto select = [&](bool by_count, unsigned count, u64 mass, auto key, auto take, u64 *mass_upto) {
        if (kept_here && listed <= unsigned(kRank)) {
            int width = 64;  // threads of a round: one a token
            while (width < int(listed)) width *= 2;
            const int i = tid & (width - 1), rounds = kThreads / width;
            if (tid < kRank) {
                sh.before[tid] = 0;
                sh.tokens[tid] = 0;
            }
            __syncthreads();
            if (tid < kRank) {
                const bool taken = tid < int(listed) && take(sh.key[tid], sh.weight[tid], sh.bin[tid]);
                sh.ranked[tid] = taken ? ulonglong2{key(sh.key[tid]), sh.weight[tid]} : ulonglong2{~0ull, 0};
            }
            __syncthreads();
            const u64 q = sh.ranked[i].x;
            const bool mine = q != ~0ull;
            if (mine) {
                u64 m = 0;
                unsigned n = 0;
#pragma unroll 4
                for (int j = tid / width; j < width; j += rounds) {
                    const ulonglong2 other = sh.ranked[j];
                    const bool sooner = other.x < q;
                    m += sooner ? other.y : 0;
                    n += sooner;
                }
                atomicAdd(&sh.before[i], m);
                atomicAdd(&sh.tokens[i], n);
            }
            __syncthreads();
            if (tid < width && mine) {
                const u64 m = sh.before[i], w = sh.ranked[i].y;
                if (by_count ? sh.tokens[i] + 1 == count : m <= mass && m + w > mass) {
                    sh.chosen = q;
                    sh.mass_before = m + w;
                }
            }
            __syncthreads();
            const u64 found = sh.chosen;
            *mass_upto = sh.mass_before;
            __syncthreads();
            return found;
        }
        // the bits that some key has, and that some key has not: both are where the keys differ
        if (tid < 2) sh.before[tid] = 0;
        __syncthreads();
        u64 ones = 0, zeros = 0;
        for_listed([&](u64 k, u64 w, int b) {
            if (take(k, w, b)) {
                ones |= key(k);
                zeros |= ~key(k);
            }
        });
        ones = wave_or(ones);
        zeros = wave_or(zeros);
        if (lane == 63) {
            atomicOr(&sh.before[0], ones);
            atomicOr(&sh.before[1], zeros);
        }
        __syncthreads();
        ones = sh.before[0];
        const u64 differ = ones & sh.before[1];
        const int start = differ ? max(56 - __builtin_clzll(differ), 0) : 0;
        u64 prefix = start + 8 < 64 ? ones >> (start + 8) << (start + 8) : 0, mass_before = 0;
        unsigned count_before = 0;
        for (int shift = start, above = start + 8;;) {  // the key's bits from `shift` up to `above`
            const u64 known = above < 64 ? prefix >> above : 0;
            const unsigned digits = (1u << (above - shift)) - 1;
            if (tid < 256) {
                sh.mass[tid] = 0;
                sh.count[tid] = 0;
            }
            __syncthreads();
            for_listed([&](u64 k, u64 w, int b) {
                if (!take(k, w, b)) return;
                const u64 q = key(k);
                if (above < 64 && q >> above != known) return;
                const unsigned digit = unsigned(q >> shift) & digits;
                atomicAdd(&sh.count[digit], 1u);
                atomicAdd(&sh.mass[digit], w);
            });
            __syncthreads();
            if (wave == 0) {  // four digits a lane
                u64 m[4], sum = 0;
                unsigned n[4], tokens = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    sum += m[i] = sh.mass[lane * 4 + i];
                    tokens += n[i] = sh.count[lane * 4 + i];
                }
                int all;
                u64 before = mass_before + wave_upto(sum) - sum;
                unsigned before_n = count_before + unsigned(wave_scan(int(tokens), &all)) - tokens;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (by_count ? before_n < count && before_n + n[i] >= count : before <= mass && before + m[i] > mass) {
                        sh.digit = lane * 4 + i;
                        sh.inside = n[i];
                        sh.mass_before = before;
                        sh.count_before = before_n;
                        sh.chosen = m[i];
                    }
                    before += m[i];
                    before_n += n[i];
                }
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
            if (shift == 0) return prefix;
            above = shift;
            shift = max(shift - 8, 0);
        }
    };
    auto order = [](u64 k) { return k; };
    u64 cut = ~0ull, total = c.mass_last;
    if (c.last < kBins) {
        u64 upto;
        cut = select(true, unsigned(c.top_k) - c.before_last, 0, order, [&](u64, u64, int b) { return b == c.last; }, &upto);
        total = c.mass_last + upto;
    }
    if (c.by_p) {
        u64 over = weight_over(c, total);
        over = over > c.mass_low ? over - c.mass_low : 0;
        u64 upto;
        const u64 k = select(false, 0, over, order, [&](u64 q, u64, int b) { return b >= c.low && b <= c.high && q <= cut; }, &upto);
        cut = k < cut ? k : cut;
    }
    // the kept weight: the chunks', and the listed tokens up to the cut
    auto kept = [&](u64 k, double e) { return k <= cut && !(e < least); };
    auto keeps = [&](u64 k, u64, int b) {
        return k <= cut && (least == 0.0 || kept(k, weight(bins_of(unordered(~unsigned(k >> 32)), top, scale), b)));
    };
    const bool whole = c.low > 0;  // some bins are kept whole
    if (tid < 256) sh.mass[tid] = whole && tid < p.chunks ? whole_of(tid) : 0;
    __syncthreads();
    for_listed([&](u64 k, u64 w, int b) {
        if (keeps(k, w, b)) atomicAdd(&sh.mass[whole ? unsigned(k) / unsigned(p.chunk) : 0], w);
    });
    __syncthreads();
    u64 all;
    const u64 m = tid < 256 ? sh.mass[tid] : 0, before = block_before<kWaves>(m, sh.part, &all);
    u64 goal = goal_of(p, row, all);
    if (!whole) {
        u64 upto;
        const u64 k = select(false, 0, goal, [](u64 q) { return q & 0xFFFFFFFFull; }, keeps, &upto);
        for_listed([&](u64 q, u64 w, int) {
            if ((q & 0xFFFFFFFFull) == k) sh.mass_before = w;  // the token's weight
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
    sh.middles[tid] = middle_of(tid) * p.unit;
    // the chunk again: which wave's part of it, then which token of that
    __syncthreads();
    const int begin = int(sh.digit) * p.chunk, end = min(begin + p.chunk, p.vocab);
    goal -= sh.mass_before;
    const float floor = floor_of(c);
    auto units = [&](float x, int i) {
        if (!(x >= floor)) return u64(0);
        const float v = plain_logit(x);
        const double t = bins_of(v, top, scale);
        const int b = bin_of(t);
        if (b == kBins - 1 || !(b < c.low || is_listed(c, b))) return u64(0);
        const double e = weight_of(t, sh.middles[b]);
        if (b >= c.low && !kept(u64(~ordered(v)) << 32 | unsigned(i), e)) return u64(0);
        return units_of(e);
    };
    const int share = (p.chunk + kThreads * 4 - 1) / (kThreads * 4) * 256;  // tokens of a wave's part
    u64 sum = 0, ignored;
    for_tokens(x, begin + wave * share, min(begin + (wave + 1) * share, end), lane, 64, [&](float v, int i) { sum += units(v, i); });
    sum = lane_of(wave_upto(sum), 63);
    const u64 first = block_before<kWaves>(lane == 0 ? sum : 0, sh.part, &ignored);
    if (lane == 0 && first <= goal && first + sum > goal) {
        sh.digit = wave;
        sh.mass_before = first;
    }
    __syncthreads();
    goal -= sh.mass_before;
    const int part = begin + int(sh.digit) * share, part_end = min(part + share, end);
    const int run = (share + kThreads - 1) / kThreads, i0 = part + tid * run, i1 = min(i0 + run, part_end);
    u64 mine = 0;
    for (int i = i0; i < i1; i++) mine += units(x[i], i);
    u64 running = block_before<kWaves>(mine, sh.part, &ignored);
    if (running <= goal && running + mine > goal) {
        for (int i = i0; i < i1; i++) {
            const u64 w = units(x[i], i);
            running += w;
            if (running > goal) {
                p.tokens[row] = i;
                if (p.chances) p.chances[row] = float(double(w) / double(all));
                break;
            }
        }
    }
}

// One workgroup a row.
__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleParams p)
{
    __shared__ DrawShared sh;
    const int row = int(blockIdx.x);
    const Cut c = p.cuts[row];
    if (c.done) return;
    const unsigned listed = c.lists ? p.listed[row] : 0;
    for (unsigned i = threadIdx.x; i < min(listed, unsigned(kList)); i += kThreads) sh.key[i] = p.list[size_t(row) * kList + i];
    draw_token(p, row, c, listed, sh, [&](int k) { return p.whole[size_t(row) * p.chunks + k]; });
}

// All of it for a row in one workgroup, for many rows: each row's passes over its logits and its arithmetic
// run beside the other rows', and nothing but the chunks' bins goes through memory.
struct RowShared {
    union {
        DrawShared draw;
        struct {
            u64 mass[kBins];
            unsigned count[kBins];
        } bins;
    };
    CutShared cut;
    unsigned listed;
};
static_assert(sizeof(RowShared) <= 64 * 1024, "within the default limit of LDS");

__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleParams p)
{
    __shared__ RowShared sh;
    const int row = int(blockIdx.x), tid = threadIdx.x;
    const Row r = row_of(p, row);
    const float *x = p.logits + size_t(row) * p.stride;
    const u64 first = top_of_tokens(x, 0, p.vocab, p.vocab, sh.cut.part);
    const float top = unordered(unsigned(first >> 32));
    if (r.greedy || top == -INFINITY) {
        if (tid == 0) write_first(p, row, first);
        return;
    }
    // (the middles lie behind the bins in the union)
    double *middles = sh.draw.middles;
    sh.bins.mass[tid] = 0;
    sh.bins.count[tid] = 0;
    middles[tid] = middle_of(tid) * p.unit;
    u64 *upto = p.mass + size_t(row) * p.chunks * kBins + tid;  // this bin's weight up to each chunk's end
    u64 m = 0;
    const double largest = top_of(top);
    __syncthreads();
    constexpr int kAhead = 4, kRun = kSampleRun;  // runs of a chunk, asked for together whatever chunks they are of
    for (int c = 0, begin = 0; c < p.chunks;) {
        v4f v[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; a++) {
            const int i = begin + a * kRun + tid * 4;
            if (i + 4 <= p.vocab) {
                v[a] = *reinterpret_cast<const v4f_any *>(x + i);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) v[a][j] = i + j < p.vocab ? x[i + j] : -INFINITY;
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; a++) {
            if (c == p.chunks) break;
#pragma unroll
            for (int j = 0; j < 4; j++) add_to_bins(v[a][j], largest, r.scale, r.has_k, sh.bins.mass, sh.bins.count, middles);
            begin += kRun;
            if (begin == (c + 1) * p.chunk || begin >= p.vocab) {  // the chunk's end
                __syncthreads();
                upto[c * kBins] = m = sh.bins.mass[tid];
                __syncthreads();
                c++;
            }
        }
    }
    const Cut c = cut_of(p, r, top, m, r.has_k ? sh.bins.count[tid] : 0, sh.cut, p.mass + size_t(row) * p.chunks * kBins, true);
    if (tid == 0) sh.listed = 0;
    __syncthreads();  // (the bins are read: the list takes their place)
    if (c.lists) list_tokens(x, 0, p.vocab, c, sh.draw.key, &sh.listed);
    __syncthreads();
    draw_token(p, row, c, sh.listed, sh.draw, [&](int k) { return sh.cut.whole[k]; });
}

}  // namespace
}  // namespace fg

using namespace fg;

namespace {

// How a call's rows are taken: the rows of a batch, the chunks of a row, and the scratch.
struct Shape {
    bool by_rows;
    size_t batch;
    int chunks, chunk;
    size_t at[8];  // where the scratch's parts start, and its end
};

Shape shape_of(size_t rows, size_t vocab)
{
    Shape s{};
    s.by_rows = sample_by_rows(rows, vocab);
    // rows of a batch: bounded scratch; by chunks, what the Infinity Cache (256 MB) holds beside the rest
    size_t most = std::min<size_t>(rows, 2048);
    if (!s.by_rows) most = std::max<size_t>(1, std::min(most, (size_t(192) << 20) / (vocab * 4)));
    const size_t batches = (rows + most - 1) / most;
    s.batch = (rows + batches - 1) / batches;
    s.chunks = sample_chunks(s.batch, vocab, s.by_rows);
    s.chunk = sample_chunk(vocab, s.by_rows, &s.chunks);
    const size_t work = s.batch * s.chunks;
    size_t sizes[7] = {work * 8, work * kBins * 8, work * kBins * 4, work * 8, s.batch * sizeof(Cut), s.batch * 4, s.batch * kList * 8};
    for (int i = 0; i < 7; i++) s.at[i + 1] = s.at[i] + (s.by_rows && i != 1 ? 0 : (sizes[i] + 255) / 256 * 256);
    return s;
}

}  // namespace

extern "C" size_t fg_sample_scratch(size_t rows, size_t vocab)
{
    return rows && vocab && rows <= (size_t(1) << 20) && vocab <= (size_t(1) << 22) ? shape_of(rows, vocab).at[7] : 0;
}

extern "C" int fg_sample(const float *logits, size_t rows, size_t vocab, size_t stride, const fg_sampling *settings, int32_t *tokens,
                         float *chances, void *scratch, size_t scratch_bytes, void *stream)
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
    const Shape shape = shape_of(rows, vocab);
    const size_t batch = shape.batch;
    p.chunks = shape.chunks;
    p.chunk = shape.chunk;
    void *ws = nullptr;
    bool owned = false;
    int rc = stream_scratch(scratch, scratch_bytes, shape.at[7], "fg_sample", s, &ws, &owned);
    if (rc) return rc;
    char *base = static_cast<char *>(ws);
    p.top = reinterpret_cast<u64 *>(base + shape.at[0]);
    p.mass = reinterpret_cast<u64 *>(base + shape.at[1]);
    p.count = reinterpret_cast<unsigned *>(base + shape.at[2]);
    p.whole = reinterpret_cast<u64 *>(base + shape.at[3]);
    p.cuts = reinterpret_cast<Cut *>(base + shape.at[4]);
    p.listed = reinterpret_cast<unsigned *>(base + shape.at[5]);
    p.list = reinterpret_cast<u64 *>(base + shape.at[6]);
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
        if (shape.by_rows) {
            sample_row_kernel<<<n, kThreads, 0, s>>>(p);
        } else {
            sample_top_kernel<<<grid, kThreads, 0, s>>>(p);
            sample_bins_kernel<<<grid, kThreads, 0, s>>>(p);
            sample_cut_kernel<<<n, kThreads, 0, s>>>(p);
            if (p.top_k || p.top_p || p.min_p) sample_collect_kernel<<<grid, kThreads, 0, s>>>(p);
            sample_draw_kernel<<<n, kThreads, 0, s>>>(p);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) rc = check_hip(e, "fg_sample");
    }
    if (owned) {
        const hipError_t e = hipFreeAsync(ws, s);
        if (rc == FG_OK && e != hipSuccess) rc = check_hip(e, "hipFreeAsync");
    }
    return rc;
}
