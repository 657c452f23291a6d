// Attention of a step's new tokens over the paged 8-bit cache where groups of sequences begin with the same pages
// (fg_cache_attend_shared): a group's pages once for all rows of its sequences, each sequence's own pages, and the join of
// both. cache_attend.h has what a workgroup does with a task.
#include <algorithm>
#include <atomic>

#include "cache_attend.h"

namespace fg {
namespace {

// ---------------------------------------------------------------------------- the plan
//
// Spans of rows to work through: the groups' (the rows of all of a group's sequences, over the shared pages), then the
// sequences' (over the pages behind them). A span's (row, query head) pairs lie in tiles as in cache_attend.hip, of 128 or, in
// spans of few pairs, of 16, and a tile's pages are split into parts of about the same work; a part is a task, a
// workgroup's for each key head. Every workgroup finds its task from the arrays, all 256 threads together.

// Where the sums of a row's pairs are, in the order in which the tasks lie: tile t's part s at slot base + (tiles - 1 - t)
// parts + s of the large tiles' or the small ones'.
struct RowNote {
    int base, begin;  // begin: the span's first row
    int tiles;
    int parts;        // of a tile; 0: its outputs are written already
};
constexpr int kLargeTiles = 1 << 16, kAfterShared = 1 << 17;  // flags in `parts`

struct SharedParams : AttendParams {
    const int32_t *starts, *counts;
    int groups;
    int limit;        // pairs of a span that small tiles take
    int large_slots, small_slots;
    float *small_partial;
    RowNote *own, *shared;  // [rows]
};

struct Entity {
    Span span;
    int tiles, pages;  // pages: that a tile sees at most
    int first_page;    // of the span's
    bool large, joined;
};

// How many of a group's sequences' first pages are shared, within what any table holds.
__device__ __forceinline__ int shared_pages(const SharedParams &p, int count) { return max(0, min(count, p.b.max_pages)); }

__device__ __forceinline__ int sequence_index(const SharedParams &p, int start) { return max(0, min(start, p.b.sequences)); }

// Span e, the groups' first. Every lane of the wave takes part.
__device__ __forceinline__ Entity entity_of(const SharedParams &p, int e)
{
    Entity n{};
    const int lane = threadIdx.x & 63, s = e - p.groups;
    // the shared pages of sequence s: those of the last group that starts at or before it
    int before = 0;
    for (int g0 = 0; g0 <= p.groups; g0 += 64) {
        const int start = g0 + lane <= p.groups ? p.starts[g0 + lane] : INT_MAX;
        const int count = g0 + lane < p.groups ? p.counts[g0 + lane] : 0;
        const int here = min(64, p.groups + 1 - g0);
        for (int i = 0; i < here; i++) {
            const int at = __builtin_amdgcn_readlane(start, i), pages = __builtin_amdgcn_readlane(count, i);
            before = s >= at ? pages : before;
        }
    }
    if (e < p.groups) {
        const int a = sequence_index(p, p.starts[e]), b = sequence_index(p, p.starts[e + 1]);
        if (b <= a) return n;
        n.span = span_of(p.b.row_starts[a], p.b.row_starts[b], 0, p.b.rows);
        n.pages = shared_pages(p, p.counts[e]);
        // (each row sees less than a window of the pages before its sequence's own)
        if (p.window > 0) n.pages = min(n.pages, p.window / kPage + 2);
        if (n.pages == 0) return n;
    } else if (s < p.b.sequences) {
        n.span = sequence_span(p.b, s);
        n.first_page = shared_pages(p, before);
        n.joined = n.first_page > 0;
    }
    if (n.span.rows == 0) return n;
    const int pairs = n.span.rows * p.group;
    n.large = pairs > p.limit;
    const int tm = n.large ? 128 : 16;
    n.tiles = (pairs + tm - 1) / tm;
    if (e >= p.groups) {
        const PageRange r = pages_seen(n.span, 0, n.span.rows - 1, p.window, p.b.max_pages);
        n.pages = max(0, r.hi - max(r.lo, n.first_page));
        if (p.window > 0) n.pages = min(n.pages, p.window / kPage + tm / p.group / kPage + 3);
    }
    return n;
}

__device__ __forceinline__ float wave_total(float v) { return wave_allsum(v); }
__device__ __forceinline__ int wave_total(int v)
{
    int total;
    (void)wave_scan(v, &total);
    return total;
}

// A sum over the workgroup's threads, in an order that is always the same.
template <class T>
__device__ __forceinline__ T block_sum(T v, T *wave_totals)
{
    v = wave_total(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) wave_totals[threadIdx.x >> 6] = v;
    __syncthreads();
    return wave_totals[0] + wave_totals[1] + wave_totals[2] + wave_totals[3];
}

struct Found {
    Task task;
    int entity, first_page, joined, large;
};

__device__ __forceinline__ int splits_of(int pages, int part) { return pages <= part ? 1 : min((pages + part - 1) / part, kMaxSplit); }

// The task of index x into *found (its entity -1 where there is none).
__device__ __forceinline__ void find_task(const SharedParams &p, int x, Found *found)
{
    __shared__ float works[4];
    __shared__ int counts[4];
    const int tid = threadIdx.x, all = p.groups + p.b.sequences;
    Entity n = entity_of(p, tid);
    float work = 0.0f;
    for (int e0 = 0;;) {
        work = work + float(n.tiles) * float(n.pages);
        e0 += 256;
        if (e0 >= all) break;
        n = entity_of(p, e0 + tid);
    }
    // (a little more than a share: the sum is in f32)
    const float share = block_sum(work, works) * 1.00001f / float(p.target) + 1.0f;
    const int part = share < float(kMinPages) ? kMinPages : share > 1e9f ? 1000000000 : int(share);
    auto units = [&]() { return n.tiles ? n.tiles * splits_of(n.pages, part) : 0; };
    // the tasks of large tiles come first
    int large = 0;
    for (int e0 = 0; e0 < all; e0 += 256) {
        if (all > 256) n = entity_of(p, e0 + tid);
        large += n.large ? units() : 0;
    }
    large = block_sum(large, counts);
    const bool is_large = x < large;
    const int index = is_large ? x : x - large;
    if (tid == 0) found->entity = -1;
    int before = 0;
    for (int e0 = 0; e0 < all; e0 += 256) {
        if (all > 256) n = entity_of(p, e0 + tid);
        const int mine = n.large == is_large ? units() : 0;
        int total;
        const int upto = wave_scan(mine, &total);
        __syncthreads();
        if ((tid & 63) == 0) counts[tid >> 6] = total;
        __syncthreads();
        int start = before + upto - mine;
        for (int w = 0; w < (tid >> 6); w++) start += counts[w];
        before += counts[0] + counts[1] + counts[2] + counts[3];
        const int within = index - start;
        if (within >= 0 && within < mine) {
            const int nsplit = splits_of(n.pages, part);
            Task t{};
            t.seq = e0 + tid < p.groups ? sequence_index(p, p.starts[e0 + tid]) : e0 + tid - p.groups;
            t.tile = n.tiles - 1 - within / nsplit;
            t.split = within % nsplit;
            t.nsplit = nsplit;
            t.slot = index;
            t.span = n.span;
            *found = Found{t, e0 + tid, n.first_page, n.joined, n.large};
        }
        if (before > index) break;
    }
    __syncthreads();
}

// ------------------------------------------------------------------------------ the tasks

// The positions of a tile's rows, by the row within the span (those of a group's are its sequences'), and of its pairs.
struct InTile {
    const int *positions, *pairs;
    int row0, low, high;
    __device__ __forceinline__ int of(int at) const { return positions[at - row0]; }
    __device__ __forceinline__ int again(const Pair &, int pair) const { return pairs[pair]; }
};

constexpr int kTileRows = 129;  // that 128 pairs lie in, at most

template <int DP>
constexpr size_t shared_lds() { return many_lds<DP>() > sizeof(FewJoin<DP>) ? many_lds<DP>() : sizeof(FewJoin<DP>); }

// A workgroup a task and key head.
template <int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void shared_tasks_kernel(SharedParams p)
{
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ Found found;
    __shared__ int positions[kTileRows + 3], pair_positions[128];
    const int tid = threadIdx.x, lane = tid & 63, kv = int(blockIdx.x % unsigned(p.kv_heads));
    find_task(p, int(blockIdx.x / unsigned(p.kv_heads)), &found);
    auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int entity = same(found.entity);
    if (entity < 0) return;  // the whole workgroup
    const Task task = uniform(found.task);
    const bool large = same(found.large), own = entity >= p.groups, joined = same(found.joined);
    const int first_page = same(found.first_page), tm = large ? 128 : 16;
    if (task.slot >= (large ? p.large_slots : p.small_slots)) return;  // (starts that fall: more tiles than the rows have)
    // the tile's rows, within the span
    const int row0 = task.tile * tm / p.group, row1 = min((task.tile * tm + tm - 1) / p.group, task.span.rows - 1);
    // (a large tile always leaves parts: what its lanes would need to find their outputs does not fit their registers)
    const bool direct = own && !joined && task.nsplit == 1 && !large;
    if (kv == 0 && task.split == 0) {
        // rows whose first pair lies in the tile
        const int parts = direct ? 0 : task.nsplit | (large ? kLargeTiles : 0) | (joined ? kAfterShared : 0);
        const int tiles = (task.span.rows * p.group + tm - 1) / tm, base = task.slot - (tiles - 1 - task.tile) * task.nsplit;
        for (int r = row0 + tid; r <= row1; r += 256)
            if (r * p.group >= task.tile * tm) (own ? p.own : p.shared)[task.span.begin + r] = RowNote{base, task.span.begin, tiles, parts};
    }
    const int32_t *table = p.b.pages + size_t(task.seq) * p.b.max_pages;
    if (own) {
        for (int i = tid; i <= row1 - row0; i += 256) positions[i] = task.span.first + row0 + i;
    } else {
        for (int i = tid; i <= row1 - row0; i += 256) positions[i] = -1;
        __syncthreads();
        const int begin = sequence_index(p, p.starts[entity]), end = sequence_index(p, p.starts[entity + 1]);
        for (int s = begin + tid; s < end; s += 256) {
            const Span span = sequence_span(p.b, s);
            const int from = max(span.begin, task.span.begin + row0), to = min(span.begin + span.rows - 1, task.span.begin + row1);
            for (int r = from; r <= to; r++) positions[r - task.span.begin - row0] = span.first + (r - span.begin);
        }
    }
    __syncthreads();
    // (past the pairs the last again)
    const int pairs = task.span.rows * p.group;
    if (tid < tm) pair_positions[tid] = positions[min(task.tile * tm + tid, pairs - 1) / p.group - row0];
    __syncthreads();
    // the first and last position of the tile, and of a wave's pairs
    auto ends = [&](int first, int last, int &low, int &high) {
        low = INT_MAX, high = INT_MIN;
        for (int i = first + lane; i < last; i += 64) {
            low = min(low, pair_positions[i]);
            high = max(high, pair_positions[i]);
        }
#pragma unroll
        for (int step = 32; step; step >>= 1) {
            low = min(low, __shfl_xor(low, step));
            high = max(high, __shfl_xor(high, step));
        }
        low = same(low), high = same(high);
    };
    InTile places{positions, pair_positions, row0, 0, 0};
    ends(0, tm, places.low, places.high);
    PageRange range;
    range.lo = own ? first_page : 0;
    range.hi = own ? p.b.max_pages : shared_pages(p, p.counts[entity]);
    range.hi = min(range.hi, places.high < 0 ? 0 : places.high / kPage + 1);
    range.lo = min(max(first_seen(places.low, p.window) / kPage, range.lo), range.hi);
    const int n = (range.hi - range.lo + task.nsplit - 1) / task.nsplit;
    range.lo = min(range.lo + task.split * n, range.hi);
    range.hi = same(min(range.lo + n, range.hi)), range.lo = same(range.lo);
    if (large) {
        ends(same(tid >> 6) * 32, same(tid >> 6) * 32 + 32, places.low, places.high);
        float *parts = p.partial + (size_t(task.slot) * p.kv_heads + kv) * 4 * many_floats(DP);
        __builtin_assume(parts != nullptr);
        attend_many<DP>(p, task, range, table, kv, places, lds, parts);
    } else {
        float *part = direct ? nullptr : p.small_partial + (size_t(task.slot) * p.kv_heads + kv) * few_floats(DP);
        attend_few<DP>(p, task, range, table, kv, places, *reinterpret_cast<FewJoin<DP> *>(lds), part);
    }
}

// ------------------------------------------------------------------------------- the join

// A row and head's parts, one after the other: those over the shared pages, then its own.
struct Parts {
    const float *at;  // the first one's
    size_t step;
    int count;
    int sums, values;  // where in a part this lane's reference and four values are (the totals 64 behind the references)
};

template <int DP>
__device__ __forceinline__ Parts parts_of(const SharedParams &p, const RowNote &note, int row, int kv, int in_group, int quad)
{
    const bool large = note.parts & kLargeTiles;
    Parts r{};
    r.count = note.parts & (kLargeTiles - 1);
    // (64 bits and every check, for the notes of a batch whose starts fall may hold anything)
    const int64_t m = (int64_t(row) - note.begin) * p.group + in_group, tm = large ? 128 : 16, tile = m / tm;
    int64_t slot = note.base + (note.tiles - 1 - tile) * r.count;
    if (r.count > kMaxSplit || m < 0 || tile >= note.tiles || slot < 0 || slot + r.count > (large ? p.large_slots : p.small_slots))
        r.count = 0, slot = 0;
    const int pair = int(m & (tm - 1));
    if (large) {
        r.at = p.partial + ((size_t(slot) * p.kv_heads + kv) * 4 + pair / 32) * many_floats(DP);
        r.step = size_t(p.kv_heads) * 4 * many_floats(DP);
        r.sums = pair % 32;
        r.values = 128 + (quad / 2) * 256 + (pair % 32 + 32 * (quad & 1)) * 4;
    } else {
        r.at = p.small_partial + (size_t(slot) * p.kv_heads + kv) * few_floats(DP);
        r.step = size_t(p.kv_heads) * few_floats(DP);
        r.sums = pair;
        r.values = 128 + (quad / 4) * 256 + (pair + 16 * (quad & 3)) * 4;
    }
    return r;
}

struct Joined {
    float r = -INFINITY, total = 0.0f;
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
};

__device__ __forceinline__ void join_parts(Joined &j, const Parts &parts)
{
    constexpr int kAhead = 8;
    for (int s0 = 0; s0 < parts.count; s0 += kAhead) {
        float rs[kAhead], totals[kAhead];
        v4f os[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const float *from = parts.at + size_t(min(s0 + i, parts.count - 1)) * parts.step;
            rs[i] = from[parts.sums];
            totals[i] = from[64 + parts.sums];
            os[i] = *reinterpret_cast<const v4f *>(from + parts.values);
        }
        float top = j.r;
#pragma unroll
        for (int i = 0; i < kAhead; i++) top = s0 + i < parts.count ? fmaxf(top, rs[i]) : top;
        const float a = part_factor(j.r, top);
        j.r = top;
        j.total = j.total * a;
#pragma unroll
        for (int e = 0; e < 4; e++) j.o[e] = j.o[e] * a;
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (s0 + i >= parts.count) continue;
            const float b = part_factor(rs[i], top);
            j.total = j.total + totals[i] * b;
#pragma unroll
            for (int e = 0; e < 4; e++) j.o[e] = j.o[e] + os[i][e] * b;
        }
    }
}

// A team of lanes a row and query head, four dimensions a lane.
template <int DP>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedParams p)
{
    constexpr int kTeam = DP == 32 ? 8 : DP == 64 ? 16 : DP <= 128 ? 32 : 64;
    const int quad = threadIdx.x & (kTeam - 1);
    const int first = p.b.row_starts[0], last = min(p.b.row_starts[p.b.sequences], p.b.rows);
    const unsigned units = unsigned(p.b.rows) * unsigned(p.heads);
    for (unsigned unit = blockIdx.x * (256 / kTeam) + threadIdx.x / kTeam; unit < units; unit += gridDim.x * (256 / kTeam)) {
        const int row = int(unit / unsigned(p.heads)), head = int(unit % unsigned(p.heads));
        if (row < first || row >= last || 4 * quad >= p.head_dim) continue;
        const RowNote own = p.own[row];
        if ((own.parts & (kLargeTiles - 1)) == 0) continue;
        const int kv = head / p.group, in_group = head - kv * p.group;
        Joined j;
        if (own.parts & kAfterShared) join_parts(j, parts_of<DP>(p, p.shared[row], row, kv, in_group, quad));
        join_parts(j, parts_of<DP>(p, own, row, kv, in_group, quad));
        v4f x;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = j.total == 0.0f ? 0.0f : j.o[e] / j.total;
        *reinterpret_cast<v4f_any *>(p.out + size_t(row) * p.out_stride + size_t(head) * p.head_dim + 4 * quad) = x;
    }
}

// ------------------------------------------------------------------------------- the host

struct Launch {
    bool shared;  // or each sequence by itself
    int limit;
    size_t large_slots, small_slots, grid;  // a key head's
    int target;
    size_t note_bytes, large_bytes, small_bytes;
    size_t bytes() const { return 2 * note_bytes + large_bytes + small_bytes; }
};

size_t up(size_t bytes) { return (bytes + 255) / 256 * 256; }

Launch plan_launch(const fg_cache *c, const fg_batch *b, const fg_prefixes *f, size_t heads)
{
    Launch l{};
    const size_t group = heads / c->kv_heads, pairs = b->rows * group, sequences = std::min(b->sequences, b->rows);
    const size_t groups = std::min(f->groups, sequences);
    l.limit = c->padded <= 128 ? 96 : 64;
    l.shared = groups && sequences > groups && b->max_pages > 16 && pairs <= size_t(l.limit) * sequences;
    if (!l.shared) return l;
    const size_t units = std::max<size_t>(kUnits / c->kv_heads, 1);
    l.target = int((c->padded <= 128 ? 2 : 1) * units);
    // spans of n pairs have at most n / 128 + 1 large tiles, n / 16 + 1 small ones; the parts beyond a tile's first are the target
    size_t large = 0, small = 0;
    for (size_t spans : {groups, sequences}) {
        large += pairs > size_t(l.limit) ? pairs / 128 + std::min(spans, pairs / (l.limit + 1)) : 0;
        small += std::min(pairs / 16 + spans, size_t(l.limit / 16) * spans);
    }
    l.large_slots = large ? large + l.target : 0;
    l.small_slots = small + l.target;
    l.grid = large + small + l.target;
    l.note_bytes = up(b->rows * sizeof(RowNote));
    l.large_bytes = up(l.large_slots * c->kv_heads * 4 * many_floats(c->padded) * 4);
    l.small_bytes = up(l.small_slots * c->kv_heads * few_floats(c->padded) * 4);
    return l;
}

template <int DP>
int launch_shared(const SharedParams &p, const Launch &l, hipStream_t s)
{
    if (shared_lds<DP>() > 60 * 1024) {  // more than the default limit, with what the plan takes: raised once a device
        static std::atomic<unsigned long long> raised{0};
        int device = 0;
        FG_HIP(hipGetDevice(&device));
        const unsigned long long bit = 1ull << (device & 63);
        if (device > 63 || !(raised.load() & bit)) {
            FG_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(shared_tasks_kernel<DP>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                       int(shared_lds<DP>())));
            raised.fetch_or(bit);
        }
    }
    shared_tasks_kernel<DP><<<unsigned(p.kv_heads * l.grid), 256, shared_lds<DP>(), s>>>(p);
    FG_HIP(hipGetLastError());
    constexpr int kTeam = DP == 32 ? 8 : DP == 64 ? 16 : DP <= 128 ? 32 : 64;
    const size_t units = size_t(p.b.rows) * p.heads, grid = (units + 256 / kTeam - 1) / (256 / kTeam);
    shared_join_kernel<DP><<<unsigned(std::min(grid, size_t(1) << 20)), 256, 0, s>>>(p);
    FG_HIP(hipGetLastError());
    return FG_OK;
}

int check_prefixes(const fg_prefixes *f, const char *who)
{
    if (!f) return set_error(FG_ERR_ARG, std::string(who) + ": null prefixes");
    if (f->groups > 65536) return set_error(FG_ERR_SHAPE, std::string(who) + ": at most 65536 groups");
    if (f->groups && (!f->starts || !f->pages)) return set_error(FG_ERR_ARG, std::string(who) + ": a null array of the prefixes");
    return FG_OK;
}

}  // namespace
}  // namespace fg

using namespace fg;

extern "C" size_t fg_cache_attend_shared_scratch(const fg_cache *c, const fg_batch *b, const fg_prefixes *f, size_t heads)
{
    if (!c || !b || !f || !heads || heads % c->kv_heads) return 0;
    const Launch l = plan_launch(c, b, f, heads);
    return l.shared ? l.bytes() : fg_cache_attend_scratch(c, b, heads);
}

extern "C" int fg_cache_attend_shared(const fg_cache *c, const fg_batch *b, const fg_prefixes *f, const float *query, size_t query_stride,
                                      size_t heads, float scale, size_t window, float *out, size_t out_stride, void *scratch,
                                      size_t scratch_bytes, void *stream)
{
    const char *who = "fg_cache_attend_shared";
    int rc = check_prefixes(f, who);
    if (rc) return rc;
    rc = check_attend(c, b, query, heads, scale, out, out_stride, who);
    if (rc) return rc;
    if (!b->rows || !b->sequences) return FG_OK;
    const Launch l = plan_launch(c, b, f, heads);
    if (!l.shared)
        return fg_cache_attend(c, b, query, query_stride, heads, scale, window, out, out_stride, scratch, scratch_bytes, stream);
    if (l.grid * c->kv_heads > kMaxGrid || b->rows * heads > 0xf0000000)
        return set_error(FG_ERR_SHAPE, std::string(who) + ": more sequences times heads than a launch takes");
    const hipStream_t s = as_stream(stream);
    void *ws = nullptr;
    bool owned = false;
    rc = stream_scratch(scratch, scratch_bytes, l.bytes(), who, s, &ws, &owned);
    if (rc) return rc;
    SharedParams p = attend_params<SharedParams>(c, b, query, query_stride, heads, scale, window, out, out_stride);
    p.starts = f->starts;
    p.counts = f->pages;
    p.groups = int(f->groups);
    p.limit = l.limit;
    p.target = l.target;
    p.large_slots = int(l.large_slots);
    p.small_slots = int(l.small_slots);
    char *at = static_cast<char *>(ws);
    p.own = reinterpret_cast<RowNote *>(at);
    p.shared = reinterpret_cast<RowNote *>(at + l.note_bytes);
    p.partial = reinterpret_cast<float *>(at + 2 * l.note_bytes);
    p.small_partial = reinterpret_cast<float *>(at + 2 * l.note_bytes + l.large_bytes);
    switch (c->padded) {
    case 32: rc = launch_shared<32>(p, l, s); break;
    case 64: rc = launch_shared<64>(p, l, s); break;
    case 96: rc = launch_shared<96>(p, l, s); break;
    case 128: rc = launch_shared<128>(p, l, s); break;
    case 192: rc = launch_shared<192>(p, l, s); break;
    default: rc = launch_shared<256>(p, l, s); break;
    }
    if (owned) {
        const hipError_t e = hipFreeAsync(ws, s);
        if (rc == FG_OK && e != hipSuccess) rc = check_hip(e, "hipFreeAsync");
    }
    return rc;
}
