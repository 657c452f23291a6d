// Attention of a step's new tokens over the paged 8-bit cache where groups of sequences begin with the same pages
// (fg_cache_attend_shared): a group's pages once for all rows of its sequences, each sequence's own pages, and the join of
// both. cache_attend.h has what a workgroup, or a wave, does with a task.
#include <algorithm>
#include <atomic>

#include "cache_attend.h"

namespace fg {
namespace {

// ---------------------------------------------------------------------------- the plan
//
// Spans of rows to work through: the groups' (the rows of all of a group's sequences, over the shared pages), then the
// sequences' (over the pages behind them). A span's (row, query head) pairs lie in tiles as in cache_attend.hip: large ones of
// 128, a workgroup's, or, in spans of few pairs, small ones of 16, a wave's. A tile's pages are split into parts of about the
// same time; a part of a tile is a task, for each key head. One workgroup lists the tasks from the batch's arrays, and what
// the join then does: nothing about the lengths is known on the host. (Each task's workgroup looking for itself, as in
// cache_attend.hip, took 2.7 us of each one's time, and 6.7 from 257 spans on: 256 sequences in five groups 98 us, listed 76.)

struct SpanRecord {
    int table;         // the sequence whose table has the pages
    int begin, rows;
    int first;         // the position of a sequence's first row
    int lo, hi;        // pages [lo, hi) at most
    int tiles, nsplit;
    int base;          // the first of its tasks: tile t's part s is base + (tiles - 1 - t) nsplit + s (the last tiles see the most keys)
    int flags;
    int fill[6];
};
// large tiles; a group's; a sequence's whose rows see shared pages too; a sequence's of small tiles whose tasks are single and
// write its outputs
constexpr int kLarge = 1, kShared = 2, kJoined = 4, kWhole = 8;

// A span's task `at`.
struct Place {
    int span, at;
};

// A small tile, or a quarter of a large one, whose parts are to be joined.
struct JoinRecord {
    int begin, rows;  // the span's
    int at;           // its pairs are 16 at, or 32 at, on
    int slot, parts;  // its first part's task, and how many
    int flags;
    int fill[2];
};

// Where a row's own parts are: a sequence's `base`, first row, tiles and nsplit.
struct OwnRecord {
    int base, begin, tiles, parts;  // parts with kOwnLarge: of large tiles
};
constexpr int kOwnLarge = 1 << 16;

struct PlanHeader {
    int large, small, joins;
};

struct SharedParams : AttendParams {
    const int32_t *starts, *counts;
    int groups;
    int limit;  // pairs of a sequence that small tiles take
    int large_slots, small_slots, join_slots;
    PlanHeader *header;
    SpanRecord *spans;  // the groups', the sequences'
    Place *large_tasks, *small_tasks;
    JoinRecord *joins;
    int *positions;     // [rows]
    OwnRecord *own;     // [rows]
    float *small_partial;
    uint4 *pieces;           // the queries' two f16 pieces (piece_at)
    float *factors;          // [key head][pair]: of its scores
};

// What a part takes: at least so many pages, and of the whole work, in units of a small tile's page, a share of the target, two
// workgroups a CU. Microseconds of 64 conversations behind 128 pages / 32 questions behind 940 / 256 in five groups, 16 heads
// of 128 over 4: 36 / 58 / 72; at least 2, 8 pages of a large tile 40 / 63 / 79 and 42 / 58 / 73; 4, 8 of a small one 39 / 64 / 77
// and 44 / 63 / 78; a large tile's page for one, three small ones' 37 / 64 / 88 and 37 / 64 / 83; three or four workgroups a CU 37 /
// 73 / 81 and 37 / 77 / 82 (the second and later ones taken when these read 36.7 / 63.6 / 77.8).
// A group's small tiles, whose pages are many, lie in fewer parts, and a group of more than 48 pairs, three small tiles, takes large
// ones: in 38 cases of 9 to 128 sequences in groups of 20 to 96 pairs behind 60 to 1500 pages at least 5 pages are 1.5 % faster than 2 on
// average (12 sequences behind 400 pages, 16 heads of 128 over 4, 34 and 28), 8 are 20 % slower in some; and with large tiles from 32 /
// 48 / 64 / 80 pairs on 1.5 / 2.6 / 0.6 / 0.7 % faster than from 96 on (24 sequences behind 900 pages 70 and 50).
constexpr int kLargePages = 4, kSmallPages = 2, kGroupPages = 5, kLargeCost = 2;
constexpr int kGroupLimit = 48;  // pairs of a group that small tiles take
constexpr int kSharedSplit = 256;  // parts of a tile, at most

struct Entity {
    Span span;
    int tiles, lo, hi, pages;  // pages [lo, hi) at most, and how many of them a tile sees at most
    int table;
    bool large, shared, joined;  // joined: a sequence's whose rows see shared pages too
};

__device__ __forceinline__ int shared_pages(const SharedParams &p, int count) { return max(0, min(count, p.b.max_pages)); }
__device__ __forceinline__ int sequence_index(const SharedParams &p, int start) { return max(0, min(start, p.b.sequences)); }

// The groups' arrays and the sequences', in LDS where they fit: a group's rows are found by its starts, and one load after the other
// is most of the plan's time.
constexpr int kHeld = 1024;
struct Groups {
    const int *starts, *counts, *rows, *lengths;
};

// Span e, the groups' first.
__device__ __forceinline__ Entity entity_of(const SharedParams &p, const Groups &groups, int e)
{
    Entity n{};
    const int s = e - p.groups;
    int before = 0;
    if (s >= 0) {
        if (s >= p.b.sequences) return n;
        n.span = span_of(groups.rows[s], groups.rows[s + 1], groups.lengths[s], p.b.rows);
        // the shared pages of sequence s: those of the last group that starts at or before it
        int upto = 0;  // so many starts are
        for (int step = 1 << (31 - __builtin_clz(p.groups + 1)); step; step >>= 1)
            if (upto + step <= p.groups + 1 && groups.starts[upto + step - 1] <= s) upto += step;
        if (upto > 0 && upto <= p.groups) before = groups.counts[upto - 1];
    }
    n.table = s;
    if (s < 0) {
        const int a = sequence_index(p, groups.starts[e]), b = sequence_index(p, groups.starts[e + 1]);
        if (b <= a) return n;
        n.span = span_of(groups.rows[a], groups.rows[b], 0, p.b.rows);
        n.table = a;
        n.shared = true;
        n.pages = n.hi = shared_pages(p, groups.counts[e]);
        // (each row sees less than a window of the pages before its sequence's own)
        if (p.window > 0) n.pages = min(n.pages, p.window / kPage + 2);
        if (n.hi == 0) return n;
    } else {
        n.lo = shared_pages(p, before);
        n.joined = n.lo > 0;
    }
    if (n.span.rows == 0) return n;
    const int pairs = n.span.rows * p.group;
    n.large = pairs > (n.shared ? kGroupLimit : p.limit);
    const int tm = n.large ? 128 : 16;
    n.tiles = (pairs + tm - 1) / tm;
    if (!n.shared) {
        const PageRange r = pages_seen(n.span, 0, n.span.rows - 1, p.window, p.b.max_pages);
        n.hi = r.hi;
        n.pages = max(0, r.hi - max(r.lo, n.lo));
        if (p.window > 0) n.pages = min(n.pages, p.window / kPage + tm / p.group / kPage + 3);
    }
    return n;
}

constexpr int kPlanThreads = 1024, kFewSpans = 512;  // half as many threads up to so many spans: fewer waves to wait for

// Where the high piece of eight dimensions, block `block` of them, of a pair is, in 16 bytes (the low one 64 further on). `pair` is its
// place among all rows' of the key head; 32 in a row lie as a large tile's step takes them, a kilobyte of 64 lanes (pair, half of
// the step's 32 dimensions), whatever the tile's first pair is: at most two runs. (One pair after the other, each lane of a load
// asked for a line of its own, and a tile's queries took 6000 cycles.)
__host__ __device__ __forceinline__ size_t pair_blocks(size_t rows, int group) { return (rows * size_t(group) + 31) / 32; }
__device__ __forceinline__ size_t piece_at(int DP, size_t blocks32, int kv, int pair, int block)
{
    const int step = 2 * (block >> 2) + (block & 1), half = (block >> 1) & 1;
    return (((size_t(kv) * blocks32 + (pair >> 5)) * (DP / 16) + step) * 4 + half) * 32 + (pair & 31);
}

// The queries split into their two pieces, once for all tasks that multiply them: a team of lanes a row and head, eight
// dimensions a lane.
__device__ __forceinline__ void split_queries(const SharedParams &p, int padded)
{
    const int blocks = padded / 8;
    int team = 4;
    while (team < blocks) team *= 2;
    const int first = max(0, p.b.row_starts[0]), rows = min(p.b.row_starts[p.b.sequences], p.b.rows) - first;
    if (rows <= 0) return;
    const unsigned units = unsigned(rows) * unsigned(p.heads), step = (gridDim.x - 1) * (blockDim.x / team);
    const int block = threadIdx.x & (team - 1);
    for (unsigned unit = (blockIdx.x - 1) * (blockDim.x / team) + threadIdx.x / team; unit < units; unit += step) {  // whole teams
        const int row = first + int(unit / unsigned(p.heads)), head = int(unit % unsigned(p.heads));
        float x[8];
        load8(p.query + size_t(row) * p.query_stride + size_t(head) * p.head_dim, 8 * block, p.head_dim, x);
        float amax = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) amax = fmaxf(amax, fabsf(x[k]));
        for (int m = 1; m < team; m *= 2) amax = fmaxf(amax, __shfl_xor(amax, m));
        const int shift = query_shift(amax);
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = ldexpf(x[k], shift);
        v8h hi, lo;
        split8(x, hi, lo);
        const int kv = head / p.group, pair = row * p.group + (head - kv * p.group);
        const size_t blocks32 = pair_blocks(p.b.rows, p.group);
        if (block < blocks) {
            const size_t at = piece_at(padded, blocks32, kv, pair, block);
            p.pieces[at] = __builtin_bit_cast(uint4, hi);
            p.pieces[at + 64] = __builtin_bit_cast(uint4, lo);
        }
        if (block == 0) p.factors[size_t(kv) * blocks32 * 32 + pair] = ldexpf(p.scale2, -shift);
    }
}

struct SplitQueries {
    const uint4 *pieces;
    const float *factors;
    template <int DP>
    __device__ __forceinline__ void few(const AttendParams &p, const Pair &, int kv, int pair, int g, v8h (&qh)[(DP + 63) / 64][2],
                                        v8h (&ql)[(DP + 63) / 64][2], float &f) const
    {
        const size_t blocks32 = pair_blocks(p.b.rows, p.group);
        f = factors[size_t(kv) * blocks32 * 32 + pair];
#pragma unroll
        for (int j = 0; j < (DP + 63) / 64; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int block = 8 * j + 2 * g + e;
                uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
                if (DP % 64 == 0 || block < DP / 8) {
                    const size_t at = piece_at(DP, blocks32, kv, pair, block);
                    hi = pieces[at];
                    lo = pieces[at + 64];
                }
                qh[j][e] = __builtin_bit_cast(v8h, hi);
                ql[j][e] = __builtin_bit_cast(v8h, lo);
            }
    }
    template <int DP>
    __device__ __forceinline__ void many(const AttendParams &p, const Pair &, int kv, int pair, int h, v8h (&qh)[DP / 16], v8h (&ql)[DP / 16],
                                         float &f) const
    {
        const size_t blocks32 = pair_blocks(p.b.rows, p.group);
        f = factors[size_t(kv) * blocks32 * 32 + pair];
        const uint4 *from = pieces + piece_at(DP, blocks32, kv, pair, 2 * h);
#pragma unroll
        for (int k = 0; k < DP / 16; k++) {
            qh[k] = __builtin_bit_cast(v8h, from[k * 128]);
            ql[k] = __builtin_bit_cast(v8h, from[k * 128 + 64]);
        }
    }
};

// The first workgroup lists the tasks, a thread a span; the others split the queries. Bounded by its launch and a chain of waits:
// the groups, their rows, two sums over the workgroup. 65 spans 5.3 us, 261 6.2, 1040 12.0; with the
// sequences' rows looked up in memory behind the groups, and sums over the waves one after the other, 5.8, 6.6 and 13.7.
__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(SharedParams p, int padded)
{
    if (blockIdx.x > 0) {
        split_queries(p, padded);
        return;
    }
    __shared__ float works[2][kPlanThreads / 64];
    __shared__ int totals[3][kPlanThreads / 64], held[4][kHeld + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), all = p.groups + p.b.sequences;
    const int threads = int(blockDim.x), waves = threads / 64;
    Groups groups{p.starts, p.counts, p.b.row_starts, p.b.lengths};
    if (p.groups <= kHeld && p.b.sequences <= kHeld) {
        for (int i = tid; i <= max(p.groups, p.b.sequences); i += threads) {
            int x[4] = {};
            if (i <= p.groups) x[0] = p.starts[i];
            if (i < p.groups) x[1] = p.counts[i];
            if (i <= p.b.sequences) x[2] = p.b.row_starts[i];
            if (i < p.b.sequences) x[3] = p.b.lengths[i];
            for (int k = 0; k < 4; k++) held[k][i] = x[k];
        }
        groups = Groups{held[0], held[1], held[2], held[3]};
        __syncthreads();
    }
    // write(item, i) for each lane's `item` and i from 0 to its `count`: a lane does its own few, and the wave those of one
    // that has many after the other
    auto each = [&](int count, const auto &item, auto write) {
        constexpr int kOwn = 8, kInts = sizeof(item) / 4;
        for (int i = 0; i < min(count, kOwn); i++) write(item, i);
        unsigned long long many = __ballot(count > kOwn);
        while (many) {
            const int l = __builtin_ctzll(many);
            many &= many - 1;
            const int end = __builtin_amdgcn_readlane(count, l);
            auto of_lane = item;
            int ints[kInts];
            __builtin_memcpy(ints, &item, sizeof(item));
            for (int k = 0; k < kInts; k++) ints[k] = __builtin_amdgcn_readlane(ints[k], l);
            __builtin_memcpy(&of_lane, ints, sizeof(item));
            for (int i = kOwn + lane; i < end; i += 64) write(of_lane, i);
        }
    };
    Entity n{};
    float work = 0.0f, rows = 0.0f;
    for (int e0 = 0; e0 < all; e0 += threads) {
        n = entity_of(p, groups, e0 + tid);
        work = work + float(n.tiles) * float(n.pages) * (n.large ? float(kLargeCost) : 1.0f);
        rows = rows + float(n.span.rows);
    }
    work = wave_allsum(work);
    rows = wave_allsum(rows);
    if (lane == 0) works[0][wave] = work, works[1][wave] = rows;
    __syncthreads();
    work = wave_allsum(lane < waves ? works[0][lane] : 0.0f);
    rows = wave_allsum(lane < waves ? works[1][lane] : 0.0f);
    // Spans apart have each row twice at most, a sequence's and a group's. A batch whose starts fall may have it thousands of
    // times: no room holds, nor any int counts, what that would be to do, and nothing is done.
    if (rows > 2.01f * float(p.b.rows) + 1.0f) {
        if (tid == 0) *p.header = PlanHeader{0, 0, 0};
        return;
    }
    // (a little more than a share: the sum is in f32)
    const float share = work * 1.00001f / float(p.target);
    auto pages_of = [&](float share, int least) { return share + 1.0f < float(least) ? least : share > 1e9f ? 1000000000 : int(share + 1.0f); };
    const int large_part = pages_of(share / float(kLargeCost), kLargePages), small_part = pages_of(share / 4.0f, kSmallPages);
    int done[3] = {0, 0, 0};
    for (int e0 = 0; e0 < all; e0 += threads) {
        if (all > threads) n = entity_of(p, groups, e0 + tid);
        const int part = n.large ? large_part : n.shared ? max(small_part, kGroupPages) : small_part;
        const int nsplit = n.pages <= part ? 1 : min((n.pages + part - 1) / part, kSharedSplit);
        const int units = n.tiles * nsplit;
        const bool whole = !n.shared && !n.joined && !n.large && nsplit == 1;
        const int pairs = n.span.rows * p.group;
        const int joins = n.tiles == 0 || (!n.shared && n.joined) || whole ? 0 : n.large ? (pairs + 31) / 32 : n.tiles;
        const int mine[3] = {n.large ? units : 0, n.large ? 0 : units, joins};
        int at[3];  // the span's first
        if (e0) __syncthreads();  // (what the last round read is read)
        for (int k = 0; k < 3; k++) {
            int total;
            at[k] = wave_scan(mine[k], &total) - mine[k];
            if (lane == 0) totals[k][wave] = total;
        }
        __syncthreads();
        for (int k = 0; k < 3; k++) {
            const int of_wave = lane < waves ? totals[k][lane] : 0;
            int total;
            const int upto = wave_scan(of_wave, &total);
            at[k] += done[k] + __builtin_amdgcn_readlane(upto - of_wave, wave);
            done[k] += total;
        }
        const int e = e0 + tid, base = n.large ? at[0] : at[1];
        const int flags = (n.large ? kLarge : 0) | (n.shared ? kShared : 0) | (n.joined ? kJoined : 0) | (whole ? kWhole : 0);
        if (e < all) p.spans[e] = SpanRecord{n.table, n.span.begin, n.span.rows, n.span.first, n.lo, n.hi, n.tiles, nsplit, base, flags, {}};
        // (more tasks than there is room for are those of a batch whose starts fall)
        struct Tasks {
            int span, base, large;
        };
        each(units, Tasks{e, base, n.large}, [&](const Tasks &u, int i) {
            if (u.base + i < (u.large ? p.large_slots : p.small_slots)) (u.large ? p.large_tasks : p.small_tasks)[u.base + i] = Place{u.span, i};
        });
        struct Joins {
            int to, begin, rows, base, tiles, parts, flags;
        };
        each(joins, Joins{at[2], n.span.begin, n.span.rows, base, n.tiles, nsplit, flags}, [&](const Joins &u, int i) {
            const int tile = u.flags & kLarge ? i / 4 : i, slot = u.base + (u.tiles - 1 - tile) * u.parts;
            // (nor has a tile parts past that room)
            const int parts = slot + u.parts <= (u.flags & kLarge ? p.large_slots : p.small_slots) ? u.parts : 0;
            if (u.to + i < p.join_slots) p.joins[u.to + i] = JoinRecord{u.begin, u.rows, i, slot, parts, u.flags, {}};
        });
        struct Rows {
            OwnRecord own;
            int first;
        };
        each(n.shared ? 0 : n.span.rows, Rows{OwnRecord{base, n.span.begin, n.tiles, nsplit | (n.large ? kOwnLarge : 0)}, n.span.first},
             [&](const Rows &u, int i) {
                 p.positions[u.own.begin + i] = u.first + i;
                 p.own[u.own.begin + i] = u.own;
             });
    }
    if (tid == 0) *p.header = PlanHeader{min(done[0], p.large_slots), min(done[1], p.small_slots), min(done[2], p.join_slots)};
}

// ------------------------------------------------------------------------------ the tasks

// The positions of a tile's rows: one after the other in a sequence, in a group's span its sequences'. A lane's
// pair has its position in LDS too, from where it is read in every page rather than kept.
struct InTile {
    const int *positions;  // the span's rows'; null: a sequence's
    int first, low, high;
    const int *pairs;
    __device__ __forceinline__ int of(int at) const { return positions ? positions[at] : first + at; }
    __device__ __forceinline__ int again(const Pair &, int pair) const { return pairs[pair]; }
};

// The least and the largest of the wave's values.
__device__ __forceinline__ void wave_ends(int v, int &low, int &high)
{
    low = high = v;
#pragma unroll
    for (int step = 32; step; step >>= 1) {
        low = min(low, __shfl_xor(low, step));
        high = max(high, __shfl_xor(high, step));
    }
    low = __builtin_amdgcn_readfirstlane(low), high = __builtin_amdgcn_readfirstlane(high);
}

// The pages of a task: of those from lo to hi that rows at positions low to high see, its part.
__device__ __forceinline__ PageRange part_of(const SpanRecord &t, int split, int low, int high, int window)
{
    PageRange r;
    r.hi = min(t.hi, high < 0 ? 0 : high / kPage + 1);  // (the largest int: all)
    r.lo = min(max(first_seen(low, window) / kPage, t.lo), r.hi);
    const int n = (r.hi - r.lo + t.nsplit - 1) / t.nsplit;
    r.lo = min(r.lo + split * n, r.hi);
    r.hi = min(r.lo + n, r.hi);
    r.lo = __builtin_amdgcn_readfirstlane(r.lo), r.hi = __builtin_amdgcn_readfirstlane(r.hi);
    return r;
}

// A workgroup a large task and key head, or a wave a small one and key head: both kinds in one launch, the large ones first,
// so that the sequences' own pages are read while the shared ones multiply.
// Bounded by the matrix cores and vector units in turns, like attend_many_kernel: a large tile's page takes 4900 cycles with one
// workgroup a CU and 5800 to 7000 with two, after 8500 to 10500 for the record, the queries and the first page, 3000 to 4000 more in
// the first page, whose code is not in the instruction cache yet, and 2200 for the part. 32 questions behind 60160 tokens (16 heads of
// 128 over 4): 42 us, 31.6 GF of two-piece products, 745 TFLOP/s; the matrix cores are busy 42 % of the cycles, the vector
// units 46, waits are 23. 64 conversations behind 8192, whose four pages a part are mostly the first: 21 us, 417 TFLOP/s, 24 %.
// 256 sequences in five groups, 73 MB of their own pages beside them: 57 us.
// (Eight waves a workgroup, four every second page, which halves the parts: 37 / 55 / 72 us for these against 36 / 57 / 72, and
// where parts are few 10 % slower; waves of the same SIMD at different priorities, or started apart, the queries asked for before
// the page table's entries, the next page stored after the products instead of before: no difference. A large task a CU, small
// ones beside them, then the other large ones: 256 sequences 70, the last large ones starting late.)
template <int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void shared_tasks_kernel(SharedParams p)
{
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ int pair_positions[128];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const PlanHeader header = *p.header;
    const unsigned large_blocks = unsigned(header.large) * unsigned(p.kv_heads);
    const bool large = blockIdx.x < large_blocks;
    const unsigned unit = large ? blockIdx.x : (blockIdx.x - large_blocks) * 4 + unsigned(wave);
    const int index = int(unit / unsigned(p.kv_heads)), kv = int(unit % unsigned(p.kv_heads));
    if (!large && index >= header.small) return;  // the wave
    const Place place = (large ? p.large_tasks : p.small_tasks)[index];
    const SpanRecord t = p.spans[__builtin_amdgcn_readfirstlane(place.span)];
    const int split = place.at % t.nsplit, tile = t.tiles - 1 - place.at / t.nsplit;
    const bool shared = t.flags & kShared;
    Task task{};
    task.seq = t.table;
    task.tile = tile;
    task.nsplit = t.nsplit;
    task.span = Span{t.begin, t.rows, t.first, 0};
    task = uniform(task);
    const int32_t *table = p.b.pages + size_t(task.seq) * p.b.max_pages;
    InTile places{shared ? p.positions + t.begin : nullptr, t.first, 0, 0, pair_positions};
    const int pairs = t.rows * p.group, tm = large ? 128 : 16;
    auto row_of = [&](int pair) { return min(tile * tm + pair, pairs - 1) / p.group; };
    // the positions of the tile's first and last row, of a group's only where a window asks for them: with none its rows see
    // all shared pages (or the mask hides what they do not)
    int low = 0, high = INT_MAX;
    if (!shared) low = t.first + row_of(0), high = t.first + row_of(tm - 1);
    if (large) {
        const int mine = places.of(row_of(wave * 32 + (lane & 31)));
        if (lane < 32) pair_positions[wave * 32 + lane] = mine;
        if (shared && p.window > 0) {
            __syncthreads();
            int other;
            wave_ends(min(pair_positions[lane], pair_positions[64 + lane]), low, other);
        }
        const PageRange range = part_of(t, split, low, high, p.window);
        wave_ends(mine, places.low, places.high);
        float *parts = p.partial + size_t(blockIdx.x) * 4 * many_floats(DP);
        __builtin_assume(parts != nullptr);
        attend_many<DP, true>(p, task, range, table, kv, places, SplitQueries{p.pieces, p.factors}, lds, parts);
    } else {
        wave_ends(places.of(row_of(lane & 15)), places.low, places.high);
        const PageRange range = part_of(t, split, shared ? places.low : low, high, p.window);
        attend_few<DP, 1>(p, task, range, table, kv, places, SplitQueries{p.pieces, p.factors}, static_cast<FewJoin<DP> *>(nullptr),
                          t.flags & kWhole ? nullptr : p.small_partial + size_t(unit) * few_floats(DP));
    }
}

// ------------------------------------------------------------------------------- the join

constexpr int kPieces = 2;  // of a part, a kilobyte each, that a wave has at once
constexpr int kJoinWaves = 8;

struct Sums {
    float r, total;
    v4f o[kPieces];
};

// The sums of both in `to`.
__device__ __forceinline__ void add_sums(Sums &to, const Sums &from)
{
    const float r = fmaxf(to.r, from.r);
    const float a = part_factor(to.r, r), b = part_factor(from.r, r);
    to.r = r;
    to.total = to.total * a + from.total * b;
#pragma unroll
    for (int i = 0; i < kPieces; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) to.o[i][e] = to.o[i][e] * a + from.o[i][e] * b;
}

// `count` parts, from the one at `part` on, `step` floats apart: the row's sums are at `row` in each, the pieces' values at
// `values` and `next`.
__device__ __forceinline__ void add_parts(Sums &to, const float *part, size_t step, int count, int row, int values, int next)
{
    constexpr int kAhead = 4;
    for (int s0 = 0; s0 < count; s0 += kAhead) {
        Sums from[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const float *at = part + size_t(min(s0 + i, count - 1)) * step;
            from[i].r = at[row];
            from[i].total = at[64 + row];
            from[i].o[0] = *reinterpret_cast<const v4f *>(at + values);
            from[i].o[1] = *reinterpret_cast<const v4f *>(at + next);
        }
        float top = to.r;
#pragma unroll
        for (int i = 0; i < kAhead; i++) top = s0 + i < count ? fmaxf(top, from[i].r) : top;
        const float a = part_factor(to.r, top);
        to.r = top;
        to.total = to.total * a;
#pragma unroll
        for (int k = 0; k < kPieces; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) to.o[k][e] = to.o[k][e] * a;
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (s0 + i >= count) continue;
            const float b = part_factor(from[i].r, top);
            to.total = to.total + from[i].total * b;
#pragma unroll
            for (int k = 0; k < kPieces; k++)
#pragma unroll
                for (int e = 0; e < 4; e++) to.o[k][e] = to.o[k][e] + from[i].o[k][e] * b;
        }
    }
}

// Eight waves, or where there are many of them four, a join, key head and two kilobytes of a part: lane l has a pair and four
// dimensions of each, as the tasks left them, so that parts are read whole lines at a time. The waves take the parts in
// turn, but the last one the rows' own where these are apart.
// Bounded by waits: its record, a row's own, the parts, the exchange, one after the other, 80 % of the waves' cycles. 1024 pairs
// of 32 parts, 17 MB, 7.9 us; 512 of 118, 31 MB, 9.9; 3920 of up to 23 9.6. (A team of lanes a row and head, whose parts
// lie in lines that others read too: 12.5, 18.1 and 13.0.)
template <int DP>
__global__ __launch_bounds__(kJoinWaves * 64) void shared_join_kernel(SharedParams p)
{
    constexpr unsigned kSteps = DP / 16;  // of a large tile's quarter; a small tile has half
    __shared__ Sums sums[kJoinWaves][64];
    const int lane = threadIdx.x & 63, all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned units = unsigned(p.header->joins) * unsigned(p.kv_heads) * kSteps;
    const int waves = units <= 2 * kUnits ? kJoinWaves : kJoinWaves / 2;
    const int wave = all_waves % waves;
    const unsigned at_once = unsigned(kJoinWaves / waves);
    for (unsigned unit0 = blockIdx.x * at_once; unit0 < units; unit0 += gridDim.x * at_once) {
        const unsigned unit = unit0 + unsigned(all_waves / waves);
        const int piece = int(unit % kSteps) * kPieces, kv = int(unit / kSteps % unsigned(p.kv_heads));
        JoinRecord t = p.joins[min(unit / kSteps / unsigned(p.kv_heads), unsigned(p.join_slots - 1))];  // (asked for beside their number)
        const bool there = unit < units, large = t.flags & kLarge, shared = t.flags & kShared;
        const int rows = large ? 32 : 16, width = 256 / rows, pairs = there ? t.rows * p.group : 0;
        const int pair = t.at * rows + (lane & (rows - 1)), dim = piece * width + 4 * (lane / rows);
        const bool live = there && pair < pairs && piece < rows * DP / 256;
        const int at = min(pair, pairs - 1) / p.group, row = t.begin + at, in_group = min(pair, pairs - 1) - at * p.group;
        Sums mine{-INFINITY, 0.0f, {}};
        const int others = shared ? waves - 1 : waves;
        if (wave < others) {
            const size_t floats = large ? many_floats(DP) : few_floats(DP), task = large ? 4 * floats : floats;
            const float *part = (large ? p.partial : p.small_partial) + (size_t(t.slot + wave) * p.kv_heads + kv) * task + (large ? t.at % 4 * floats : 0);
            const int values = 128 + piece * 256 + lane * 4;
            if (there && wave < t.parts && piece < rows * DP / 256)
                add_parts(mine, part, size_t(others) * p.kv_heads * task, (t.parts - wave + others - 1) / others, lane, values, values + 256);
        } else if (live) {
            // (64 bits and every check: a row that no sequence holds, of a batch whose starts fall, may have any record)
            const OwnRecord o = p.own[row];
            const bool own_large = o.parts & kOwnLarge;
            const int tm = own_large ? 128 : 16, parts = o.parts & (kOwnLarge - 1);
            const int64_t m = (int64_t(row) - o.begin) * p.group + in_group, tile = m / tm;
            const int64_t slot = o.base + (int64_t(o.tiles) - 1 - tile) * parts;
            const int own = int(m & (tm - 1));
            // where in a part the four values from dimension d on are
            auto values = [&](int d) {
                const int q = d / 4;
                return own_large ? 128 + (q / 2) * 256 + (own % 32 + 32 * (q & 1)) * 4 : 128 + (q / 4) * 256 + (own + 16 * (q & 3)) * 4;
            };
            const size_t floats = own_large ? many_floats(DP) : few_floats(DP), task = own_large ? 4 * floats : floats;
            if (m >= 0 && tile < o.tiles && parts <= kSharedSplit && slot >= 0 &&
                slot + parts <= (own_large ? p.large_slots : p.small_slots)) {
                const float *part = (own_large ? p.partial : p.small_partial) + (size_t(slot) * p.kv_heads + kv) * task +
                                    (own_large ? own / 32 * floats : 0);
                add_parts(mine, part, p.kv_heads * task, parts, own_large ? own % 32 : own, values(dim), values(dim + width));
            }
        }
        sums[all_waves][lane] = mine;
        __syncthreads();
        if (wave == 0 && live) {
            for (int w = 1; w < waves; w++) add_sums(mine, sums[all_waves + w][lane]);
            float *to = p.out + size_t(row) * p.out_stride + size_t(kv * p.group + in_group) * p.head_dim + dim;
#pragma unroll
            for (int i = 0; i < kPieces; i++) {
                v4f x;
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = mine.total == 0.0f ? 0.0f : mine.o[i][e] / mine.total;
                if (dim + i * width < p.head_dim) *reinterpret_cast<v4f_any *>(to + i * width) = x;
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------- the host

struct Launch {
    bool shared;  // or each sequence by itself
    int limit, target;
    size_t large_slots, small_slots, join_slots, blocks;  // of a key head but the blocks
    size_t at[11];  // where in the scratch the arrays are, and its size
};

// Whether a step's shared pages are worked through apart: three launches, of which the plan and the join cost 10 to 15 us, pay
// where what all sequences may see of their tables together, all of them or a window, holds 224 MiB (the host knows no more of the
// lengths). Microseconds, each sequence by itself and shared, of S sequences of one new token behind P shared pages and up to 5 of
// their own: 16 heads of 128 over 4 (a page is 66 KiB), S = 8: P = 115 19 and 24, 400 32 and 32, 1000 56 and 46; S = 32: 45 23 and 28, 115 34 and 30, 400 78
// and 42, 1000 171 and 60; S = 256: 8 31 and 31, 20 45 and 33, 200 260 and 81; 14 of 64 over 2 (17 KiB), S = 32: 400 32
// and 36, 1000 61 and 46; S = 128: 45 22 and 26, 115 36 and 36, 400 91 and 55. With windows over 400 pages of 66 KiB: S = 64, 800
// tokens 18 and 30, 3000 28 and 31, 8000 53 and 36; S = 256: 100 21 and 28, 800 36 and 35, 3000 77 and 46.
// Of 220 steps of 4 to 256 sequences in 1 to 5 groups behind 10 to 900 pages, 1 to 10 rows each (as many in all sequences of a
// step), heads of 36 to 256, the way chosen so takes 1.9 % longer than the faster one on average (from 160 or 256 MiB on 2.5 and 3.0; always the one way or the other 17 and 16).
// (How many groups are named says nothing: arrays with room for a group a sequence may hold one group of all. Such arrays and arrays of
// one group take the same time, 16 of 128 over 4, S = 8: P = 1301 49 and 49, 64 by itself; S = 128: 79 37 and 37, 58. Where
// nothing is shared the two launches and the single waves cost, groups of one sequence each: S = 8: P = 478 60, 52 by itself, 1304 145 and
// 137; S = 128: 30 68 and 46, 82 153 and 130; S = 256: 41 166 and 128.)
// Nor where the sequences have more than 96 pairs of a new token and a head of a key head on average (64 of heads past 128): a
// prompt's chunks fill tiles of their own, and the parts cost what is left to gain: 17 chunks of 1 to 512 tokens behind 94
// pages, 14 heads of 64 over 2, 95 and 124; 16 of 60 tokens behind 100, 16 of 128 over 4, 123 and 156. One long chunk among single tokens
// takes their sharing away so: 63 behind 940 pages beside 2048 rows 2498, where the two apart take 76 and 1286.
constexpr double kSharedBytes = 7 * 0x1p25;

Launch plan_launch(const fg_cache *c, const fg_batch *b, const fg_prefixes *f, size_t heads, size_t window)
{
    Launch l{};
    const size_t group = heads / c->kv_heads, pairs = b->rows * group, sequences = std::min(b->sequences, b->rows);
    const size_t groups = std::min(f->groups, sequences);
    l.limit = c->padded <= 128 ? 96 : 64;
    const size_t pages = window ? std::min(b->max_pages, window / kPage + 2) : b->max_pages;
    const double bytes_held = double(sequences) * double(pages) * double(c->kv_heads) * double(record_bytes(c->padded));
    l.shared = groups && sequences > 1 && bytes_held >= kSharedBytes && pairs <= size_t(l.limit) * sequences;
    if (!l.shared) return l;
    const size_t units = std::max<size_t>(kUnits / c->kv_heads, 1);
    l.target = int((c->padded <= 128 ? 2 : 1) * units);
    // spans of n pairs have at most n / 128 + 1 large tiles, or n / 16 + 1 small ones; what a share of the target
    // leaves of the work are its tiles' further parts, of small tiles four times as many
    size_t large = 0, small = 0;
    auto add = [&](size_t spans, size_t limit) {
        large += pairs > limit ? pairs / 128 + std::min(spans, pairs / (limit + 1)) : 0;
        small += std::min(pairs / 16 + spans, limit / 16 * spans);
    };
    add(groups, kGroupLimit);
    add(sequences, size_t(l.limit));
    l.large_slots = large ? large + l.target : 0;
    l.small_slots = small + 4 * l.target;
    l.join_slots = 4 * large + small;
    l.blocks = l.large_slots * c->kv_heads + (l.small_slots * c->kv_heads + 3) / 4;
    const size_t floats = 4 * size_t(many_floats(c->padded));
    const size_t bytes[10] = {sizeof(PlanHeader), l.large_slots * sizeof(Place), l.small_slots * sizeof(Place),
                             l.join_slots * sizeof(JoinRecord), b->rows * (sizeof(int) + sizeof(OwnRecord)), (f->groups + b->sequences) * sizeof(SpanRecord),
                             l.large_slots * c->kv_heads * floats * 4, l.small_slots * c->kv_heads * size_t(few_floats(c->padded)) * 4,
                             pair_blocks(b->rows, int(group)) * 32 * c->kv_heads * size_t(c->padded) * 4,
                             pair_blocks(b->rows, int(group)) * 32 * c->kv_heads * 4};
    for (int i = 0; i < 10; i++) l.at[i + 1] = l.at[i] + (bytes[i] + 255) / 256 * 256;
    return l;
}

template <int DP>
int launch_shared(const SharedParams &p, const Launch &l, hipStream_t s)
{
    if (many_lds<DP>() > 60 * 1024) {  // more than the default limit, with the positions: raised once a device
        static std::atomic<unsigned long long> raised{0};
        int device = 0;
        FG_HIP(hipGetDevice(&device));
        const unsigned long long bit = 1ull << (device & 63);
        if (device > 63 || !(raised.load() & bit)) {
            FG_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(shared_tasks_kernel<DP>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                       int(many_lds<DP>())));
            raised.fetch_or(bit);
        }
    }
    const unsigned threads = size_t(p.groups) + p.b.sequences <= kFewSpans ? kPlanThreads / 2 : kPlanThreads;
    const size_t per = size_t(threads / (DP <= 32 ? 4 : DP == 64 ? 8 : DP <= 128 ? 16 : 32));  // rows and heads of a workgroup
    shared_plan_kernel<<<unsigned(1 + std::min<size_t>((size_t(p.b.rows) * p.heads + per - 1) / per, 2 * kUnits)), threads, 0, s>>>(p, DP);
    FG_HIP(hipGetLastError());
    shared_tasks_kernel<DP><<<unsigned(l.blocks), 256, many_lds<DP>(), s>>>(p);
    FG_HIP(hipGetLastError());
    shared_join_kernel<DP><<<unsigned(std::min(l.join_slots * p.kv_heads * (DP / 16), 4 * kUnits)), kJoinWaves * 64, 0, s>>>(p);
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
    // (either way: with a window the call may take the other one)
    const Launch l = plan_launch(c, b, f, heads, 0);
    return std::max(l.at[10], fg_cache_attend_scratch(c, b, heads));
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
    const Launch l = plan_launch(c, b, f, heads, window);
    if (!l.shared)
        return fg_cache_attend(c, b, query, query_stride, heads, scale, window, out, out_stride, scratch, scratch_bytes, stream);
    if (l.blocks > kMaxGrid || l.join_slots * c->kv_heads * (c->padded / 16) > 0xf0000000)
        return set_error(FG_ERR_SHAPE, std::string(who) + ": more sequences times heads than a launch takes");
    const hipStream_t s = as_stream(stream);
    void *ws = nullptr;
    bool owned = false;
    rc = stream_scratch(scratch, scratch_bytes, l.at[10], who, s, &ws, &owned);
    if (rc) return rc;
    SharedParams p = attend_params<SharedParams>(c, b, query, query_stride, heads, scale, window, out, out_stride);
    p.starts = f->starts;
    p.counts = f->pages;
    p.groups = int(f->groups);
    p.limit = l.limit;
    p.target = l.target;
    p.large_slots = int(l.large_slots);
    p.small_slots = int(l.small_slots);
    p.join_slots = int(l.join_slots);
    char *at = static_cast<char *>(ws);
    p.header = reinterpret_cast<PlanHeader *>(at);
    p.large_tasks = reinterpret_cast<Place *>(at + l.at[1]);
    p.small_tasks = reinterpret_cast<Place *>(at + l.at[2]);
    p.joins = reinterpret_cast<JoinRecord *>(at + l.at[3]);
    p.own = reinterpret_cast<OwnRecord *>(at + l.at[4]);
    p.positions = reinterpret_cast<int *>(at + l.at[4] + b->rows * sizeof(OwnRecord));
    p.spans = reinterpret_cast<SpanRecord *>(at + l.at[5]);
    p.partial = reinterpret_cast<float *>(at + l.at[6]);
    p.small_partial = reinterpret_cast<float *>(at + l.at[7]);
    p.pieces = reinterpret_cast<uint4 *>(at + l.at[8]);
    p.factors = reinterpret_cast<float *>(at + l.at[9]);
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
