// Attention of a step's new tokens over the paged 8-bit cache (fg_cache_attend), each sequence by itself: the tasks of a
// step, the kernels' routing and the join of a tile's parts. cache_attend.h has what a workgroup does with a task.
#include <algorithm>
#include <atomic>

#include "cache_attend.h"

namespace fg {
namespace {

// ---------------------------------------------------------------------------- the plan
//
// The rows of a tile are (new token, query head of the key head's group) pairs, token-major: tile t of a
// sequence holds pairs t·TM .. of its rows·group. A tile's pages are split over the sequence's nsplit
// tasks. Every workgroup finds its task from the batch's arrays by itself: nothing about the lengths is
// known on the host.
__device__ __forceinline__ int tiles_of(const AttendParams &p, const Span &s, int TM) { return (s.rows * p.group + TM - 1) / TM; }

// Pages that a tile of the sequence sees at most.
__device__ __forceinline__ int tile_pages(const AttendParams &p, const Span &s, int TM)
{
    if (s.rows <= 0) return 0;
    const PageRange r = pages_seen(s, 0, s.rows - 1, p.window, p.b.max_pages);
    const int all = r.hi - r.lo;
    return p.window > 0 ? min(all, p.window / kPage + TM / p.group / kPage + 3) : all;
}

// Pages a part takes: the whole work spread over the target (a little more than its share: the sum is
// in f32).
__device__ __forceinline__ int part_pages(const AttendParams &p, int TM)
{
    if (!p.target) return INT_MAX;
    const int lane = threadIdx.x & 63;
    float work = 0.0f;
    for (int s0 = 0; s0 < p.b.sequences; s0 += 64) {
        if (s0 + lane >= p.b.sequences) continue;
        const Span span = sequence_span(p.b, s0 + lane);
        work = work + float(tiles_of(p, span, TM)) * float(tile_pages(p, span, TM));
    }
    const float part = wave_allsum(work) * 1.00001f / float(p.target) + 1.0f;
    return __builtin_amdgcn_readfirstlane(part < float(kMinPages) ? kMinPages : part > 1e9f ? 1000000000 : int(part));
}

__device__ __forceinline__ int splits_of(int pages, int part)
{
    return pages <= part ? 1 : min((pages + part - 1) / part, kMaxSplit);
}

// The task of index x, or seq -1.
__device__ __forceinline__ Task find_task(const AttendParams &p, int x, int TM)
{
    const int part = part_pages(p, TM);
    Task t{};
    int within;
    t.seq = find_unit(p.b.sequences, x, &within, [&](int s) {
        const Span span = sequence_span(p.b, s);
        return tiles_of(p, span, TM) * splits_of(tile_pages(p, span, TM), part);
    });
    if (t.seq < 0) return t;
    t.span = sequence_span(p.b, t.seq);
    t.nsplit = splits_of(tile_pages(p, t.span, TM), part);
    // the last tiles see the most keys: they come first
    t.tile = tiles_of(p, t.span, TM) - 1 - within / t.nsplit;
    t.split = within % t.nsplit;
    t.slot = x;
    return t;
}

// What the join takes of a task, by its slot: the parts that start here (0: none, or one alone) and the
// tile's rows. Every workgroup of the grid leaves a note, those without a task too.
struct Note {
    int parts, tile, begin, rows, first;
};
__device__ __forceinline__ void leave_note(const AttendParams &p, const Task &t, int x, int kv)
{
    if (!p.target || kv != 0 || threadIdx.x != 0) return;
    const bool starts = t.seq >= 0 && t.split == 0 && t.nsplit > 1;
    p.notes[x] = Note{starts ? t.nsplit : 0, t.tile, t.span.begin, t.span.rows, t.span.first};
}

// The pages [lo, hi) of a task.
__device__ __forceinline__ PageRange task_pages(const AttendParams &p, const Task &t, int TM)
{
    const int row = t.tile * TM / p.group, last = min((t.tile * TM + TM - 1) / p.group, t.span.rows - 1);
    PageRange r = pages_seen(t.span, row, last, p.window, p.b.max_pages);
    const int n = (r.hi - r.lo + t.nsplit - 1) / t.nsplit;
    r.lo = min(r.lo + t.split * n, r.hi);
    r.hi = min(r.lo + n, r.hi);
    return r;
}

template <int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void attend_few_kernel(AttendParams p)
{
    constexpr int TM = 16;
    __shared__ __align__(16) FewJoin<DP> join;
    const int x = int(blockIdx.x / unsigned(p.kv_heads)), kv = int(blockIdx.x % unsigned(p.kv_heads));
    const Task task = uniform(find_task(p, x, TM));
    leave_note(p, task, x, kv);
    if (task.seq < 0) return;  // the whole workgroup
    const int low = task.span.first + task.tile * TM / p.group;
    const int high = task.span.first + min((task.tile * TM + TM - 1) / p.group, task.span.rows - 1);
    float *part = task.nsplit > 1 ? p.partial + (size_t(task.slot) * p.kv_heads + kv) * few_floats(DP) : nullptr;
    attend_few<DP, 4>(p, task, task_pages(p, task, TM), p.b.pages + size_t(task.seq) * p.b.max_pages, kv,
                      InSequence{task.span.first, low, high}, RawQueries{}, &join, part);
}

template <int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void attend_many_kernel(AttendParams p)
{
    constexpr int TM = 128;
    extern __shared__ __align__(16) uint8_t lds[];
    const int x = int(blockIdx.x / unsigned(p.kv_heads)), kv = int(blockIdx.x % unsigned(p.kv_heads));
    const Task task = uniform(find_task(p, x, TM));
    leave_note(p, task, x, kv);
    if (task.seq < 0) return;  // the whole workgroup
    // the positions of the wave's first and last pairs
    const int pairs = task.span.rows * p.group, m0 = task.tile * TM + int(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 32;
    const int low = task.span.first + min(m0, pairs - 1) / p.group, high = task.span.first + min(m0 + 31, pairs - 1) / p.group;
    float *parts = task.nsplit > 1 ? p.partial + (size_t(task.slot) * p.kv_heads + kv) * 4 * many_floats(DP) : nullptr;
    attend_many<DP, false>(p, task, task_pages(p, task, TM), p.b.pages + size_t(task.seq) * p.b.max_pages, kv,
                    InSequence{task.span.first, low, high}, RawQueries{}, lds, parts);
}

// The parts of split tiles joined: per slot where a tile's parts start and head, a wave for each tile of
// ROWS pairs and piece of dimensions (four a lane, the lanes as the kernels above hold them). Launch and
// the chain of note, parts, division bound it: 4.2 us for 64 sequences of up to 8000 tokens, 8 for 500 parts of 8
// long ones, 7 for chunks of 1300 rows, 14 heads of 64.
template <int DP, int ROWS, int TILES>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendParams p)
{
    constexpr int TM = ROWS * TILES, C = ROWS * DP / 256;  // pieces
    const int lane = threadIdx.x & 63, kv = int(blockIdx.x % unsigned(p.kv_heads)), x = int(blockIdx.x / unsigned(p.kv_heads));
    const int unit = __builtin_amdgcn_readfirstlane(int(blockIdx.y) * 4 + int(threadIdx.x >> 6));
    const Note note = p.notes[x];
    const int parts = __builtin_amdgcn_readfirstlane(note.parts);
    if (parts == 0 || x + parts > p.grid || unit >= TILES * C) return;  // (the second: starts that fall)
    const int tile = unit / C, c = unit % C;
    constexpr size_t kPart = ROWS == 16 ? few_floats(DP) : many_floats(DP);
    const size_t step = size_t(p.kv_heads) * TILES * kPart;
    const float *part = p.partial + ((size_t(x) * p.kv_heads + kv) * TILES + tile) * kPart;
    Task t{};
    t.span = Span{note.begin, note.rows, note.first, note.first + note.rows};
    const Pair pair = pair_of(p, t, kv, note.tile * TM + tile * ROWS + (lane & (ROWS - 1)), InSequence{note.first, 0, 0});
    if (!pair.live) return;  // (its sums are not written)
    // eight parts at a time, joined like the waves' sums
    constexpr int kAhead = 8;
    float r = -INFINITY, total = 0.0f;
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < parts; s0 += kAhead) {
        float rs[kAhead], totals[kAhead];
        v4f os[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const float *from = part + min(s0 + i, parts - 1) * step;
            rs[i] = from[lane];
            totals[i] = from[64 + lane];
            os[i] = *reinterpret_cast<const v4f *>(from + 128 + c * 256 + lane * 4);
        }
        float top = r;
#pragma unroll
        for (int i = 0; i < kAhead; i++) top = s0 + i < parts ? fmaxf(top, rs[i]) : top;
        const float a = part_factor(r, top);
        r = top;
        total = total * a;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = o[e] * a;
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (s0 + i >= parts) continue;
            const float b = part_factor(rs[i], top);
            total = total + totals[i] * b;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = o[e] + os[i][e] * b;
        }
    }
    const int dim = c * (256 / ROWS) + 4 * (lane / ROWS);
    if (dim >= p.head_dim) return;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = total == 0.0f ? 0.0f : o[e] / total;
    *reinterpret_cast<v4f_any *>(p.out + size_t(pair.row) * p.out_stride + size_t(pair.head) * p.head_dim + dim) = o;
}

// ------------------------------------------------------------------------------ the host

struct Launch {
    bool few;
    size_t grid;  // a bound on the tasks of a head
    int target;
    size_t note_bytes, partial_bytes;
};

// Which kernel a step takes, and whether its tiles are split, from what the host knows of it: microseconds of
// decode steps and chunks over caches of random or equal lengths, 16 query heads of 128 over 4 key heads (a), 14 of
// 64 over 2 (b), 8 of 128 over 1 (c).
//
// attend_few_kernel up to 96 pairs a sequence, few's time and many's: 64 sequences of up to 3200 tokens, 48 pairs
// (a) 66 and 91, 84 pairs (b) 32 and 43, 96 pairs (a) 92 and 100, (c) 43 and 38; 128 pairs (a) 112 and 114, (c) 50
// and 40. Up to 64 for heads past 128: 8 heads of 256 over 2, 48 pairs 89 and 94, 64 pairs 104 and 96, 96 pairs 134
// and 101; 8 of 192 over 1, 64 pairs 50 and 51, 96 73 and 56.
//
// Tiles are split when there are at most as many as CUs, all heads together: 64 sequences of up to 8000 tokens
// (a) 71 whole and 56 split, (b) 42 and 21; all of 8000, which a CU each serves evenly, (a) 98 and 108; 128 sequences
// (a), two a CU, 132 and 135. Of small tiles not over tables of up to 16 pages: joining costs about 4 us, as
// much as ten pages, and as much again on the host (500 tokens: 10.3 whole, 11.2 split). A large tile's page costs 1.5 to 3.5 us,
// and what joining costs grows with the tiles: they are split over more than 4 pages, or more than 32 pages times the share of the
// CUs that they fill (to 16). A chunk of 102 rows over 5 / 7 / 11 pages, whole and split: (b) 15.4 14.5 / 18.4 15.8 / 24.5 16.3,
// (a) 19.8 17.7 / 24.3 19.9 / 32.4 19.9, 8 of 256 over 2 32 26 / 39 29 / 54 30 (the host knows the table, not the
// length: the same rows with nothing before them, two pages, pay for the join, 13.0 and 10.8, (a) 16.1 and 13.7); four of 120 over 7 / 9 / 13 (a) 25 25 / 29 24 / 37 32;
// 13 of 78, half of the CUs, over 7 / 16 (a) 25 35 / 44 40, (b) 19 24 / 33 38. Two workgroups a CU read at once what memory
// gives, so the parts aimed at are two a CU, less half of one a tile, whose last part is half a part on average:
// fewer leave some CUs two parts and others one (eight documents of 30000 to 70000 tokens: 288 parts 105, 350 98,
// 512 88), more start and end too often (1024: 104). 64 sequences as above (a): 384 parts 61 and of equal lengths
// 130, 512 56 and 108, 640 64 and 130. Heads past 128 leave one workgroup a CU, and as many parts: 8 heads of 256 over 2,
// 8 sequences of 8000 tokens, 25 us and for two a CU 38, 64 of up to 2000 28 and 38, a chunk of 512 rows 55 and 72.
//
// Both rules go by a step's means, all that the host knows, and cost uneven steps: 64 sequences of 6 to 8000 tokens, even
// over their logarithm,
// (a) 26.5 and 65 of them 59.7; one of 70000 beside 100 of 500 (a) 485, alone 32 (slots without rows are no sequences: with
// 100 of those 33); 63 tokens after 2000 others each and a chunk of 512 (a) 45, of 2048 97, where the two apart take
// 30 + 35 and 30 + 64, (b) 25 and 60, apart 15 + 33 and 15 + 43. And every workgroup looks through all sequences for
// its task, 64 at a time: 256 sequences of 500 tokens (a) 34, 1024 177, 4096 1430, of which memory's share is 417.
Launch plan_launch(const fg_cache *c, const fg_batch *b, size_t heads)
{
    Launch l{};
    const size_t group = heads / c->kv_heads, pairs = b->rows * group, sequences = std::min(b->sequences, b->rows);
    l.few = pairs <= (c->padded <= 128 ? 96 : 64) * sequences;
    const size_t tm = l.few ? 16 : 128, units = std::max<size_t>(kUnits / c->kv_heads, 1);
    const size_t tiles = std::max(pairs / tm, sequences);  // about
    l.grid = pairs / tm + sequences;
    if (tiles <= units && b->max_pages > (l.few ? 16 : std::min<size_t>(std::max<size_t>(32 * tiles / units, 4), 16))) {
        l.target = int((c->padded <= 128 ? 2 : 1) * units - tiles / 2);
        const size_t most = std::min<size_t>((b->max_pages + kMinPages - 1) / kMinPages, kMaxSplit);
        l.grid = std::min(l.grid * most, l.grid + l.target);
        l.note_bytes = (l.grid * sizeof(Note) + 255) / 256 * 256;
        l.partial_bytes = l.grid * c->kv_heads * (tm * c->padded + (l.few ? 1 : 4) * 128) * 4;
    }
    return l;
}

template <int DP>
int launch_attend(const AttendParams &p, const Launch &l, hipStream_t s)
{
    const unsigned grid = unsigned(p.kv_heads * l.grid);
    if (l.few) {
        attend_few_kernel<DP><<<grid, 256, 0, s>>>(p);
        FG_HIP(hipGetLastError());
        if (l.target) attend_join_kernel<DP, 16, 1><<<dim3(grid, (16 * DP / 256 + 3) / 4), 256, 0, s>>>(p);
    } else {
        if (many_lds<DP>() > 64 * 1024) {  // more than the default limit: raised once a device
            static std::atomic<unsigned long long> raised{0};
            int device = 0;
            FG_HIP(hipGetDevice(&device));
            const unsigned long long bit = 1ull << (device & 63);
            if (device > 63 || !(raised.load() & bit)) {
                FG_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(attend_many_kernel<DP>),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, int(many_lds<DP>())));
                raised.fetch_or(bit);
            }
        }
        attend_many_kernel<DP><<<grid, 256, many_lds<DP>(), s>>>(p);
        FG_HIP(hipGetLastError());
        if (l.target) attend_join_kernel<DP, 32, 4><<<dim3(grid, 128 * DP / 256 / 4), 256, 0, s>>>(p);
    }
    FG_HIP(hipGetLastError());
    return FG_OK;
}

}  // namespace

int check_attend(const fg_cache *c, const fg_batch *b, const float *query, size_t heads, float scale, const float *out, size_t out_stride,
                 const char *who)
{
    const std::string name(who);
    const int rc = check_batch(c, b, who);
    if (rc) return rc;
    if (!heads || heads % c->kv_heads || heads > 65536)
        return set_error(FG_ERR_SHAPE, name + ": the heads must be a positive multiple of the cache's, at most 65536");
    if (!(std::fabs(scale) <= 2e38f))  // (times log2 e it is in f32's range)
        return set_error(FG_ERR_ARG, name + ": the scale must be a number of at most 2e38");
    if (!b->rows || !b->sequences) return FG_OK;
    if (!query || !out) return set_error(FG_ERR_ARG, name + ": a null query or output");
    const size_t width = heads * c->head_dim;
    if (b->rows > 1 && out_stride < width) return set_error(FG_ERR_SHAPE, name + ": a row's heads run past the row stride");
    if (b->rows * (heads / c->kv_heads) > (size_t(1) << 30))
        return set_error(FG_ERR_SHAPE, name + ": at most 2^30 rows times heads of a key head");
    return FG_OK;
}

}  // namespace fg

using namespace fg;

extern "C" size_t fg_cache_attend_scratch(const fg_cache *c, const fg_batch *b, size_t heads)
{
    if (!c || !b || !heads || heads % c->kv_heads) return 0;
    const Launch l = plan_launch(c, b, heads);
    return l.note_bytes + l.partial_bytes;
}

extern "C" int fg_cache_attend(const fg_cache *c, const fg_batch *b, const float *query, size_t query_stride, size_t heads,
                               float scale, size_t window, float *out, size_t out_stride, void *scratch, size_t scratch_bytes,
                               void *stream)
{
    int rc = check_attend(c, b, query, heads, scale, out, out_stride, "fg_cache_attend");
    if (rc) return rc;
    if (!b->rows || !b->sequences) return FG_OK;
    const hipStream_t s = as_stream(stream);
    const Launch l = plan_launch(c, b, heads);
    if (l.grid * c->kv_heads > kMaxGrid) return set_error(FG_ERR_SHAPE, "fg_cache_attend: more sequences times heads than a launch takes");
    AttendParams p = attend_params<AttendParams>(c, b, query, query_stride, heads, scale, window, out, out_stride);
    p.grid = int(l.grid);
    p.target = l.target;
    void *ws = nullptr;
    bool owned = false;
    rc = stream_scratch(scratch, scratch_bytes, l.note_bytes + l.partial_bytes, "fg_cache_attend", s, &ws, &owned);
    if (rc) return rc;
    p.notes = static_cast<Note *>(ws);
    p.partial = reinterpret_cast<float *>(static_cast<char *>(ws) + l.note_bytes);
    switch (c->padded) {
    case 32: rc = launch_attend<32>(p, l, s); break;
    case 64: rc = launch_attend<64>(p, l, s); break;
    case 96: rc = launch_attend<96>(p, l, s); break;
    case 128: rc = launch_attend<128>(p, l, s); break;
    case 192: rc = launch_attend<192>(p, l, s); break;
    default: rc = launch_attend<256>(p, l, s); break;
    }
    if (owned) {
        const hipError_t e = hipFreeAsync(ws, s);
        if (rc == FG_OK && e != hipSuccess) rc = check_hip(e, "hipFreeAsync");
    }
    return rc;
}
