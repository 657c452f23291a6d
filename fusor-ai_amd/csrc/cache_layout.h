// Where the paged cache keeps a token's levels, and which keys a step's rows see (plain C++: the
// kernels and the host share it).
#pragma once

#include <cstddef>
#include <cstdint>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define FG_BOTH __host__ __device__ __forceinline__
#else
#define FG_BOTH inline
#endif

namespace fg {

constexpr int kPage = 64;  // FG_CACHE_PAGE

// A page's record of one head is one run of bytes: the keys' levels, the values' levels, the 64 keys'
// scales, the 64 values'. Levels are stored as level + 128 (what the widening to f16 starts from), in
// the order in which the matrix cores' first operand takes them, blocks of 1 KiB of 64 lanes of 16 bytes:
//   keys   block (32 tokens, 32 dimensions): lane l holds token l % 32, dimensions 16 (l / 32) on;
//   values block (32 dimensions, 32 tokens): lane l holds dimension l % 32 and, with h = l / 32, the
//          tokens 8 j + 4 h + i at byte 4 j + i: those whose scores the same lane holds after a
//          32 x 32 product of keys and queries, so the weights are the next product's operand in place.
// The blocks of a token's keys are the record's [token / 32][dimension / 32], of its values
// [dimension / 32][token / 32]. head_dim is padded to one of the sizes that the kernels are built for.
FG_BOTH int padded_head(int d) { return d <= 128 ? (d + 31) / 32 * 32 : d <= 192 ? 192 : 256; }
FG_BOTH int record_bytes(int padded) { return 2 * kPage * padded + 2 * kPage * 4; }
FG_BOTH int key_byte(int padded, int token, int dim)
{
    return ((token >> 5) * (padded >> 5) + (dim >> 5)) * 1024 + (((dim >> 4) & 1) * 32 + (token & 31)) * 16 + (dim & 15);
}
FG_BOTH int value_byte(int padded, int token, int dim)
{
    return kPage * padded + ((dim >> 5) * 2 + (token >> 5)) * 1024 + (((token >> 2) & 1) * 32 + (dim & 31)) * 16 +
           ((token >> 3) & 3) * 4 + (token & 3);
}
FG_BOTH int key_scale_byte(int padded, int token) { return 2 * kPage * padded + token * 4; }
FG_BOTH int value_scale_byte(int padded, int token) { return 2 * kPage * padded + kPage * 4 + token * 4; }

// The scale kept beside a value all of whose levels are 0 (a key's is 1). It changes no product, but attention sets
// a row's reference from its largest weight times scale, and what adds nothing may not hide what does: at a scale
// of 1, zeros beside values of 1e-6 cost these all but 11 bits. Small enough for that, and large enough that a
// weight is bounded by it: weights reach 2^15 / 2^-80 = 2^95 at most, and 2^30 of them stay in f32's range.
constexpr float kNoValueScale = 0x1p-80f;

// The new rows of a sequence: rows begin .. begin + rows - 1 of the operands at positions first on
// (negative ones have no token). The arrays' values are clamped to the operands, so no row outside
// them is touched whatever the arrays hold.
struct Span {
    int begin, rows, first, length;
};
FG_BOTH Span span_of(int start, int stop, int length, int total)
{
    Span s;
    s.begin = start < 0 ? 0 : start > total ? total : start;
    const int end = stop < s.begin ? s.begin : stop > total ? total : stop;
    s.rows = end - s.begin;
    s.length = length < 0 ? 0 : length;
    s.first = s.length - s.rows;
    return s;
}

// The page of a sequence's table that holds its tokens 64 index on, or -1.
FG_BOTH int valid_page(int id, int pages) { return id >= 0 && id < pages ? id : -1; }
FG_BOTH int page_at(const int32_t *table, int index, int max_pages, int pages)
{
    return index >= 0 && index < max_pages ? valid_page(table[index], pages) : -1;
}

// The first position that a row at `position` sees. (No difference is formed that a window longer than any
// sequence, or a position before 0, could take out of range.)
FG_BOTH int first_seen(int position, int window) { return window > 0 && position >= window ? position - window + 1 : 0; }

// Pages [lo, hi) of a sequence that the rows row .. last see (hi at most max_pages).
struct PageRange {
    int lo, hi;
};
FG_BOTH PageRange pages_seen(const Span &s, int row, int last, int window, int max_pages)
{
    PageRange r;
    const int end = s.first + last + 1;  // one past the last row's position
    r.lo = first_seen(s.first + row, window) / kPage;
    r.hi = end <= 0 ? 0 : (end - 1) / kPage + 1;
    if (r.hi > max_pages) r.hi = max_pages;
    if (r.lo > r.hi) r.lo = r.hi;
    return r;
}

// Runs of 64 positions [lo, hi) that the new rows lie in, those without a page included (a row before
// position 0, or past the sequence's table).
FG_BOTH PageRange pages_of_new(const Span &s)
{
    PageRange r;
    r.lo = s.first >= 0 ? s.first / kPage : -((kPage - 1 - s.first) / kPage);
    const int last = s.first + s.rows - 1;
    r.hi = s.rows <= 0 ? r.lo : (last >= 0 ? last / kPage : -((kPage - 1 - last) / kPage)) + 1;
    return r;
}

}  // namespace fg
