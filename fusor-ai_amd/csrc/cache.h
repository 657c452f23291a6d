// The paged cache's handle and what its kernels share.
#pragma once

#include "cache_layout.h"
#include "common.h"

struct fg_cache {
    int device;
    int pages, kv_heads, head_dim, padded;
    uint8_t *records;  // [page][head] of record_bytes(padded)
};

namespace fg {

// Workgroups of 256 that a launch takes (2^32 threads are too many).
constexpr size_t kMaxGrid = 0xffffff;

// What the kernels take of a batch.
struct BatchParams {
    const int32_t *row_starts, *lengths, *pages;
    int sequences, rows, max_pages;
};

// The arguments that every call over a batch checks.
int check_batch(const fg_cache *cache, const fg_batch *batch, const char *who);

inline BatchParams batch_params(const fg_batch *b)
{
    return BatchParams{b->row_starts, b->lengths, b->pages, int(b->sequences), int(b->rows), int(b->max_pages)};
}

__device__ __forceinline__ Span sequence_span(const BatchParams &b, int s)
{
    return span_of(b.row_starts[s], b.row_starts[s + 1], b.lengths[s], b.rows);
}

// The sum over the wave's lanes up to this one, and over all of them: within rows of 16 lanes, then
// each row's last lane to the rows behind it (DPP throughout).
__device__ __forceinline__ int wave_scan(int v, int *total)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15: to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast 31: to rows 2 and 3
    *total = __builtin_amdgcn_readlane(v, 63);
    return v;
}

// Finds which sequence's unit `index` is when sequence s has count(s) units, in order: the sequence
// (-1 past the last) and the index within it. Every lane of the wave takes part and gets the result.
template <class F>
__device__ __forceinline__ int find_unit(int sequences, int index, int *within, F count)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = 0; s0 < sequences; s0 += 64) {
        const int n = s0 + lane < sequences ? count(s0 + lane) : 0;
        int total;
        const int upto = before + wave_scan(n, &total);
        const unsigned long long here = __ballot(index < upto);
        if (here) {
            const int at = __builtin_ctzll(here);
            *within = index - __builtin_amdgcn_readlane(upto - n, at);
            return s0 + at;
        }
        before += total;
    }
    return -1;
}

// The sequence that holds operand row `row`, or -1: 64 starts at a time (they do not fall).
__device__ __forceinline__ int sequence_of_row(const BatchParams &b, int row)
{
    const int lane = threadIdx.x & 63;
    int lo = 0, n = b.sequences + 1;  // the last start that is <= row lies in [lo, lo + n)
    if (b.row_starts[0] > row) return -1;
    while (n > 1) {
        const int step = (n + 63) / 64, at = lo + lane * step;
        const int k = __popcll(__ballot(lane * step < n && b.row_starts[at] <= row));
        if (k == 0) return -1;  // starts that fall: no sequence's row
        const int end = lo + n;
        lo += (k - 1) * step;
        n = lo + step < end ? step : end - lo;
        if (step == 1) n = 1;
    }
    return lo < b.sequences ? lo : -1;
}

}  // namespace fg
