// Pages of the paged cache copied to other pages (fg_cache_copy): forks, compactions.
#include <algorithm>

#include "cache.h"

namespace fg {
namespace {

typedef unsigned v4u __attribute__((ext_vector_type(4)));  // (an array of uint4 would lie in LDS)

constexpr int kCopyCaches = 64;        // of a launch
constexpr int kCopyLoads = 4;  // of 16 bytes a thread, on their way at once
constexpr unsigned kCopyPiece = kCopyLoads * 4096;  // bytes of a workgroup, about

struct CopyParams {
    const int32_t *sources, *targets;
    unsigned pages, pieces;  // pieces of a page
    unsigned piece_bytes;    // of the first ones
    size_t page_bytes;
    uint8_t *records[kCopyCaches];
    int limit[kCopyCaches];  // the cache's pages
};

// A workgroup a piece of a page: a page of all heads is one run of bytes, whole 512s. Bounded by memory: 1000 pages of 4 heads
// of 128 in two caches, 270 MB read and written, 48.6 us, 5.6 TB/s. Loads that keep nothing in the caches (the sources are
// read no more) are what that takes, 70 without; stores that do not keep the copies, which the next step reads, cost 55.9, and the
// read after them no less. One to eight loads a thread: no difference. Eight pages of 24 caches: 5 us, a launch and three loads
// one after the other.
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyParams p)
{
    const unsigned cache = blockIdx.y, units = p.pages * p.pieces;
    uint8_t *records = p.records[cache];
    for (unsigned unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const unsigned pair = unit / p.pieces, piece = unit % p.pieces;
        const int source = valid_page(p.sources[pair], p.limit[cache]), target = valid_page(p.targets[pair], p.limit[cache]);
        if (source < 0 || target < 0 || source == target) continue;
        const unsigned begin = piece * p.piece_bytes, end = min(begin + p.piece_bytes, unsigned(p.page_bytes));
        const uint8_t *from = records + size_t(source) * p.page_bytes;
        uint8_t *to = records + size_t(target) * p.page_bytes;
        for (unsigned at = begin + threadIdx.x * 16; at < end; at += kCopyPiece) {
            v4u x[kCopyLoads];
#pragma unroll
            for (int i = 0; i < kCopyLoads; i++)
                if (at + i * 4096 < end) x[i] = __builtin_nontemporal_load(reinterpret_cast<const v4u *>(from + at + i * 4096));
#pragma unroll
            for (int i = 0; i < kCopyLoads; i++)
                if (at + i * 4096 < end) *reinterpret_cast<v4u *>(to + at + i * 4096) = x[i];
        }
    }
}

size_t page_bytes_of(const fg_cache *c) { return size_t(c->kv_heads) * record_bytes(c->padded); }

// As many as leave each about kCopyPiece bytes.
unsigned pieces_of(size_t page_bytes) { return unsigned(std::max<size_t>((page_bytes + kCopyPiece / 2) / kCopyPiece, 1)); }

}  // namespace
}  // namespace fg

using namespace fg;

extern "C" int fg_cache_copy(fg_cache *const *caches, size_t count, const int32_t *sources, const int32_t *targets, size_t pages,
                             void *stream)
{
    if (!count || !pages) return FG_OK;
    if (!caches || !sources || !targets) return set_error(FG_ERR_ARG, "fg_cache_copy: null caches, sources or targets");
    if (count > 65536 || pages > (size_t(1) << 24)) return set_error(FG_ERR_SHAPE, "fg_cache_copy: at most 65536 caches and 2^24 pages");
    int device = 0;
    FG_HIP(hipGetDevice(&device));
    for (size_t i = 0; i < count; i++) {
        if (!caches[i]) return set_error(FG_ERR_ARG, "fg_cache_copy: a null cache");
        if (caches[i]->device != device)
            return set_error(FG_ERR_ARG, "fg_cache_copy: a cache is on device " + std::to_string(caches[i]->device) +
                                             ", the current one is " + std::to_string(device));
        if (pages * pieces_of(page_bytes_of(caches[i])) > 0xf0000000)
            return set_error(FG_ERR_SHAPE, "fg_cache_copy: more pages than a launch takes");
    }
    // a launch a run of caches whose pages are of one size
    for (size_t first = 0; first < count;) {
        CopyParams p{};
        p.page_bytes = page_bytes_of(caches[first]);
        size_t n = 0;
        while (first + n < count && n < size_t(kCopyCaches)) {
            const fg_cache *c = caches[first + n];
            if (page_bytes_of(c) != p.page_bytes) break;
            p.records[n] = c->records;
            p.limit[n++] = c->pages;
        }
        p.sources = sources;
        p.targets = targets;
        p.pages = unsigned(pages);
        p.pieces = pieces_of(p.page_bytes);
        p.piece_bytes = unsigned((p.page_bytes + p.pieces * 256 - 1) / (p.pieces * size_t(256)) * 256);
        copy_pages_kernel<<<dim3(unsigned(std::min<size_t>(pages * p.pieces, 65536)), unsigned(n)), 256, 0, as_stream(stream)>>>(p);
        FG_HIP(hipGetLastError());
        first += n;
    }
    return FG_OK;
}
