// Pages of the paged cache copied to other pages (fg_cache_copy): forks, compactions.
#include <algorithm>

#include "cache.h"

namespace fg {
namespace {

constexpr int kCopyCaches = 64;        // of a launch
constexpr unsigned kCopyPiece = 8192;  // bytes of a workgroup: two loads of 16 a thread, both on their way at once

struct CopyParams {
    const int32_t *sources, *targets;
    unsigned pages, pieces;  // pieces of a page
    size_t page_bytes;
    uint8_t *records[kCopyCaches];
    int limit[kCopyCaches];  // the cache's pages
};

// A workgroup a piece of a page: a page of all heads is one run of bytes, whole 512s.
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyParams p)
{
    const unsigned cache = blockIdx.y, units = p.pages * p.pieces;
    uint8_t *records = p.records[cache];
    for (unsigned unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const unsigned pair = unit / p.pieces, piece = unit % p.pieces;
        const int source = valid_page(p.sources[pair], p.limit[cache]), target = valid_page(p.targets[pair], p.limit[cache]);
        if (source < 0 || target < 0 || source == target) continue;
        const size_t begin = size_t(piece) * kCopyPiece + threadIdx.x * 16;
        const uint8_t *from = records + size_t(source) * p.page_bytes;
        uint8_t *to = records + size_t(target) * p.page_bytes;
        uint4 x[kCopyPiece / 4096];
#pragma unroll
        for (int i = 0; i < int(kCopyPiece / 4096); i++)
            if (begin + i * 4096 < p.page_bytes) x[i] = *reinterpret_cast<const uint4 *>(from + begin + i * 4096);
#pragma unroll
        for (int i = 0; i < int(kCopyPiece / 4096); i++)
            if (begin + i * 4096 < p.page_bytes) *reinterpret_cast<uint4 *>(to + begin + i * 4096) = x[i];
    }
}

size_t page_bytes_of(const fg_cache *c) { return size_t(c->kv_heads) * record_bytes(c->padded); }

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
        if (pages * ((page_bytes_of(caches[i]) + kCopyPiece - 1) / kCopyPiece) > 0xf0000000)
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
        p.pieces = unsigned((p.page_bytes + kCopyPiece - 1) / kCopyPiece);
        copy_pages_kernel<<<dim3(unsigned(std::min<size_t>(pages * p.pieces, 65536)), unsigned(n)), 256, 0, as_stream(stream)>>>(p);
        FG_HIP(hipGetLastError());
        first += n;
    }
    return FG_OK;
}
