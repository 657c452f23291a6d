// Which of fg_sample's two forms a call takes, and how a row is cut into chunks, from its sizes alone (plain C++).
#pragma once

#include <cstddef>

namespace fg {

constexpr int kSampleChunks = 16;  // of a row, at most
constexpr int kSampleRun = 4096;   // logits that a workgroup takes at once

// Whether each row is one workgroup's (sample_row_kernel) rather than its chunks' (five launches): the first
// walks 256 rows at a time, a row's arithmetic on one CU, the second spreads few rows over the chip. Both in
// microseconds, rows' against chunks': 64 rows of 5000 logits 17 and 30, 16 rows of 32003 28 and 31, 200 rows
// 34 and 53; of 151936 logits 16 rows 82 and 41, 64 rows 91 and 65, 128 rows 95 and 86, 200 rows 101 and 108,
// 512 rows 199 and 255.
inline bool sample_by_rows(size_t rows, size_t vocab)
{
    const double logits = double(rows) * double(vocab), rounds = rows > 256 ? double(rows) / 256.0 : 1.0;
    const double by_rows = rounds * (14.0 + 4.5e-4 * double(vocab)) + 6e-7 * logits;
    const double by_chunks = 35.0 + 2.4e-6 * logits;
    return by_rows <= by_chunks;
}

// Chunks of a row, for `rows` rows at once. Each row a workgroup: the parts of a row whose weight under a cut
// is known apart, so that the draw walks one of them: a run each, or as many runs as 16 parts of a row ask for
// (512 rows of 151936 in parts of four runs 205 us, of three 200; 200 rows of 32003 in parts of four 35.5, of
// one 34.9). Else the workgroups of a row: the chip takes 512 at once, each of which costs about 2 us and 0.6 ns a
// logit (the bins of 64 rows of 151936: 8 chunks, one round, 13 us; 16 chunks, two rounds, 16 us), and the draw
// walks one chunk of every row, 0.4 ns a logit (331 rows: 3 chunks 44 us, 6 chunks 32).
inline int sample_chunks(size_t rows, size_t vocab, bool by_rows)
{
    if (by_rows) {
        const size_t runs = (vocab + kSampleRun - 1) / kSampleRun;
        return int(runs < size_t(kSampleChunks) ? runs : size_t(kSampleChunks));
    }
    double best = 0.0;
    int chunks = 1;
    for (size_t c = 1; c <= size_t(kSampleChunks) && (c == 1 || (vocab + c - 1) / c >= 4096); c++) {
        const double share = double(vocab) / double(c);
        const double cost = double((rows * c + 511) / 512) * (2000.0 + 0.6 * share) + 0.4 * share;
        if (c == 1 || cost < best) {
            best = cost;
            chunks = int(c);
        }
    }
    return chunks;
}

// Logits of a chunk, and the chunks that this leaves: whole runs of a workgroup that takes a row, whole 256 of one
// that takes a chunk.
inline int sample_chunk(size_t vocab, bool by_rows, int *chunks)
{
    const size_t unit = by_rows ? kSampleRun : 256, n = size_t(*chunks);
    const size_t chunk = ((vocab + n - 1) / n + unit - 1) / unit * unit;
    *chunks = int((vocab + chunk - 1) / chunk);
    return int(chunk);
}

}  // namespace fg
