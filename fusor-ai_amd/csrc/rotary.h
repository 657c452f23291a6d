// Rotary positions: the handle, and what the kernels that turn pairs share.
#pragma once

#include "cache.h"
#include "rotary_phase.h"

struct fg_rotary {
    int device;
    int dims, halves;  // the values of a head that are turned, and whether value i's partner is i + dims / 2
    double magnitude;
    fg::RotaryPair *pairs;  // [dims / 2]
};

namespace fg {

struct RotaryParams {
    const RotaryPair *pairs;
    int dims, halves;
    double magnitude;
};

typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));  // four floats at any float's address

// A pair's factors in f32: each rounded once, from 64 bits.
struct Turn {
    float c, s;
};
__device__ __forceinline__ Turn turn_of(const Angle &a, double magnitude) { return Turn{float(a.c * magnitude), float(a.s * magnitude)}; }
__device__ __forceinline__ Turn turn_at(const RotaryParams &r, int pair, int position)
{
    return turn_of(angle_at(r.pairs[pair], position), r.magnitude);
}

// Rows to turn out of place or in place: rows * units of `unit_heads` heads, a wave each.
struct RotateParams {
    BatchParams b;
    RotaryParams r;
    const float *x;
    size_t x_stride;
    float *out;
    size_t out_stride;
    int heads, head_dim, units, unit_heads;
    bool keep;  // `out` is `x`: what is not turned stays where it is
};

// One value a, its partner b: a c - b s where a is the pair's first, a c + b s where it is the second. Products and
// sums are f32, rounded one by one, so that turned keys have the same 8-bit levels wherever they are computed.
__device__ __forceinline__ float turned(float a, float b, Turn t, bool first)
{
    const float own = a * t.c, other = b * t.s;
    return first ? own - other : own + other;
}

// The unit's heads of one row, a wave. A team of lanes, a power of two, has a head's items: a pair of quads (halves), a quad of two
// pairs, or, where pairs do not come in quads (QUADS false), one pair; then the head's values that are not turned. A lane's
// angles, some 60 f64 operations each, serve all heads of the unit.
constexpr int kAhead = 4;  // heads of a lane whose loads are on their way at once

template <bool QUADS>
__device__ __forceinline__ void rotate_unit(const RotateParams &p, unsigned unit)
{
    const int lane = threadIdx.x & 63;
    const int row = int(unit / unsigned(p.units)), head0 = int(unit % unsigned(p.units)) * p.unit_heads;
    const int s = sequence_of_row(p.b, row);
    if (s < 0) return;
    const Span span = sequence_span(p.b, s);
    const int at = row - span.begin;
    if (at < 0 || at >= span.rows) return;
    const int position = span.first + at;
    const int half = p.r.dims / 2;
    const int turning = QUADS ? (p.r.halves ? half / 4 : p.r.dims / 4) : half;
    const int items = turning + (QUADS ? (p.head_dim - p.r.dims) / 4 : p.head_dim - p.r.dims);
    const int wanted = p.keep && position >= 0 ? turning : items;
    int team = 1;
    while (team < wanted && team < 64) team *= 2;
    const int heads_end = min(head0 + p.unit_heads, p.heads);
    const float *x = p.x + size_t(row) * p.x_stride;
    float *out = p.out + size_t(row) * p.out_stride;
    for (int item = lane & (team - 1); item < wanted; item += team) {
        const bool turns = item < turning;
        if (QUADS) {
            const int dim = turns ? 4 * item : p.r.dims + 4 * (item - turning);
            const bool pair = turns && p.r.halves;
            Turn t[4] = {};
            if (turns && position >= 0) {
                if (p.r.halves) {
#pragma unroll
                    for (int j = 0; j < 4; j++) t[j] = turn_at(p.r, dim + j, position);
                } else {
#pragma unroll
                    for (int j = 0; j < 2; j++) t[j] = turn_at(p.r, dim / 2 + j, position);
                }
            }
            const int step = 64 / team;
            for (int head = head0 + lane / team; head < heads_end; head += kAhead * step) {
                // (all loads before the first store: `out` may be `x`, so the compiler keeps their order)
                v4f a[kAhead], b[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; i++) {
                    a[i] = b[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                    if (position < 0 || head + i * step >= heads_end) continue;
                    const float *from = x + size_t(head + i * step) * p.head_dim + dim;
                    a[i] = *reinterpret_cast<const v4f_any *>(from);
                    if (pair) b[i] = *reinterpret_cast<const v4f_any *>(from + half);
                }
#pragma unroll
                for (int i = 0; i < kAhead; i++) {
                    if (head + i * step >= heads_end) break;
                    float *to = out + size_t(head + i * step) * p.head_dim + dim;
                    v4f u = a[i], v;
                    if (pair) {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            u[j] = turned(a[i][j], b[i][j], t[j], true);
                            v[j] = turned(b[i][j], a[i][j], t[j], false);
                        }
                    } else if (turns) {
#pragma unroll
                        for (int j = 0; j < 4; j++) u[j] = turned(a[i][j], a[i][j ^ 1], t[j / 2], j % 2 == 0);
                    }
                    *reinterpret_cast<v4f_any *>(to) = u;
                    if (pair) *reinterpret_cast<v4f_any *>(to + half) = v;
                }
            }
        } else {
            const int first = !turns ? p.r.dims + item - turning : p.r.halves ? item : 2 * item;
            const int second = p.r.halves ? first + half : first + 1;
            Turn t = {};
            if (turns && position >= 0) t = turn_at(p.r, item, position);
            for (int head = head0 + lane / team; head < heads_end; head += 64 / team) {
                const size_t place = size_t(head) * p.head_dim;
                const float a = position >= 0 ? x[place + first] : 0.0f;
                const float b = position >= 0 && turns ? x[place + second] : 0.0f;
                out[place + first] = turns ? turned(a, b, t, true) : a;
                if (turns) out[place + second] = turned(b, a, t, false);
            }
        }
    }
}

// Whether a head's pairs come in whole quads.
inline bool whole_quads(const fg_rotary *r) { return r->dims % (r->halves ? 8 : 4) == 0; }

inline RotaryParams rotary_params(const fg_rotary *r) { return RotaryParams{r->pairs, r->dims, r->halves, r->magnitude}; }

// A batch's rows of `heads` heads for rotate_unit.
RotateParams rotate_params(const fg_rotary *r, const fg_batch *b, const float *x, size_t x_stride, size_t heads, size_t head_dim,
                           float *out, size_t out_stride);
int launch_rotate(const RotateParams &p, bool quads, hipStream_t s);

// Whether `rows` rows of a and of b share memory (rows of different strides among each other: not told).
bool rows_meet(const float *a, size_t a_stride, size_t a_width, const float *b, size_t b_stride, size_t b_width, size_t rows);

// The arguments that rotating calls check; `device` is the current one.
int check_rotary(const fg_rotary *r, int device, size_t head_dim, const std::string &who);
int check_rotated(const fg_batch *b, const float *x, size_t x_stride, size_t heads, size_t head_dim, const float *out, size_t out_stride,
                  const std::string &who);

}  // namespace fg
