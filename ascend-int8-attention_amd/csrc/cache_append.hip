// MI355X (gfx950) append of rows to the paged 8-bit caches, their position
// rotation applied on the way.
//
// Mathematics (sharedkv_hip.h).  A row's last R channels are rotated by the
// angles of its position,
//   a' = a cos - b sin,  b' = a sin + b cos
// and all channels are encoded: with frozen channel scales as the writer does,
// or with one scale for the 32 rows of a page and KV head, that of the page's
// first appended rows, later doubled as often as larger rows need.  Doubling
// moves a code by at most half a step of the new scale, and all doublings of a
// page together by less than one of its last; any other factor would add half
// a step for every row that passes the ones before.
//
// Codes are those of the rotated value itself, not of its rounding to FP32.
// Values and quotients are made in FP32 with bounds on what they are off by
// (below); where a code or the page's largest value could come out another way
// within them, that row or page is done again in FP64.  (FP64 throughout takes
// 26.5 us where this takes 18.8: 48 requests of 1-200 rows of four heads.)
//
// What bounds it.  1024 bytes read and 512 written for a row and head, beside
// 185 vector instructions for a lane's eight values, all told (e4m3 214); with
// few rows one chain of round trips (the requests' ends; the rows, their positions and
// page; the angles and the old scale; the codes).  One row takes 4.2 us, 256
// requests' 6.3 (7.0 where each one's scale grows and the page's codes are rounded
// again), five prompts of 700-2600 rows 8.1, 65536 rows 31 (3.8 TB/s).  A
// work-group takes a page: the rows that share a scale are in its registers from
// the first read on, so they are read once and a launch needs no second pass.
// Eight waves with four rows each: with two rows each 9.9 and 39 us for the last
// two, with eight 10.3 and 30.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "sharedkv_hip.h"

namespace {

constexpr int D = 512;
constexpr int PAGE_ROWS = 32;
constexpr int WAVES = 8, THREADS = 64 * WAVES;
constexpr int EACH = PAGE_ROWS / WAVES;          // rows of a page for a wave
constexpr uint32_t MAX_HEADS = 128;
constexpr uint32_t MAX_WIDTH = 0x7fffffffu / PAGE_ROWS;
constexpr uint64_t MAX_GROUPS = 0xffffffffu / THREADS;
constexpr float FLOOR = 1e-8f;                   // smallest scale, as of calibrated channels

enum Codes { INT8, E4M3, CHANNEL };
enum Rotation { NONE, PAIRS, HALVES };           // channels 2k and 2k + 1 turn together, or k and k + R / 2

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <typename T>
__device__ __forceinline__ const __attribute__((address_space(1))) T *gptr(uint64_t a)
{
    return reinterpret_cast<const __attribute__((address_space(1))) T *>(a);
}
template <typename T>
__device__ __forceinline__ __attribute__((address_space(1))) T *gout(uint64_t a)
{
    return reinterpret_cast<__attribute__((address_space(1))) T *>(a);
}

// First work-group of request b: n rows behind any others touch at most n / 32 + 2 pages, no matter where they begin,
// and where n % 32 is 0 or 1 one less, so requests' ranges never overlap.
__host__ __device__ constexpr uint64_t first_of(uint64_t cu, uint64_t b) { return cu / PAGE_ROWS + 2 * b; }

// Maximum over a wave of values from 0 on.
__device__ __forceinline__ float wave_max(float v)
{
    auto step = [&](auto control, auto rows) {
        const int x = __builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(control)::value, decltype(rows)::value, 0xf, false);
        v = fmaxf(v, __int_as_float(x));
    };
    using std::integral_constant;
    step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});     // row_shr 1, 2, 4, 8
    step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});     // row_bcast 15, 31
    step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// a b + c d.  FP32: the second product's rounding is taken back, so that the sum is off by 2^-23 of itself and 2^-47 of the
// products at most, also where they nearly cancel.  Where a product is infinite it is no number, though the sum may be one:
// rows that have such a value are done in FP64.
__device__ __forceinline__ double sum_of(double a, double b, double c, double d) { return fma(a, b, c * d); }
__device__ __forceinline__ float sum_of(float a, float b, float c, float d)
{
    const float product = c * d;
    return __builtin_fmaf(a, b, product) + __builtin_fmaf(c, d, -product);
}

// Rounded to FP32 such that another rounding to fewer bits is that of the value itself: inexact ones end in a set bit.
// `larger`: the nearest number's size is larger than the value's, so it is none of the zeros.
__device__ __forceinline__ float to_odd(float nearest, bool larger, bool inexact)
{
    return __uint_as_float((__float_as_uint(nearest) - (larger ? 1u : 0u)) | (inexact ? 1u : 0u));
}
__device__ __forceinline__ float to_odd(double x)
{
    const float f = (float)x;
    return to_odd(f, fabs((double)f) > fabs(x), (double)f != x);
}

__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ uint32_t pack_bytes(const int (&x)[4])
{
    return (uint32_t)(x[0] & 255) | (uint32_t)(x[1] & 255) << 8 | (uint32_t)(x[2] & 255) << 16 | (uint32_t)x[3] << 24;
}

struct Shared {
    int32_t found[4];                            // request, its first and end token, its rows
    uint32_t odd[WAVES];                         // rows with a rotated value that is no number in FP32
    int32_t begin[WAVES];                        // first row that is written
    float peak[2][WAVES];                        // of channels as they are, of rotated ones
};

template <int CODES, int ROTATION>
__global__ void __launch_bounds__(THREADS, 4) cache_append(const uint64_t cu_q, const uint64_t seq_lens, const uint32_t batch,
               const uint32_t tokens, const CacheAppendArgs p)
{
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), head = blockIdx.y;
    // ---- whose page this is ----
    if (tid == 0) s.found[0] = -1;
    __syncthreads();
    const auto *cu = gptr<int32_t>(cu_q), *lens = gptr<int32_t>(seq_lens);
    for (uint32_t b = tid; b < batch; b += THREADS) {
        const int c0 = min(max(cu[b], 0), (int)tokens), c1 = min(max(cu[b + 1], c0), (int)tokens), length = lens[b];
        const uint64_t item = blockIdx.x;
        if (item >= first_of(c0, b) && item < first_of(c1, b + 1)) {
            s.found[0] = (int)b, s.found[1] = c0, s.found[2] = c1, s.found[3] = length;
        }
    }
    __syncthreads();
    const int b = __builtin_amdgcn_readfirstlane(s.found[0]);
    if (b < 0) return;
    const int first = __builtin_amdgcn_readfirstlane(s.found[1]), count = __builtin_amdgcn_readfirstlane(s.found[2]) - first;
    const int length = __builtin_amdgcn_readfirstlane(s.found[3]);
    if (length <= 0 || count <= 0) return;       // graph padding
    const int start = length - count, begin = max(start, 0);          // logical rows
    const int column = begin / PAGE_ROWS + (int)(blockIdx.x - first_of(first, b)), row0 = column * PAGE_ROWS;
    if (column >= (int)p.tableWidth || row0 >= length) return;
    const int low = max(begin - row0, 0), high = min(length - row0, PAGE_ROWS);     // the page's rows to write

    // ---- rows, positions and the page; then angles and the old scale: each kind's loads at once ----
    const int page = __builtin_amdgcn_readfirstlane(gptr<int32_t>(p.table)[(uint64_t)b * p.tableWidth + column]);
    const uint32_t half = p.rotary / 2;
    const int from = 64 - (int)p.rotary / 8;     // first lane that is rotated
    const bool turned = ROTATION != NONE && lane >= from;
    // Channel k of the first half goes with k of the second, R / 16 lanes on.
    const int apart = (int)p.rotary / 16;
    const bool second = ROTATION == HALVES && lane >= from + apart;
    constexpr int ANGLES = ROTATION == NONE ? 0 : ROTATION == PAIRS ? 1 : 2;    // times four cosines and sines of a lane
    struct Row {
        u32x4 raw;
        f32x4 cosine[ANGLES ? ANGLES : 1], sine[ANGLES ? ANGLES : 1];
    };
    auto read_row = [&](uint32_t token) {
        return *gptr<u32x4>(p.updates + ((uint64_t)token * p.updateStride + (uint64_t)head * p.updateHeadStride + lane * 8) * 2);
    };
    auto read_angles = [&](Row &row, int64_t place) {   // lanes that are not rotated read what the first that is reads
        const int at = max(lane - from, 0) - (second ? apart : 0);
        const uint64_t angles = p.rotation + ((uint64_t)place * p.rotationStride + (uint32_t)(at * 4 * ANGLES)) * 4;
#pragma unroll
        for (int q = 0; q < ANGLES; ++q) row.cosine[q] = gptr<f32x4>(angles)[q], row.sine[q] = gptr<f32x4>(angles + half * 4)[q];
    };
    // The row's values, in T.
    auto values = [&](const Row &row, auto (&y)[8]) {
        using T = std::remove_reference_t<decltype(y[0])>;
        auto value = [](const u32x4 &w, int e) { return (T)__uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16); };
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = value(row.raw, e);
        if constexpr (ROTATION == PAIRS) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const T u = y[2 * e], v = y[2 * e + 1], c = row.cosine[0][e], n = row.sine[0][e];
                const T a = sum_of(u, c, -v, n), b = sum_of(u, n, v, c);
                y[2 * e] = turned ? a : u, y[2 * e + 1] = turned ? b : v;
            }
        }
        if constexpr (ROTATION == HALVES) {
            u32x4 other;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                other[e] = (uint32_t)__shfl((int)row.raw[e], turned ? second ? lane - apart : lane + apart : lane);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const T u = y[e], v = value(other, e), c = row.cosine[e / 4][e % 4], n = row.sine[e / 4][e % 4];
                const T a = sum_of(u, c, second ? v : -v, n);
                y[e] = turned ? a : u;
            }
        }
    };
    // A row's token (for one that is not to be written, the page's first) and position.
    auto token_of = [&](int row, bool mine) { return (uint32_t)(first + (mine ? row0 + row - start : begin - start)); };
    auto place_of = [&](int row, uint32_t token) {
        return !p.positions        ? (int64_t)(row0 + row)
               : p.int64Positions ? gptr<int64_t>(p.positions)[token]
                                  : (int64_t)gptr<int32_t>(p.positions)[token];
    };
    Row rows[EACH];
    int64_t place[EACH];
    bool mine[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int row = wave + WAVES * i;
        mine[i] = row >= low && row < high;
        rows[i].raw = read_row(token_of(row, mine[i]));
    }
    if constexpr (ROTATION != NONE) {
        const bool wide = p.positions && p.int64Positions;
        int32_t words[EACH][2];                  // the low word, and the high one of wide ones, all at once
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const uint32_t token = token_of(wave + WAVES * i, mine[i]);
            const uint64_t at = p.positions ? p.positions + (uint64_t)token * (wide ? 8 : 4) : p.cuQ;
            words[i][0] = gptr<int32_t>(at)[0], words[i][1] = gptr<int32_t>(at)[wide ? 1 : 0];
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            place[i] = !p.positions ? (int64_t)(row0 + wave + WAVES * i)
                       : wide       ? (int64_t)((uint64_t)(uint32_t)words[i][1] << 32 | (uint32_t)words[i][0])
                                    : (int64_t)words[i][0];
    }
    if ((uint32_t)page >= p.pages) return;
    const uint64_t scale_at = p.scale + ((uint64_t)page * p.scaleStride + head) * 4;
    float old = 0.0f;
    if (CODES != CHANNEL) old = *gptr<float>(scale_at);
    if constexpr (ROTATION != NONE) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const bool there = place[i] >= 0 && place[i] < (int64_t)p.rotationRows;
            mine[i] = mine[i] && there;
            place[i] = there ? place[i] : 0;
            read_angles(rows[i], place[i]);
        }
    }
    float y[EACH][8];
#pragma unroll
    for (int i = 0; i < EACH; ++i) values(rows[i], y[i]);
    // In FP64, of a row that is written, all of it read again: kept, it would cost half the waves.
    auto exactly = [&](int row, double (&y)[8]) {
        const uint32_t token = token_of(row, true);
        Row its;
        its.raw = read_row(token);
        if constexpr (ROTATION != NONE) read_angles(its, place_of(row, token));
        values(its, y);
    };
    const uint64_t to = p.cache + (uint64_t)page * p.pageStride + ((uint64_t)head * D + lane * 8);
    const uint64_t row_bytes = (uint64_t)p.heads * D;

    // ---- frozen channel scales: the writer's codes ----
    if constexpr (CODES == CHANNEL) {
        const f32x4 inverse[2] = {gptr<f32x4>(p.inverseScale)[2 * lane], gptr<f32x4>(p.inverseScale)[2 * lane + 1]};
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            double exact[8];                     // FP32 takes the value's own rounding
            values(rows[i], exact);
            u32x2 w;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                int code[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = (float)exact[4 * q + e] * inverse[q][e];
                    code[e] = (int)__builtin_rintf(fminf(fmaxf(v, -127.0f), 127.0f));
                }
                w[q] = pack_bytes(code);
            }
            if (mine[i]) *gout<u32x2>(to + (uint64_t)(wave + WAVES * i) * row_bytes) = w;
        }
        return;
    }

    // ---- the page's scale ----
    constexpr float LARGEST = CODES == E4M3 ? 448.0f : 127.0f;
    // NaN values do not count, infinities as the largest number.
    float its = 0.0f, most[EACH], all = 0.0f;    // `most` and `all` keep a NaN
    int begin_row = PAGE_ROWS;                   // first row that is written
    uint32_t odd = 0;                            // rows of the wave with a rotated value that is no number in FP32
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        most[i] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) most[i] = __builtin_elementwise_maximum(most[i], mine[i] ? fabsf(y[i][e]) : 0.0f);
        all = __builtin_elementwise_maximum(all, most[i]);
        begin_row = min(begin_row, mine[i] ? wave + WAVES * i : PAGE_ROWS);
    }
    if (__ballot(!(all < INFINITY))) {           // seldom
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const bool none = !(most[i] < INFINITY);
            odd |= __ballot(none && turned) ? 1u << i : 0u;
            float others = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) others = fmaxf(others, turned ? 0.0f : fabsf(y[i][e]));
            most[i] = none ? others : most[i];
        }
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) its = fmaxf(its, most[i]);
    const float still = wave_max(turned ? 0.0f : its), rotated = wave_max(turned ? its : 0.0f);
    if (lane == 0) s.peak[0][wave] = still, s.peak[1][wave] = rotated, s.odd[wave] = odd, s.begin[wave] = begin_row;
    asm volatile("" : "+v"(old));                // read before any wave may store the new one
    __syncthreads();
    float peak = 0.0f, other = 0.0f;
    uint32_t any_odd = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) peak = fmaxf(peak, s.peak[0][w]), other = fmaxf(other, s.peak[1][w]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) any_odd |= s.odd[w], begin_row = min(begin_row, s.begin[w]);
    if (begin_row == PAGE_ROWS) return;          // all are skipped: the page stays as it is, its scale too
    if (any_odd || !(peak >= other * (1.0f + 0x1p-20f))) {  // the page's largest value may be a rotated one: exactly
        uint32_t rest = odd;
#pragma unroll
        for (int i = 0; i < EACH; ++i) rest |= __ballot(turned && most[i] * (1.0f + 0x1p-20f) >= other) && mine[i] ? 1u << i : 0u;
        its = 0.0f;
        for (; rest; rest &= rest - 1) {
            double exact[8];
            exactly(wave + WAVES * __builtin_ctz(rest), exact);
#pragma unroll
            for (int e = 0; e < 8; ++e) its = fmaxf(its, fabsf((float)exact[e]));
        }
        const float rotated = wave_max(turned ? its : 0.0f);
        __syncthreads();
        if (lane == 0) s.peak[1][wave] = rotated;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) peak = fmaxf(peak, s.peak[1][w]);
    }
    const bool infinite = !(peak < INFINITY);
    const float needed = fmaxf(fminf(peak, 0x1.fffffep127f) / LARGEST, FLOOR);
    const bool begun = begin_row > 0 && old > 0.0f && old < INFINITY;
    int power = 0;
    float scale = needed;
    if (begun) {
        // The least power of two by which the old scale holds the new rows.
        power = __builtin_amdgcn_frexp_expf(needed) - __builtin_amdgcn_frexp_expf(old);
        if (ldexpf(old, power) < needed) ++power;
        power = max(power, 0);
        scale = ldexpf(old, power);
    }

    // ---- codes ----
    const float reciprocal = 1.0f / scale;
    // A quotient made in FP32 is off by 2^-24 of itself for each of the reciprocal, the product and, rotated, two roundings
    // of the value; the products' 2^-47 are below 2^-37 of a code.
    constexpr float OFF = 0x1p-22f, SLACK = 0x1p-36f;
    // Codes of quotients; false where another one is within what they are off by (0: nothing).
    auto encode = [&](const float (&v)[8], bool exact, u32x2 &w) {
        bool certain = true;
        if (CODES == E4M3) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float low[4], high[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = v[4 * q + e], off = exact ? 0.0f : __builtin_fmaf(fabsf(x), OFF, SLACK);
                    low[e] = x - off, high[e] = x + off;
                }
                w[q] = pack_e4m3(low[0], low[1], low[2], low[3]);
                certain = certain && w[q] == pack_e4m3(high[0], high[1], high[2], high[3]);
            }
            return certain;
        }
        // With 1.5 * 2^23 more, the nearest whole number sits in the low bits.
        float most = 0.0f;                       // keeps a NaN
        uint32_t bits[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float sum = v[e] + 12582912.0f, off = exact ? -1.0f : __builtin_fmaf(fabsf(v[e]), OFF, SLACK);
            most = __builtin_elementwise_maximum(most, fabsf(v[e] - (sum - 12582912.0f)) + off);
            bits[e] = __float_as_uint(sum);
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t ab = __builtin_amdgcn_perm(bits[4 * q + 1], bits[4 * q], 0x0c0c0400u);
            w[q] = ab | __builtin_amdgcn_perm(bits[4 * q + 3], bits[4 * q + 2], 0x04000c0cu);
        }
        return most < 0.5f;
    };
    uint32_t rest = odd;                         // rows that have a code to be made in FP64
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (!mine[i]) continue;
        u32x2 w;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = y[i][e] * reciprocal;
        bool certain = encode(v, false, w) && !infinite;
        if (__ballot(!certain && !turned)) {
            // Values as they are leave a remainder that FP32 holds: the quotient's rounding that keeps ties apart.
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = __builtin_fmaf(__builtin_fmaf(-v[e], scale, y[i][e]), reciprocal, v[e]);
                const float rest = __builtin_fmaf(-v[e], scale, y[i][e]);
                const bool apart = (int)(__float_as_uint(rest) ^ __float_as_uint(v[e])) < 0;
                v[e] = to_odd(v[e], apart & (rest != 0.0f) & (v[e] != 0.0f), rest != 0.0f);
            }
            u32x2 other;
            const bool some = encode(v, true, other);
            if (!turned) w = other, certain = some && !infinite;
        }
        if (__ballot(!certain)) rest |= 1u << i;
        *gout<u32x2>(to + (uint64_t)(wave + WAVES * i) * row_bytes) = w;
    }
    for (; rest; rest &= rest - 1) {
        const int row = wave + WAVES * __builtin_ctz(rest);
        const double step = (double)scale, inverse = 1.0 / step;
        double exact[8];
        exactly(row, exact);
        u32x2 w;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            int code[4];
            float value[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double x = fmin(fmax(exact[4 * q + e], -0x1.fffffep127), 0x1.fffffep127);
                // The quotient, rounded once: a tie stays one.
                double v = x * inverse;
                v = fma(fma(-v, step, x), inverse, v);
                v = fmin(fmax(v, -(double)LARGEST), (double)LARGEST);
                const bool number = exact[4 * q + e] == exact[4 * q + e];
                code[e] = number ? (int)rint(v) : 0;
                value[e] = number ? to_odd(v) : __builtin_nanf("");
            }
            w[q] = CODES == E4M3 ? pack_e4m3(value[0], value[1], value[2], value[3]) : pack_bytes(code);
        }
        *gout<u32x2>(to + (uint64_t)row * row_bytes) = w;
    }
    if (power) {                                 // the rows that were there, in the new scale; rows behind the last stay
        const float f = ldexpf(1.0f, -power);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int row = wave + WAVES * i;
            if (mine[i] || row >= high) continue;
            const u32x2 was = *gptr<u32x2>(to + (uint64_t)row * row_bytes);
            u32x2 w;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if (CODES == E4M3) {
                    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)was[q], false);
                    const auto c = __builtin_amdgcn_cvt_pk_f32_fp8((int)was[q], true);
                    w[q] = pack_e4m3(a[0] * f, a[1] * f, c[0] * f, c[1] * f);
                } else {
                    int code[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) code[e] = (int)__builtin_rintf((float)(int8_t)(was[q] >> (8 * e)) * f);
                    w[q] = pack_bytes(code);
                }
            }
            *gout<u32x2>(to + (uint64_t)row * row_bytes) = w;
        }
    }
    if (tid == 0 && (power || !begun)) *gout<float>(scale_at) = scale;
}

bool rejected(const CacheAppendArgs *a)
{
    if (!a || !a->cache || !a->updates || !a->table || !a->cuQ || !a->seqLens || (!a->scale == !a->inverseScale)) return true;
    if (!a->batch || !a->heads || a->heads > MAX_HEADS || !a->pages || !a->tableWidth || a->tableWidth > MAX_WIDTH) return true;
    if (a->codes > 1 || a->interleaved > 1 || a->int64Positions > 1 || a->tokens > 0x7fffffffu || a->batch > 0xffffffu)
        return true;
    if (a->inverseScale && (a->codes || a->heads != 1)) return true;
    if (a->pageStride < (uint64_t)PAGE_ROWS * D * a->heads || a->pageStride % 8 || a->cache % 8 || a->updates % 16 ||
        a->updateStride % 8 || a->updateHeadStride % 8 || a->inverseScale % 16 || a->scale % 4)
        return true;
    if (a->rotary > D || a->rotary % 16 || (a->rotary && (!a->rotation || a->rotation % 16 || a->rotationStride % 4 ||
                                                          a->rotationStride < a->rotary || !a->rotationRows)))
        return true;
    // Work-groups of a launch: the threads are counted in 32 bits.
    return first_of(a->tokens, a->batch) * a->heads > MAX_GROUPS;
}

}  // namespace

extern "C" {

int launch_sharedkv_append(void *stream, const CacheAppendArgs *a)
{
    if (rejected(a)) return (int)hipErrorInvalidValue;
    if (!a->tokens) return (int)hipSuccess;
    const auto of_codes = [&](auto rotation) {
        return a->inverseScale ? &cache_append<CHANNEL, rotation.value>
               : a->codes      ? &cache_append<E4M3, rotation.value>
                               : &cache_append<INT8, rotation.value>;
    };
    const auto kernel = !a->rotary       ? of_codes(std::integral_constant<int, NONE>{})
                        : a->interleaved ? of_codes(std::integral_constant<int, PAIRS>{})
                                         : of_codes(std::integral_constant<int, HALVES>{});
    hipLaunchKernelGGL(kernel, dim3((uint32_t)first_of(a->tokens, a->batch), a->heads), dim3(THREADS), 0,
                       static_cast<hipStream_t>(stream), a->cuQ, a->seqLens, a->batch, a->tokens, *a);
    return (int)hipGetLastError();
}

uint32_t sharedkv_append_args_size(void) { return (uint32_t)sizeof(CacheAppendArgs); }

}  // extern "C"
