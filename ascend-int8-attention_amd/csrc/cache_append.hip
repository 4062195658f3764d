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
// Codes are those of the rotated value itself: the rotation and the quotient
// run in FP64 (a few instructions for a value, far from what bounds the
// kernel), so no rounding to FP32 puts a value on the other side of a border.
//
// What bounds it.  1024 bytes read and 512 written for a row and head: bytes,
// from some thousand rows on, and below that one chain of round trips (the
// requests' ends; the rows, their positions and page; the angles and the old
// scale; the codes).  A work-group takes a page: the rows that share a scale
// are in its registers from the first read on, so they are read once and a
// launch needs no second pass.
#include <hip/hip_runtime.h>
#include <stdint.h>

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

// Rounded to FP32 such that another rounding to fewer bits is that of the value itself: inexact ones end in a set bit.
__device__ __forceinline__ float to_odd(double x)
{
    const float f = (float)x;
    uint32_t bits = __float_as_uint(f);
    bits -= fabs((double)f) > fabs(x) ? 1u : 0u;
    return __uint_as_float(bits | ((double)f != x ? 1u : 0u));
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
    float peak[WAVES];
};

template <int CODES>
__global__ void __launch_bounds__(THREADS) cache_append(const uint64_t cu_q, const uint64_t seq_lens, const uint32_t batch,
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

    // ---- rows, angles ----
    const int page = __builtin_amdgcn_readfirstlane(gptr<int32_t>(p.table)[(uint64_t)b * p.tableWidth + column]);
    const uint32_t half = p.rotary / 2;
    const int from = 64 - (int)p.rotary / 8;     // first lane that is rotated
    u32x4 raw[EACH];
    int64_t place[EACH];
    bool mine[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int row = wave + WAVES * i;
        mine[i] = row >= low && row < high;
        const uint64_t token = (uint64_t)(first + (mine[i] ? row0 + row - start : begin - start));
        raw[i] = *gptr<u32x4>(p.updates + (token * p.updateStride + (uint64_t)head * p.updateHeadStride + lane * 8) * 2);
        place[i] = 0;
        if (p.rotary)
            place[i] = !p.positions        ? (int64_t)(row0 + row)
                       : p.int64Positions ? gptr<int64_t>(p.positions)[token]
                                          : (int64_t)gptr<int32_t>(p.positions)[token];
    }
    if ((uint32_t)page >= p.pages) return;
    const uint64_t scale_at = p.scale + ((uint64_t)page * p.scaleStride + head) * 4;
    float old = 0.0f;
    if (CODES != CHANNEL) old = *gptr<float>(scale_at);
    double y[EACH][8];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            y[i][e] = (double)__uint_as_float(e & 1 ? raw[i][e / 2] & 0xffff0000u : raw[i][e / 2] << 16);
        if (!p.rotary) continue;
        const bool there = place[i] >= 0 && place[i] < (int64_t)p.rotationRows;
        mine[i] = mine[i] && there;
        const uint64_t angles = p.rotation + (uint64_t)(there ? place[i] : 0) * p.rotationStride * 4;
        if (p.interleaved) {
            if (lane >= from) {
                const uint64_t at = angles + (uint64_t)(lane - from) * 16;
                const f32x4 cosine = *gptr<f32x4>(at), sine = *gptr<f32x4>(at + half * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double u = y[i][2 * e], v = y[i][2 * e + 1], c = cosine[e], n = sine[e];
                    y[i][2 * e] = fma(u, c, -(v * n)), y[i][2 * e + 1] = fma(u, n, v * c);
                }
            }
        } else {
            // Channel k of the first half goes with k of the second, R / 16 lanes on.
            const int apart = (int)p.rotary / 16;
            const bool second = lane >= from + apart;
            u32x4 other;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                other[e] = (uint32_t)__shfl((int)raw[i][e], lane < from ? lane : second ? lane - apart : lane + apart);
            if (lane >= from) {
                const uint64_t at = angles + (uint64_t)(lane - from - (second ? apart : 0)) * 32;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const f32x4 cosine = *gptr<f32x4>(at + 16 * q), sine = *gptr<f32x4>(at + half * 4 + 16 * q);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t w = other[2 * q + e / 2];
                        const double u = y[i][4 * q + e], v = (double)__uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
                        const double c = cosine[e], n = sine[e];
                        y[i][4 * q + e] = second ? fma(v, n, u * c) : fma(u, c, -(v * n));
                    }
                }
            }
        }
    }
    const uint64_t to = p.cache + (uint64_t)page * p.pageStride + ((uint64_t)head * D + lane * 8);
    const uint64_t row_bytes = (uint64_t)p.heads * D;

    // ---- frozen channel scales: the writer's codes ----
    if constexpr (CODES == CHANNEL) {
        const f32x4 inverse[2] = {gptr<f32x4>(p.inverseScale)[2 * lane], gptr<f32x4>(p.inverseScale)[2 * lane + 1]};
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (!mine[i]) continue;
            u32x2 w;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                int code[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = (float)y[i][4 * q + e] * inverse[q][e];
                    code[e] = (int)__builtin_rintf(fminf(fmaxf(v, -127.0f), 127.0f));
                }
                w[q] = pack_bytes(code);
            }
            *gout<u32x2>(to + (uint64_t)(wave + WAVES * i) * row_bytes) = w;
        }
        return;
    }

    // ---- the page's scale ----
    constexpr float LARGEST = CODES == E4M3 ? 448.0f : 127.0f;
    float peak = 0.0f;                           // NaN values do not count, infinities as the largest number
#pragma unroll
    for (int i = 0; i < EACH; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) peak = fmaxf(peak, mine[i] ? fabsf((float)y[i][e]) : 0.0f);
#pragma unroll
    for (int step = 1; step < 64; step *= 2) peak = fmaxf(peak, __shfl_xor(peak, step));
    if (lane == 0) s.peak[wave] = peak;
    asm volatile("" : "+v"(old));                // read before any wave may store the new one
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) peak = fmaxf(peak, s.peak[w]);
    const float needed = fmaxf(fminf(peak, 0x1.fffffep127f) / LARGEST, FLOOR);
    const bool begun = low > 0 && old > 0.0f && old < INFINITY;
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
    const double step = (double)scale, inverse = 1.0 / step;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (!mine[i]) continue;
        u32x2 w;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            int code[4];
            float value[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double x = fmin(fmax(y[i][4 * q + e], -0x1.fffffep127), 0x1.fffffep127);
                // The quotient, rounded once: a tie stays one.
                double v = x * inverse;
                v = fma(fma(-v, step, x), inverse, v);
                v = fmin(fmax(v, -(double)LARGEST), (double)LARGEST);
                const bool number = y[i][4 * q + e] == y[i][4 * q + e];
                code[e] = number ? (int)rint(v) : 0;
                value[e] = number ? to_odd(v) : __builtin_nanf("");
            }
            w[q] = CODES == E4M3 ? pack_e4m3(value[0], value[1], value[2], value[3]) : pack_bytes(code);
        }
        *gout<u32x2>(to + (uint64_t)(wave + WAVES * i) * row_bytes) = w;
    }
    if (power) {                                 // the rows before, in the new scale; rows behind the last stay
        const float f = ldexpf(1.0f, -power);
        for (int row = wave; row < low; row += WAVES) {
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
    const auto kernel = a->inverseScale ? &cache_append<CHANNEL> : a->codes ? &cache_append<E4M3> : &cache_append<INT8>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)first_of(a->tokens, a->batch), a->heads), dim3(THREADS), 0,
                       static_cast<hipStream_t>(stream), a->cuQ, a->seqLens, a->batch, a->tokens, *a);
    return (int)hipGetLastError();
}

uint32_t sharedkv_append_args_size(void) { return (uint32_t)sizeof(CacheAppendArgs); }

}  // extern "C"
