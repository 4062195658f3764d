// MI355X (gfx950) attention over paged 8-bit caches with one scale for each
// page of 32 rows and KV head.
//
// Mathematics.  Query row (token at position P, head h) sees the compressed rows
// and the window of original rows up to P (sharedkv_hip.h).  With code[j][c] the
// codes of key j and scale_j its page's scale,
//   s_j   = softmaxScale * scale_j * sum_c q[c] code[j][c]
//   out_c = sum_j e^{s_j} scale_j code[j][c] / (e^{sink} + sum_j e^{s_j})
// in one pass over the keys with a running maximum and sum.  A page's scale goes
// into the exponent: weights are 2^(s_j + log2 scale_j - m), so that P V runs on
// the codes as they lie in the cache, a weight beside a page of far larger values
// loses 2^-33 of the largest e^{s_j} scale_j at most, and neither scale costs an
// instruction for a key.  The sum of e^{s_j} takes a page's weights times
// 1 / scale_j.
//
// Q K.  INT8 codes run on v_mfma_i32_16x16x64_i8: Q times a power of two of its
// row becomes whole numbers, off by half of one at most, and the sums are exact.
// Two signed bytes hold the row's values up to the smaller of its largest and 8
// times its mean |q| (normal values' largest of 512 is some 4-5 times), so a unit is
// at most 1 / 16256 of that.  What is larger, in rows of which a few channels are,
// has a third byte: those blocks of 64 channels take one more matrix instruction for
// each sixteen keys; where LDS has no room for that byte (units of 64 rows have it
// for one block, of 32 for four) it is made from Q again for each tile.  (With 16
// bits for the row's largest a channel of 300 beside normal ones moves scores by
// 0.03.  Two chunks of 1900-2048 tokens take 730 us without such channels, 772 with
// one block of them, 920 with two and 1907 with eight; launches of few rows 0.35 us
// for the mean and 0.5 for a block.)  e4m3 codes, exact in BF16, run on v_mfma_f32_16x16x32_bf16
// against Q as it is.  (Q in two e4m3 terms would spare the conversion, at the same
// rate, but that matrix instruction sums eight products with 13 bits below their
// largest: scores up to 1e-4 off.)  P V runs on v_mfma_f32_16x16x32_f16: codes are
// exact in FP16, weights are rounded to its 11 bits (the output has 8); sums are of
// the weights before rounding.
//
// A unit is 16 RT query rows of one request and KV head (a row is a token and a
// head, heads innermost), which share every key tile of 64 rows (two pages).  A
// work-group of four waves takes an item, a run of a unit's tiles: for Q K a wave
// has sixteen of the rows and 16 RT of the keys, for P V all rows and 128 of the
// channels, the weights passing between them in LDS.  Tiles come by LDS DMA into
// a ring of two, one in flight while the other is used.  Every work-group makes
// the same plan from the live lengths.  Where units are split, a second launch
// joins their items' states.
//
// What bounds it.  Few query rows: the cache's bytes, 5.1 TB/s for 16 requests
// of one token and 8 heads over 32-128 K rows (130-138 us).  64 rows a unit: the
// vector instructions beside the matrix ones (codes to FP16 and the softmax): a wave
// and INT8 tile counts 512 SQ_INSTS_VALU and 128 SQ_INSTS_MFMA, and the matrix
// cores are busy for 44 % of the time.  512 tokens of one request over 64 K rows
// reach 1120-1183 TFLOP/s by the card, a large library FP16 product 1200-1240, and
// two prompts' chunks of 1900-2048 tokens over 8-16 K rows 1010-1035 (715-735 us).
// Between them, split contexts: the states of all items, written and read (up to
// 67 MB of 64-row units: 32 requests of 64 heads over 6-16 K rows 79-86 us, 12-15.5
// of them the join), and the launch's chain of round trips (lengths, pages and Q,
// scales, a tile; the join): one request of 4096 rows takes 12.5 us; in a trace the two kernels take 9.2 and 4.1.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "lds_dma.h"
#include "sharedkv_hip.h"

namespace {

constexpr int D = 512;
constexpr int KEYS = 64;           // keys of a tile: two pages
constexpr int PAGE_ROWS = 32;
constexpr int THREADS = 256;
constexpr int WAVES = THREADS / 64;
constexpr int P_STRIDE = KEYS + 8; // halves; 144 bytes keep the 16-byte reads of 16 rows on different banks
constexpr int WHOLE = 0x3fffffff;  // tiles of an item where units are not split
constexpr uint32_t MAX_HEADS = 128;
constexpr uint32_t MAX_WIDTH = (0x7fffffffu - KEYS) / PAGE_ROWS;
constexpr uint32_t MAX_GROUPS = 0xffffffffu / THREADS;   // the threads of a launch are counted in 32 bits
constexpr uint32_t SLOTS = 512;    // work-groups that run at once: two on each of 256 CUs
constexpr uint32_t MAX_SPLIT_UNITS = SLOTS * 3 / 4;       // launches of more units fill the slots as they are
// Tiles of a launch's units together, up to which a launch is split: they are summed over 64 lanes in 32 bits.
constexpr uint64_t MAX_SPLIT_WORK = 0x1ffffff;
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.69314718055994531f;
// Weights are 2^(s - m) with m the row's maximum less HEAD when it was last
// set, so they start at 2^HEAD and m moves only when a score passes it by
// LIMIT: 2^15 is below FP16's largest, and weights down to 2^-22 of the
// largest stay normal.
constexpr float HEAD = 8.0f, LIMIT = 15.0f;
// Least scale that weighs values: 2^15 / 2^-80 times any number of keys is an FP32 number.
constexpr float LEAST = 0x1p-80f;

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) v2i lds_v2i;
typedef __attribute__((address_space(3))) v4i lds_v4i;

template <typename T>
__device__ __forceinline__ const __attribute__((address_space(1))) T *gptr(uint64_t a)
{
    return reinterpret_cast<const __attribute__((address_space(1))) T *>(a);
}
// For stores: a flat store, which may reach LDS too, makes every later wait for an LDS read wait for all of them.
template <typename T>
__device__ __forceinline__ __attribute__((address_space(1))) T *gout(uint64_t a)
{
    return reinterpret_cast<__attribute__((address_space(1))) T *>(a);
}
// A value that the compiler takes for another: what is made of it is made anew where it is used and holds no register
// meanwhile.  (128 of a thread's 256 registers hold the output and 64 the codes of Q where a unit has 64 rows.)
__device__ __forceinline__ int again(int x)
{
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t uni64(uint64_t x)
{
    return (uint64_t)(uint32_t)uni((int)(x >> 32)) << 32 | (uint32_t)uni((int)x);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The launch's sizes.
struct Sizes {
    uint32_t tokens, ratioBits, window, oriTableWidth, cmpTableWidth, group, kvHeads;
    uint32_t groupInverse, groupBits;  // n / group is n * groupInverse >> groupBits for n below 2^31
};
__device__ __forceinline__ int by_group(const Sizes &p, int n) { return (int)((uint64_t)(uint32_t)n * p.groupInverse >> p.groupBits); }

// a / b, rounded down, for a from 0 and b from 1 on, with `inverse` about 1 / b: a step by the remainder for what FP32
// cannot hold, and one for its rounding.  (Divisions are most of the plan's instructions, and this one is half of a
// 32-bit division's.)
__device__ __forceinline__ int quotient(int a, int b, float inverse)
{
    int q = (int)((float)a * inverse), r = a - q * b;
    const int more = (int)((float)r * inverse);
    q += more, r -= more * b;
    return q + (r >= b) - (r < 0);
}

// A split unit as the join finds it: its parts' states are those of items first, first + stride, ...
struct Unit {
    int32_t first, stride, parts, rows;
    int32_t token, row0, head0, unused;   // first token of the request, the unit's first row in it, its first head
};

// A request's rows of the launch, made safe: nothing below reads or writes past
// the arrays whatever cuQ and seqLens hold.
struct Request {
    int32_t first, count, length;      // first token, tokens, all rows
    int32_t per_head, units, tiles;    // units of a KV head, of all; tiles of a unit, at most
    int32_t work, most;                // tiles of all units, about and at most
};

__device__ __forceinline__ int compressed_at(const Sizes &p, int position)
{
    const int64_t rows = (int64_t)p.cmpTableWidth * PAGE_ROWS;
    return p.ratioBits ? (int)min((int64_t)((uint32_t)max(position + 1, 0) >> p.ratioBits), rows) : 0;
}

template <int ROWS>
__device__ __forceinline__ Request request_of(const Sizes &p, int c0, int c1, int length)
{
    Request r;
    const int tokens = (int)p.tokens;
    r.first = min(max(c0, 0), tokens);
    r.count = min(max(c1, r.first), tokens) - r.first;
    r.length = length;
    r.per_head = (int)((r.count * (int64_t)p.group + ROWS - 1) / ROWS);
    r.units = r.per_head * (int)p.kvHeads;
    r.tiles = r.work = r.most = 0;
    if (length > 0 && r.count > 0) {
        const int64_t near = (int64_t)p.window + by_group(p, ROWS - 1) + 1 + PAGE_ROWS;
        const int64_t rows = min(min((int64_t)length, (int64_t)p.oriTableWidth * PAGE_ROWS), near);
        const int compressed = compressed_at(p, length - 1);
        r.tiles = (compressed + KEYS - 1) / KEYS + (int)((rows + KEYS - 1) / KEYS);
        // The first unit lacks the rows behind its tokens: half of that on average.
        const int less = (int)min(rows, max((int64_t)0, (int64_t)r.count - (length - rows))) + (compressed - compressed_at(p, length - r.count));
        r.work = (int)min((int64_t)r.units * max(1, r.tiles - less / (2 * KEYS)), (int64_t)MAX_SPLIT_WORK);
        r.most = (int)min((int64_t)r.units * r.tiles, (int64_t)MAX_SPLIT_WORK);
    }
    return r;
}

// Maximum over the four lanes of a query row (lane modulo 16).
__device__ __forceinline__ float row_max(float v)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __builtin_elementwise_maxnum(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_elementwise_maxnum(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// Sum over them.
__device__ __forceinline__ float row_total(float v)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Sum over the lanes up to and with this one.
__device__ __forceinline__ int wave_upto(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);    // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}
__device__ __forceinline__ int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_upto(v), 63); }

// Q of a lane's row as the matrix instructions take it: INT8, in two terms of whole numbers relative to a power of two
// of its own, most significant first (third terms above them are kept apart); e4m3, the first and the last eight of
// sixteen channels as they are.
template <bool E4M3>
struct Query {
    static constexpr float LARGEST = 127.0f * 256.0f;
    v4i term[2][8];                    // of channels 64 j + 16 g on
    float inverse, step;               // units of one; score (base 2) of one unit and scale 1

    // `peak`: of the values that two terms hold.
    __device__ __forceinline__ void set(float peak, float softmax2)
    {
        // Rows below 2^-90 score zero to FP32 against any code; their inverse would overflow.  The units' sign is the
        // softmax scale's, so that the largest sum has the largest score.
        const bool some = !(peak <= 0x1p-90f), odd = !(peak < INFINITY);
        int power = 15 - __builtin_amdgcn_frexp_expf(peak);
        if (ldexpf(peak, power) > LARGEST) --power;
        inverse = some && !odd ? (softmax2 < 0.0f ? -1.0f : 1.0f) * ldexpf(1.0f, power) : 0.0f;
        step = odd ? __builtin_nanf("") : some ? ldexpf(fabsf(softmax2), -power) : 1.0f;
    }
    // With 1.5 * 2^23 more, the nearest whole number sits in the low bits; with half of a byte's range more too,
    // the second byte is rounded as the first, signed, byte wants it, and that one has its sign bit flipped.
    static __device__ __forceinline__ uint32_t whole(const u32x4 &w, int e, float inverse)
    {
        return __float_as_uint(__builtin_fmaf(e & 1 ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2]), inverse, 12582912.0f + 128.0f));
    }
    // Eight channels' whole numbers: words [term][0 and 1].
    __device__ __forceinline__ void make(uint32_t (&out)[2][2], const u32x4 &w) const
    {
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = whole(w, e, inverse);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t *u = v + 4 * q;
            const uint32_t ab = __builtin_amdgcn_perm(u[1], u[0], 0x05040100u), cd = __builtin_amdgcn_perm(u[3], u[2], 0x05040100u);
            out[0][q] = __builtin_amdgcn_perm(cd, ab, 0x07050301u);
            out[1][q] = __builtin_amdgcn_perm(cd, ab, 0x06040200u) ^ 0x80808080u;
        }
    }
    // What sixteen channels have beyond the two terms, in 65536 units: at most 32, as no value is more than 512 times
    // the row's mean and the two terms hold 8 times that or all.
    static __device__ __forceinline__ v4i beyond(const u32x4 &a, const u32x4 &b, float inverse)
    {
        v4i out;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t word = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                word |= (((whole(q < 2 ? a : b, 4 * (q & 1) + e, inverse) - 0x4b400000u + 0x8000u) >> 16) & 255u) << (8 * e);
            out[q] = (int)word;
        }
        return out;
    }
};

// Eight e4m3 codes to BF16, exactly.
__device__ __forceinline__ bf16x8 to_bf16(int a, int b)
{
    const bf16x2 w0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)a, 1.0f, false);
    const bf16x2 w1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)a, 1.0f, true);
    const bf16x2 w2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)b, 1.0f, false);
    const bf16x2 w3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)b, 1.0f, true);
    return bf16x8{w0[0], w0[1], w1[0], w1[1], w2[0], w2[1], w3[0], w3[1]};
}

// Eight codes to FP16, exactly.  INT8: 1024 + (code + 128) has the byte as its low mantissa bits.
template <bool E4M3>
__device__ __forceinline__ f16x8 to_f16(v2i w)
{
    f16x8 out;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        f16x2 a, b;
        if (E4M3) {
            a = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)w[k], 1.0f, false));
            b = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)w[k], 1.0f, true));
        } else {
            const uint32_t u = (uint32_t)w[k] ^ 0x80808080u;
            a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - (_Float16)1152.0f;
            b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - (_Float16)1152.0f;
        }
        out[4 * k] = a[0], out[4 * k + 1] = a[1], out[4 * k + 2] = b[0], out[4 * k + 3] = b[1];
    }
    return out;
}

// Floats of an item's state: a row's numerators, then the rows' maxima and sums.
__host__ __device__ constexpr uint64_t state_floats(int rt) { return 16ull * rt * (D + 2); }

// Share of the sum of e^{s_j} 2^-m, `sum`, among it and the sink's, and the log-sum-exp (base 2).
struct Final {
    float give, lse2;
    __device__ __forceinline__ Final(float m, float sum, float sink2)
    {
        const float keys = sum == 0.0f ? -INFINITY : m + __builtin_amdgcn_logf(sum);
        const float most = keys != keys ? keys : fmaxf(keys, sink2);
        // Where both are -infinity no key was seen and there is no sink; an infinite sink takes everything.
        const float share = keys == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(keys - most);
        const float rest = sink2 == most ? (most == -INFINITY ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(sink2 - most);
        const float whole = share + rest;
        give = share == 0.0f ? 0.0f : share / (whole * sum);
        lse2 = whole == 0.0f ? most : most + __builtin_amdgcn_logf(whole);
    }
};

// Tile addresses below are made by XOR within a row's 512 bytes.
template <int RT>
struct alignas(1024) Shared {
    static constexpr int ROWS = 16 * RT, PARTS = WAVES / RT;
    int8_t tile[2][KEYS * D];          // key rows, their 16-byte chunks XOR-swizzled with the row
    _Float16 p[ROWS * P_STRIDE];       // weights [row][key]
    float factor[ROWS], top[ROWS], sum[PARTS][ROWS], peak[PARTS][ROWS];
    uint32_t far[WAVES];               // INT8: blocks of 64 channels where a row of the wave's has values beyond two terms
    int32_t moved[RT];                 // whether a row tile moved its maximum in this tile
    int32_t scan[3][WAVES];
    int32_t found[6];
    int32_t token[ROWS];               // of the unit's rows, counted in the request
    int32_t place[ROWS];               // their rows of q and out
};
// INT8: for rows of Q with values beyond two terms.
template <int RT>
struct Beyond {
    static constexpr int BLOCKS = RT == 1 ? 8 : RT == 2 ? 4 : 1;   // as many as leave two work-groups a CU
    v4i third[RT][BLOCKS][64];         // third terms of a row tile's first blocks that have some
    uint64_t query[16 * RT];           // the rows' addresses in q
    float inverse[16 * RT];            // units of one
};

template <bool E4M3, int RT>
__global__ void __launch_bounds__(THREADS, 2) block_attention(const uint64_t cu_q, const uint64_t seq_lens, const uint32_t batch_arg, const uint32_t split_arg,
                const uint32_t tokens_arg, const uint32_t ratio_bits, const uint32_t window_rows, const uint32_t ori_width,
                const uint32_t cmp_width, const uint32_t group_arg, const uint32_t kv_heads, const uint32_t group_inverse,
                const uint32_t group_bits, const BlockAttentionArgs p)
{
    const Sizes size = {tokens_arg, ratio_bits, window_rows, ori_width, cmp_width, group_arg, kv_heads, group_inverse, group_bits};
    using S = Shared<RT>;
    constexpr int ROWS = S::ROWS, PARTS = S::PARTS;
    constexpr int MIN_TILES = RT == 4 ? 8 : RT; // of an item; 1 to 12 differ little
    __shared__ S s;
    __shared__ Beyond<RT> beyond;
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), g = lane >> 4, n = lane & 15;
    // The leading arguments are the ones that the first loads need: the build preloads them into SGPRs.  split_arg: the units
    // and, from bit 16 on, the work-groups that the launch has scratch for; 0 where it is not split.
    const uint32_t split = split_arg & 0xffff;
    const int group = (int)group_arg, heads = group * (int)kv_heads, batch = (int)batch_arg;
    const auto *cu = gptr<int32_t>(cu_q), *lens = gptr<int32_t>(seq_lens);

    // ---- plan: units and tiles of the live requests, tiles of an item, this work-group's item ----
    const bool one_step = batch <= THREADS, one_wave = batch <= 64;
    Request mine = {};
    int units = 0, work = 0, most = 0;                 // units, times their tiles, about and at most
    for (int b = one_wave ? lane : tid; b < batch; b += THREADS) {
        mine = request_of<ROWS>(size, cu[b], cu[b + 1], lens[b]);
        units += mine.units;
        work = min(mine.work + work, (int)MAX_SPLIT_WORK);
        most = min(mine.most + most, (int)MAX_SPLIT_WORK);
    }
    const int end = min(max(cu[batch], 0), (int)size.tokens) * heads;
    const int all_rows = (int)size.tokens * heads, pad_units = (all_rows - end + ROWS - 1) / ROWS;
    units = wave_sum(units);
    uint32_t all_work = (uint32_t)wave_sum(work);      // of launches that may be split at most MAX_SPLIT_WORK
    uint32_t all_most = (uint32_t)wave_sum(most);      // likewise
    if (!one_wave) {
        if (lane == 0) s.scan[0][wave] = units, s.scan[1][wave] = (int)all_work, s.scan[2][wave] = (int)all_most;
        if (tid == 0) s.found[0] = -1;
        __syncthreads();
        units = 0, all_work = 0, all_most = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) units += s.scan[0][w], all_work += (uint32_t)s.scan[1][w], all_most += (uint32_t)s.scan[2][w];
    }
    // Tiles of an item: the fewest of five that leave no more than SLOTS items, as the scratch has room for no more.  Four
    // go by the tiles of average units and are counted where a wave holds all requests.  The last always fits: units of t
    // tiles make ceil(t / per_item) <= 1 + (t - 1) / per_item items each, and it divides all their tiles (a prompt's first
    // units see fewer, but count as the others do) by the slots that the units and the padding leave.  (It alone takes
    // 95.8 us for a prompt of 2048 tokens, and 86.4 with the four before it.)  `split` is the number of units that the
    // launch has scratch for: requests that lie one behind the other are never more, and others are not split.
    int per_item = WHOLE;
    if (units + pad_units <= (int)split) {
        const int whole = units + pad_units;
        auto share = [&](uint32_t tiles, int room) {
            return max(MIN_TILES, quotient((int)tiles + room - 1, room, __builtin_amdgcn_rcpf((float)room)));
        };
        per_item = share(all_most, (int)SLOTS - whole);
        if (one_wave) {
            int tries[4], items[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                tries[i] = share(all_work, (int)SLOTS - whole * i / 3);
                items[i] = wave_sum(mine.units * max(1, quotient(mine.tiles + tries[i] - 1, tries[i], __builtin_amdgcn_rcpf((float)tries[i]))));
            }
#pragma unroll
            for (int i = 3; i >= 0; --i) per_item = items[i] + pad_units <= (int)SLOTS ? tries[i] : per_item;
        }
    }
    per_item = uni(per_item), units = uni(units);
    const bool may_split = per_item != WHOLE;
    if (split && blockIdx.x == 0 && tid == 0) *gout<int32_t>(p.units) = may_split ? units : 0;
    const float item_inverse = __builtin_amdgcn_rcpf((float)per_item);
    auto parts_of = [&](int tiles) { return max(1, quotient(tiles + per_item - 1, per_item, item_inverse)); };
    // Where units are split, the work-groups of one XCD (blockIdx modulo 8) take neighbouring items, which read the same
    // rows.
    int item = 0, items = 0, unit0 = 0, b = -1, local = 0, first = 0, past = 0, length = 0;
    auto take = [&](int number) {                      // the work-group's item of `number`; false: none
        items = number;
        const int share = (items + 7) / 8;
        item = may_split ? (int)(blockIdx.x & 7) * share + (int)(blockIdx.x >> 3) : (int)blockIdx.x;
        return item < (may_split ? min(items, (int)(split_arg >> 16)) : items) && !(may_split && (int)(blockIdx.x >> 3) >= share);
    };
    if (one_wave) {                                    // every wave for itself
        const int n_items = mine.units * parts_of(mine.tiles), upto = wave_upto(n_items), at_units = wave_upto(mine.units);
        if (!take(__builtin_amdgcn_readlane(upto, 63) + pad_units)) return;
        const uint64_t its = __ballot(item < upto && item >= upto - n_items);
        if (its) {
            b = __builtin_ctzll(its);
            local = item - __builtin_amdgcn_readlane(upto - n_items, b), unit0 = __builtin_amdgcn_readlane(at_units - mine.units, b);
            first = __builtin_amdgcn_readlane(mine.first, b), past = first + __builtin_amdgcn_readlane(mine.count, b);
            length = __builtin_amdgcn_readlane(mine.length, b);
        }
    } else {
        int upto = 0, at_units = 0;
        for (int pass = 0; pass < 2 && b < 0; ++pass) {
            // First the number of items (pass 0 ends there where one step holds all requests), then whose this one is.
            int before = 0, units_before = 0;
            for (int at = 0; at < batch; at += THREADS) {
                const int b0 = at + tid;
                if (!one_step) mine = b0 < batch ? request_of<ROWS>(size, cu[b0], cu[b0 + 1], lens[b0]) : Request{};
                const bool there = b0 < batch;
                const int u = there ? mine.units : 0, n_items = there ? u * parts_of(mine.tiles) : 0;
                upto = wave_upto(n_items), at_units = wave_upto(u);
                __syncthreads();
                if (lane == 63) s.scan[0][wave] = upto, s.scan[1][wave] = at_units;
                __syncthreads();
                int total = 0, total_units = 0;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    if (w < wave) upto += s.scan[0][w], at_units += s.scan[1][w];
                    total += s.scan[0][w], total_units += s.scan[1][w];
                }
                upto += before, at_units += units_before;
                before += total, units_before += total_units;
                if (one_step || pass) {
                    if (!take(one_step ? before + pad_units : items)) return;
                    if (item < upto && item >= upto - n_items) {
                        s.found[0] = b0, s.found[1] = item - (upto - n_items), s.found[2] = at_units - u;
                        s.found[3] = mine.first, s.found[4] = mine.first + mine.count, s.found[5] = mine.length;
                    }
                }
            }
            items = before + pad_units;
            if (one_step) break;
        }
        __syncthreads();
        b = s.found[0];
        if (b >= 0) local = s.found[1], unit0 = s.found[2], first = s.found[3], past = s.found[4], length = s.found[5];
    }
    item = uni(item), items = uni(items);
    auto zero_row = [&](int64_t place) {               // by one wave
        *gout<u32x4>(p.out + (uint64_t)place * (D * 2) + lane * 16) = u32x4{0, 0, 0, 0};
        if (p.lse && lane == 0) gout<float>(p.lse)[place] = 0.0f;
    };
    if (b < 0) {                                       // rows behind the last request
        const int64_t first = (int64_t)end + (int64_t)(item - (items - pad_units)) * ROWS;
        for (int i = wave; i < ROWS; i += WAVES)
            if (first + i >= end && first + i < all_rows) zero_row(first + i);
        return;
    }
    b = uni(b), local = uni(local), unit0 = uni(unit0);
    const Request r = request_of<ROWS>(size, uni(first), uni(past), uni(length));
    const int slots = uni(parts_of(r.tiles));
    // Items of a request: by KV head, part, unit.  Whole units go from the last, which see most.
    const int of_parts = uni(quotient(local, r.per_head, __builtin_amdgcn_rcpf((float)r.per_head)));
    const int kv_head = uni(quotient(of_parts, slots, __builtin_amdgcn_rcpf((float)slots))), part = of_parts - kv_head * slots;
    const int from_first = local - of_parts * r.per_head, in_head = slots == 1 ? r.per_head - 1 - from_first : from_first;
    const int row0 = in_head * ROWS;                   // of the request and KV head
    const int rows = min((int64_t)ROWS, r.count * (int64_t)group - row0);
    const int t0 = by_group(size, row0), t1 = by_group(size, row0 + rows - 1);
    // ---- the unit's tiles: compressed rows, then original ones, upwards ----
    const int start = r.length - r.count, at0 = start + t0, at1 = start + t1;     // positions
    const int window = (int)min(size.window, 0x7fffffffu);
    const int cmp_rows = uni(compressed_at(size, at1)), cmp_tiles = (cmp_rows + KEYS - 1) / KEYS;
    const int low = (at0 >= window ? at0 - window + 1 : 0) & ~(PAGE_ROWS - 1);
    const int high = (int)min((int64_t)at1 + 1, (int64_t)size.oriTableWidth * PAGE_ROWS);
    const int tiles = r.length > 0 ? cmp_tiles + max(0, high - low + KEYS - 1) / KEYS : 0;
    const int parts = uni(min(slots, parts_of(tiles)));
    const int its_unit = unit0 + kv_head * r.per_head + in_head;
    if (may_split && part == 0 && tid == 0 && (uint32_t)its_unit < split) {
        auto *to = gout<int32_t>(p.units + sizeof(Unit) * (uint64_t)(1 + its_unit));
        const Unit u = {item, r.per_head, parts, rows, r.first, row0, kv_head * group, 0};
        to[0] = u.first, to[1] = u.stride, to[2] = u.parts, to[3] = u.rows, to[4] = u.token, to[5] = u.row0, to[6] = u.head0;
    }
    if (part >= parts) return;
    const int share = parts == 1 ? tiles : uni(quotient(tiles, parts, __builtin_amdgcn_rcpf((float)parts)));
    const int more = tiles - share * parts;            // equal shares, the first ones a tile more
    const int k0 = part * share + min(part, more), k1 = k0 + share + (part < more);
    if (tid < ROWS) {
        const int at = row0 + min(tid, rows - 1), token = by_group(size, at);
        s.token[tid] = token;
        s.place[tid] = (r.first + token) * heads + kv_head * group + (at - token * group);
    }
    lds_barrier();
    if (r.length <= 0) {                               // graph padding
        for (int i = wave; i < rows; i += WAVES) zero_row(s.place[i]);
        return;
    }

    auto base_of = [&](int k) { return k < cmp_tiles ? k * KEYS : low + (k - cmp_tiles) * KEYS; };
    int entries = -1;                                  // page of half (lane & 1) of tile 32 block + lane / 2
    float scales = 1.0f;                               // and its scale
    auto read_entries = [&](int block) {
        const int lx = again(tid) & 63, k = 32 * block + (lx >> 1);
        const bool ori = k >= cmp_tiles;
        const int e = base_of(k) / PAGE_ROWS + (lx & 1), width = (int)(ori ? p.oriTableWidth : p.cmpTableWidth);
        entries = k < k1 && e < width ? gptr<int32_t>(ori ? p.oriTable : p.cmpTable)[(int64_t)b * width + e] : -1;
        scales = 1.0f;
        if ((uint32_t)entries < (ori ? p.oriPages : p.cmpPages))
            scales = gptr<float>(ori ? p.oriScale : p.cmpScale)[(uint64_t)(uint32_t)entries *
                                                                     (ori ? p.oriScaleStride : p.cmpScaleStride) + kv_head];
    };
    // Starts the copies of tile k and returns its rows that lie on a page.  Wave w moves rows 4 w .. 4 w + 3 of every
    // sixteen, two an instruction, so that a lane's place in a row (the swizzle goes by the row modulo 16) is the same
    // for all sixteens, and differs by one bit between the pairs.
    const uint32_t row_bytes = kv_heads * D;
    auto copy_tile = [&](int k) -> uint64_t {
        const int at = 2 * (k & 31);
        const bool ori = k >= cmp_tiles;
        const uint64_t pool = (ori ? p.ori : p.cmp) + (uint64_t)kv_head * D, stride = ori ? p.oriStride : p.cmpStride;
        const uint32_t pages = ori ? p.oriPages : p.cmpPages;
        const int lx = again(tid) & 63;
        const uint32_t lane_offset =
            (uint32_t)(4 * wave + (lx >> 5)) * row_bytes + (uint32_t)(((lx & 31) ^ (4 * wave + (lx >> 5))) << 4);
        const uint32_t to = (uint32_t)(uintptr_t)s.tile[k & 1] + 4 * wave * D;
        uint64_t rows_there = 0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int page = __builtin_amdgcn_readlane(entries, at + half);
            if ((uint32_t)page >= pages) continue;
            rows_there |= 0xffffffffull << (32 * half);
            const uint64_t from = uni64(pool + (uint64_t)page * stride);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t lds = (uint32_t)uni((int)(to + (32 * half + 16 * i) * D));
                lds_dma16(from + 16 * i * row_bytes, lane_offset, lds);
                lds_dma16(from + 16 * i * row_bytes, (lane_offset ^ 32u) + 2 * row_bytes, lds + 2 * D);
            }
        }
        return rows_there;
    };

    // ---- Q; the first tile is on its way while Q is encoded ----
    const int row = 16 * (wave % RT) + n;              // the lane's row in Q K
    const int key0 = wave / RT * 16 * RT;              // the wave's first key there
    // The waves of a row tile encode a share of its channels each (64 j .. 64 j + 63, j from j0 on) and pass the codes
    // round in the tile buffer that is free.
    constexpr bool SHARE = PARTS > 1 && !E4M3;
    constexpr int AT_ONCE = KEYS * D / (RT * 8 * 64 * 16) < 2 ? 1 : 2;   // terms that the buffer holds
    constexpr int JN = SHARE ? 8 / PARTS : 8;
    const int j0 = SHARE ? wave / RT * JN : 0;
    Query<E4M3> q = {};
    auto stage_at = [&](int8_t *stage, int t, int j) { return stage + ((((wave % RT) * AT_ONCE + t) * 8 + j) * 64 + lane) * 16; };
    uint64_t seen = 0, next_seen = 0;
    uint32_t far = 0;                                  // INT8: blocks of 64 channels where a row has values beyond two terms
    if (k0 < k1) {
        const float softmax2 = p.softmaxScale * LOG2E;
        const auto *q_row = gptr<u32x4>(p.q + (uint64_t)(uint32_t)s.place[row] * (D * 2)) + 2 * g + 8 * j0;
        u32x4 raw[JN][2];
#pragma unroll
        for (int j = 0; j < JN; ++j) raw[j][0] = q_row[8 * j], raw[j][1] = q_row[8 * j + 1];
        read_entries(k0 >> 5);
        // The copies come last: a wait for an earlier load does not wait for them.
#pragma unroll
        for (int j = 0; j < JN; ++j) asm volatile("" : "+v"(raw[j][0]), "+v"(raw[j][1]));
        next_seen = copy_tile(k0);
        if constexpr (E4M3) {
            const uint32_t flip = softmax2 < 0.0f ? 0x80008000u : 0u;
            q.step = fabsf(softmax2);
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) q.term[h][j] = __builtin_bit_cast(v4i, raw[j][h] ^ flip);
        } else {
            float peak = 0.0f, sums[2] = {0.0f, 0.0f}; // keeps a NaN; sums of |q|
#pragma unroll
            for (int j = 0; j < JN; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float lo = fabsf(bf16_lo(raw[j][h][e])), hi = fabsf(bf16_hi(raw[j][h][e]));
                        peak = __builtin_elementwise_maximum(__builtin_elementwise_maximum(peak, lo), hi);
                        sums[0] += lo, sums[1] += hi;
                    }
            peak = row_max(peak == peak ? peak : INFINITY);   // from here on infinity stands for both
            float mean = row_total(sums[0] + sums[1]);
            if (SHARE) {
                if (g == 0) s.peak[wave / RT][row] = peak, s.sum[wave / RT][row] = mean;
                lds_barrier();
                mean = 0.0f;
#pragma unroll
                for (int part = 0; part < PARTS; ++part) peak = fmaxf(peak, s.peak[part][row]), mean += s.sum[part][row];
                lds_barrier();
            }
            // Two terms hold 8 times the mean, whatever a few channels have: those go into a third.
            const float most = peak < INFINITY ? fminf(peak, mean * (8.0f / D)) : peak;
            q.set(most, softmax2);
            if (__ballot(peak > most)) {               // in all waves of these rows
                if (wave < RT && g == 0)
                    beyond.inverse[row] = q.inverse, beyond.query[row] = p.q + (uint64_t)(uint32_t)s.place[row] * (D * 2);
#pragma unroll
                for (int j = 0; j < JN; ++j) {
                    float its = 0.0f;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            its = fmaxf(its, fmaxf(fabsf(bf16_lo(raw[j][h][e])), fabsf(bf16_hi(raw[j][h][e]))));
                    far |= __ballot(its * fabsf(q.inverse) > Query<false>::LARGEST) ? 1u << (j0 + j) : 0u;
                }
            }
            if (SHARE && lane == 0) s.far[wave] = far;
            int8_t *stage = s.tile[(k0 + 1) & 1];
            v4i own[SHARE ? 2 : 1][SHARE ? JN : 1];
#pragma unroll
            for (int j = 0; j < JN; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t out[2][2];
                    q.make(out, raw[j][h]);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        v4i &to = SHARE ? own[SHARE ? t : 0][SHARE ? j : 0] : q.term[t][j];
                        to[2 * h] = (int)out[t][0], to[2 * h + 1] = (int)out[t][1];
                    }
                    if (!SHARE) __builtin_amdgcn_sched_barrier(0);
                }
            if (SHARE) {
#pragma unroll
                for (int t0 = 0; t0 < 2; t0 += AT_ONCE) {
                    if (t0) lds_barrier();
#pragma unroll
                    for (int t = t0; t < t0 + AT_ONCE; ++t)
#pragma unroll
                        for (int j = 0; j < JN; ++j)
                            *reinterpret_cast<v4i *>(stage_at(stage, t - t0, j0 + j)) = own[SHARE ? t : 0][SHARE ? j : 0];
                    lds_barrier();
#pragma unroll
                    for (int t = t0; t < t0 + AT_ONCE; ++t)
#pragma unroll
                        for (int j = 0; j < 8; ++j) q.term[t][j] = *reinterpret_cast<const v4i *>(stage_at(stage, t - t0, j));
                }
#pragma unroll
                for (int part = 0; part < PARTS; ++part) far |= s.far[wave % RT + part * RT];
                far = (uint32_t)uni((int)far);
            }
        }
    }
    if constexpr (!E4M3) {
        int n = 0;
        for (uint32_t rest = far; rest && n < Beyond<RT>::BLOCKS; rest &= rest - 1, ++n) {   // seldom
            if (wave / RT != n % PARTS) continue;
            const auto *from = gptr<u32x4>(p.q + (uint64_t)(uint32_t)s.place[row] * (D * 2)) + 2 * g + 8 * __builtin_ctz(rest);
            const u32x4 low = from[0], high = from[1];
            beyond.third[wave % RT][n][lane] = Query<E4M3>::beyond(low, high, q.inverse);
        }
    }
    // Tiles whose rows all of the unit's tokens see need no masks.
    auto is_plain = [&](int k) {
        const int base = base_of(k);
        if (k < cmp_tiles) return base + KEYS <= compressed_at(size, at0);
        return base > at1 - window && base + KEYS <= at0 + 1;
    };
    f32x4 acc[8][RT] = {};
    float m = -INFINITY, sum = 0.0f;
#pragma nounroll
    for (int k = k0; k < k1; ++k) {
        seen = next_seen;
        const int scale0 = __builtin_amdgcn_readlane(__float_as_int(scales), 2 * (k & 31));
        const int scale1 = __builtin_amdgcn_readlane(__float_as_int(scales), 2 * (k & 31) + 1);
        vm_wait_all();
        lds_barrier();                                 // tile k is there; nobody uses tile k - 1 or its weights any more
        if (k + 1 < k1) {
            if (!((k + 1) & 31)) read_entries((k + 1) >> 5);
            next_seen = copy_tile(k + 1);
        }
        const int lx = again(tid) & 63, its_row = 16 * (wave % RT) + (lx & 15);
        const uint32_t tile = (uint32_t)(uintptr_t)s.tile[k & 1];

        // S = Q K^T: query row n, keys key0 + 16 kt + 4 g + i.
        float w[RT][4];
        {
            const uint32_t at = tile + (uint32_t)((key0 + (lx & 15)) * D + (((lx >> 4) ^ (lx & 15)) << 4));
            if constexpr (E4M3) {
                // Step st: keys of tile st / 8, channels 64 (st % 8) on; reads run two steps ahead, conversions half a one.
                constexpr int STEPS = 8 * RT, AHEAD = 3;
                v4i key[AHEAD];
                bf16x8 value[2];
                auto fetch = [&](int st) {
                    key[st % AHEAD] = *(const lds_v4i *)(uintptr_t)((at ^ (uint32_t)(64 * (st & 7))) + (uint32_t)(16 * (st >> 3) * D));
                };
                fetch(0);
                fetch(1);
                value[0] = to_bf16(key[0][0], key[0][1]);
                f32x4 dots[2];
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    if (st + 2 < STEPS) fetch(st + 2);
                    const int j = st & 7;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (h == 0) value[1] = to_bf16(key[st % AHEAD][2], key[st % AHEAD][3]);
                        if (h == 1 && st + 1 < STEPS) value[0] = to_bf16(key[(st + 1) % AHEAD][0], key[(st + 1) % AHEAD][1]);
                        dots[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value[h], __builtin_bit_cast(bf16x8, q.term[h][j]),
                                                                          j ? dots[h] : f32x4{0, 0, 0, 0}, 0, 0, 0);
                    }
                    if (j == 7)
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[st >> 3][i] = dots[0][i] + dots[1][i];
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                constexpr int PAIR = RT == 2 ? 2 : 1, STEPS = 8 * RT / PAIR, AHEAD = 3;
                // Step st: keys of tiles PAIR (st / 8) on, channels 64 (st % 8) on; reads run two steps ahead.
                v4i key[AHEAD][PAIR];
                auto fetch = [&](int st) {
#pragma unroll
                    for (int kt = 0; kt < PAIR; ++kt)
                        key[st % AHEAD][kt] = *(const lds_v4i *)(uintptr_t)((at ^ (uint32_t)(64 * (st & 7))) +
                                                                           (uint32_t)(16 * (PAIR * (st >> 3) + kt) * D));
                };
                fetch(0);
                fetch(1);
                v4i dots[2][PAIR];
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    if (st + 2 < STEPS) fetch(st + 2);
                    const int j = st & 7;
#pragma unroll
                    for (int kt = 0; kt < PAIR; ++kt)
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            dots[t][kt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(key[st % AHEAD][kt], q.term[t][j],
                                                                                j ? dots[t][kt] : v4i{0, 0, 0, 0}, 0, 0, 0);
                    if (j == 7)
#pragma unroll
                        for (int kt = 0; kt < PAIR; ++kt)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                // At most 512 * 32512 * 128 + 512 * 128 * 128, and far less where there is a third
                                // term (fewer than 64 channels pass 8 times the mean): within 32 bits.
                                w[PAIR * (st >> 3) + kt][i] = (float)(dots[0][kt][i] * 256 + dots[1][kt][i]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                for (uint32_t rest = far; rest; rest &= rest - 1) {         // seldom
                    const int n = __builtin_popcount(far) - __builtin_popcount(rest);
                    const int j = __builtin_ctz(rest);
                    v4i third;
                    if (Beyond<RT>::BLOCKS == 8 || n < Beyond<RT>::BLOCKS) {
                        third = beyond.third[wave % RT][n][lx];
                    } else {
                        const auto *from = gptr<u32x4>(beyond.query[its_row]) + 2 * (lx >> 4) + 8 * j;
                        const u32x4 low = from[0], high = from[1];
                        third = Query<E4M3>::beyond(low, high, beyond.inverse[its_row]);
                    }
#pragma unroll
                    for (int kt = 0; kt < RT; ++kt) {
                        const v4i code = *(const lds_v4i *)(uintptr_t)((at ^ (uint32_t)(64 * j)) + (uint32_t)(16 * kt * D));
                        const v4i dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(code, third, v4i{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[kt][i] = __builtin_fmaf((float)dot[i], 65536.0f, w[kt][i]);
                    }
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
        const bool edge = !is_plain(k) || seen != ~0ull;
        if (edge) {
            const int position = start + s.token[its_row], base = base_of(k);
            const int to = k < cmp_tiles ? compressed_at(size, position) - base : position + 1 - base;
            const int from = k < cmp_tiles || position < window ? 0 : max(0, position - window + 1 - base);
            uint64_t bits = seen;
            bits &= to >= KEYS ? ~0ull : to <= 0 ? 0ull : ~0ull >> (KEYS - to);
            bits &= from >= KEYS ? 0ull : ~0ull << from;
#pragma unroll
            for (int kt = 0; kt < RT; ++kt) {
                const uint32_t its = (uint32_t)(bits >> (key0 + 16 * kt + 4 * (lx >> 4))) & 15u;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[kt][i] = its >> i & 1 ? w[kt][i] : -INFINITY;
            }
        }
        // Of the pages that the wave's keys are on (one, or for units of 64 rows both): a unit's score, log2 of the scale that
        // weighs values, and its inverse.
        constexpr int PAGES = RT == 4 ? 2 : 1;
        float step[PAGES], lift[PAGES], drop[PAGES];
#pragma unroll
        for (int h = 0; h < PAGES; ++h) {
            const float its = __int_as_float((PAGES == 2 ? h : wave >> 1) ? scale1 : scale0);
            step[h] = __builtin_elementwise_maximum(q.step * its, 0x1p-126f);   // never 0: masked keys score -infinity; keeps a NaN
            lift[h] = __builtin_amdgcn_logf(its < LEAST ? LEAST : its);
            drop[h] = __builtin_amdgcn_exp2f(-lift[h]);
        }
        float peak = -INFINITY, most = -INFINITY;      // of score + lift
#pragma unroll
        for (int kt = 0; kt < RT; ++kt) {
            // (These maxima pass over a NaN and take two values an instruction.)
            if (PAGES == 1 || !(kt & 1)) most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; i += 2) most = __builtin_elementwise_maxnum(__builtin_elementwise_maxnum(most, w[kt][i]), w[kt][i + 1]);
            if (PAGES == 1 || kt & 1) {
                const int h = PAGES == 2 ? kt >> 1 : 0;
                peak = __builtin_elementwise_maxnum(peak, __builtin_fmaf(most, step[h], lift[h]));
            }
        }
        peak = row_max(peak);
        if (PARTS > 1) {                               // the row's keys are spread over waves
            if (lx < 16) s.peak[wave / RT][its_row] = peak;
            lds_barrier();
#pragma unroll
            for (int part = 0; part < PARTS; ++part) peak = fmaxf(peak, s.peak[part][its_row]);
        }
        const bool move = peak > m + LIMIT;            // and where m is still -infinity
        const bool any = __ballot(move) != 0;
        if (wave < RT && lx == 0) s.moved[wave] = any;
        if (any) {                                     // seldom
            const float factor = move ? __builtin_amdgcn_exp2f(m - (peak - HEAD)) : 1.0f;
            if (move) m = peak - HEAD;
            sum *= factor;
            if (wave < RT && lx < 16) s.factor[its_row] = factor;
        }
        // Weights 2^(score + lift - m): 0 for masked keys, also where all have been masked so far.
        auto weigh = [&](auto masked) {
            const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int kt = 0; kt < RT; ++kt) {
                f16x4 half;
                const int h = PAGES == 2 ? kt >> 1 : 0;
                const float less = lift[h] - from;
                float together = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = __builtin_amdgcn_exp2f(__builtin_fmaf(w[kt][i], step[h], less));
                    if (masked.value) x = w[kt][i] == -INFINITY ? 0.0f : x;   // whatever the page's scale is
                    together += x;
                    half[i] = (_Float16)x;
                }
                if (!masked.value || together != 0.0f) sum = __builtin_fmaf(together, drop[h], sum);
                *reinterpret_cast<f16x4 *>(s.p + its_row * P_STRIDE + key0 + 16 * kt + 4 * (lx >> 4)) = half;
            }
        };
        if (edge)
            weigh(std::true_type{});
        else
            weigh(std::false_type{});
        if (E4M3 && edge) {
            // A code that is no number may lie in a row that some token does not see, and 0 times it is none either.
            // Rows that see it have weights that are no numbers already.
            lds_barrier();                             // all scores are made
            for (int i = again(tid); i < KEYS * D / 16; i += THREADS) {
                u32x4 v = reinterpret_cast<u32x4 *>(s.tile[k & 1])[i];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] &= ~((((v[e] & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u) * 255u);
                reinterpret_cast<u32x4 *>(s.tile[k & 1])[i] = v;
            }
        }
        lds_barrier();

        // acc[ct][rt]: channels 128 wave + 16 ct + 4 g + i, row 16 rt + n.
        {
            const int lx = again(tid) & 63;
            const int slot = 8 * (lx >> 4) + ((lx & 15) >> 1);
            const uint32_t from = tile + (uint32_t)(slot * D + 8 * (lx & 1) + (((8 * wave) ^ (slot & 15)) << 4));
            const _Float16 *its = s.p + (lx & 15) * P_STRIDE + 8 * (lx >> 4);
            // Step st: channels 16 (st % 8) on of keys 32 (st / 8) on.  Reads run AHEAD steps ahead, and the next step's
            // codes are converted between this step's matrix instructions.
            constexpr int AHEAD = 4;
            v2i code[AHEAD];
            auto fetch = [&](int st) {
                code[st % AHEAD] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                    (lds_v2i *)(uintptr_t)((from ^ (uint32_t)((st & 7) << 4)) + (uint32_t)(32 * (st >> 3) * D)));
            };
            f16x8 weight[RT], value[2];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) weight[rt] = *reinterpret_cast<const f16x8 *>(its + 16 * rt * P_STRIDE);
#pragma unroll
            for (int st = 0; st < AHEAD; ++st) fetch(st);
            int moved = 0;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) moved |= s.moved[rt];
            if (uni(moved)) {
                float f[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) f[rt] = s.moved[rt] ? s.factor[16 * rt + (lx & 15)] : 1.0f;
#pragma unroll
                for (int ct = 0; ct < 8; ++ct)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) acc[ct][rt] *= f[rt];
            }
            value[0] = to_f16<E4M3>(code[0]);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int st = 0; st < 16; ++st) {
                if (st == 8)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) weight[rt] = *reinterpret_cast<const f16x8 *>(its + 16 * rt * P_STRIDE + 32);
                if (st + AHEAD < 16) fetch(st + AHEAD);
                if (st + 1 < 16) value[(st + 1) & 1] = to_f16<E4M3>(code[(st + 1) % AHEAD]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    acc[st & 7][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value[st & 1], weight[rt], acc[st & 7][rt], 0, 0, 0);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);              // one matrix instruction,
                    __builtin_amdgcn_sched_group_barrier(0x2, 12 / RT, 0);         // then others
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
        }
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    const int last = again(tid), lx = last & 63, gx = lx >> 4, nx = lx & 15;
    if (gx == 0) {
        s.sum[wave / RT][16 * (wave % RT) + nx] = sum;
        if (wave < RT) s.top[16 * (wave % RT) + nx] = m;
    }
    lds_barrier();
    auto row_sum = [&](int at) {
        float total = s.sum[0][at];
#pragma unroll
        for (int part = 1; part < PARTS; ++part) total += s.sum[part][at];
        return total;
    };
    if (parts > 1) {                                   // joined by the next launch
        const uint64_t state = p.partial + (uint64_t)item * state_floats(RT) * 4;
#pragma unroll
        for (int ct = 0; ct < 8; ++ct)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                if (16 * rt + nx < rows)
                    *gout<f32x4>(state + ((16 * rt + nx) * D + 128 * wave + 16 * ct + 4 * gx) * 4) = acc[ct][rt];
        if (last < rows) {
            gout<float>(state)[ROWS * D + last] = s.top[last];
            gout<float>(state)[ROWS * (D + 1) + last] = row_sum(last);
        }
        return;
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int at = 16 * rt + nx;
        if (at >= rows) continue;
        const uint32_t place = (uint32_t)s.place[at];
        const Final f(s.top[at], row_sum(at), gptr<float>(p.sinks)[place % (uint32_t)heads] * LOG2E);
#pragma unroll
        for (int ct = 0; ct < 8; ++ct) {
            const f32x4 v = acc[ct][rt] * f.give;
            *gout<u32x2>(p.out + (uint64_t)place * (D * 2) + (128 * wave + 16 * ct + 4 * gx) * 2) =
                u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
        }
        if (p.lse && wave == 0 && gx == 0) gout<float>(p.lse)[place] = f.lse2 * LN2;
    }
}

// Joins the states of a split unit's items, in the parts' order: a row, all channels of it where there are few parts and
// 128 where there are many.  What bounds it is the chain of its reads (the unit; all maxima, sums and the first
// numerators), so each is started as soon as it can be.
constexpr int AT_ONCE = 4;                             // parts that a thread reads at once

template <int CHANNELS>
__global__ void __launch_bounds__(THREADS) block_join(const uint64_t partial, const uint64_t units, const uint32_t rt, const uint32_t group,
                                                      const uint32_t heads, const BlockAttentionArgs p)
{
    constexpr int LANES = CHANNELS / 4, JOINERS = THREADS / LANES;        // of a part; parts read side by side
    __shared__ float factor[SLOTS];
    __shared__ float most_of[THREADS / 64], sum_of[THREADS / 64];
    __shared__ f32x4 sums[JOINERS][LANES];
    const uint32_t rows = 16 * rt;
    const int unit = (int)(blockIdx.x / rows), row = (int)(blockIdx.x % rows), tid = threadIdx.x;
    const auto *u = gptr<int32_t>(units + sizeof(Unit) * (uint64_t)(1 + unit));
    const int number = *gptr<int32_t>(units), first = u[0], stride = u[1], parts = min(u[2], (int)SLOTS), its_rows = u[3];
    const int token0 = u[4], row0 = u[5], head0 = u[6];
    if (unit >= number || parts < 2 || row >= its_rows) return;
    const uint64_t size = 16ull * rt * (D + 2);
    auto state = [&](int part) { return gptr<float>(partial) + (uint64_t)(first + part * stride) * size; };
    const int channel = CHANNELS * (int)blockIdx.y + 4 * (tid % LANES), joiner = tid / LANES;
    auto numerators = [&](int part) {
        return *reinterpret_cast<const __attribute__((address_space(1))) f32x4 *>(state(part) + row * D + channel);
    };
    constexpr int EACH = SLOTS / THREADS;
    float m[EACH], l[EACH], most = -INFINITY, total = 0.0f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int part = tid + i * THREADS;
        m[i] = -INFINITY, l[i] = 0.0f;
        if (part < parts) m[i] = state(part)[rows * D + row], l[i] = state(part)[rows * (D + 1) + row];
    }
    f32x4 v[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) v[i] = numerators(min(joiner + i * JOINERS, parts - 1));
#pragma unroll
    for (int i = 0; i < EACH; ++i) most = fmaxf(most, m[i]);
#pragma unroll
    for (int step = 1; step < 64; step *= 2) most = fmaxf(most, __shfl_xor(most, step));
    if ((tid & 63) == 0) most_of[tid >> 6] = most;
    lds_barrier();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) most = fmaxf(most, most_of[w]);
    const float from = most == -INFINITY ? 0.0f : most;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int part = tid + i * THREADS;
        const float f = __builtin_amdgcn_exp2f(m[i] - from);
        factor[part] = f;                              // 0 past the parts
        total += l[i] * f;
    }
#pragma unroll
    for (int step = 1; step < 64; step *= 2) total += __shfl_xor(total, step);
    if ((tid & 63) == 0) sum_of[tid >> 6] = total;
    lds_barrier();
    total = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) total += sum_of[w];
    f32x4 sum = {};
#pragma nounroll
    for (int part = joiner; part < parts; part += AT_ONCE * JOINERS) {
        f32x4 next[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) next[i] = numerators(min(part + (AT_ONCE + i) * JOINERS, parts - 1));
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
            if (part + i * JOINERS < parts) sum += v[i] * factor[part + i * JOINERS];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) v[i] = next[i];
    }
    sums[joiner][tid % LANES] = sum;
    lds_barrier();
    if (joiner) return;
#pragma unroll
    for (int i = 1; i < JOINERS; ++i) sum += sums[i][tid];
    const int at = row0 + row, token = at / (int)group;
    const uint32_t place = (uint32_t)((token0 + token) * (int)heads + head0 + at - token * (int)group);
    const Final f(most, total, gptr<float>(p.sinks)[place % heads] * LOG2E);
    sum *= f.give;
    *gout<u32x2>(p.out + (uint64_t)place * (D * 2) + channel * 2) = u32x2{pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3])};
    if (p.lse && tid == 0 && blockIdx.y == 0) gout<float>(p.lse)[place] = f.lse2 * LN2;
}

bool rejected(const BlockAttentionArgs *a)
{
    if (!a || !a->heads || a->heads > MAX_HEADS || !a->kvHeads || a->heads % a->kvHeads || !a->batch || !a->window || !a->ratio)
        return true;
    if (!a->q || !a->ori || !a->oriScale || !a->oriTable || !a->cuQ || !a->seqLens || !a->sinks || !a->out) return true;
    if (a->ratio > 0x40000000u || (a->ratio & (a->ratio - 1)) || a->codes > 1) return true;
    const uint64_t page = (uint64_t)PAGE_ROWS * D * a->kvHeads;
    if (!a->oriPages || !a->oriTableWidth || (a->oriStride & 15) || a->oriStride < page) return true;
    if ((a->q | a->ori | a->out) & 15 || a->oriScale & 3) return true;
    if (a->ratio > 1 && (!a->cmp || !a->cmpScale || !a->cmpTable || !a->cmpPages || !a->cmpTableWidth ||
                         (a->cmpStride & 15) || a->cmpStride < page || a->cmp & 15 || a->cmpScale & 3))
        return true;
    // Rows and pages are counted in 32 bits, signed: a table's rows and a tile more.
    return a->batch > 0xffffffu || (uint64_t)a->tokens * a->heads > 0x7fff0000ull || a->oriTableWidth > MAX_WIDTH ||
           a->cmpTableWidth > MAX_WIDTH;
}

struct Plan {
    int rt;
    bool split;
    uint32_t units, grid;
};
Plan plan_of(const BlockAttentionArgs *a)
{
    Plan plan;
    const uint64_t rows = (uint64_t)a->tokens * a->heads;
    const uint64_t near = (uint64_t)a->window + 2 * PAGE_ROWS + 64;
    const uint64_t tiles = (a->ratio > 1 ? (a->cmpTableWidth + 1) / 2 : 0) +
                           ((near / PAGE_ROWS < a->oriTableWidth ? near / PAGE_ROWS : a->oriTableWidth) + 1) / 2;
    // Units of 16 rows spread few rows over more work-groups and have the smallest states; units of 64 rows convert a key
    // for more of them, so that the matrix instructions bound them, but split contexts move four times the states.  With R
    // tiles of 64 rows in a launch and `tiles` of 64 keys in a unit (by the block tables' width, as lengths are not known
    // here: tables far wider than the contexts take larger units than these would, 8 requests of 64 heads over 4 K rows
    // 25.7 us with a table of 4 K rows, 28.4 of 32 K and 39.0 of 128 K), the better one goes by R * R * tiles, and for units of
    // 64 rows by the tiles too (microseconds of 16, 32 and 64 rows a unit):
    //        64  1 request, 64 heads, 4 K      16.6, 18.5, 33.7     131 K  16 of 16 tokens, 8 K         82.3, 64.3, 63.7
    //       4 K  8, 64 heads, 4 K              25.5, 28.9, 38.2     131 K  1 of 128 tokens, 32 K         144,  101, 89.3
    //      16 K  8 of 8 tokens, 16 K           50.0, 42.7, 42.4     131 K  64 of 8 tokens, 2 K          53.0, 44.5, 45.2
    //      32 K  8, 64 heads, 32 K             83.3, 69.6, 69.5     262 K  32, 64 heads, 6-16 K          120, 89.9, 85.0
    //      65 K  4 of 32 tokens, 16 K          81.3, 61.1, 62.6     262 K  8 of 256 tokens, window      33.4, 24.4, 32.9
    //     1.0 M  2 of 2048 tokens, window      65.3, 47.1, 38.3     4.2 M  4 of 512 tokens, 4 K          256,  160,  158
    const uint64_t each = (rows / a->kvHeads + a->batch - 1) / a->batch;        // rows of a request and KV head, on average
    const uint64_t score = (rows + 63) / 64 * ((rows + 63) / 64) * tiles;
    const bool wide = score >= 400000 || (score >= 130000 && tiles >= 128);
    plan.rt = each <= 16 || score < 8000 ? 1 : each <= 32 || !wide ? 2 : 4;
    // The last unit of a request and KV head may be short, and so may the padding's; a token's rows are in few units.
    const uint64_t group = a->heads / a->kvHeads, unit = 16 * plan.rt;
    const uint64_t short_last = rows / unit + (uint64_t)a->batch * a->kvHeads;
    const uint64_t by_token = (uint64_t)a->tokens * a->kvHeads * ((group + unit - 1) / unit);
    const uint64_t units = (short_last < by_token ? short_last : by_token) + 1;
    plan.units = units > MAX_GROUPS ? MAX_GROUPS + 1 : (uint32_t)units;
    plan.split = plan.units <= MAX_SPLIT_UNITS && tiles > 1 && plan.units * tiles <= MAX_SPLIT_WORK;
    const uint64_t items = plan.split ? plan.units * tiles : plan.units;
    plan.grid = (uint32_t)((plan.split && items > SLOTS ? SLOTS : items) + 7) & ~7u;
    return plan;
}

}  // namespace

extern "C" {

int launch_sharedkv_block(void *stream, const BlockAttentionArgs *a)
{
    if (rejected(a)) return (int)hipErrorInvalidValue;
    if (!a->tokens) return (int)hipSuccess;
    const Plan plan = plan_of(a);
    if (plan.grid > MAX_GROUPS) return (int)hipErrorInvalidValue;
    if (plan.split && (!a->partial || !a->units || ((a->partial | a->units) & 15))) return (int)hipErrorInvalidValue;
    const auto of_rows = [&](auto e4m3) {
        return plan.rt == 4   ? &block_attention<e4m3.value, 4>
               : plan.rt == 2 ? &block_attention<e4m3.value, 2>
                              : &block_attention<e4m3.value, 1>;
    };
    const auto kernel = a->codes ? of_rows(std::true_type{}) : of_rows(std::false_type{});
    const uint32_t group = a->heads / a->kvHeads;
    uint32_t bits = 0;                                 // 2^31 * 2^bits / group, rounded up, is exact for 31 bits
    while ((1u << bits) < group) ++bits;
    const uint32_t inverse = (uint32_t)(((0x80000000ull << bits) + group - 1) / group);
    hipLaunchKernelGGL(kernel, dim3(plan.grid), dim3(THREADS), 0, static_cast<hipStream_t>(stream), a->cuQ, a->seqLens,
                       a->batch, plan.split ? plan.grid << 16 | plan.units : 0u, a->tokens, (uint32_t)__builtin_ctz(a->ratio), a->window,
                       a->oriTableWidth, a->ratio > 1 ? a->cmpTableWidth : 0u, group, a->kvHeads, inverse, 31 + bits, *a);
    if (plan.split) {
        // By the parts of a unit where all are alike: few rows of many parts take more work-groups.
        const uint32_t parts = plan.grid / plan.units, channels = parts <= 16 ? 512 : parts <= 64 ? 128 : 32;
        hipLaunchKernelGGL(channels == 512 ? &block_join<512> : channels == 128 ? &block_join<128> : &block_join<32>,
                           dim3(plan.units * 16 * plan.rt, D / channels), dim3(THREADS), 0, static_cast<hipStream_t>(stream),
                           a->partial, a->units, (uint32_t)plan.rt, group, a->heads, *a);
    }
    return (int)hipGetLastError();
}

int sharedkv_block_scratch(const BlockAttentionArgs *a, uint64_t *partial, uint64_t *units)
{
    if (!partial || !units || rejected(a)) return (int)hipErrorInvalidValue;
    const Plan plan = plan_of(a);
    if (plan.grid > MAX_GROUPS) return (int)hipErrorInvalidValue;
    *partial = plan.split ? plan.grid * state_floats(plan.rt) * 4 : 0;
    *units = plan.split ? sizeof(Unit) * (1 + (uint64_t)plan.units) : 0;
    return (int)hipSuccess;
}

uint32_t sharedkv_block_args_size(void) { return (uint32_t)sizeof(BlockAttentionArgs); }

}  // extern "C"
