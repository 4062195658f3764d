// MI355X (gfx950) attention of drafted-token trees over the paged INT8 caches.
//
// Mathematics.  Query row (token i, head h) of request b sees the compressed
// rows, the window rows and its ancestors' rows (sharedkv_hip.h).  With
// code[j][c] the INT8 codes of key j and scale[c] the channel scales,
//   s_j   = softmaxScale * sum_c q[c] scale[c] code[j][c]
//   out_c = scale[c] * sum_j e^{s_j} code[j][c] / (e^{sink} + sum_j e^{s_j})
// one pass over the keys with the running maximum and sum of the softmax.
//
// Q K runs on v_mfma_i32_16x16x64_i8: q * scale becomes a whole number of 16
// bits per channel (24 where the log-sum-exp is asked for) relative to its
// row's largest, split into signed bytes, so the keys are used as they lie in
// the cache and the sums are exact integers.  16 bits leave a score within
// 2^-16 of its row's scale, far below the output's BF16; the log-sum-exp is an
// FP32 result and takes 24.  P V runs on v_mfma_f32_16x16x32_f16: codes are
// exact in FP16, weights are rounded to its 11 bits (the output has 8).
//
// A unit is 16 RT query rows of one request (a row is a token and a head, heads
// innermost), which share every key tile of 64 rows (two pages).  A work-group
// of four waves takes an item, a run of a unit's tiles: for Q K a wave has
// sixteen of the rows and 16 RT of the keys, for P V all rows and 128 of the
// channels, the weights passing between them in LDS.  Tiles come by LDS DMA into
// a ring of two, one in flight while the other is used.  Every work-group makes
// the same plan from the live lengths (which requests there are, how many tiles
// an item gets), and the last item of a unit to finish joins the unit's states.
//
// What bounds it.  4 * 512 flops for every 512-byte key and query row: from some
// hundred rows a request on, the matrix instructions and the vector ones beside
// them (a key's codes to FP16, the softmax).  4 requests of 57-61 tokens and 16
// heads over 20-32 K rows take 231-246 us by the card, 824-880 TFLOP/s, three quarters of
// a large library FP16 product's rate; a SIMD takes about 4960 cycles for a wave's tile,
// 2048 of them busy with matrix instructions, beside some 420 vector ones.  Small launches are a chain of
// round trips (lengths, Q and tables, tiles, states): one request of 8 tokens and
// 4096 rows takes 13.5 us, 32 of 4-16 tokens 22.6.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "lds_dma.h"
#include "sharedkv_hip.h"
#include "xcd_local.h"

namespace {

constexpr int D = 512;
constexpr int KEYS = 64;           // keys of a tile: two pages
constexpr int PAGE_ROWS = 32;
constexpr int THREADS = 256;
constexpr int WAVES = THREADS / 64;
constexpr int P_STRIDE = KEYS + 8; // halves; 144 bytes keep the 16-byte reads of 16 rows on different banks
constexpr int PARENTS = 1024;      // parents kept in LDS; larger trees read theirs from memory
constexpr int ROOT = 0xffff;
constexpr int WHOLE = 0x3fffffff;  // tiles of an item where units are not split
constexpr uint32_t MAX_HEADS = 128;
constexpr int CUS = 256;
constexpr uint32_t MAX_WIDTH = (0x7fffffffu - KEYS) / PAGE_ROWS;
constexpr uint32_t MAX_GROUPS = 0xffffffffu / THREADS;   // the threads of a launch are counted in 32 bits
// Items of a launch: two work-groups on each of 256 CUs; of small units, whose items differ most, half as many again (32
// requests of 4-16 nodes: 24.8 us in at most 512 items, 22.7 in 768, 30.1 in 1024).
__host__ __device__ constexpr uint32_t items_for(int rt) { return rt == 1 ? 768 : 512; }
// Tiles of a launch's units together, up to which a launch is split: they are summed over 64 lanes in 32 bits.
constexpr uint64_t MAX_SPLIT_WORK = 0x1ffffff;
constexpr uint32_t XCD_LOCAL = 0x80000000u;   // bit of `split`: work-groups with one blockIdx modulo 8 share an XCD
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.69314718055994531f;
// Weights are 2^(s - m) with m the row's maximum less HEAD when it was last
// set, so they start at 2^HEAD and m moves only when a score passes it by
// LIMIT: 2^15 is below FP16's largest, and weights down to 2^-22 of the
// largest stay normal.
constexpr float HEAD = 8.0f, LIMIT = 15.0f;
// Cache policies of the states that items exchange: past the XCD's L2, where items of other XCDs see them, or in it.
constexpr int SC1 = 16, SC0 = 1;

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i lds_v2i;
typedef __attribute__((address_space(3))) v4i lds_v4i;

template <typename T>
__device__ __forceinline__ const __attribute__((address_space(1))) T *gptr(uint64_t a)
{
    return reinterpret_cast<const __attribute__((address_space(1))) T *>(a);
}
// A value that the compiler takes for another: what is made of it is made anew where it is used and holds no register
// meanwhile.  (128 of a thread's 256 registers hold the output and 64 the codes of Q where a unit has 64 rows.)
__device__ __forceinline__ int again(int x)
{
    asm volatile("" : "+v"(x));
    return x;
}
// For stores: a flat store, which may reach LDS too, makes every later wait for an LDS read wait for all of them.
template <typename T>
__device__ __forceinline__ __attribute__((address_space(1))) T *gout(uint64_t a)
{
    return reinterpret_cast<__attribute__((address_space(1))) T *>(a);
}
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Scale in which a channel's numerator is held once original rows have joined the compressed ones: the original one,
// unless that is so far below the compressed one that the quotient could overflow.  Raised, it is at most 2^-60 of the
// compressed one, and so is what the original codes add.
__device__ __forceinline__ f32x4 joint_scale(f32x4 cmp, f32x4 ori)
{
    f32x4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = fmaxf(fmaxf(ori[i], cmp[i] * 0x1p-60f), 0x1p-149f);
    return out;
}

// Tile addresses below are made by XOR within a row's 512 bytes.
template <int RT>
struct alignas(1024) Shared {
    static constexpr int ROWS = 16 * RT, PARTS = WAVES / RT;
    int8_t tile[2][KEYS * D];          // key rows, their 16-byte chunks XOR-swizzled with the row
    union {
        _Float16 p[ROWS * P_STRIDE];   // weights [row][key]
        float scale[2][D];             // channel scales (compressed, original) while Q is encoded
    };
    uint64_t mask[ROWS];               // the tile's rows that each of the unit's tokens sees
    float factor[ROWS], top[ROWS], sum[PARTS][ROWS], peak[PARTS][ROWS];
    int32_t moved[RT];                 // whether a row tile moved its maximum in this tile
    int32_t scan[3][WAVES];
    int32_t found[7];
    // Of the unit's tokens: node that the walk is at, steps to it, depth, compressed rows it sees.
    int32_t walk[ROWS], steps[ROWS], depth[ROWS], compressed[ROWS];
    uint8_t token[ROWS];               // of the unit's rows
    uint16_t parent[PARENTS];
};

// A request's rows of the launch, made safe: nothing below reads past the
// arrays whatever cuQ and seqLens hold.
struct Request {
    int32_t first, nodes, length, committed;   // first token, drafted tokens, all rows, committed rows
    bool live;
    int32_t compressed, shared;        // compressed rows that some token may see, that all do
    int32_t low, end;                  // original rows [low, end), low a multiple of PAGE_ROWS
    int32_t cmp_tiles, ori_tiles;
};

// The launch's sizes.
struct Sizes {
    uint32_t tokens, ratio, window, oriTableWidth, cmpTableWidth;
};
template <bool CAUSAL>
__device__ __forceinline__ Request request_of(const Sizes &p, int c0, int c1, int length)
{
    Request r;
    const int tokens = (int)p.tokens;
    r.first = min(max(c0, 0), tokens);
    r.nodes = min(max(c1, r.first), tokens) - r.first;
    r.length = length;
    r.live = length > 0 && r.nodes > 0;
    r.committed = max(0, length - r.nodes);
    const int64_t ori_rows = (int64_t)p.oriTableWidth * PAGE_ROWS, cmp_rows = (int64_t)p.cmpTableWidth * PAGE_ROWS;
    r.shared = p.ratio > 1 ? (int)min((int64_t)(r.committed / (int)p.ratio), cmp_rows) : 0;
    r.compressed = CAUSAL ? (int)min((int64_t)((r.committed + r.nodes) / (int)p.ratio), cmp_rows) : r.shared;
    r.low = max(0, r.committed - (int)min(p.window, 0x7fffffffu) + 1) & ~(PAGE_ROWS - 1);
    r.end = (int)min((int64_t)r.committed + r.nodes, ori_rows);
    r.cmp_tiles = r.live ? (r.compressed + KEYS - 1) / KEYS : 0;
    r.ori_tiles = r.live ? max(0, r.end - r.low + KEYS - 1) / KEYS : 0;
    return r;
}

// Maximum over the four lanes of a query row (lane modulo 16).
__device__ __forceinline__ float row_max(float v)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// Products q * scale of the lane's channels 64 j + 16 g + 8 h on.
struct Products {
    float x[8];
};
__device__ __forceinline__ Products products(const u32x4 &w, const float *scale)
{
    Products out;
#pragma unroll
    for (int e = 0; e < 8; ++e) out.x[e] = (e & 1 ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2])) * scale[e];
    return out;
}

// q * scale as whole numbers of 8 * TERMS bits relative to the row's largest.
template <int TERMS>
struct Codes {
    static constexpr float LARGEST = TERMS == 2 ? 127.0f * 256.0f : 127.0f * 65536.0f;
    v4i term[TERMS][8];                // most significant first
    float inverse, step;               // units of one q * scale; score (base 2) of one unit

    __device__ __forceinline__ void set(float peak, float softmax2)
    {
        // Rows below 2^-90 score zero to FP32 against any code; their inverse would overflow.  The units' sign is the
        // softmax scale's, so that the largest sum has the largest score.
        const bool some = !(peak <= 0x1p-90f), odd = !(peak < INFINITY);
        inverse = some && !odd ? (softmax2 < 0.0f ? -LARGEST : LARGEST) / peak : 0.0f;
        // Never 0, so that masked keys score -infinity.
        step = odd ? __builtin_nanf("") : some ? fmaxf(peak / LARGEST * fabsf(softmax2), 0x1p-126f) : 1.0f;
    }
    // Eight channels' codes: words [term][0 and 1].
    __device__ __forceinline__ void make(uint32_t (&out)[TERMS][2], const Products &from) const
    {
        uint32_t v[8];
        if (TERMS == 2) {
            // With 1.5 * 2^23 more, the nearest whole number sits in the low bits; with half of a byte's range more too,
            // the second byte is rounded as the first, signed, byte wants it, and that one has its sign bit flipped.
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = __float_as_uint(__builtin_fmaf(from.x[e], inverse, 12582912.0f + 128.0f));
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t *u = v + 4 * q;
                const uint32_t ab = __builtin_amdgcn_perm(u[1], u[0], 0x05040100u), cd = __builtin_amdgcn_perm(u[3], u[2], 0x05040100u);
                out[0][q] = __builtin_amdgcn_perm(cd, ab, 0x07050301u);
                out[1][q] = __builtin_amdgcn_perm(cd, ab, 0x06040200u) ^ 0x80808080u;
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (uint32_t)(int)__builtin_rintf(from.x[e] * inverse);
#pragma unroll
        for (int t = TERMS - 1; t >= 0; --t)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t *u = v + 4 * q;
                const uint32_t ab = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), cd = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
                out[t][q] = ab | cd;
#pragma unroll
                for (int e = 0; e < 4; ++e) u[e] = (u[e] + 128) >> 8;
            }
    }
};

// Eight codes to FP16, exactly: 1024 + (code + 128) has the byte as its low mantissa bits.  (Left unsubtracted, as a
// subnormal code + 128, the offset would save two fifths of these instructions, and round the sums of a long context
// at 128 times their size.)
__device__ __forceinline__ f16x8 to_f16(v2i w)
{
    f16x8 out;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t u = (uint32_t)w[k] ^ 0x80808080u;
        const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - (_Float16)1152.0f;
        const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - (_Float16)1152.0f;
        out[4 * k] = a[0], out[4 * k + 1] = a[1], out[4 * k + 2] = b[0], out[4 * k + 3] = b[1];
    }
    return out;
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

// Floats of an item's state: numerators in the order the waves hold them, then
// the rows' maxima and sums.
__host__ __device__ constexpr uint64_t state_floats(int rt) { return 16ull * rt * (D + 2); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t state_at(uint64_t partial, uint64_t item, int rt)
{
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<float *>(partial) + item * state_floats(rt), 0, 0x7fffffff,
                                             0x00020000);
}

// Place of a work-group's unit among `units` in falling length.
__device__ __forceinline__ int by_length(int group, int units)
{
    if (group >= units || units <= CUS || units > 2 * CUS) return group;
    const int shared = units - CUS;                    // CUs with two units: the first work-groups'
    return group < shared ? CUS - shared + group : group < CUS ? group - shared : units - 1 - (group - CUS);
}

// CAUSAL: compressed rows go by a token's own position.  A kernel of its own: the masks' scalars, kept over the tile loop,
// cost whole contexts 2 % (243.3 to 248.1 us, 16 requests of 24 nodes and 64 heads 79.6 to 80.4), which launches without
// them need not pay.
template <int TERMS, int RT, bool CAUSAL>
__global__ void __launch_bounds__(THREADS, TERMS == 2 || RT < 4 ? 2 : 1) tree_attention(const uint64_t cu_q, const uint64_t seq_lens, const uint32_t batch_arg, const uint32_t heads_arg,
               const uint32_t split, const uint32_t tokens_arg, const uint32_t ratio, const uint32_t window_rows,
               const uint32_t ori_width, const uint32_t cmp_width, const TreeAttentionArgs p)
{
    const Sizes size = {tokens_arg, ratio, window_rows, ori_width, cmp_width};
    using S = Shared<RT>;
    constexpr int ROWS = S::ROWS, PARTS = S::PARTS;
    __shared__ S s;
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), g = lane >> 4, n = lane & 15;
    // The leading arguments are the ones that the first loads need: the build preloads them into SGPRs.
    const int heads = (int)heads_arg, batch = (int)batch_arg;
    const auto *cu = gptr<int32_t>(cu_q), *lens = gptr<int32_t>(seq_lens);

    // ---- plan: units and tiles of the live requests, tiles of an item, this work-group's item ----
    auto units_of = [&](const Request &r) { return (r.nodes * heads + ROWS - 1) / ROWS; };
    Request mine = {};
    int units = 0, kinds = 0, work = 0;                // units, times their kinds, times their tiles
    for (int b = tid; b < batch; b += THREADS) {
        mine = request_of<CAUSAL>(size, cu[b], cu[b + 1], lens[b]);
        const int u = units_of(mine);
        units += u;
        kinds += u * max(1, (mine.cmp_tiles > 0) + (mine.ori_tiles > 0));
        work = (int)min((int64_t)u * (mine.cmp_tiles + mine.ori_tiles) + work, (int64_t)MAX_SPLIT_WORK);
    }
    const int end = min(max(cu[batch], 0), (int)size.tokens) * heads;
    const int all_rows = (int)size.tokens * heads, pad_units = (all_rows - end + ROWS - 1) / ROWS;
    units = wave_sum(units), kinds = wave_sum(kinds), work = wave_sum(work);
    if (lane == 0) s.scan[0][wave] = units, s.scan[1][wave] = kinds, s.scan[2][wave] = work;
    if (tid == 0) s.found[0] = -1;
    __syncthreads();
    units = kinds = pad_units;
    int64_t all_work = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) units += s.scan[0][w], kinds += s.scan[1][w], all_work += s.scan[2][w];
    // Tiles of an item: as many as leave no more than items_for items (a unit's last of either kind may be short).
    // `split` is the number of units that the launch has scratch for: requests that lie one behind the other are never
    // more, and others are not split.
    int per_item = WHOLE;
    if (units <= (int)(split & ~XCD_LOCAL)) {
        const int64_t room = (int64_t)items_for(RT) - kinds;
        per_item = (int)min((int64_t)WHOLE - 1, max((int64_t)1, (all_work + room - 1) / room));
    }
    // A unit that is split is split between its kinds too: Q is encoded with a kind's scales.
    auto parts_of = [&](int tiles) { return (tiles + per_item - 1) / per_item; };
    auto items_of = [&](const Request &r) {
        return per_item == WHOLE ? 1 : max(1, parts_of(r.cmp_tiles) + parts_of(r.ori_tiles));
    };
    // Work-groups of one XCD (blockIdx modulo 8) take neighbouring items, which read the same rows.  Whole units of 64
    // rows go by their length instead, the longest first, and where there are more than one and at most two for a CU, the
    // longest run alone and the shortest share a CU: work-groups come to CUs in order, the first 256 to one each (16
    // requests of 24 nodes and 64 heads over 64-128 K rows, 384 units: 87.4 us in the requests' order, 80.9 so, 89.7 with
    // the longest sharing).  Requests past a wave's lanes keep their order.
    const bool ranked = RT == 4 && per_item == WHOLE && batch <= 64;
    int item, items = 0, share = 0, unit = 0, unit0 = 0, b = -1;
    {
        int upto = 0, at_units = 0;
        for (int pass = 0; pass < 2 && b < 0; ++pass) {
            // First the number of items (pass 0 ends there where one step holds all requests), then whose this one is.
            int before = 0, units_before = 0;
            const bool one_step = batch <= THREADS;
            for (int at = 0; at < batch; at += THREADS) {
                const int b0 = at + tid;
                if (!one_step) mine = b0 < batch ? request_of<CAUSAL>(size, cu[b0], cu[b0 + 1], lens[b0]) : Request{};
                const bool there = b0 < batch;
                const int u = there ? units_of(mine) : 0, n_items = there ? u * items_of(mine) : 0;
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
                if (ranked) {                      // items of the requests before it by length, in the first wave
                    const int rank = min(mine.cmp_tiles + mine.ori_tiles, 0xffffff) << 6 | (63 - lane);
                    upto = n_items;
                    if (wave == 0)
                        for (int i = 0; i < batch; ++i) {
                            const int other = __builtin_amdgcn_readlane(n_items, i);
                            upto += __builtin_amdgcn_readlane(rank, i) > rank ? other : 0;
                        }
                }
                if (one_step || pass) {
                    if (one_step) items = before + pad_units;
                    share = (items + 7) / 8;
                    item = (int)(blockIdx.x & 7) * share + (int)(blockIdx.x >> 3);
                    if (!ranked && (int)(blockIdx.x >> 3) >= share) return;
                    if (ranked) item = by_length((int)blockIdx.x, items);
                    if (item >= items) return;
                    if (item < upto && item >= upto - n_items) {
                        s.found[0] = b0, s.found[1] = item - (upto - n_items), s.found[2] = at_units - u;
                        s.found[3] = mine.first, s.found[4] = mine.first + mine.nodes, s.found[5] = mine.length;
                    }
                }
            }
            items = before + pad_units;
            if (one_step) break;
        }
        __syncthreads();
        b = s.found[0];
    }
    auto zero_rows = [&](int first, int count) {
        for (int i = tid; i < count * (D / 8); i += THREADS)
            gout<u32x4>(p.out)[(int64_t)first * (D / 8) + i] = u32x4{0, 0, 0, 0};
        if (p.lse)
            for (int i = tid; i < count; i += THREADS) gout<float>(p.lse)[first + i] = 0.0f;
    };
    if (b < 0) {                                       // rows behind the last request
        const int64_t first = (int64_t)end + (int64_t)(item - (items - pad_units)) * ROWS;
        if (first < all_rows) zero_rows((int)first, (int)min((int64_t)ROWS, all_rows - first));
        return;
    }
    b = uni(b);
    const Request r = request_of<CAUSAL>(size, uni(s.found[3]), uni(s.found[4]), uni(s.found[5]));
    const int splits = items_of(r), local = uni(s.found[1]);
    const int part_no = local % splits;                // which of the unit's items
    unit = local / splits;
    unit0 = uni(s.found[2]);
    const int row0 = unit * ROWS;                      // of the request
    const int rows = min(ROWS, r.nodes * heads - row0);
    const int64_t out0 = (int64_t)r.first * heads + row0;
    if (!r.live) {
        zero_rows((int)out0, rows);
        return;
    }
    const int tiles = r.cmp_tiles + r.ori_tiles;
    int k0 = 0, k1 = tiles;
    if (splits > 1) {                                  // equal shares of the kind's tiles
        const int first = parts_of(r.cmp_tiles), second = parts_of(r.ori_tiles);
        const bool window = part_no >= first;
        const int at = window ? part_no - first : part_no, of = window ? second : first;
        const int its_tiles = window ? r.ori_tiles : r.cmp_tiles;
        k0 = (window ? r.cmp_tiles : 0) + (int)((int64_t)its_tiles * at / of);
        k1 = (window ? r.cmp_tiles : 0) + (int)((int64_t)its_tiles * (at + 1) / of);
    }

    // ---- tiles: k < cmp_tiles compressed rows upwards, then the original rows downwards (walks go up the tree) ----
    auto base_of = [&](int k) { return k < r.cmp_tiles ? k * KEYS : r.low + (tiles - 1 - k) * KEYS; };
    int entries = -1;                                  // page of half (lane & 1) of tile 32 block + lane / 2
    auto read_entries = [&](int block) {
        const int k = 32 * block + (lane >> 1);
        const bool window = k >= r.cmp_tiles;
        const int e = base_of(k) / PAGE_ROWS + (lane & 1), width = (int)(window ? p.oriTableWidth : p.cmpTableWidth);
        entries = k < k1 && e < width ? gptr<int32_t>(window ? p.oriTable : p.cmpTable)[(int64_t)b * width + e] : -1;
    };
    // Starts the copies of tile k and returns its rows that lie on a page.  Wave w moves rows 4 w .. 4 w + 3 of every
    // sixteen, two an instruction, so that a lane's place in a row (the swizzle goes by the row modulo 16) is the same
    // for all sixteens, and differs by one bit between the pairs.
    auto copy_tile = [&](int k) -> uint64_t {
        const int at = 2 * (k & 31);
        const bool window = k >= r.cmp_tiles;
        const uint64_t pool = window ? p.ori : p.cmp, stride = window ? p.oriStride : p.cmpStride;
        const uint32_t pages = window ? p.oriPages : p.cmpPages;
        const int lx = again(lane);
        const uint32_t lane_offset =
            (uint32_t)((4 * wave + (lx >> 5)) * D + (((lx & 31) ^ (4 * wave + (lx >> 5))) << 4));
        const uint32_t to = (uint32_t)(uintptr_t)s.tile[k & 1] + 4 * wave * D;
        uint64_t rows_there = 0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int page = __builtin_amdgcn_readlane(entries, at + half);
            if ((uint32_t)page >= pages) continue;
            rows_there |= 0xffffffffull << (32 * half);
            const uint64_t from = pool + (uint64_t)page * stride;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t lds = (uint32_t)uni((int)(to + (32 * half + 16 * i) * D));
                lds_dma16(from + 16 * i * D, lane_offset, lds);
                lds_dma16(from + 16 * i * D, (lane_offset ^ 32u) + 2 * D, lds + 2 * D);
            }
        }
        return rows_there;
    };

    // ---- Q, scales and parents; the first tile is on its way while Q is encoded ----
    const int row = 16 * (wave % RT) + n;              // the lane's row in Q K
    const int key0 = wave / RT * 16 * RT;              // the wave's first key there
    auto q_at = [&](int j) {                           // its channels 64 j + 16 g on; rows past the unit's take the first's
        const int lx = again(lane), at = 16 * (wave % RT) + (lx & 15);
        return gptr<u32x4>(p.q + (uint64_t)(out0 + (at < rows ? at : 0)) * (D * 2)) + 2 * (lx >> 4) + 8 * j;
    };
    const int token0 = row0 / heads, tokens = (row0 + rows - 1) / heads - token0 + 1;
    const float softmax2 = p.softmaxScale * LOG2E;
    const bool has_cmp = k0 < r.cmp_tiles && k0 < k1, has_ori = k1 > r.cmp_tiles;
    const bool walks = has_ori || (CAUSAL && r.shared != r.compressed);
    // The waves of a row tile encode a share of its channels each (64 j .. 64 j + 63, j from j0 on) and pass the codes
    // round in the tile buffer that is free.
    constexpr bool SHARE = PARTS > 1;
    constexpr int AT_ONCE = KEYS * D / (RT * 8 * 64 * 16) > 0 ? KEYS * D / (RT * 8 * 64 * 16) : 1;   // terms that the buffer holds
    constexpr int JN = SHARE ? 8 / PARTS : 8;
    const int j0 = SHARE ? wave / RT * JN : 0;
    auto load_scales = [&]() {
        for (int i = RT == 4 ? again(tid) : tid; i < D / 4; i += THREADS) {
            if (has_cmp) reinterpret_cast<f32x4 *>(s.scale[0])[i] = gptr<f32x4>(p.cmpScale)[i];
            if (has_ori) reinterpret_cast<f32x4 *>(s.scale[1])[i] = gptr<f32x4>(p.oriScale)[i];
        }
    };
    auto kept = [](float peak) { return peak == peak ? peak : INFINITY; };   // from here on infinity stands for both
    auto row_peak = [&](float mine_peak) {             // over the waves of the row tile
        if (!SHARE) return mine_peak;
        if (g == 0) s.peak[wave / RT][row] = mine_peak;
        lds_barrier();
        float peak = s.peak[0][row];
#pragma unroll
        for (int part = 1; part < PARTS; ++part) peak = fmaxf(peak, s.peak[part][row]);
        lds_barrier();
        return peak;
    };
    Codes<TERMS> q = {};
    auto stage_at = [&](int8_t *stage, int t, int j) { return stage + ((((wave % RT) * AT_ONCE + t) * 8 + j) * 64 + lane) * 16; };
    // Codes of eight of the wave's channels; `own` are the wave's shares, j from j0 on.
    v4i own[SHARE ? TERMS : 1][SHARE ? JN : 1];
    auto put = [&](int j, int h, const Products &x) {
        uint32_t out[TERMS][2];
        q.make(out, x);
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
            v4i &to = SHARE ? own[SHARE ? t : 0][SHARE ? j : 0] : q.term[t][j];
            to[2 * h] = (int)out[t][0], to[2 * h + 1] = (int)out[t][1];
        }
    };
    // Every wave of a row tile gets all codes, some terms at a time through the staging buffer.
    auto take = [&](int8_t *stage) {
        if (!SHARE) return;
#pragma unroll
        for (int t0 = 0; t0 < TERMS; t0 += AT_ONCE) {
            if (t0) lds_barrier();
#pragma unroll
            for (int t = t0; t < TERMS && t < t0 + AT_ONCE; ++t)
#pragma unroll
                for (int j = 0; j < JN; ++j) *reinterpret_cast<v4i *>(stage_at(stage, t - t0, j0 + j)) = own[SHARE ? t : 0][SHARE ? j : 0];
            lds_barrier();
#pragma unroll
            for (int t = t0; t < TERMS && t < t0 + AT_ONCE; ++t)
#pragma unroll
                for (int j = 0; j < 8; ++j) q.term[t][j] = *reinterpret_cast<const v4i *>(stage_at(stage, t - t0, j));
        }
    };
    uint64_t seen = 0, next_seen = 0;
    float ori_peak = 0.0f;
    if (k0 < k1) {
        u32x4 raw[JN][2];
#pragma unroll
        for (int j = 0; j < JN; ++j) raw[j][0] = q_at(j0 + j)[0], raw[j][1] = q_at(j0 + j)[1];
        read_entries(k0 >> 5);
        load_scales();
        if (tid < ROWS) s.token[tid] = (uint8_t)((row0 + min(tid, rows - 1)) / heads - token0);
        if (walks)
            for (int i = tid; i < min(r.nodes, PARENTS); i += THREADS) {
                const int up = gptr<int32_t>(p.parents)[r.first + i];
                s.parent[i] = (uint16_t)(up >= 0 && up < i ? up : ROOT);
            }
        // The copies come last: a wait for an earlier load does not wait for them.
#pragma unroll
        for (int j = 0; j < JN; ++j) asm volatile("" : "+v"(raw[j][0]), "+v"(raw[j][1]));
        next_seen = copy_tile(k0);
        lds_barrier();
        const float *scale = s.scale[has_cmp ? 0 : 1] + 64 * j0 + 16 * g;
        int8_t *stage = s.tile[(k0 + 1) & 1];
        constexpr bool KEEP = JN <= 4;                 // few enough products to hold them
        Products x[KEEP ? JN : 1][2];
        float first_peak = 0.0f, second_peak = 0.0f;   // maxima that keep a NaN
#pragma unroll
        for (int j = 0; j < JN; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Products &at = x[KEEP ? j : 0][h];
                at = products(raw[j][h], scale + 64 * j + 8 * h);
#pragma unroll
                for (int e = 0; e < 8; ++e) first_peak = __builtin_elementwise_maximum(first_peak, fabsf(at.x[e]));
                if (!KEEP) __builtin_amdgcn_sched_barrier(0);
            }
        if (has_cmp && has_ori)
#pragma unroll
            for (int j = 0; j < JN; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Products at = products(raw[j][h], s.scale[1] + 64 * (j0 + j) + 16 * g + 8 * h);
#pragma unroll
                    for (int e = 0; e < 8; ++e) second_peak = __builtin_elementwise_maximum(second_peak, fabsf(at.x[e]));
                    if (!KEEP) __builtin_amdgcn_sched_barrier(0);
                }
        first_peak = row_peak(row_max(kept(first_peak)));
        if (has_cmp && has_ori) ori_peak = row_peak(row_max(kept(second_peak)));
        q.set(first_peak, softmax2);
#pragma unroll
        for (int j = 0; j < JN; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!KEEP) {
                    asm volatile("" : "+v"(raw[j][h]));   // made again, not held
                    x[0][h] = products(raw[j][h], scale + 64 * j + 8 * h);
                }
                put(j, h, x[KEEP ? j : 0][h]);
                if (!KEEP) __builtin_amdgcn_sched_barrier(0);
            }
        take(stage);
    }
    auto parent_of = [&](int node) {
        if (r.nodes <= PARENTS) {
            const int up = s.parent[node];
            return up == ROOT ? -1 : up;
        }
        const int up = gptr<int32_t>(p.parents)[r.first + node];
        return up >= 0 && up < node ? up : -1;
    };
    // Thread t < tokens walks token t's chain, and says which of an original tile's rows the token sees.
    if ((CAUSAL || has_ori) && tid < tokens) {
        int depth = 0;
        if (walks)
            for (int a = parent_of(token0 + tid); a >= 0; a = parent_of(a)) ++depth;
        s.walk[tid] = token0 + tid, s.steps[tid] = 0, s.depth[tid] = depth;
        if (CAUSAL) s.compressed[tid] = min(r.compressed, (r.committed + depth + 1) / (int)p.ratio);
    }
    // Original tiles of committed rows that the deepest token's window still holds need no masks, nor do compressed ones
    // whose rows all tokens see.
    const int plain_from = max(0, r.committed + r.nodes - (int)min(p.window, 0x7fffffffu));
    auto is_plain = [&](int k) {
        const int base = base_of(k);
        if (k < r.cmp_tiles) return !CAUSAL || base + KEYS <= r.shared;
        return base >= plain_from && base + KEYS <= r.committed;
    };
    auto make_mask = [&](int k, uint64_t rows_there) {
        const int at = tid;
        if (is_plain(k) || at >= tokens) return;
        const int base = base_of(k);
        if (CAUSAL && k < r.cmp_tiles) {
            const int left = s.compressed[at] - base;
            s.mask[at] = left > 0 ? (~0ull >> (KEYS - min(left, KEYS))) & rows_there : 0;
            return;
        }
        // Committed rows (C + depth - window, C), then the ancestors.
        const int from = max(0, max(0, r.committed + s.depth[at] + 1 - (int)min(p.window, 0x7fffffffu)) - base);
        const int to = min(KEYS, r.committed - base);
        uint64_t bits = 0;
        if (from < to) bits = (~0ull >> (KEYS - to)) & (~0ull << from);
        if (r.committed + r.nodes > base) {
            int walk = s.walk[at], steps = s.steps[at];
            for (; walk >= 0 && r.committed + walk >= base && (uint32_t)steps < p.window; walk = parent_of(walk), ++steps)
                if (r.committed + walk < base + KEYS) bits |= 1ull << (r.committed + walk - base);
            s.walk[at] = walk, s.steps[at] = steps;
        }
        s.mask[at] = bits & rows_there;
    };
    if (k0 < k1) make_mask(k0, next_seen);

    f32x4 acc[8][RT] = {};
    float m = -INFINITY, sum = 0.0f;
#pragma nounroll
    for (int k = k0; k < k1; ++k) {
        const bool window = k >= r.cmp_tiles;
        seen = next_seen;
        vm_wait_all();
        lds_barrier();                                 // tile k is there; nobody uses tile k - 1 or its weights any more
        if (window && k == r.cmp_tiles && k > k0) {
            // From the compressed rows' channel scales to the original ones'.
            u32x4 raw[JN][2];                          // in the registers of the compressed kind's codes
#pragma unroll
            for (int j = 0; j < JN; ++j) raw[j][0] = q_at(j0 + j)[0], raw[j][1] = q_at(j0 + j)[1];
            load_scales();
            lds_barrier();
#pragma unroll
            for (int ct = 0; ct < 8; ++ct) {
                const int at = 128 * wave + 16 * ct + 4 * (again(lane) >> 4);
                const f32x4 cmp = *reinterpret_cast<const f32x4 *>(s.scale[0] + at);
                const f32x4 ratio = cmp / joint_scale(cmp, *reinterpret_cast<const f32x4 *>(s.scale[1] + at));
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[ct][rt] *= ratio;
                __builtin_amdgcn_sched_barrier(0);
            }
            q.set(ori_peak, softmax2);
            int8_t *stage = s.tile[(k + 1) & 1];
#pragma unroll
            for (int j = 0; j < JN; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    put(j, h, products(raw[j][h], s.scale[1] + 64 * (j0 + j) + 16 * (again(lane) >> 4) + 8 * h));
                __builtin_amdgcn_sched_barrier(0);
            }
            take(stage);
            lds_barrier();
        }
        if (k + 1 < k1) {
            if (!((k + 1) & 31)) read_entries((k + 1) >> 5);
            next_seen = copy_tile(k + 1);
        }
        const int lx = again(lane), its_row = 16 * (wave % RT) + (lx & 15);
        const uint32_t tile = (uint32_t)(uintptr_t)s.tile[k & 1];

        // S = Q K^T: query row n, keys key0 + 16 kt + 4 g + i.
        const bool plain = is_plain(k);
        if (!CAUSAL && !window) {
            const int left = r.compressed - k * KEYS;
            if (left < KEYS) seen &= (1ull << left) - 1;
        }
        float w[RT][4];
        {
            const uint32_t at = tile + (uint32_t)((key0 + (lx & 15)) * D + (((lx >> 4) ^ (lx & 15)) << 4));
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
            v4i dots[TERMS][PAIR];
            // Matrix instructions before the other work-group's vector ones, here and in P V (16 requests of 24 nodes and
            // 64 heads, and 4 of 61 over 32 K rows: 80.6 and 236 us, 83.7 and 252 without).
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                if (st + 2 < STEPS) fetch(st + 2);
                const int j = st & 7;
#pragma unroll
                for (int kt = 0; kt < PAIR; ++kt)
#pragma unroll
                    for (int t = 0; t < TERMS; ++t)
                        dots[t][kt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(key[st % AHEAD][kt], q.term[t][j],
                                                                            j ? dots[t][kt] : v4i{0, 0, 0, 0}, 0, 0, 0);
                if (j == 7)
#pragma unroll
                    for (int kt = 0; kt < PAIR; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            // At most 512 * 32512 * 128 + 512 * 128 * 128: within 32 bits.
                            float x = (float)(dots[0][kt][i] * 256 + dots[1][kt][i]);
                            if (TERMS == 3) x = __builtin_fmaf(x, 256.0f, (float)dots[TERMS - 1][kt][i]);
                            w[PAIR * (st >> 3) + kt][i] = x;
                        }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if (!plain || seen != ~0ull) {
            const uint64_t its = plain ? seen : s.mask[s.token[its_row]];
#pragma unroll
            for (int kt = 0; kt < RT; ++kt) {
                const uint32_t bits = (uint32_t)(its >> (key0 + 16 * kt + 4 * (lx >> 4))) & 15u;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[kt][i] = bits >> i & 1 ? w[kt][i] : -INFINITY;
            }
        }
        float peak = -INFINITY;                        // scores are no NaN: units, or -infinity
#pragma unroll
        for (int kt = 0; kt < RT; ++kt)
#pragma unroll
            for (int i = 0; i < 4; i += 2) peak = __builtin_elementwise_maxnum(__builtin_elementwise_maxnum(peak, w[kt][i]), w[kt][i + 1]);
        peak = row_max(peak);
        if (PARTS > 1) {                               // the row's keys are spread over waves
            if (lx < 16) s.peak[wave / RT][its_row] = peak;
            lds_barrier();
#pragma unroll
            for (int part = 0; part < PARTS; ++part) peak = fmaxf(peak, s.peak[part][its_row]);
        }
        peak *= q.step;
        float factor = 1.0f;
        const bool move = peak > m + LIMIT;            // and where m is still -infinity
        if (move) {
            factor = __builtin_amdgcn_exp2f(m - (peak - HEAD));
            m = peak - HEAD;
            sum *= factor;
        }
        const bool any = __ballot(move) != 0;
        if (wave < RT) {
            if (lx == 0) s.moved[wave] = any;
            if (any && lx < 16) s.factor[its_row] = factor;
        }
        {
            // Weights 2^(x step - m): 0 for masked keys, also where all have been masked so far.
            const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int kt = 0; kt < RT; ++kt) {
                f16x4 half;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(w[kt][i], q.step, -from));
                    if (TERMS == 3) sum += x;          // the log-sum-exp's sum is of the weights before rounding
                    half[i] = (_Float16)x;
                }
                if (TERMS == 2) {                      // the output's, of the weights as P V takes them
                    const f16x2 ones = {(_Float16)1.0f, (_Float16)1.0f};
                    sum = __builtin_amdgcn_fdot2(f16x2{half[0], half[1]}, ones, sum, false);
                    sum = __builtin_amdgcn_fdot2(f16x2{half[2], half[3]}, ones, sum, false);
                }
                *reinterpret_cast<f16x4 *>(s.p + its_row * P_STRIDE + key0 + 16 * kt + 4 * (lx >> 4)) = half;
            }
        }
        lds_barrier();
        if (k + 1 < k1) make_mask(k + 1, next_seen);

        // acc[ct][rt]: channels 128 wave + 16 ct + 4 g + i, row 16 rt + n.
        {
            const int lx = again(lane);
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
            value[0] = to_f16(code[0]);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int st = 0; st < 16; ++st) {
                if (st == 8)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) weight[rt] = *reinterpret_cast<const f16x8 *>(its + 16 * rt * P_STRIDE + 32);
                if (st + AHEAD < 16) fetch(st + AHEAD);
                if (st + 1 < 16) value[(st + 1) & 1] = to_f16(code[(st + 1) % AHEAD]);
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
    if (g == 0) {
        s.sum[wave / RT][row] = sum;
        if (wave < RT) s.top[row] = m;
    }
    lds_barrier();
    auto row_sum = [&](int at) {
        float total = s.sum[0][at];
#pragma unroll
        for (int part = 1; part < PARTS; ++part) total += s.sum[part][at];
        return total;
    };
    // Values from code units.
    {
        const uint64_t scales = has_cmp && !has_ori ? p.cmpScale : p.oriScale;
#pragma unroll
        for (int ct = 0; ct < 8; ++ct) {
            f32x4 scale = gptr<f32x4>(scales)[(128 * wave + 16 * ct + 4 * g) / 4];
            if (has_cmp && has_ori) scale = joint_scale(gptr<f32x4>(p.cmpScale)[(128 * wave + 16 * ct + 4 * g) / 4], scale);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[ct][rt] *= scale;
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    float top[RT], total[RT];
    if (splits == 1) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) top[rt] = s.top[16 * rt + n], total[rt] = row_sum(16 * rt + n);
    } else {
        // ---- states of the unit's items, joined by the last of them to finish ----
        // Every store has completed (at the point where all XCDs see it) before the ticket is taken, and the states
        // are added in the items' order, whichever is last.
        const uint64_t first_item = (uint64_t)(item - part_no);
        const bool near = (split & XCD_LOCAL) && (item - part_no) / share == (item - part_no + splits - 1) / share;
        auto exchange = [&](auto policy_c) {
            constexpr int POLICY = decltype(policy_c)::value;
            {
                const auto to = state_at(p.partial, (uint64_t)item, RT);
#pragma unroll
                for (int ct = 0; ct < 8; ++ct)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[ct][rt]), to,
                                                               ((ct * RT + rt) * THREADS + tid) * 16, 0, POLICY);
                if (tid < ROWS) {
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s.top[tid]), to, (ROWS * D + tid) * 4, 0, POLICY);
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(row_sum(tid)), to, (ROWS * (D + 1) + tid) * 4, 0,
                                                          POLICY);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            auto *ticket = gout<uint32_t>(p.workspace) + unit0 + unit;
            if (tid == 0) s.found[6] = (int)__hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (s.found[6] != splits - 1) return false;
            if (tid == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
            auto statistic = [&](int part, int rt, int which) {
                return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                    state_at(p.partial, first_item + (uint64_t)part, RT), (ROWS * (D + which) + 16 * rt + n) * 4, 0, POLICY));
            };
            // One pass, some channels and several states at a time: as many loads in flight as there are registers for.
            constexpr int GROUP = RT == 4 ? 1 : 4 / RT, HALF = 8 / RT;
#pragma unroll
            for (int c0 = 0; c0 < 8; c0 += HALF) {
                float high[RT], whole[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    high[rt] = -INFINITY, whole[rt] = 0.0f;
#pragma unroll
                    for (int ct = 0; ct < HALF; ++ct) acc[c0 + ct][rt] = f32x4{0, 0, 0, 0};
                }
#pragma nounroll
                for (int part = 0; part < splits; part += GROUP) {
                    float its[GROUP][RT], its_sum[GROUP][RT];
                    f32x4 v[GROUP][HALF][RT];
#pragma unroll
                    for (int u = 0; u < GROUP; ++u) {
                        const int at = min(part + u, splits - 1);
                        const auto from = state_at(p.partial, first_item + (uint64_t)at, RT);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) its[u][rt] = statistic(at, rt, 0), its_sum[u][rt] = statistic(at, rt, 1);
#pragma unroll
                        for (int ct = 0; ct < HALF; ++ct)
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt)
                                v[u][ct][rt] = __builtin_bit_cast(
                                    f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                               from, (((c0 + ct) * RT + rt) * THREADS + tid) * 16, 0, POLICY));
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        float most = high[rt];
#pragma unroll
                        for (int u = 0; u < GROUP; ++u) most = fmaxf(most, its[u][rt]);
                        const float from = most == -INFINITY ? 0.0f : most, keep = __builtin_amdgcn_exp2f(high[rt] - from);
                        whole[rt] *= keep;
#pragma unroll
                        for (int ct = 0; ct < HALF; ++ct) acc[c0 + ct][rt] *= keep;
#pragma unroll
                        for (int u = 0; u < GROUP; ++u) {
                            if (part + u >= splits) continue;
                            const float f = __builtin_amdgcn_exp2f(its[u][rt] - from);
                            whole[rt] += its_sum[u][rt] * f;
#pragma unroll
                            for (int ct = 0; ct < HALF; ++ct) acc[c0 + ct][rt] += v[u][ct][rt] * f;
                        }
                        high[rt] = most;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) top[rt] = high[rt], total[rt] = whole[rt];
            }
            return true;
        };
        if (!(near ? exchange(std::integral_constant<int, SC0>{}) : exchange(std::integral_constant<int, SC1>{}))) return;
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int at = 16 * rt + n;
        if (at >= rows) continue;
        const float sink = gptr<float>(p.sinks)[(row0 + at) % heads] * LOG2E;
        const float most = top[rt], higher = fmaxf(most, sink);
        // Where both are -infinity no key was seen and there is no sink; an infinite sink takes everything.
        const float share = most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(most - higher);
        const float rest = sink == higher ? (higher == -INFINITY ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(sink - higher);
        const float whole = total[rt] * share + rest;
        const float give = share == 0.0f && !(whole != whole) ? 0.0f : share / whole;
#pragma unroll
        for (int ct = 0; ct < 8; ++ct) {
            const f32x4 v = acc[ct][rt] * give;
            *gout<u32x2>(p.out + (uint64_t)(out0 + at) * (D * 2) + (128 * wave + 16 * ct + 4 * g) * 2) =
                u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
        }
        if (p.lse && wave == 0 && g == 0)
            gout<float>(p.lse)[out0 + at] = higher * LN2 + (whole == 0.0f ? 0.0f : logf(whole));
    }
}

bool rejected(const TreeAttentionArgs *a)
{
    if (!a || !a->heads || a->heads > MAX_HEADS || !a->batch || !a->window || !a->ratio) return true;
    if (!a->q || !a->ori || !a->oriScale || !a->oriTable || !a->cuQ || !a->seqLens || !a->sinks || !a->parents || !a->out)
        return true;
    if (a->ratio > 0x7fffffffu || a->causalCompressed > 1) return true;
    if (!a->oriPages || !a->oriTableWidth || (a->oriStride & 15) || a->oriStride < (uint64_t)PAGE_ROWS * D) return true;
    if ((a->q | a->ori | a->oriScale | a->out) & 15) return true;
    if (a->ratio > 1 && (!a->cmp || !a->cmpScale || !a->cmpTable || !a->cmpPages || !a->cmpTableWidth ||
                         (a->cmpStride & 15) || a->cmpStride < (uint64_t)PAGE_ROWS * D || ((a->cmp | a->cmpScale) & 15)))
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
Plan plan_of(const TreeAttentionArgs *a)
{
    Plan plan;
    const uint64_t rows = (uint64_t)a->tokens * a->heads;
    const uint64_t cmp_tiles = a->ratio > 1 ? (a->cmpTableWidth + 1) / 2 : 0;
    // Tiles that a request is likely to have: the window and trees of twice the average size, as far as the tables go.
    const uint64_t near = (uint64_t)a->window + 2 * (a->tokens / a->batch + 1) + PAGE_ROWS;
    const uint64_t ori_pages = near / PAGE_ROWS + 1 < a->oriTableWidth ? near / PAGE_ROWS + 1 : a->oriTableWidth;
    const uint64_t work = (rows + 63) / 64 * (cmp_tiles + (ori_pages + 1) / 2);
    // Units of 16 rows spread few rows over more work-groups and join smaller states, in more work-groups at once; units
    // of 64 rows read and convert a key's row for more of them.  With R tiles of 64 rows and `work` tiles of 64 rows and 64
    // keys, the better one goes by R * work (microseconds of 16, 32 and 64 rows a unit, whole contexts but for two):
    //        1 K  64 rows, 65536 keys           97, 220,  906      16 K  256 rows, 65536 keys       122, 115, 352
    //       16 K  1024 rows, 4096 keys        46.7, 46.5, 103      17 K  32 requests of 4-16 nodes  19.5, 26.1, 38.7
    //       66 K  2048 rows, 4096 keys          69, 49.5,  85      90 K  48 of 25 nodes, window     29.8, 23.3, 30.5
    //      263 K  2048 rows, 16384 keys        204, 112,  130       1 M  2048 rows, 65536 keys      749, 364, 296
    //      1.8 M  4 of 57-61 nodes, 32 K keys  609, 313,  243       3 M  16 of 24 nodes, 64 heads   152, 115, 86
    // Of 173 launches (8 to 98304 rows, windows of 128 to 262144 keys) its choice is 1 % behind the best of the three on
    // average and 23 % at worst; bounds on `work` alone, whatever units share it, are 21 % behind, and 7 times at worst.
    // Measured without the log-sum-exp.  With it units of 64 rows hold one work-group a CU, and units of 32 are faster where
    // they are chosen too (the last two: 326 against 429, and 122 against 155): still chosen, as for the output alone, since
    // the scratch is the same for both.
    const uint64_t score = (rows + 63) / 64 * work;
    plan.rt = score < 28000 ? 1 : score < 400000 ? 2 : 4;
    // A request's last unit may be short, and so may the padding's.
    plan.units = (uint32_t)(rows / (16 * plan.rt)) + a->batch + 1;
    const uint64_t tiles = cmp_tiles + (a->oriTableWidth + 1) / 2;
    const uint32_t most = items_for(plan.rt);
    plan.split = plan.units <= most * 3 / 8 && tiles > 1 && plan.units * tiles <= MAX_SPLIT_WORK;
    const uint64_t items = plan.split ? plan.units * tiles : plan.units;
    plan.grid = (uint32_t)((plan.split && items > most ? most : items) + 7) & ~7u;
    return plan;
}

}  // namespace

extern "C" {

int launch_sharedkv_tree(void *stream, const TreeAttentionArgs *a)
{
    if (rejected(a)) return (int)hipErrorInvalidValue;
    if (!a->tokens) return (int)hipSuccess;
    const Plan plan = plan_of(a);
    if (plan.grid > MAX_GROUPS) return (int)hipErrorInvalidValue;
    if (plan.split && (!a->workspace || !a->partial || ((a->workspace | a->partial) & 15))) return (int)hipErrorInvalidValue;
    const auto of_rows = [&](auto terms, auto causal) {
        return plan.rt == 4   ? &tree_attention<terms.value, 4, causal.value>
               : plan.rt == 2 ? &tree_attention<terms.value, 2, causal.value>
                              : &tree_attention<terms.value, 1, causal.value>;
    };
    const auto of_terms = [&](auto causal) {
        return a->lse ? of_rows(std::integral_constant<int, 3>{}, causal) : of_rows(std::integral_constant<int, 2>{}, causal);
    };
    const auto kernel = a->ratio > 1 && a->causalCompressed ? of_terms(std::true_type{}) : of_terms(std::false_type{});
    const bool local = plan.split && sharedkv::xcd_local(static_cast<hipStream_t>(stream));
    hipLaunchKernelGGL(kernel, dim3(plan.grid), dim3(THREADS), 0, static_cast<hipStream_t>(stream), a->cuQ, a->seqLens,
                       a->batch, a->heads, (plan.split ? plan.units : 0u) | (local ? XCD_LOCAL : 0u), a->tokens, a->ratio,
                       a->window, a->oriTableWidth, a->ratio > 1 ? a->cmpTableWidth : 0u, *a);
    return (int)hipGetLastError();
}

int sharedkv_tree_scratch(const TreeAttentionArgs *a, uint64_t *workspace, uint64_t *partial)
{
    if (!workspace || !partial || rejected(a)) return (int)hipErrorInvalidValue;
    const Plan plan = plan_of(a);
    if (plan.grid > MAX_GROUPS) return (int)hipErrorInvalidValue;
    *workspace = plan.split ? plan.units * 4ull : 0;
    *partial = plan.split ? plan.grid * state_floats(plan.rt) * 4 : 0;
    return (int)hipSuccess;
}

uint32_t sharedkv_tree_args_size(void) { return (uint32_t)sizeof(TreeAttentionArgs); }

}  // extern "C"
