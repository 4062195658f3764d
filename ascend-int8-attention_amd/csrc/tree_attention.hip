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
// A unit is 64 query rows of one request (a row is a token and a head, heads
// innermost), which share every key tile of 64 rows (two pages).  Four waves:
// for Q K each has sixteen of the rows, for P V each has 128 of the channels,
// the weights passing between them in LDS.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sharedkv_hip.h"

namespace {

constexpr int D = 512;
constexpr int ROWS = 64;           // query rows of a unit
constexpr int KEYS = 64;           // keys of a tile: two pages
constexpr int PAGE_ROWS = 32;
constexpr int THREADS = 256;
constexpr int WAVES = THREADS / 64;
constexpr int P_STRIDE = KEYS + 8; // halves; 144 bytes keep the 16-byte reads of 16 rows on different banks
constexpr int PARENTS = 1024;      // parents kept in LDS; larger trees read theirs from memory
constexpr uint32_t MAX_HEADS = 128;
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.69314718055994531f;
// Weights are 2^(s - m) with m the row's maximum less HEAD when it was last
// set, so they start at 2^HEAD and m moves only when a score passes it by
// LIMIT: 2^15 is below FP16's largest, and weights down to 2^-22 of the
// largest stay normal.
constexpr float HEAD = 8.0f, LIMIT = 15.0f;

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
typedef __attribute__((address_space(3))) v2i lds_v2i;

template <typename T>
__device__ __forceinline__ const __attribute__((address_space(1))) T *gptr(uint64_t a)
{
    return reinterpret_cast<const __attribute__((address_space(1))) T *>(a);
}
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}

struct alignas(16) Shared {
    int8_t tile[KEYS * D];             // key rows, their 16-byte chunks XOR-swizzled with the row
    _Float16 p[ROWS * P_STRIDE];       // weights [row][key]
    uint64_t mask[ROWS];               // the tile's keys that each of the unit's tokens sees
    float factor[ROWS], top[ROWS], sum[ROWS];
    int32_t moved[WAVES];              // whether a wave's rows moved their maximum in this tile
    int32_t scan[WAVES];
    int32_t found[2];
    int32_t parent[PARENTS];
};

// A request's rows of the launch, made safe: nothing below reads past the
// arrays whatever cuQ and seqLens hold.
struct Request {
    int32_t first, nodes, committed;   // first token, drafted tokens, committed rows
    bool live;
    int32_t compressed;                // visible compressed rows
    int32_t low, end;                  // original rows [low, end), low a multiple of PAGE_ROWS
    int32_t cmp_tiles, ori_tiles;
};

__device__ __forceinline__ Request request_of(const TreeAttentionArgs &p, int c0, int c1, int length)
{
    Request r;
    const int tokens = (int)p.tokens;
    r.first = min(max(c0, 0), tokens);
    r.nodes = min(max(c1, r.first), tokens) - r.first;
    r.live = length > 0 && r.nodes > 0;
    r.committed = max(0, length - r.nodes);
    const int64_t ori_rows = (int64_t)p.oriTableWidth * PAGE_ROWS, cmp_rows = (int64_t)p.cmpTableWidth * PAGE_ROWS;
    r.compressed = p.ratio > 1 ? (int)min((int64_t)(r.committed / (int)p.ratio), cmp_rows) : 0;
    r.low = max(0, r.committed - (int)min(p.window, 0x7fffffffu) + 1) & ~(PAGE_ROWS - 1);
    r.end = (int)min((int64_t)r.committed + r.nodes, ori_rows);
    r.cmp_tiles = r.live ? (r.compressed + KEYS - 1) / KEYS : 0;
    r.ori_tiles = r.live ? max(0, r.end - r.low + KEYS - 1) / KEYS : 0;
    return r;
}

template <int TERMS>
struct Codes {
    v4i term[TERMS][8];                // most significant first; channels 64 j + 16 g .. + 15 of row n
    float step;                        // score (base 2) of one unit
};

// q * scale of the lane's row as whole numbers of 8 * TERMS bits.
template <int TERMS>
__device__ __forceinline__ void encode(Codes<TERMS> &c, uint64_t q_row, uint64_t scale, int g, float softmax2)
{
    asm volatile("" : "+v"(g));        // keeps the addresses below from being held in registers across tiles
    constexpr float LARGEST = TERMS == 2 ? 127.0f * 256.0f : 127.0f * 65536.0f;
    float peak = 0.0f;
    bool odd = false;                  // an infinity or NaN
    const auto *qp = gptr<u32x4>(q_row);
    const auto *sp = gptr<f32x4>(scale);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const u32x4 w = qp[(64 * j + 16 * g + 8 * half) / 8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float s = sp[(64 * j + 16 * g + 8 * half) / 4 + e / 4][e & 3];
                const float x = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16) * s;
                peak = fmaxf(peak, fabsf(x));
                odd |= !(fabsf(x) < INFINITY);
            }
        }
        __builtin_amdgcn_sched_barrier(0);   // a few loads at a time: registers are short here
    }
    peak = fmaxf(peak, __shfl_xor(peak, 16));
    peak = fmaxf(peak, __shfl_xor(peak, 32));
    const uint64_t any = __ballot(odd);
    const int n = threadIdx.x & 15;
    const bool bad = ((any >> n) | (any >> (n + 16)) | (any >> (n + 32)) | (any >> (n + 48))) & 1;
    // Rows below 2^-90 score zero to FP32 against any code; their inverse would overflow.
    asm volatile("" : "+v"(g));
    const float inverse = peak > 0x1p-90f ? LARGEST / peak : 0.0f;
    c.step = bad ? __builtin_nanf("") : peak > 0x1p-90f ? peak / LARGEST * softmax2 : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const u32x4 w = qp[(64 * j + 16 * g + 8 * half) / 8];
#pragma unroll
            for (int word = 0; word < 2; ++word) {
                uint32_t packed[TERMS] = {};
#pragma unroll
                for (int e = 4 * word; e < 4 * word + 4; ++e) {
                    const float s = sp[(64 * j + 16 * g + 8 * half) / 4 + e / 4][e & 3];
                    const float x = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16) * s;
                    const float y = fminf(fmaxf(x * inverse, -LARGEST), LARGEST);
                    int v = bad ? 0 : (int)__builtin_rintf(y);
#pragma unroll
                    for (int t = TERMS - 1; t >= 0; --t) {
                        const int low = t ? (int)(int8_t)v : v;
                        packed[t] |= (uint32_t)(low & 255) << (8 * (e & 3));
                        v = (v - low) >> 8;
                    }
                }
#pragma unroll
                for (int t = 0; t < TERMS; ++t) c.term[t][j][2 * half + word] = (int)packed[t];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
}

// Eight codes to FP16, exactly: 1024 + (code + 128) has the byte as its low
// mantissa bits.
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

// Inclusive sum over the work-group; `total` gets the whole.
__device__ __forceinline__ int block_scan(Shared &s, int v, int &total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const int other = __shfl_up(v, step);
        if (lane >= step) v += other;
    }
    __syncthreads();
    if (lane == 63) s.scan[wave] = v;
    __syncthreads();
    total = 0;
    int before = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) before += s.scan[w];
        total += s.scan[w];
    }
    return v + before;
}

template <int TERMS>
__global__ void __launch_bounds__(THREADS, TERMS == 2 ? 2 : 1) tree_attention(const TreeAttentionArgs p)
{
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), g = lane >> 4, n = lane & 15;
    const int heads = (int)p.heads, batch = (int)p.batch;
    const auto *cu = gptr<int32_t>(p.cuQ), *lens = gptr<int32_t>(p.seqLens);

    // The unit of this work-group: units of the requests in order, then the
    // rows of graph padding behind the last request.
    int unit = (int)blockIdx.x, b = -1;
    {
        int done = 0;
        if (tid < 2) s.found[tid] = -1;
        for (int at = 0; at < batch && unit >= done; at += THREADS) {
            const int mine = at + tid;
            int units = 0;
            if (mine < batch) units = (request_of(p, cu[mine], cu[mine + 1], 1).nodes * heads + ROWS - 1) / ROWS;
            int total;
            const int upto = block_scan(s, units, total) + done;
            if (unit < upto && unit >= upto - units) s.found[0] = mine, s.found[1] = unit - (upto - units);
            done += total;
            __syncthreads();
        }
        __syncthreads();
        b = s.found[0];
        if (b >= 0) unit = s.found[1];
        else unit -= done;
    }
    const int all_rows = (int)p.tokens * heads;
    auto zero_rows = [&](int first, int count) {
        for (int i = tid; i < count * (D / 8); i += THREADS)
            reinterpret_cast<u32x4 *>(p.out)[(int64_t)first * (D / 8) + i] = u32x4{0, 0, 0, 0};
        if (p.lse)
            for (int i = tid; i < count; i += THREADS) reinterpret_cast<float *>(p.lse)[first + i] = 0.0f;
    };
    if (b < 0) {
        const int live = min(max(cu[batch], 0), (int)p.tokens) * heads;
        const int64_t first = (int64_t)live + (int64_t)unit * ROWS;
        if (first < all_rows) zero_rows((int)first, (int)min((int64_t)ROWS, all_rows - first));
        return;
    }
    const Request r = request_of(p, cu[b], cu[b + 1], lens[b]);
    const int row0 = unit * ROWS;                      // of the request
    const int rows = min(ROWS, r.nodes * heads - row0);
    const int64_t out0 = (int64_t)r.first * heads + row0;
    if (!r.live) {
        zero_rows((int)out0, rows);
        return;
    }

    // Tokens of the unit: thread t < tokens walks token t's chain.
    const int token0 = row0 / heads, tokens = (row0 + rows - 1) / heads - token0 + 1;
    for (int i = tid; i < min(r.nodes, PARENTS); i += THREADS) s.parent[i] = gptr<int32_t>(p.parents)[r.first + i];
    __syncthreads();
    auto parent_of = [&](int node) {
        const int up = r.nodes <= PARENTS ? s.parent[node] : gptr<int32_t>(p.parents)[r.first + node];
        return up >= 0 && up < node ? up : -1;
    };
    int walk = -1, steps = 0, depth = 0;
    if (tid < tokens) {
        walk = token0 + tid;
        for (int a = parent_of(walk); a >= 0; a = parent_of(a)) ++depth;
    }

    const int row = 16 * wave + n;                     // the lane's row in Q K
    const bool there = row < rows;
    const int token = there ? (row0 + row) / heads - token0 : 0;
    const uint64_t q_row = p.q + (uint64_t)(out0 + (there ? row : 0)) * (D * 2);
    const float softmax2 = p.softmaxScale * LOG2E;

    Codes<TERMS> q;
    f32x4 acc[8][4] = {};
    float m = -INFINITY, sum = 0.0f;
    const int tiles = r.cmp_tiles + r.ori_tiles;
    auto run_tile = [&](int k, const bool window) {
        // Original tiles run from the last to the first: the walks go from a token up.
        const int base = window ? r.low + (tiles - 1 - k) * KEYS : k * KEYS;
        uint64_t seen = 0;                             // the tile's rows that lie on a page of the pool
        {
            const uint64_t table = window ? p.oriTable : p.cmpTable;
            const int width = (int)(window ? p.oriTableWidth : p.cmpTableWidth);
            const uint32_t pages = window ? p.oriPages : p.cmpPages;
            const uint64_t pool = window ? p.ori : p.cmp, stride = window ? p.oriStride : p.cmpStride;
            __syncthreads();
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int e = base / PAGE_ROWS + half;
                const int page = e < width ? gptr<int32_t>(table)[(int64_t)b * width + e] : -1;
                const bool good = (uint32_t)page < pages;
                if (good) seen |= 0xffffffffull << (32 * half);
                const auto *from = gptr<v4i>(pool + (good ? (uint64_t)page : 0) * stride);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = tid + i * THREADS, slot = PAGE_ROWS * half + at / 32, chunk = at & 31;
                    *reinterpret_cast<v4i *>(s.tile + slot * D + ((chunk ^ (slot & 15)) << 4)) = from[at];
                }
            }
        }
        if (!window) {
            const int left = r.compressed - base;
            if (left < KEYS) seen &= (1ull << left) - 1;
            if (tid < ROWS) s.mask[tid] = seen;
        } else if (tid < tokens) {
            // Committed rows (C + depth - window, C), then the ancestors.
            uint64_t mine = 0;
            const int64_t from = max((int64_t)0, (int64_t)r.committed + depth - p.window + 1 - base);
            const int64_t to = min((int64_t)KEYS, (int64_t)r.committed - base);
            if (from < to) mine = (to == KEYS ? ~0ull : (1ull << to) - 1) & ~((1ull << from) - 1);
            for (; walk >= 0 && r.committed + walk >= base && (uint32_t)steps < p.window; walk = parent_of(walk), ++steps)
                if (r.committed + walk < base + KEYS) mine |= 1ull << (r.committed + walk - base);
            s.mask[tid] = mine & seen;
        }
        __syncthreads();

        // S = Q K^T: query row n, keys 16 kt + 4 g + i.
        int lx = lane;
        asm volatile("" : "+v"(lx));   // addresses from here on are made anew: registers are short
        const int gx = lx >> 4, nx = lx & 15;
        const int8_t *at = s.tile + nx * D;
        const uint64_t mask = s.mask[token];
        float w[4][4], peak = -INFINITY;
#pragma unroll
        for (int kp = 0; kp < 2; ++kp) {
            v4i dots[TERMS][2] = {};
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const v4i key =
                        *reinterpret_cast<const v4i *>(at + 16 * (2 * kp + kt) * D + (((4 * j + gx) ^ nx) << 4));
#pragma unroll
                    for (int t = 0; t < TERMS; ++t)
                        dots[t][kt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(key, q.term[t][j], dots[t][kt], 0, 0, 0);
                }
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const uint32_t bits = (uint32_t)(mask >> (16 * (2 * kp + kt) + 4 * g)) & 15u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // At most 512 * 32512 * 128 + 512 * 128 * 128: within 32 bits.
                    float x = (float)(dots[0][kt][i] * 256 + dots[1][kt][i]);
                    if (TERMS == 3) x = __builtin_fmaf(x, 256.0f, (float)dots[TERMS - 1][kt][i]);
                    w[2 * kp + kt][i] = bits >> i & 1 ? x * q.step : -INFINITY;
                    peak = fmaxf(peak, w[2 * kp + kt][i]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        peak = fmaxf(peak, __shfl_xor(peak, 16));
        peak = fmaxf(peak, __shfl_xor(peak, 32));
        float factor = 1.0f;
        const bool move = peak > m + LIMIT;            // and where m is still -infinity
        if (move) {
            factor = __builtin_amdgcn_exp2f(m - (peak - HEAD));
            m = peak - HEAD;
            sum *= factor;
        }
        const bool any = __ballot(move) != 0;
        if (lane == 0) s.moved[wave] = any;
        if (any && g == 0) s.factor[row] = factor;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            const uint32_t bits = (uint32_t)(mask >> (16 * kt + 4 * g)) & 15u;
            f16x4 half;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = bits >> i & 1 ? __builtin_amdgcn_exp2f(w[kt][i] - m) : 0.0f;
                sum += x;
                half[i] = (_Float16)x;
            }
            *reinterpret_cast<f16x4 *>(s.p + row * P_STRIDE + 16 * kt + 4 * g) = half;
        }
        __syncthreads();

        // acc[ct][rt]: channels 128 wave + 16 ct + 4 g + i, row 16 rt + n.
        if (uni(s.moved[0] | s.moved[1] | s.moved[2] | s.moved[3])) {
            f32x4 f;
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) f[rt] = s.moved[rt] ? s.factor[16 * rt + n] : 1.0f;
#pragma unroll
            for (int ct = 0; ct < 8; ++ct)
#pragma unroll
                for (int rt = 0; rt < 4; ++rt) acc[ct][rt] *= f[rt];
        }
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" : "+v"(lx));
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int gx = lx >> 4, nx = lx & 15;
            f16x8 weight[4];
#pragma unroll
            for (int rt = 0; rt < 4; ++rt)
                weight[rt] = *reinterpret_cast<const f16x8 *>(s.p + (16 * rt + nx) * P_STRIDE + 32 * kb + 8 * gx);
            const int slot = 32 * kb + 8 * gx + (nx >> 1);
            const int8_t *from = s.tile + slot * D + 8 * (nx & 1);
#pragma unroll
            for (int ct = 0; ct < 8; ++ct) {
                const v2i code = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                    (lds_v2i *)(from + (((8 * wave + ct) ^ (slot & 15)) << 4)));
                const f16x8 value = to_f16(code);
#pragma unroll
                for (int rt = 0; rt < 4; ++rt)
                    acc[ct][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value, weight[rt], acc[ct][rt], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (r.cmp_tiles) {
        encode<TERMS>(q, q_row, p.cmpScale, g, softmax2);
        for (int k = 0; k < r.cmp_tiles; ++k) run_tile(k, false);
    }
    if (r.ori_tiles) {
        encode<TERMS>(q, q_row, p.oriScale, g, softmax2);
        if (r.cmp_tiles) {
            // From the compressed rows' channel scales to the original ones'.
#pragma unroll
            for (int ct = 0; ct < 8; ++ct) {
                const int at = (128 * wave + 16 * ct + 4 * g) / 4;
                const f32x4 ratio = gptr<f32x4>(p.cmpScale)[at] / gptr<f32x4>(p.oriScale)[at];
#pragma unroll
                for (int rt = 0; rt < 4; ++rt) acc[ct][rt] *= ratio;
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        for (int k = r.cmp_tiles; k < tiles; ++k) run_tile(k, true);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (g == 0) s.top[row] = m, s.sum[row] = sum;
    __syncthreads();
    const uint64_t scales = r.ori_tiles ? p.oriScale : p.cmpScale;
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
        const int mine = 16 * rt + n;
        if (mine >= rows) continue;
        const float sink = gptr<float>(p.sinks)[(row0 + mine) % heads] * LOG2E;
        const float most = s.top[mine];
        const float top = fmaxf(most, sink);
        // Where both are -infinity no key was seen and there is no sink; an infinite sink takes everything.
        const float share = most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(most - top);
        const float rest = sink == top ? (top == -INFINITY ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(sink - top);
        const float total = s.sum[mine] * share + rest;
        const float give = share == 0.0f && !(total != total) ? 0.0f : share / total;
#pragma unroll
        for (int ct = 0; ct < 8; ++ct) {
            const int c = 128 * wave + 16 * ct + 4 * g;
            const f32x4 v = acc[ct][rt] * give * gptr<f32x4>(scales)[c / 4];
            *reinterpret_cast<u32x2 *>(p.out + (uint64_t)(out0 + mine) * (D * 2) + c * 2) =
                u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
        }
        if (p.lse && wave == 0 && g == 0)
            reinterpret_cast<float *>(p.lse)[out0 + mine] = top * LN2 + (total == 0.0f ? 0.0f : logf(total));
    }
}

bool rejected(const TreeAttentionArgs *a)
{
    if (!a || !a->heads || a->heads > MAX_HEADS || !a->batch || !a->window || !a->ratio) return true;
    if (!a->q || !a->ori || !a->oriScale || !a->oriTable || !a->cuQ || !a->seqLens || !a->sinks || !a->parents || !a->out)
        return true;
    if (!a->oriPages || !a->oriTableWidth || (a->oriStride & 15) || a->oriStride < (uint64_t)PAGE_ROWS * D) return true;
    if ((a->q | a->ori | a->oriScale | a->out) & 15) return true;
    if (a->ratio > 1 && (!a->cmp || !a->cmpScale || !a->cmpTable || !a->cmpPages || !a->cmpTableWidth ||
                         (a->cmpStride & 15) || a->cmpStride < (uint64_t)PAGE_ROWS * D || ((a->cmp | a->cmpScale) & 15)))
        return true;
    // Rows and pages are counted in 32 bits.
    return (uint64_t)a->tokens * a->heads > 0x7fff0000ull || a->oriTableWidth > 0x3ffffffu || a->cmpTableWidth > 0x3ffffffu;
}

}  // namespace

extern "C" {

int launch_sharedkv_tree(void *stream, const TreeAttentionArgs *a)
{
    if (rejected(a)) return (int)hipErrorInvalidValue;
    if (!a->tokens) return (int)hipSuccess;
    // A request's last unit may be short, and so may the padding's.
    const uint32_t units = (uint32_t)((uint64_t)a->tokens * a->heads / ROWS) + a->batch + 1;
    const auto kernel = a->lse ? &tree_attention<3> : &tree_attention<2>;
    hipLaunchKernelGGL(kernel, dim3(units), dim3(THREADS), 0, static_cast<hipStream_t>(stream), *a);
    return (int)hipGetLastError();
}

uint32_t sharedkv_tree_args_size(void) { return (uint32_t)sizeof(TreeAttentionArgs); }

}  // extern "C"
