// kv8_decode.hip — batched decode attention over the 8-bit cache (gfx950).
//
// One query row per sequence (or few, which the prefill hands over: their (row,
// head) pairs then stand in for heads).  A segment is one (sequence, kv head,
// group of up to 16 q heads); its keys are cut into tiles of 64 positions, four
// subtiles of 16, each inside one cache block and so with one K and one V
// scale.  Per tile a wavefront computes, on v_mfma_f32_16x16x32_f16,
//   S^T[16 tokens][16 heads] += K . Q^T     per subtile, K codes as binary16
//   O^T[16 dims][16 heads]   += V^T . P^T   per 16 dims, over 32 tokens a time
// Codes are exact in binary16; q and the weights p * (V scale) are two
// binary16 terms each, which keeps 22 bits, so what is lost is below the f32
// sums' own rounding.  Each takes two MFMAs for one, on a matrix unit that the
// memory leaves idle for the most part.
//
// No operand passes through LDS or between lanes.  K arrives as 16 bytes per
// lane in A's layout (row = token, 8 + 8 dims).  Row m of a subtile's A is
// token 4 (m % 4) + m / 4, so the lane group g = lane / 16 of the result holds
// tokens 4 i + g, i = 0..3: in V those are, for each i, four neighbouring rows,
// which one load per i reads whole.  V^T's A operand needs one dim and eight
// tokens per lane: the eight loads give a lane 4 (8 at head_dim 128) dims of
// its eight tokens, and two byte permutes per pair of words put two tokens'
// bytes side by side before the conversion that they need anyway.
//
// Scales: a subtile's K scale multiplies its scores (with the row's own power
// of two, that of q, and 1/sqrt(D) log2(e)).  A V scale multiplies its weights
// relative to the largest of the scales seen, times 2^14: every product is at
// most 2^14 and keeps its 22 bits down to 2^-18 of the largest.
//
// Softmax in log2 units with a running maximum; O and the sum are rescaled
// only in tiles that raise it.
//
// Split over keys: as many pieces as fill the chip, in one launch.  Batches
// lay their segments' tiles end to end and cut the list into equal ranges, one
// per workgroup, whatever the spread of the lengths; launches of few segments
// cut each by itself, which needs no sums over the batch.  Pieces of a segment
// leave their maximum, sum and O in the workspace (stored and loaded past the
// L2s, which the XCDs do not share) and the last one to arrive joins them in
// the order of the pieces, so that the order of arrival changes nothing.
//
// Bound: the cache's bytes at batch (64 sequences of 16640 tokens, 32/4 heads of
// 64: 95.5 us, 5.7 TB/s; 24 of 200-16000, 32/8 of 128: 82.5 us, 4.8 TB/s, int8 with
// capped scores 92); for single sequences the chain length -> table -> rows ->
// partials -> join (4 kv heads of 64: 128 tokens 4.5 us, 4096 9.2, 32768 15.1).
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "kv8.hpp"

namespace nyion {

constexpr int kTile = 64;            // tokens
constexpr int kMaxSeqs = 1024;       // sequences per launch
constexpr int kMaxWgs = kKv8Counters / 2;  // workgroups per launch, two partials each
constexpr int kWaves = 4;
constexpr float kWeightUnit = 16384.f;
constexpr float kLeastScale = 7.888609052210118e-31f;  // 2^-100

struct Kv8DecodeArgs {
    Kv8 c;
    ScoreArgs s;
    const int32_t* tables;
    const int32_t* ctx_lens;
    const void* q;
    void* out;
    long long q_stride;
    float* ws_acc;   // [slots][16][D]
    float2* ws_ml;   // [slots][16]
    int* counters;   // [kKv8Counters], by the slot of a segment's first piece
    int max_blocks;
    int span;        // tokens that a table covers
    int batch;
    int n_heads;
    int group;       // q heads per kv head
    int n_hg;        // groups of 16 heads, or (row, head) pairs, per kv head
    int pieces;      // > 0: each segment is cut into up to this many pieces
    int min_tiles;   // fewest tiles of a workgroup
    int slots;       // partials that the workspace holds
    int bf16;
    int n_rows;      // with several rows per sequence only
    const int32_t* row_starts;
};

// max(v, v of lane ^ 16), then ^ 32: the lanes of one head
__device__ __forceinline__ float max_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float lane_value(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

// What two f32 values have beyond their binary16 parts, as binary16: exact
// differences, each one mixed-precision FMA instead of a conversion and a
// subtraction.
__device__ __forceinline__ half2_t rest_of_pair(half2_t hi, float a, float b) {
    const uint32_t h = __builtin_bit_cast(uint32_t, hi);
    float x, y;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(x) : "v"(h), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(y) : "v"(h), "v"(b));
    return half2_t{(_Float16)x, (_Float16)y};
}

// tanh: the odd series to x^11 below 0.35 (the next term is 2e-8 of x there),
// 1 - 2 / (e^2x + 1) above, where that difference loses nothing.
__device__ __forceinline__ float tanh_series(float x) {
    const float y = x * x;
    float t = -0.00886323553f;  // -1382/155925
    t = __builtin_fmaf(t, y, 0.0218694885f);    // 62/2835
    t = __builtin_fmaf(t, y, -0.0539682540f);   // -17/315
    t = __builtin_fmaf(t, y, 0.133333333f);     // 2/15
    t = __builtin_fmaf(t, y, -0.333333333f);
    return __builtin_fmaf(t * y, x, x);
}
__device__ __forceinline__ float tanh_exp(float x) {
    return 1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * 2.885390081777927f) + 1.f);
}

template <int D>
struct Kv8Tile {
    static constexpr int KC = D / 64;  // 16-byte chunks of a K row per lane
    static constexpr int VW = D / 64;  // words of a V row per lane
    u32x4_t k[4][KC];
    uint32_t v[4][4][VW];
};

// The range of keys of a sequence and its tiles.
struct Kv8Span {
    int lo, hi;      // keys [lo, hi)
    int first;       // tile of lo
    int tiles;       // at least 1: an empty range has a tile with every key masked
};
__device__ __forceinline__ Kv8Span kv8_span(const Kv8DecodeArgs& a, int ctx) {
    Kv8Span r;
    r.hi = max(min(ctx, a.span), 0);
    r.lo = a.s.window > 0 && ctx > a.s.window ? ctx - a.s.window : 0;
    if (r.lo > r.hi) r.lo = r.hi;
    r.first = r.lo / kTile;
    r.tiles = max((int)(((unsigned)r.hi + kTile - 1) / kTile) - r.first, 1);
    return r;
}

// The same for a sequence of several rows: the keys that any of them sees.
__device__ __forceinline__ Kv8Span kv8_span(const Kv8DecodeArgs& a, const Kv8Rows& s) {
    Kv8Span r;
    r.hi = s.rows > 0 ? s.key_end(s.pos0 + s.rows - 1) : 0;
    r.lo = a.s.window > 0 ? min(max(s.pos0 - a.s.window + 1, 0), r.hi) : 0;
    r.first = r.lo / kTile;
    r.tiles = max((int)(((unsigned)r.hi + kTile - 1) / kTile) - r.first, 1);
    return r;
}

// ROWS: several rows per sequence, as few as the prefill hands over: a segment is 16
// (row, head) pairs of a kv head, numbered row-major.
template <int D, int CODE, bool MODS, bool PASSING, bool ROWS>
__global__ __launch_bounds__(64 * kWaves, 2) void kv8_decode_kernel(Kv8DecodeArgs a) {
    using Tile = Kv8Tile<D>;
    constexpr int KC = Tile::KC, VW = Tile::VW;
    constexpr int MT = D / 16;       // 16-dim tiles of O^T
    constexpr int PAD = 4;
    __shared__ float sm_acc[kWaves][16][D + PAD];
    __shared__ float2 sm_ml[kWaves][16];
    __shared__ int sm_ends[kMaxSeqs];
    __shared__ int sm_wave[kWaves];
    __shared__ struct {
        int n_pieces, slot0, slot1, b, head0, heads;
    } sm_shared[2];
    __shared__ int sm_last[2];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15;   // head of the group / row of an A operand
    const int g = lane >> 4;   // lane group
    const int units = a.c.n_kv_heads * a.n_hg;
    const auto rows_of = [&](int b) {
        return kv8_rows(a.row_starts, a.ctx_lens, a.s.prefix_lens, a.n_rows, a.span, b);
    };
    const auto span_of = [&](int b, int ctx) {
        if constexpr (ROWS)
            return kv8_span(a, rows_of(b));
        else
            return kv8_span(a, ctx);
    };

    // Where this workgroup's tiles lie: of `total` tiles each of `wgs`
    // workgroups takes total / wgs, the first total % wgs one more.
    uint32_t pos = 0, end = 0, wgs = 0, share = 0, extra = 0;
    int seq_ctx = 0, seq_end = 0;  // up to 64 sequences: lane b holds b's length, and the tiles up to and with b
    if (a.pieces == 0) {
        uint32_t total;
        if (a.batch <= 64) {
            seq_ctx = lane < a.batch ? a.ctx_lens[lane] : 0;
            seq_end = lane < a.batch ? span_of(lane, seq_ctx).tiles : 0;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int y = __shfl_up(seq_end, d);
                if (lane >= d) seq_end += y;
            }
            total = (uint32_t)__builtin_amdgcn_readlane(seq_end, 63) * units;
        } else {
            int before = 0;
            for (int b0 = 0; b0 < a.batch; b0 += 64 * kWaves) {
                const int b = b0 + tid;
                int x = b < a.batch ? span_of(b, a.ctx_lens[b]).tiles : 0;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int y = __shfl_up(x, d);
                    if (lane >= d) x += y;
                }
                if (lane == 63) sm_wave[wave] = x;
                __syncthreads();
                int all = 0;
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    if (w < wave) x += sm_wave[w];
                    all += sm_wave[w];
                }
                if (b < a.batch) sm_ends[b] = before + x;
                before += all;
                __syncthreads();
            }
            total = (uint32_t)__builtin_amdgcn_readfirstlane(before) * units;
        }
        wgs = min((uint32_t)gridDim.x, (total + a.min_tiles - 1) / a.min_tiles);
        if (blockIdx.x >= wgs) return;
        share = total / wgs;
        extra = total - share * wgs;
        pos = share * blockIdx.x + min(blockIdx.x, extra);
        end = pos + share + (blockIdx.x < extra ? 1 : 0);
    }
    bool first_segment = true;
    // the workgroup that holds tile t, and the first tile of workgroup w
    const auto holder = [&](uint32_t t) {
        const uint32_t longer = extra * (share + 1);
        return t < longer ? t / (share + 1) : extra + (t - longer) / share;
    };
    const auto first_tile = [&](uint32_t w) { return share * w + min(w, extra); };

    // results: a thread holds DPT dims of a head
    constexpr int DPT = D / 16;
    const int row = tid >> 4;
    const int d0 = (tid & 15) * DPT;
    // b: the sequence's (first) row of out; head0: the segment's first head, with
    // several rows per sequence its unit
    const auto write_out = [&](const float (&o)[DPT], float ol, int b, int head0, int heads) __attribute__((always_inline)) {
        if (row >= heads) return;
        const float inv = ol == 0.f ? 0.f : 1.f / ol;  // nothing seen: zeros
        long long at;
        if constexpr (ROWS) {
            const int kvh = head0 / a.n_hg, x = (head0 - kvh * a.n_hg) * 16 + row, i = x / a.group;
            at = ((long long)(b + i) * a.n_heads + kvh * a.group + (x - i * a.group)) * D + d0;
        } else {
            at = ((long long)b * a.n_heads + head0 + row) * D + d0;
        }
        if (a.bf16) {
#pragma unroll
            for (int e = 0; e < DPT; e += 4) {
                typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
                *(bf16x4_t*)((uint16_t*)a.out + at + e) =
                    bf16x4_t{(__bf16)(o[e] * inv), (__bf16)(o[e + 1] * inv), (__bf16)(o[e + 2] * inv),
                             (__bf16)(o[e + 3] * inv)};
            }
        } else {
#pragma unroll
            for (int e = 0; e < DPT; e += 4)
                *(float4_t*)((float*)a.out + at + e) =
                    float4_t{o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv};
        }
    };
    const __amdgpu_buffer_rsrc_t racc = partial_rsrc(a.ws_acc, (uint32_t)a.slots * 16 * D * 4);
    const __amdgpu_buffer_rsrc_t rml = partial_rsrc(a.ws_ml, (uint32_t)a.slots * 16 * 8);
    int n_shared = 0;  // segments that other workgroups have pieces of
    const int slot_step = a.pieces > 0 ? 1 : 2;

    while (true) {
        int seg, t0, t1, n_pieces;
        int slot_mine, slot0, slot1;  // partials: piece 0's, and piece p >= 1's less slot_step (p - 1)
        Kv8Span sp;
        int b, ctx;
        if (a.pieces > 0) {
            seg = (int)blockIdx.x / a.pieces;
            const int p = (int)blockIdx.x - seg * a.pieces;
            b = seg / units;
            ctx = __builtin_amdgcn_readfirstlane(a.ctx_lens[b]);
            sp = span_of(b, ctx);
            n_pieces = min(a.pieces, (sp.tiles + a.min_tiles - 1) / a.min_tiles);
            if (p >= n_pieces) return;
            // pieces of tiles / n_pieces, the first ones one more
            const int part = sp.tiles / n_pieces, more = sp.tiles - part * n_pieces;
            t0 = part * p + min(p, more);
            t1 = t0 + part + (p < more ? 1 : 0);
            slot0 = seg * a.pieces;
            slot1 = slot0 + 1;
            slot_mine = slot0 + p;
        } else {
            int before;  // tiles of the sequences in front
            if (a.batch <= 64) {
                b = (int)__builtin_ctzll(__ballot((uint32_t)seq_end * units > pos));
                before = b > 0 ? __builtin_amdgcn_readlane(seq_end, b - 1) : 0;
                ctx = __builtin_amdgcn_readlane(seq_ctx, b);
            } else {
                int lo = 0, hi = a.batch - 1;  // first sequence whose tiles end behind pos
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if ((uint32_t)sm_ends[mid] * units > pos)
                        hi = mid;
                    else
                        lo = mid + 1;
                }
                b = __builtin_amdgcn_readfirstlane(lo);
                before = b > 0 ? __builtin_amdgcn_readfirstlane(sm_ends[b - 1]) : 0;
                ctx = __builtin_amdgcn_readfirstlane(a.ctx_lens[b]);
            }
            sp = span_of(b, ctx);
            const uint32_t seq0 = (uint32_t)before * units;
            const uint32_t unit = (pos - seq0) / (uint32_t)sp.tiles;
            const uint32_t start = seq0 + unit * sp.tiles;  // of the segment
            seg = b * units + (int)unit;
            t0 = (int)(pos - start);
            t1 = (int)min((uint32_t)sp.tiles, end - start);
            if (t0 == 0 && t1 == sp.tiles) {
                n_pieces = 1;
                slot0 = slot1 = slot_mine = 0;
            } else {
                const uint32_t w0 = holder(start), w1 = holder(start + sp.tiles - 1);
                n_pieces = (int)(w1 - w0) + 1;
                slot0 = 2 * (int)w0 + (first_tile(w0) >= start ? 0 : 1);
                slot1 = 2 * (int)(w0 + 1);
                slot_mine = 2 * (int)blockIdx.x + (first_segment ? 0 : 1);
            }
        }
        const int unit = seg - b * units;
        const int kvh = unit / a.n_hg;
        const int hg = unit - kvh * a.n_hg;
        const int32_t* table = a.tables + (long long)b * a.max_blocks;
        const int head0 = kvh * a.group + (ROWS ? 0 : hg * 16);
        int heads = min(16, a.group - hg * 16);
        int qpos = ctx - 1;
        int row0 = 0, i = 0, mine = n;  // ROWS: the sequence's first row, this lane's of it, its head of the group
        int key_lo, key_hi, all_lo, all_hi;  // ROWS: what this lane's pair sees, what all pairs see
        if constexpr (ROWS) {
            const Kv8Rows rows = rows_of(b);
            const int x0 = hg * 16;
            row0 = rows.row0;
            heads = max(min(16, rows.rows * a.group - x0), 0);
            const int last = max(heads - 1, 0), x = x0 + min(n, last);
            i = x / a.group;
            mine = x - i * a.group;
            const int first_pos = rows.pos0 + x0 / a.group, last_pos = rows.pos0 + (x0 + last) / a.group;
            qpos = rows.pos0 + i;
            key_hi = rows.key_end(qpos);
            all_hi = rows.key_end(first_pos);
            key_lo = a.s.window > 0 ? max(qpos - a.s.window + 1, 0) : 0;
            all_lo = a.s.window > 0 ? max(last_pos - a.s.window + 1, 0) : 0;
        }

        float slope = 0.f;
        if (MODS && a.s.slopes && n < heads) slope = a.s.slopes[head0 + mine] * 1.4426950408889634f;

        float4_t acc[MT];
#pragma unroll
        for (int j = 0; j < MT; j++) acc[j] = float4_t{};
        float m = -INFINITY, l = 0.f;
        float unit_scale = 0.f;  // largest V scale so far, what acc is measured in

        // this wavefront's tiles
        const int tn = t1 - t0;
        const int tw0 = sp.first + t0 + tn * wave / kWaves;
        int te = sp.first + t0 + tn * (wave + 1) / kWaves;
        if (ROWS && heads == 0) te = tw0;  // pairs that this sequence does not have

        const uint32_t klane = (uint32_t)((4 * (n & 3) + (n >> 2)) * D + 16 * g);
        const uint32_t vlane = (uint32_t)(g * D + 4 * VW * n);

        // the last 16 tiles, 64 subtiles, in front of tile te, from tb on: a lane looks
        // up one subtile's place and scales
        long long off = 0;
        float ks = 0.f, vs = 0.f;
        unsigned long long absent = 0;
        int tb = 0;
        auto look_up = [&]() __attribute__((always_inline)) {
            tb = max(tw0, te - 16);
            const int tok = tb * kTile + 16 * lane;
            int block = -1;
            if (lane < 4 * (te - tb) && tok < sp.hi && tok + 16 > sp.lo) block = kv8_block(a.c, table, a.max_blocks, tok);
            const bool present = block >= 0;
            off = 0;
            ks = vs = 0.f;
            if (present) {
                off = kv8_offset(a.c, block, kvh) + (long long)(tok & ((1 << a.c.bt_log2) - 1)) * D;
                ks = a.c.k_scales[(long long)block * a.c.n_kv_heads + kvh];
                vs = a.c.v_scales[(long long)block * a.c.n_kv_heads + kvh];
            }
            absent = ~__ballot(present);
        };
        const auto get = [](const auto* p) __attribute__((always_inline)) {
            return PASSING ? __builtin_nontemporal_load(p) : *p;
        };
        auto load = [&](Tile& t, int i) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)off, 4 * i + u);
                const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(off >> 32), 4 * i + u);
                const long long at = (long long)(((unsigned long long)hi << 32) | lo);
                const uint8_t* kb = a.c.k + at;
                const uint8_t* vb = a.c.v + at;
#pragma unroll
                for (int c = 0; c < KC; c++) t.k[u][c] = get((const u32x4_t*)(kb + (klane + 64 * c)));
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if constexpr (VW == 2) {
                        const u32x2_t w = get((const u32x2_t*)(vb + (vlane + 4 * D * r)));
                        t.v[u][r][0] = w[0];
                        t.v[u][r][1] = w[1];
                    } else {
                        t.v[u][r][0] = get((const uint32_t*)(vb + (vlane + 4 * D * r)));
                    }
                }
            }
        };
        // the first tile's rows are on their way while q is split
        Tile tile_a, tile_b;
        if (tw0 < te) look_up();
        // q of head n as two binary16 terms of q * 2^-e, largest in [2^13, 2^14)
        half8_t qh[2 * KC], ql[2 * KC];
        float crow;  // what a score is multiplied with, besides the K scale
        float xq[2 * KC][8];
#pragma unroll
        for (int c = 0; c < 2 * KC; c++) {
            const long long at =
                (ROWS ? row0 + i : b) * a.q_stride + (long long)(head0 + mine) * D + 64 * (c >> 1) + 16 * g + 8 * (c & 1);
            if (n >= heads) {
#pragma unroll
                for (int e = 0; e < 8; e++) xq[c][e] = 0.f;
            } else if (a.bf16) {
                const u32x4_t w = *(const u32x4_t*)((const uint16_t*)a.q + at);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    xq[c][2 * e] = __uint_as_float(w[e] << 16);
                    xq[c][2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                }
            } else {
                const float4_t u = *(const float4_t*)((const float*)a.q + at);
                const float4_t v = *(const float4_t*)((const float*)a.q + at + 4);
#pragma unroll
                for (int e = 0; e < 4; e++) xq[c][e] = u[e], xq[c][4 + e] = v[e];
            }
        }
        if (tw0 < te) load(tile_a, te - tb - 1);
        {
            float top = 0.f;
#pragma unroll
            for (int c = 0; c < 2 * KC; c++)
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(xq[c][e]));
            top = max_groups(top);
            const int ex = top > 0.f && top <= 3.402823466e38f ? __builtin_amdgcn_frexp_expf(top) - 14 : 0;
#pragma unroll
            for (int c = 0; c < 2 * KC; c++)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float y0 = __builtin_amdgcn_ldexpf(xq[c][e], -ex), y1 = __builtin_amdgcn_ldexpf(xq[c][e + 1], -ex);
                    const half2_t hi = {(_Float16)y0, (_Float16)y1};
                    const half2_t lo = rest_of_pair(hi, y0, y1);
                    qh[c][e] = hi[0], qh[c][e + 1] = hi[1];
                    ql[c][e] = lo[0], ql[c][e + 1] = lo[1];
                }
            crow = __builtin_amdgcn_ldexpf(a.s.scale_log2, ex);
        }

        // from the last tile to the first: scores biased by distance then leave the
        // maximum alone
        while (tw0 < te) {
            // the weights' unit: the largest V scale
            {
                const float top = fmaxf(wave_reduce_dpp<true>(fabsf(vs)), kLeastScale);
                if (top > unit_scale) {
                    const float down = unit_scale / top;
#pragma unroll
                    for (int j = 0; j < MT; j++) acc[j] *= down;
                    unit_scale = top;
                }
            }
            const float cvl = vs / unit_scale * kWeightUnit;

            auto use = [&](Tile& t, int i) __attribute__((always_inline)) {
                const int p0 = (tb + i) * kTile;
                const int gone = (int)(absent >> (4 * i)) & 15;
                const bool masked = ROWS ? p0 < all_lo || p0 > all_hi - kTile || gone
                                         : p0 < sp.lo || p0 > sp.hi - kTile || gone;
                // two subtiles' chains side by side: a chain's MFMAs wait for each other
                float4_t s[4];
#pragma unroll
                for (int u = 0; u < 4; u++) s[u] = float4_t{};
#pragma unroll
                for (int u0 = 0; u0 < 4; u0 += 2)
#pragma unroll
                    for (int c = 0; c < 2 * KC; c++) {
                        half8_t kh[2];
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const uint32_t w0 = kv8_bias<CODE>(t.k[u0 + u][c >> 1][2 * (c & 1)]);
                            const uint32_t w1 = kv8_bias<CODE>(t.k[u0 + u][c >> 1][2 * (c & 1) + 1]);
                            const u32x4_t kf = {kv8_pair<CODE, false>(w0), kv8_pair<CODE, true>(w0),
                                                kv8_pair<CODE, false>(w1), kv8_pair<CODE, true>(w1)};
                            kh[u] = __builtin_bit_cast(half8_t, kf);
                            s[u0 + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[u], qh[c], s[u0 + u], 0, 0, 0);
                        }
#pragma unroll
                        for (int u = 0; u < 2; u++)
                            s[u0 + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[u], ql[c], s[u0 + u], 0, 0, 0);
                    }
                // log2 scores are s * f
                float f[4];
#pragma unroll
                for (int u = 0; u < 4; u++) f[u] = lane_value(ks, 4 * i + u) * crow;
                if constexpr (MODS) {
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        s[u] *= f[u];
                        f[u] = 1.f;
                    }
                    if (a.s.cap_log2 > 0.f) {
                        float most = 0.f;
#pragma unroll
                        for (int u = 0; u < 4; u++)
#pragma unroll
                            for (int r = 0; r < 4; r++) most = fmaxf(most, fabsf(s[u][r]));
                        const bool wide = __any(most > 0.35f);
#pragma unroll
                        for (int u = 0; u < 4; u++)
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                float y = tanh_series(s[u][r]);
                                if (wide) y = fabsf(s[u][r]) > 0.35f ? tanh_exp(s[u][r]) : y;
                                s[u][r] = y * a.s.cap_log2;
                            }
                    }
                    if (a.s.slopes) {
                        const float back = (float)(qpos - p0 - g);
#pragma unroll
                        for (int u = 0; u < 4; u++)
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                s[u][r] = __builtin_fmaf(-slope,
                                                         ROWS ? fabsf(back - (float)(16 * u + 4 * r))
                                                              : back - (float)(16 * u + 4 * r),
                                                         s[u][r]);
                    }
                }
                if (masked) {
                    asm volatile("");  // a branch: 80 instructions that few tiles need
#pragma unroll
                    for (int u = 0; u < 4; u++) {
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int key = p0 + 16 * u + 4 * r + g;
                            const bool held = key >= sp.lo && key < sp.hi && !((gone >> u) & 1);
                            bool seen = held;
                            if constexpr (ROWS) seen = held && key >= key_lo && key < key_hi;
                            s[u][r] = seen ? s[u][r] * f[u] : -INFINITY;
#pragma unroll
                            for (int x = 0; x < VW; x++) t.v[u][r][x] = held ? t.v[u][r][x] : 0u;
                        }
                        f[u] = 1.f;
                    }
                }
                float top = -INFINITY;
#pragma unroll
                for (int u = 0; u < 4; u++)
                    top = fmaxf(top, fmaxf(fmaxf(s[u][0], s[u][1]), fmaxf(s[u][2], s[u][3])) * f[u]);
                top = fmaxf(m, max_groups(top));
                const float base = top == -INFINITY ? 0.f : top;
                if (__any(top > m)) {
                    const float down = __builtin_amdgcn_exp2f(m - base);
                    l *= down;
#pragma unroll
                    for (int j = 0; j < MT; j++) acc[j] *= down;
                    m = top;
                }
                half8_t ph[2], pl[2];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const float cv = lane_value(cvl, 4 * i + u);
                    float w[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], f[u], -base));
                        l += p;
                        w[r] = p * cv;
                        // one f32 value for both terms: the compiler may otherwise
                        // round the product to binary16 by itself, a unit away from
                        // the part that the rest is taken from
                        asm("" : "+v"(w[r]));
                    }
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const half2_t hi = {(_Float16)w[r], (_Float16)w[r + 1]};
                        const half2_t lo = rest_of_pair(hi, w[r], w[r + 1]);
                        ph[u >> 1][4 * (u & 1) + r] = hi[0];
                        ph[u >> 1][4 * (u & 1) + r + 1] = hi[1];
                        pl[u >> 1][4 * (u & 1) + r] = lo[0];
                        pl[u >> 1][4 * (u & 1) + r + 1] = lo[1];
                    }
                }
#pragma unroll
                for (int pr = 0; pr < 2; pr++)
#pragma unroll
                    for (int x = 0; x < VW; x++) {
                        uint32_t f[4][4];  // [dim within the word][token pair]
#pragma unroll
                        for (int tp = 0; tp < 4; tp++) {
                            const uint32_t w0 = kv8_bias<CODE>(t.v[2 * pr + (tp >> 1)][2 * (tp & 1)][x]);
                            const uint32_t w1 = kv8_bias<CODE>(t.v[2 * pr + (tp >> 1)][2 * (tp & 1) + 1][x]);
                            const uint32_t lo = __builtin_amdgcn_perm(w1, w0, 0x05010400u);
                            const uint32_t hi = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
                            f[0][tp] = kv8_pair<CODE, false>(lo);
                            f[1][tp] = kv8_pair<CODE, true>(lo);
                            f[2][tp] = kv8_pair<CODE, false>(hi);
                            f[3][tp] = kv8_pair<CODE, true>(hi);
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const half8_t vf =
                                __builtin_bit_cast(half8_t, u32x4_t{f[e][0], f[e][1], f[e][2], f[e][3]});
                            const int j = 4 * x + e;
                            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[pr], acc[j], 0, 0, 0);
                            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[pr], acc[j], 0, 0, 0);
                        }
                    }
            };
            int i = te - tb - 1;
            for (; i > 0; i -= 2) {
                load(tile_b, i - 1);
                use(tile_a, i);
                load(tile_a, max(i - 2, 0));
                use(tile_b, i - 1);
            }
            if (i == 0) use(tile_a, 0);
            te = tb;
            if (tw0 < te) {
                look_up();
                load(tile_a, te - tb - 1);
            }
        }

        // the wavefronts' results through LDS
        l = sum_groups(l);
        {
            const float back = unit_scale / kWeightUnit;
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int x = 0; x < VW; x++)
                    *(float4_t*)&sm_acc[wave][n][16 * VW * g + 4 * VW * r + 4 * x] =
                        float4_t{acc[4 * x][r], acc[4 * x + 1][r], acc[4 * x + 2][r], acc[4 * x + 3][r]} * back;
            if (g == 0) sm_ml[wave][n] = float2{m, l};
        }
        __syncthreads();
        float o[DPT];
        float om = -INFINITY, ol = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) om = fmaxf(om, sm_ml[w][row].x);
        const float obase = om == -INFINITY ? 0.f : om;
#pragma unroll
        for (int e = 0; e < DPT; e++) o[e] = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float2 ml = sm_ml[w][row];
            const float f = __builtin_amdgcn_exp2f(ml.x - obase);
            ol = __builtin_fmaf(ml.y, f, ol);
#pragma unroll
            for (int e = 0; e < DPT; e++) o[e] = __builtin_fmaf(sm_acc[w][row][d0 + e], f, o[e]);
        }
        if (n_pieces == 1) {
            write_out(o, ol, ROWS ? row0 : b, ROWS ? unit : head0, heads);
        } else {
            if (row < heads) {
                const int mine = slot_mine * 16 + row;
#pragma unroll
                for (int e = 0; e < DPT; e += 4)
                    __builtin_amdgcn_raw_buffer_store_b128(
                        u32x4_t{__float_as_uint(o[e]), __float_as_uint(o[e + 1]), __float_as_uint(o[e + 2]),
                                __float_as_uint(o[e + 3])},
                        racc, (mine * D + d0 + e) * 4, 0, kSc1);
                if ((tid & 15) == 0)
                    __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(om), __float_as_uint(ol)}, rml,
                                                          mine * 8, 0, kSc1);
            }
            if (tid == 0) sm_shared[n_shared] = {n_pieces, slot0, slot1, ROWS ? row0 : b, ROWS ? unit : head0, heads};
            n_shared++;
        }
        if (a.pieces > 0) break;
        pos += t1 - t0;
        first_segment = false;
        if (pos >= end) break;
        __syncthreads();  // LDS is free for the next segment
    }
    if (n_shared == 0) return;

    // At most two segments of a workgroup are shared, its first and its last.
    // Their arrivals are counted here, in one round trip: every wavefront's stores
    // have completed before (the first's long ago).
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid < n_shared) {
        sm_last[tid] = __hip_atomic_fetch_add(a.counters + sm_shared[tid].slot0, 1, __ATOMIC_RELAXED,
                                              __HIP_MEMORY_SCOPE_AGENT) == sm_shared[tid].n_pieces - 1;
    }
    __syncthreads();
    const bool last0 = __builtin_amdgcn_readfirstlane(sm_last[0]) != 0;
    const bool last1 = n_shared > 1 && __builtin_amdgcn_readfirstlane(sm_last[1]) != 0;
#pragma unroll 1
    for (int k = 0; k < 2; k++) {
        if (!(k ? last1 : last0)) continue;
        if (k && last0) __syncthreads();  // LDS still holds the other's parts
        const auto sh = sm_shared[k];
        const int heads = sh.heads, n_pieces = sh.n_pieces;
        // 16 threads a head; what is left of the workgroup takes every
        // `groups`-th piece, so that one round of loads has many
        if (ROWS && heads == 0) {  // nothing to join
            if (tid == 0) __hip_atomic_store(a.counters + sh.slot0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            continue;
        }
        const int rows = heads > 8 ? 16 : heads > 4 ? 8 : heads > 2 ? 4 : heads;  // a power of two
        const int groups = 16 / rows;
        const int mrow = row & (rows - 1), mgrp = row / rows;
        const int rr = min(mrow, heads - 1);  // rows behind the last hold nothing
        float o[DPT];
        float om = -INFINITY, ol = 0.f;
#pragma unroll
        for (int e = 0; e < DPT; e++) o[e] = 0.f;
        constexpr int AHEAD = 8;
        for (int p = mgrp; p < n_pieces; p += AHEAD * groups) {
            u32x4_t w[AHEAD][DPT / 4];
            u32x2_t ml[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                const int pk = min(p + k * groups, n_pieces - 1);
                const int slot = pk == 0 ? sh.slot0 : sh.slot1 + slot_step * (pk - 1);
                // slots are at most 2 * kMaxWgs: their bytes stay in 32 bits
                ml[k] = __builtin_amdgcn_raw_buffer_load_b64(rml, (slot * 16 + rr) * 8, 0, kSc1);
#pragma unroll
                for (int e = 0; e < DPT / 4; e++)
                    w[k][e] = __builtin_amdgcn_raw_buffer_load_b128(
                        racc, ((slot * 16 + rr) * D + d0 + 4 * e) * 4, 0, kSc1);
            }
            float top = om;
#pragma unroll
            for (int k = 0; k < AHEAD; k++) top = fmaxf(top, __uint_as_float(ml[k][0]));
            const float base = top == -INFINITY ? 0.f : top;
            const float down = __builtin_amdgcn_exp2f(om - base);
            om = top;
            ol *= down;
#pragma unroll
            for (int e = 0; e < DPT; e++) o[e] *= down;
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                if (p + k * groups >= n_pieces) break;
                const float f = __builtin_amdgcn_exp2f(__uint_as_float(ml[k][0]) - base);
                ol = __builtin_fmaf(__uint_as_float(ml[k][1]), f, ol);
#pragma unroll
                for (int e = 0; e < DPT; e++)
                    o[e] = __builtin_fmaf(__uint_as_float(w[k][e >> 2][e & 3]), f, o[e]);
            }
        }
        if (groups > 1) {
            float* const part = &sm_acc[0][0][0];  // [groups * rows = 16][D + PAD]
#pragma unroll
            for (int e = 0; e < DPT; e++) part[row * (D + PAD) + d0 + e] = o[e];
            if ((tid & 15) == 0) sm_ml[0][row] = float2{om, ol};
            __syncthreads();
            om = -INFINITY;
            ol = 0.f;
#pragma unroll
            for (int e = 0; e < DPT; e++) o[e] = 0.f;
            if (row < rows) {
                for (int k = 0; k < groups; k++) om = fmaxf(om, sm_ml[0][k * rows + row].x);
                const float base = om == -INFINITY ? 0.f : om;
                for (int k = 0; k < groups; k++) {
                    const float2 ml = sm_ml[0][k * rows + row];
                    const float f = __builtin_amdgcn_exp2f(ml.x - base);
                    ol = __builtin_fmaf(ml.y, f, ol);
#pragma unroll
                    for (int e = 0; e < DPT; e++)
                        o[e] = __builtin_fmaf(part[(k * rows + row) * (D + PAD) + d0 + e], f, o[e]);
                }
            }
        }
        write_out(o, ol, sh.b, sh.head0, heads);
        if (tid == 0) __hip_atomic_store(a.counters + sh.slot0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

// ------------------------------------------------------------- host side

// Tiles per workgroup at least, one per wavefront.
constexpr int kMinTiles = 4;
// A launch of at most this many segments cuts each of them by itself, into as
// many pieces as give one workgroup per CU, 32 at most: the join reads them
// all.  Measured (us, two workgroups per CU / one / one and 32 pieces at most):
// one sequence of 32768 tokens, 32/4 heads of 64, 32.2 / 20.4 / 16.0, 32/8 of 128
// 25.4 / 21.1 / 21.1; three of 3000-9000, 32/8 of 128, 18.2 / 17.1 / 17.2.
constexpr int kDirectSegments = 64;
constexpr long long kMaxDirectPieces = 32;
// Launches that may read more than the memory-side cache holds (256 MB, by the bound of
// the lengths, each row once) read past it with nontemporal loads: their rows would be
// gone from it before the next launch.  Measured (us, through it / past it): 64 sequences
// of 16640 tokens, 32/4 heads of 64 (545 MB) 104 / 95.4, of 512-32768 111 / 102.5, 24 of
// 200-16000, 32/8 of 128 (399 MB) 86.4 / 82.5; what fits finds itself there again: 64 of
// 2048 (67 MB) 18.1 / 19.3, seven of 8000, 32/8 of 128 (115 MB) 19.2 / 23.0.
constexpr long long kPassingBytes = 1LL << 28;
// Rows that the prefill hands over: up to 16 (row, head) pairs of a kv head, one segment
// per sequence and kv head, or up to 64 in launches of few segments, whose time is the
// chain's and not that of reading the keys once for every 16 pairs.  Measured (us, the
// prefill's kernel / here; 32/8 heads of 128 behind 2000 tokens, batch x rows): 1 x 4
// behind 30000 59.5 / 27.7, 64 x 4 (16 pairs) 93 / 56; 1 x 16 behind 16000 (64 pairs, 32
// segments) 41.1 / 25.2, 4 x 16 (128 segments) 22.0 / 20.6, 16 x 8 (256) 39.1 / 31.4, 8 x 16
// (256) 30.1 / 31.2, 64 x 16 (2048) 95 / 169.
constexpr int kFewPairs = 64;
constexpr int kFewSegments = 256;

struct Kv8DecodePlan {
    int units, chunk, pieces, grid;
    int slots;
    size_t acc, ml, bytes;
    bool passing;
};

static int decode_plan(Kv8DecodePlan& p, const Kv8& c, int batch, int n_heads, int max_ctx, int window,
                       int max_rows, const char* what) {
    if (batch <= 0 || n_heads <= 0 || max_ctx <= 0)
        return set_error(NYION_ERR_INVALID, "%s: batch, n_heads and max_ctx must be positive", what);
    if (n_heads % c.n_kv_heads)
        return set_error(NYION_ERR_INVALID, "%s: n_heads %d not a multiple of n_kv_heads %d", what, n_heads,
                         c.n_kv_heads);
    if (n_heads > 16384) return set_error(NYION_ERR_UNSUPPORTED, "%s: n_heads %d", what, n_heads);
    const int group = n_heads / c.n_kv_heads;
    p.units = c.n_kv_heads * ((max_rows * group + 15) / 16);
    p.chunk = std::min(batch, kMaxSeqs);
    const long long segments = (long long)p.chunk * p.units;
    const long long keys =
        window > 0 ? std::min((long long)window + max_rows + kTile, (long long)max_ctx) : max_ctx;
    const long long tiles = (keys + kTile - 1) / kTile;
    if (segments <= kDirectSegments) {
        const long long fill = std::min(std::max(device_cu_count() / segments, 1LL), kMaxDirectPieces);
        p.pieces = (int)std::min(fill, (tiles + kMinTiles - 1) / kMinTiles);
        p.grid = (int)(segments * p.pieces);
    } else {
        p.pieces = 0;
        p.grid = (int)std::min((long long)kMaxWgs, (tiles * segments + kMinTiles - 1) / kMinTiles);
    }
    p.passing = max_rows == 1 && segments > kDirectSegments && group <= 16 && segments * tiles * kTile * 2 * c.head_dim > kPassingBytes;
    p.slots = p.pieces ? p.grid : 2 * p.grid;
    const size_t slots = (size_t)p.slots;
    p.acc = slots * 16 * c.head_dim * sizeof(float);
    p.ml = (slots * 16 * sizeof(float2) + 255) & ~(size_t)255;
    p.bytes = p.pieces == 1 ? 0 : kKv8CounterBytes + p.acc + p.ml;
    return NYION_OK;
}

template <int D, int CODE, bool MODS, bool PASSING, bool ROWS>
static int resident_wgs() {
    static std::atomic<int> cache[kMaxDevices];
    return per_device_value(
        cache,
        [] {
            int per_cu = 0;
            if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kv8_decode_kernel<D, CODE, MODS, PASSING, ROWS>, 64 * kWaves,
                                                             0) != hipSuccess) {
                (void)hipGetLastError();
                return 0;
            }
            // more than two measured slower (64 sequences of 2048 tokens 18.1 / 22.3 us)
            return std::min(std::max(per_cu, 1), 2) * device_cu_count();
        },
        512);
}

template <int D, int CODE, bool MODS, bool PASSING, bool ROWS>
static void launch_decode(const Kv8DecodeArgs& a, int grid, hipStream_t stream) {
    if (a.pieces == 0) grid = std::min(grid, resident_wgs<D, CODE, MODS, PASSING, ROWS>());
    hipLaunchKernelGGL((kv8_decode_kernel<D, CODE, MODS, PASSING, ROWS>), dim3(grid), dim3(64 * kWaves), 0, stream, a);
}

// Launches of up to p.chunk sequences each; what a.q, a.out and the lists point to is the
// first sequence's.
static int launch_chunks(Kv8DecodeArgs a, const Kv8DecodePlan& p, int code, int batch, void* d_workspace,
                         size_t workspace_bytes, hipStream_t stream, const char* what) {
    if (p.bytes) {
        if (!d_workspace || workspace_bytes < p.bytes)
            return set_error(NYION_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu", what,
                             d_workspace ? workspace_bytes : (size_t)0, p.bytes);
        if (!aligned(d_workspace, 256))
            return set_error(NYION_ERR_INVALID, "%s: workspace not 256-byte aligned", what);
    }
    a.counters = (int*)d_workspace;
    a.ws_acc = (float*)((char*)d_workspace + kKv8CounterBytes);
    a.ws_ml = (float2*)((char*)a.ws_acc + p.acc);
    a.group = a.n_heads / a.c.n_kv_heads;
    a.n_hg = p.units / a.c.n_kv_heads;
    a.pieces = p.pieces;
    a.min_tiles = kMinTiles;
    a.slots = p.slots;
    a.span = (int)std::min((long long)a.max_blocks << a.c.bt_log2, (long long)INT_MAX - 2 * kTile);
    const bool mods = a.s.cap_log2 > 0.f || a.s.slopes, rows = a.row_starts != nullptr;
    const int64_t size = a.bf16 ? 2 : 4;
    int chunk = p.chunk;
    if (!p.pieces) {  // a launch numbers its tiles in 32 bits
        const long long per_seq = (long long)p.units * (a.span / kTile + 2);
        chunk = (int)std::min((long long)chunk, (long long)INT_MAX / per_seq);
        if (chunk < 1) return set_error(NYION_ERR_UNSUPPORTED, "%s: %lld tiles per sequence", what, per_seq);
    }
    for (int b0 = 0; b0 < batch; b0 += chunk) {
        a.batch = std::min(chunk, batch - b0);
        auto pick = [&](auto d, auto code) {
            constexpr int D = decltype(d)::value, CODE = decltype(code)::value;
            if (rows)
                launch_decode<D, CODE, true, false, true>(a, p.grid, stream);
            else if (mods && p.passing)
                launch_decode<D, CODE, true, true, false>(a, p.grid, stream);
            else if (mods)
                launch_decode<D, CODE, true, false, false>(a, p.grid, stream);
            else if (p.passing)
                launch_decode<D, CODE, false, true, false>(a, p.grid, stream);
            else
                launch_decode<D, CODE, false, false, false>(a, p.grid, stream);
        };
        auto by_code = [&](auto d) {
            if (code == NYION_KV8_E4M3)
                pick(d, std::integral_constant<int, NYION_KV8_E4M3>{});
            else
                pick(d, std::integral_constant<int, NYION_KV8_INT8>{});
        };
        if (a.c.head_dim == 64)
            by_code(std::integral_constant<int, 64>{});
        else
            by_code(std::integral_constant<int, 128>{});
        int rc;
        if ((rc = check_launch(what)) != NYION_OK) return rc;
        a.tables += (int64_t)a.batch * a.max_blocks;
        a.ctx_lens += a.batch;
        if (rows) {
            a.row_starts += a.batch;
            if (a.s.prefix_lens) a.s.prefix_lens += a.batch;
        } else {
            a.q = (const char*)a.q + a.batch * a.q_stride * size;
            a.out = (char*)a.out + (int64_t)a.batch * a.n_heads * a.c.head_dim * size;
        }
    }
    return NYION_OK;
}

bool kv8_few_rows(const Kv8& c, int batch, int n_heads, int n_rows, int max_rows) {
    const long long pairs = (long long)max_rows * (n_heads / c.n_kv_heads), sets = (pairs + 15) / 16;
    return n_heads <= 16384 && n_rows <= (long long)batch * max_rows &&
           (sets == 1 || (pairs <= kFewPairs && sets * batch * c.n_kv_heads <= kFewSegments));
}

int kv8_few_rows_size(size_t& bytes, const Kv8& c, int batch, int n_heads, int max_rows, int max_ctx, int window,
                      const char* what) {
    Kv8DecodePlan p;
    const int rc = decode_plan(p, c, batch, n_heads, max_ctx, window, max_rows, what);
    bytes = p.bytes;
    return rc;
}

int kv8_few_rows_attention(const Kv8FewRows& x, const char* what) {
    Kv8DecodeArgs a = {};
    Kv8DecodePlan p;
    int rc;
    if ((rc = decode_plan(p, x.c, x.batch, x.n_heads, x.max_ctx, x.s.window, x.max_rows, what)) != NYION_OK) return rc;
    a.c = x.c;
    a.s = x.s;
    a.tables = x.tables;
    a.max_blocks = x.max_blocks;
    a.ctx_lens = x.ctx_lens;
    a.row_starts = x.row_starts;
    a.n_rows = x.n_rows;
    a.q = x.q;
    a.out = x.out;
    a.q_stride = x.q_stride;
    a.n_heads = x.n_heads;
    a.bf16 = 1;
    return launch_chunks(a, p, x.code, x.batch, x.workspace, x.workspace_bytes, x.stream, what);
}

}  // namespace nyion

using namespace nyion;

extern "C" {

size_t nyion_kv8_decode_workspace_size(const nyion_kv8_cache* cache, int batch, int n_heads,
                                       int max_ctx, int window) {
    clear_error();
    Kv8 c;
    Kv8DecodePlan p;
    if (kv8_cache_args(c, cache, "kv8_decode_workspace_size") != NYION_OK ||
        decode_plan(p, c, batch, n_heads, max_ctx, window, 1, "kv8_decode_workspace_size") != NYION_OK)
        return 0;
    return p.bytes;
}

int nyion_kv8_decode_attention(const nyion_kv8_cache* cache, const int32_t* block_tables,
                               int max_blocks_per_seq, const int32_t* ctx_lens, int batch,
                               int max_ctx, const void* q, int64_t q_stride, void* out, int n_heads,
                               int io_dtype, const nyion_score_options* options,
                               void* d_workspace, size_t workspace_bytes, nyion_stream_t stream) {
    clear_error();
    int rc;
    if ((rc = require_device()) != NYION_OK) return rc;
    const char* what = "kv8_decode";
    Kv8DecodeArgs a = {};
    Kv8DecodePlan p;
    if ((rc = kv8_cache_args(a.c, cache, what)) != NYION_OK) return rc;
    if ((rc = kv8_score_args(a.s, options, a.c.head_dim, false, what)) != NYION_OK) return rc;
    if ((rc = decode_plan(p, a.c, batch, n_heads, max_ctx, a.s.window, 1, what)) != NYION_OK) return rc;
    if (io_dtype != NYION_IO_F32 && io_dtype != NYION_IO_BF16)
        return set_error(NYION_ERR_INVALID, "%s: io_dtype %d", what, io_dtype);
    if (!block_tables || !ctx_lens || !q || !out || max_blocks_per_seq <= 0)
        return set_error(NYION_ERR_INVALID, "%s: null pointer, or max_blocks_per_seq not positive", what);
    const int64_t size = io_dtype == NYION_IO_F32 ? 4 : 2, row = (int64_t)n_heads * a.c.head_dim;
    if (q_stride < row)
        return set_error(NYION_ERR_INVALID, "%s: q_stride %lld below n_heads * head_dim", what, (long long)q_stride);
    if (!aligned(q, 16) || !aligned(out, 16) || q_stride * size % 16)
        return set_error(NYION_ERR_INVALID, "%s: rows of q and out must be 16-byte aligned", what);
    a.tables = block_tables;
    a.max_blocks = max_blocks_per_seq;
    a.ctx_lens = ctx_lens;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.n_heads = n_heads;
    a.bf16 = io_dtype == NYION_IO_BF16;
    return launch_chunks(a, p, cache->code, batch, d_workspace, workspace_bytes, (hipStream_t)stream, what);
}

}  // extern "C"
