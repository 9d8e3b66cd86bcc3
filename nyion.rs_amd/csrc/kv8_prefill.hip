// kv8_prefill.hip — attention of a ragged batch over the 8-bit cache (gfx950).
//
// Sequence b brings rows_b query rows, the last tokens of its context, and
// each kv head is read by `group` q heads.  The rows_b * group (row, head)
// pairs of a kv head are numbered row-major, whatever the group's size, and cut
// into tiles; a workgroup of four wavefronts takes one tile of 128 * NT pairs,
// 32 * NT a wavefront, through the keys that its rows see, 64 at a time:
//   S^T[32 keys][32 pairs] += K . Q^T    v_mfma_f32_32x32x16_f16
//   O^T[32 dims][32 pairs] += V^T . P^T  v_mfma_f32_32x32x16_f16
// The result layout of S^T (a lane holds one pair and 16 keys) is the B
// operand's of the second product, so weights stay in their lane, and a pair's
// maximum, sum and O are that lane's own (shared with lane ^ 32).
//
// K and V arrive as codes, 16 KB a tile less than the binary16 that the matrix
// unit wants, and are converted once per workgroup on their way into LDS: K
// row by row, V transposed (four tokens by four dims per thread: two byte
// permutes per pair of words, as the conversion takes neighbouring bytes).
// V's scales go into the staged values, relative to the largest of the keys in
// reach so that binary16 holds them; K's into the scores' factor, which the
// exponential's FMA takes anyway.
//
// Pages: a table of 128 tiles (512 subtiles of 16 tokens, each in one block)
// is kept in LDS, the place and the scales of each subtile, so that the loads
// of a tile wait for nothing but LDS; longer ranges refill it.
//
// Weights are binary16 against a running maximum that moves only when a sum
// of 16 weights passes 2^14; q is binary16 relative to its row's largest value.
//
// Few tiles: their keys are cut into pieces as well, joined through the
// workspace by the last piece to arrive, in the order of the pieces.
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "kv8.hpp"

namespace nyion {

constexpr int kKeys = 64;          // per tile
constexpr int kTableTiles = 128;   // tiles of the page table in LDS
constexpr int kSeqsMax = 1024;     // sequences per launch
constexpr float kSumLimit = 16384.f;
constexpr float kVUnit = 64.f;     // 448 * 64 stays below binary16's largest
constexpr float kVLeast = 7.888609052210118e-31f;  // 2^-100

struct Kv8PrefillArgs {
    Kv8 c;
    ScoreArgs s;
    const int32_t* tables;
    const int32_t* ctx_lens;
    const int32_t* row_starts;
    const uint16_t* q;
    uint16_t* out;
    long long q_stride;
    float* ws_o;
    float2* ws_ml;
    int* counters;
    int max_blocks;
    int span;      // tokens that a table covers
    int batch;
    int n_rows;
    int n_heads;
    int group;
    int pieces;
    int min_tiles;
    int max_items;  // (tile, kv head)s that the launch and the workspace hold
};

template <int D>
struct Kv8Lds {
    static constexpr int KROW = D * 2 + 16;      // bytes of a K row
    static constexpr int VROW = kKeys * 2 + 16;  // bytes of a V^T row
    static constexpr int KBYTES = kKeys * KROW;
    static constexpr int VBYTES = D * VROW;
    static constexpr int TILES = 2 * (KBYTES + VBYTES);
    static constexpr int SUBS = 4 * kTableTiles;
    static constexpr int OFF = TILES;               // long long [SUBS]
    static constexpr int KS = OFF + SUBS * 8;       // float [SUBS]
    static constexpr int VS = KS + SUBS * 4;        // float [SUBS]
    static constexpr int MISC = VS + SUBS * 4;      // int [16]
    static constexpr int BYTES = MISC + 64;
};

__device__ __forceinline__ float max_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int D, int CODE, bool MODS, int NT>
__global__ __launch_bounds__(256, NT == 1 ? 2 : 1) void kv8_prefill_kernel(Kv8PrefillArgs a) {
    using L = Kv8Lds<D>;
    constexpr int DT = D / 32;       // 32-dim tiles of O^T
    constexpr int KS = D / 16;       // k-steps of the S product
    constexpr int TM = 128 * NT;     // (row, head) pairs per workgroup
    constexpr int KL = D / 64;       // 16-byte K chunks per thread and tile
    constexpr int VL = D / 64;       // V units per thread and tile
    __shared__ __attribute__((aligned(16))) unsigned char lds[L::BYTES];
    long long* const sub_off = (long long*)(lds + L::OFF);  // -1: absent
    float* const sub_ks = (float*)(lds + L::KS);
    float* const sub_vs = (float*)(lds + L::VS);
    int* const misc = (int*)(lds + L::MISC);

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31;
    const int h = lane >> 5;

    // ---- this workgroup's sequence, kv head, tile of pairs and piece
    int b = 0, tile = 0, kvh = 0, piece = 0;
    long long item;
    {
        int* const ends = (int*)lds;  // tiles up to and with each sequence
        int before = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 256) {
            const int s = b0 + tid;
            int x = 0;
            if (s < a.batch) {
                const int r0 = min(max(a.row_starts[s], 0), a.n_rows);
                const int r1 = min(max(a.row_starts[s + 1], r0), a.n_rows);
                x = (int)(((long long)(r1 - r0) * a.group + TM - 1) / TM);
            }
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int y = __shfl_up(x, d);
                if (lane >= d) x += y;
            }
            if (lane == 63) misc[wave] = x;
            __syncthreads();
            int all = 0;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                if (w < wave) x += misc[w];
                all += misc[w];
            }
            if (s < a.batch) ends[s] = before + x;
            before += all;
            __syncthreads();
        }
        const int tiles = __builtin_amdgcn_readfirstlane(before);
        // an XCD (workgroup id mod 8) takes a run of the list (kv head, tile,
        // piece): its L2 then holds few heads' keys
        const long long items = (long long)tiles * a.c.n_kv_heads * a.pieces;
        const long long per = (items + 7) / 8;
        const long long at = (int)(blockIdx.x >> 3);
        item = (blockIdx.x & 7) * per + at;
        if (at >= per || item >= items || item / a.pieces >= a.max_items) return;
        const int per_head = tiles * a.pieces;
        kvh = (int)(item / per_head);
        const int rest = (int)(item - (long long)kvh * per_head);
        const int t = tiles - 1 - rest / a.pieces;  // later tiles of a sequence are longer: first
        piece = rest % a.pieces;
        int lo = 0, hi = a.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (ends[mid] > t)
                hi = mid;
            else
                lo = mid + 1;
        }
        b = __builtin_amdgcn_readfirstlane(lo);
        tile = __builtin_amdgcn_readfirstlane(t - (b > 0 ? ends[b - 1] : 0));
        // counters and partials go by (sequence's tile, head): item / pieces
        item = item / a.pieces;
        __syncthreads();
    }
    const int row0 = min(max(a.row_starts[b], 0), a.n_rows);
    const int rows = min(max(a.row_starts[b + 1], row0), a.n_rows) - row0;
    const int ctx = a.ctx_lens[b];
    const int live = max(min(ctx, a.span), 0);  // keys that can be read
    const int pos0 = ctx - rows;                // position of row 0
    const int prefix = a.s.prefix_lens ? a.s.prefix_lens[b] : 0;
    const int pairs = rows * a.group;
    const int32_t* table = a.tables + (long long)b * a.max_blocks;

    // ---- keys of the tile's rows
    const int i_first = tile * TM / a.group;
    const int i_last = min(tile * TM + TM, pairs) - 1;
    const int p_first = pos0 + i_first, p_last = pos0 + i_last / a.group;
    const int key_end = p_last < 0 ? 0 : min(max(p_last + 1, prefix), live);
    const int key_begin = a.s.window > 0 ? min(max(p_first - a.s.window + 1, 0), key_end) : 0;
    const int tile0 = key_begin / kKeys;
    const int all_tiles = (key_end + kKeys - 1) / kKeys - tile0;
    const int n_pieces = max(min(a.pieces, all_tiles / a.min_tiles), 1);
    if (piece >= n_pieces) return;
    const int t_first = tile0 + (int)((long long)all_tiles * piece / n_pieces);
    const int n_tiles = tile0 + (int)((long long)all_tiles * (piece + 1) / n_pieces) - t_first;

    // ---- the pairs of this lane: q, bounds
    half8_t qreg[NT][KS];
    float crow[NT], slope[NT];
    int key_lo[NT], key_hi[NT], qpos[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int x = min(tile * TM + (wave * NT + t) * 32 + j, pairs - 1);
        const int i = x / a.group;
        const int head = kvh * a.group + (x - i * a.group);
        qpos[t] = pos0 + i;
        key_hi[t] = qpos[t] < 0 ? 0 : min(max(qpos[t] + 1, prefix), live);  // exclusive
        key_lo[t] = a.s.window > 0 ? max(qpos[t] - a.s.window + 1, 0) : 0;
        slope[t] = MODS && a.s.slopes ? a.s.slopes[head] * 1.4426950408889634f : 0.f;
        const uint16_t* qrow = a.q + (long long)(row0 + i) * a.q_stride + head * D + 8 * h;
        u32x4_t w[KS];
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            w[s] = *(const u32x4_t*)(qrow + 16 * s);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                top = fmaxf(top, fabsf(__uint_as_float(w[s][e] << 16)));
                top = fmaxf(top, fabsf(__uint_as_float(w[s][e] & 0xffff0000u)));
            }
        }
        top = max_half(top);
        const int ex = top > 0.f && top <= 3.402823466e38f ? __builtin_amdgcn_frexp_expf(top) - 14 : 0;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                qreg[t][s][2 * e] = (_Float16)__builtin_amdgcn_ldexpf(__uint_as_float(w[s][e] << 16), -ex);
                qreg[t][s][2 * e + 1] = (_Float16)__builtin_amdgcn_ldexpf(__uint_as_float(w[s][e] & 0xffff0000u), -ex);
            }
        crow[t] = __builtin_amdgcn_ldexpf(a.s.scale_log2, ex);
    }
    // bounds of the wavefront's pairs together, for whole tiles
    int w_lo = 0, w_hi = 0;
    {
        const int x0 = min(tile * TM + wave * NT * 32, pairs - 1) / a.group;
        const int x1 = min(tile * TM + (wave * NT + NT) * 32 - 1, pairs - 1) / a.group;
        w_hi = pos0 + x0 < 0 ? 0 : min(max(pos0 + x0 + 1, prefix), live);   // smallest end
        w_lo = a.s.window > 0 ? max(pos0 + x1 - a.s.window + 1, 0) : 0;      // largest begin
    }

    float16_t o[NT][DT];
    float mrun[NT], lrun[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int d = 0; d < DT; d++) o[t][d] = float16_t{};
        mrun[t] = -1e30f;  // finite: exp2(-inf - mrun) is 0, never NaN
        lrun[t] = 0.f;
    }

    // ---- the page table of nt tiles from tile t0 on; returns the largest V scale
    auto fill = [&](int t0, int nt) __attribute__((always_inline)) {
        float top = 0.f;
#pragma unroll
        for (int x = tid; x < L::SUBS; x += 256) {
            const int tok = t0 * kKeys + 16 * x;
            int block = -1;
            if (x < 4 * nt && tok < live) block = kv8_block(a.c, table, a.max_blocks, tok);
            float ks = 0.f, vs = 0.f;
            long long off = -1;
            if (block >= 0) {
                off = kv8_offset(a.c, block, kvh) + (long long)(tok & ((1 << a.c.bt_log2) - 1)) * D;
                ks = a.c.k_scales[(long long)block * a.c.n_kv_heads + kvh];
                vs = a.c.v_scales[(long long)block * a.c.n_kv_heads + kvh];
            }
            sub_off[x] = off;
            sub_ks[x] = ks;
            sub_vs[x] = vs;
            top = fmaxf(top, fabsf(vs));
        }
        top = wave_reduce_dpp<true>(top);
        if (lane == 0) misc[wave] = __float_as_int(top);
        __syncthreads();
        return fmaxf(fmaxf(__int_as_float(misc[0]), __int_as_float(misc[1])),
                     fmaxf(__int_as_float(misc[2]), __int_as_float(misc[3])));
    };

    // ---- staging: codes in registers between their loads and the LDS
    u32x4_t kst[KL];
    uint32_t vst[VL][4];
    float vsc = 0.f;      // V scale of this thread's tokens
    bool vdead[4];        // its tokens behind the end
    unsigned char* const kslot0 = lds;
    unsigned char* const vslot0 = lds + 2 * L::KBYTES;
    // K chunk u: token (tid + 256 u) / (D / 16), 16 bytes at (tid % (D / 16))
    constexpr int CPR = D / 16;
    // V unit u: four tokens from 4 tg on, four dims from 4 (vc + 8 * u') on
    const int tg = (lane >> 3) + 8 * (wave & 1);
    const int vc = (lane & 7) + (D == 128 ? 16 * (wave >> 1) : 8 * (wave >> 1));
    auto load_tile = [&](int t0, int it) __attribute__((always_inline)) {
        const int s0 = it * 4;
#pragma unroll
        for (int u = 0; u < KL; u++) {
            const int tk = (tid + 256 * u) / CPR;
            const long long off = max(sub_off[s0 + (tk >> 4)], 0ll);  // absent: any row, masked
            kst[u] = *(const u32x4_t*)(a.c.k + off + (tk & 15) * D + 16 * (tid % CPR));
        }
        const long long off = sub_off[s0 + (tg >> 2)];
        vsc = sub_vs[s0 + (tg >> 2)];
        const uint8_t* vb = a.c.v + max(off, 0ll) + (tg & 3) * 4 * D + 4 * vc;
#pragma unroll
        for (int u = 0; u < VL; u++)
#pragma unroll
            for (int i = 0; i < 4; i++) vst[u][i] = *(const uint32_t*)(vb + i * D + 32 * u);
        const int key = (t0 + it) * kKeys + 4 * tg;
#pragma unroll
        for (int i = 0; i < 4; i++) vdead[i] = off < 0 || key + i >= live;
    };
    auto store_tile = [&](int it, float unit) __attribute__((always_inline)) {
        unsigned char* ks = kslot0 + (it & 1) * L::KBYTES;
#pragma unroll
        for (int u = 0; u < KL; u++) {
            const int tk = (tid + 256 * u) / CPR;
            u32x4_t y[2];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t w = kv8_bias<CODE>(kst[u][e]);
                y[e >> 1][2 * (e & 1)] = kv8_pair<CODE, false>(w);
                y[e >> 1][2 * (e & 1) + 1] = kv8_pair<CODE, true>(w);
            }
            u32x4_t* p = (u32x4_t*)(ks + tk * L::KROW + 32 * (tid % CPR));
            p[0] = y[0];
            p[1] = y[1];
        }
        unsigned char* vs = vslot0 + (it & 1) * L::VBYTES;
        const _Float16 f = (_Float16)(vsc * unit);
        const half2_t f2 = {f, f};
        const int col = (tg >> 2) * 16 + (tg & 1) * 8 + ((tg >> 1) & 1) * 4;
#pragma unroll
        for (int u = 0; u < VL; u++) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = kv8_bias<CODE>(vdead[i] ? 0u : vst[u][i]);
            uint32_t y[4][2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t lo = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05010400u);
                const uint32_t hi = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07030602u);
                y[0][i] = kv8_pair<CODE, false>(lo);
                y[1][i] = kv8_pair<CODE, true>(lo);
                y[2][i] = kv8_pair<CODE, false>(hi);
                y[3][i] = kv8_pair<CODE, true>(hi);
            }
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const u32x2_t z = {__builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, y[d][0]) * f2),
                                   __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, y[d][1]) * f2)};
                *(u32x2_t*)(vs + (4 * (vc + 8 * u) + d) * L::VROW + 2 * col) = z;
            }
        }
    };

    // ---- one half (32 keys) of a tile
    auto scores = [&](const unsigned char* ks, int kb, float16_t (&st)[NT]) __attribute__((always_inline)) {
        const unsigned char* kp = ks + (kb * 32 + j) * L::KROW + 16 * h;
#pragma unroll
        for (int t = 0; t < NT; t++) st[t] = float16_t{};
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const half8_t kf = __builtin_bit_cast(half8_t, *(const u32x4_t*)(kp + 32 * s));
#pragma unroll
            for (int t = 0; t < NT; t++)
                st[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qreg[t][s], st[t], 0, 0, 0);
        }
    };
    auto load_v = [&](const unsigned char* vs, int kb, half8_t (&vf)[2][DT]) __attribute__((always_inline)) {
        const unsigned char* vp = vs + j * L::VROW + 16 * h + 64 * kb;
#pragma unroll
        for (int t2 = 0; t2 < 2; t2++)
#pragma unroll
            for (int d = 0; d < DT; d++)
                vf[t2][d] = __builtin_bit_cast(half8_t, *(const u32x4_t*)(vp + 32 * d * L::VROW + 32 * t2));
    };
    // A lane's score r of half kb is that of key kt + 32 kb + 4 h + 8 (r / 4) + r % 4,
    // which lies in subtile 2 kb + r / 8.
    auto consume = [&](float16_t st, const half8_t (&vf)[2][DT], int t, int t0, int it, int kb, bool masked)
        __attribute__((always_inline)) {
        const int k0 = (t0 + it) * kKeys + 32 * kb + 4 * h;
        const int s0 = it * 4 + 2 * kb;
        float f[2];
#pragma unroll
        for (int u = 0; u < 2; u++) f[u] = sub_ks[s0 + u] * crow[t];
        if constexpr (MODS) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float x = st[r] * f[r >> 3];
                if (a.s.cap_log2 > 0.f)  // cap tanh(x), x in natural units
                    x = __builtin_fmaf(-2.f * a.s.cap_log2,
                                       __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * 2.885390081777927f) + 1.f),
                                       a.s.cap_log2);
                if (a.s.slopes) x = __builtin_fmaf(-slope[t], fabsf((float)(qpos[t] - k0) - (float)(8 * (r >> 2) + (r & 3))), x);
                st[r] = x;
            }
            f[0] = f[1] = 1.f;
        }
        if (masked) {
            const int lo = key_lo[t] - k0, hi = key_hi[t] - k0;
            const bool gone[2] = {sub_off[s0] < 0, sub_off[s0 + 1] < 0};
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int c = 8 * (r >> 2) + (r & 3);
                st[r] = c >= lo && c < hi && !gone[r >> 3] ? st[r] * f[r >> 3] : -INFINITY;
            }
            f[0] = f[1] = 1.f;
        }
        half8_t pa[2];
        float psum;
        auto exps = [&]() __attribute__((always_inline)) {
            float sa = 0.f, sb = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], f[r >> 3], -mrun[t]));
                const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r + 1], f[r >> 3], -mrun[t]));
                sa += p0;
                sb += p1;
                pa[r >> 3][r & 7] = (_Float16)p0;
                pa[r >> 3][(r & 7) + 1] = (_Float16)p1;
            }
            psum = sa + sb;
        };
        exps();
        if (__any(psum > kSumLimit)) {
            float top = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, st[r] * f[r >> 3]);
            const float mnew = fmaxf(mrun[t], max_half(top));
            const float down = __builtin_amdgcn_exp2f(mrun[t] - mnew);
            mrun[t] = mnew;
            lrun[t] *= down;
#pragma unroll
            for (int d = 0; d < DT; d++) o[t][d] *= down;
            exps();
        }
        lrun[t] += psum;
#pragma unroll
        for (int t2 = 0; t2 < 2; t2++)
#pragma unroll
            for (int d = 0; d < DT; d++)
                o[t][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[t2][d], pa[t2], o[t][d], 0, 0, 0);
    };

    float unit = 0.f;  // the largest V scale so far: what O is measured in
    for (int base = 0; base < n_tiles; base += kTableTiles) {
        const int t0 = t_first + base;
        const int nt = min(kTableTiles, n_tiles - base);
        if (base) __syncthreads();  // the table is still read
        const float top = fmaxf(fill(t0, nt), kVLeast);
        if (top > unit) {
            const float down = unit / top;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int d = 0; d < DT; d++) o[t][d] *= down;
            unit = top;
        }
        // At the top of step `it` the LDS slots it & 1 hold tile it, and the
        // registers tile it + 1, whose loads were issued a step earlier.
        load_tile(t0, 0);
        store_tile(0, kVUnit / unit);
        if (nt > 1) load_tile(t0, 1);
        __syncthreads();
        for (int it = 0; it < nt; it++) {
            if (it + 1 < nt) store_tile(it + 1, kVUnit / unit);
            if (it + 2 < nt) load_tile(t0, it + 2);
            const unsigned char* ks = kslot0 + (it & 1) * L::KBYTES;
            const unsigned char* vs = vslot0 + (it & 1) * L::VBYTES;
            const int kt = (t0 + it) * kKeys;
            const bool gone = (sub_off[4 * it] | sub_off[4 * it + 1] | sub_off[4 * it + 2] | sub_off[4 * it + 3]) < 0;
            const bool masked = gone || kt + kKeys > w_hi || kt < w_lo;
            float16_t st0[NT], st1[NT];
            half8_t vf[2][DT];
            scores(ks, 0, st0);
            load_v(vs, 0, vf);
            scores(ks, 1, st1);
#pragma unroll
            for (int t = 0; t < NT; t++) consume(st0[t], vf, t, t0, it, 0, masked);
            load_v(vs, 1, vf);
#pragma unroll
            for (int t = 0; t < NT; t++) consume(st1[t], vf, t, t0, it, 1, masked);
            __syncthreads();
        }
    }

    // ---- results
    float l[NT], m[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        l[t] = sum_half(lrun[t]);
        m[t] = mrun[t];
#pragma unroll
        for (int d = 0; d < DT; d++) o[t][d] *= unit / kVUnit;
    }
    if (n_pieces > 1) {
        // [piece][wavefront][pair tile][dim tile][4 registers][lane]
        const long long slot0 = item * a.pieces;
        constexpr int PART = TM * D;
        const auto acc_at = [&](int p) {
            return partial_rsrc(a.ws_o + (slot0 + p) * PART + wave * (PART / 4), PART);
        };
        const auto ml_at = [&](int p) {
            return partial_rsrc(a.ws_ml + ((slot0 + p) * 4 + wave) * NT * 64, NT * 64 * 8);
        };
        {
            const __amdgpu_buffer_rsrc_t ro = acc_at(piece), rm = ml_at(piece);
#pragma unroll
            for (int t = 0; t < NT; t++) {
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        __builtin_amdgcn_raw_buffer_store_b128(
                            u32x4_t{__float_as_uint(o[t][d][4 * r]), __float_as_uint(o[t][d][4 * r + 1]),
                                    __float_as_uint(o[t][d][4 * r + 2]), __float_as_uint(o[t][d][4 * r + 3])},
                            ro, (((t * DT + d) * 4 + r) * 64 + lane) * 16, 0, kSc1);
                __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(m[t]), __float_as_uint(l[t])}, rm,
                                                      (t * 64 + lane) * 8, 0, kSc1);
            }
        }
        // every wavefront's stores have completed before the arrival is counted
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (tid == 0)
            misc[8] = __hip_atomic_fetch_add(a.counters + item, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (misc[8] != n_pieces - 1) return;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            m[t] = -1e30f;
            l[t] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; d++) o[t][d] = float16_t{};
        }
        for (int p = 0; p < n_pieces; p++) {
            const __amdgpu_buffer_rsrc_t ro = acc_at(p), rm = ml_at(p);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const u32x2_t ml = __builtin_amdgcn_raw_buffer_load_b64(rm, (t * 64 + lane) * 8, 0, kSc1);
                u32x4_t w[DT][4];
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        w[d][r] = __builtin_amdgcn_raw_buffer_load_b128(
                            ro, (((t * DT + d) * 4 + r) * 64 + lane) * 16, 0, kSc1);
                const float mp = __uint_as_float(ml[0]);
                const float mnew = fmaxf(m[t], mp);
                const float f0 = __builtin_amdgcn_exp2f(m[t] - mnew), f1 = __builtin_amdgcn_exp2f(mp - mnew);
                m[t] = mnew;
                l[t] = __builtin_fmaf(__uint_as_float(ml[1]), f1, l[t] * f0);
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        o[t][d][r] = __builtin_fmaf(__uint_as_float(w[d][r >> 2][r & 3]), f1, o[t][d][r] * f0);
            }
        }
        if (tid == 0) __hip_atomic_store(a.counters + item, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int x = tile * TM + (wave * NT + t) * 32 + j;
        if (x >= pairs) continue;
        const int i = x / a.group;
        const float inv = l[t] == 0.f ? 0.f : 1.f / l[t];  // nothing seen: zeros
        uint16_t* orow = a.out + ((long long)(row0 + i) * a.n_heads + kvh * a.group + (x - i * a.group)) * D + 4 * h;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
                *(bf16x4_t*)(orow + 32 * d + 8 * r) =
                    bf16x4_t{(__bf16)(o[t][d][4 * r] * inv), (__bf16)(o[t][d][4 * r + 1] * inv),
                             (__bf16)(o[t][d][4 * r + 2] * inv), (__bf16)(o[t][d][4 * r + 3] * inv)};
            }
    }
}

// ------------------------------------------------------------- host side

constexpr int kPieceTiles = 4;   // fewest tiles of a piece
constexpr int kMaxPieces = 16;

struct Kv8PrefillPlan {
    int chunk, nt, pieces;
    long long items;  // (tile, kv head)s of a launch at most
    size_t o, ml, bytes;
};

static int prefill_plan(Kv8PrefillPlan& p, const Kv8& c, int batch, int n_heads, int n_rows, int max_rows,
                        int max_ctx, int window, const char* what) {
    if (batch <= 0 || n_heads <= 0 || n_rows < 0 || max_rows <= 0 || max_ctx <= 0)
        return set_error(NYION_ERR_INVALID, "%s: batch, n_heads, max_rows and max_ctx must be positive, n_rows not "
                         "negative", what);
    if (n_heads % c.n_kv_heads)
        return set_error(NYION_ERR_INVALID, "%s: n_heads %d not a multiple of n_kv_heads %d", what, n_heads,
                         c.n_kv_heads);
    if ((long long)n_rows * n_heads > (1 << 27))
        return set_error(NYION_ERR_UNSUPPORTED, "%s: n_rows %d * n_heads %d beyond 2^27", what, n_rows, n_heads);
    const int group = n_heads / c.n_kv_heads;
    p.chunk = std::min(batch, kSeqsMax);
    p.nt = 1;
    const int tm = 128 * p.nt;
    // tiles: one partial tile per sequence at most, besides the whole ones
    p.items = ((long long)n_rows * group / tm + std::min(p.chunk, n_rows)) * c.n_kv_heads;
    if (p.items >= (1 << 24)) return set_error(NYION_ERR_UNSUPPORTED, "%s: %lld tiles", what, p.items);
    const long long keys = window > 0 ? std::min((long long)window + max_rows, (long long)max_ctx) : max_ctx;
    const long long tiles = (keys + kKeys - 1) / kKeys;
    const long long fill = p.items > 0 ? 4LL * device_cu_count() / p.items : 1;
    p.pieces = (int)std::max(1LL, std::min({fill, tiles / kPieceTiles, (long long)kMaxPieces}));
    p.o = p.ml = p.bytes = 0;
    if (p.pieces > 1) {
        const size_t slots = (size_t)p.items * p.pieces;
        p.o = slots * tm * c.head_dim * sizeof(float);
        p.ml = slots * 4 * p.nt * 64 * sizeof(float2);
        p.bytes = p.o + p.ml + (((size_t)p.items * sizeof(int) + 255) & ~(size_t)255);
    }
    return NYION_OK;
}

}  // namespace nyion

using namespace nyion;

extern "C" {

size_t nyion_kv8_prefill_workspace_size(const nyion_kv8_cache* cache, int batch, int n_heads,
                                        int n_rows, int max_rows, int max_ctx, int window) {
    clear_error();
    const char* what = "kv8_prefill_workspace_size";
    Kv8 c;
    Kv8PrefillPlan p;
    if (kv8_cache_args(c, cache, what) != NYION_OK ||
        prefill_plan(p, c, batch, n_heads, n_rows, max_rows, max_ctx, window, what) != NYION_OK)
        return 0;
    return p.bytes;
}

int nyion_kv8_prefill_attention_bf16(const nyion_kv8_cache* cache, const int32_t* block_tables,
                                     int max_blocks_per_seq, const int32_t* ctx_lens,
                                     const int32_t* row_starts, int batch, int n_rows,
                                     int max_rows, int max_ctx, const uint16_t* q,
                                     int64_t q_stride, uint16_t* out, int n_heads,
                                     const nyion_score_options* options, void* d_workspace,
                                     size_t workspace_bytes, nyion_stream_t stream) {
    clear_error();
    int rc;
    if ((rc = require_device()) != NYION_OK) return rc;
    const char* what = "kv8_prefill";
    Kv8PrefillArgs a;
    Kv8PrefillPlan p;
    if ((rc = kv8_cache_args(a.c, cache, what)) != NYION_OK) return rc;
    if ((rc = kv8_score_args(a.s, options, a.c.head_dim, true, what)) != NYION_OK) return rc;
    if ((rc = prefill_plan(p, a.c, batch, n_heads, n_rows, max_rows, max_ctx, a.s.window, what)) != NYION_OK)
        return rc;
    if (n_rows == 0) return NYION_OK;
    if (!block_tables || !ctx_lens || !row_starts || !q || !out || max_blocks_per_seq <= 0)
        return set_error(NYION_ERR_INVALID, "%s: null pointer, or max_blocks_per_seq not positive", what);
    if (q_stride < (int64_t)n_heads * a.c.head_dim)
        return set_error(NYION_ERR_INVALID, "%s: q_stride %lld below n_heads * head_dim", what, (long long)q_stride);
    if (!aligned(q, 16) || !aligned(out, 16) || q_stride % 8)
        return set_error(NYION_ERR_INVALID, "%s: rows of q and out must be 16-byte aligned", what);
    if (p.bytes) {
        if (!d_workspace || workspace_bytes < p.bytes)
            return set_error(NYION_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu", what,
                             d_workspace ? workspace_bytes : (size_t)0, p.bytes);
        if (!aligned(d_workspace, 256))
            return set_error(NYION_ERR_INVALID, "%s: workspace not 256-byte aligned", what);
    }
    a.ws_o = (float*)d_workspace;
    a.ws_ml = (float2*)((char*)d_workspace + p.o);
    a.counters = (int*)((char*)d_workspace + p.o + p.ml);
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.max_blocks = max_blocks_per_seq;
    a.span = (int)std::min((long long)max_blocks_per_seq << a.c.bt_log2, (long long)INT_MAX - (1 << 16));
    a.n_rows = n_rows;
    a.n_heads = n_heads;
    a.group = n_heads / a.c.n_kv_heads;
    a.pieces = p.pieces;
    a.min_tiles = kPieceTiles;
    a.max_items = (int)p.items;
    const bool mods = a.s.cap_log2 > 0.f || a.s.slopes;
    const int grid = (int)((p.items * p.pieces + 7) / 8 * 8);
    const int32_t* prefix = a.s.prefix_lens;
    for (int b0 = 0; b0 < batch; b0 += p.chunk) {
        a.batch = std::min(p.chunk, batch - b0);
        a.tables = block_tables + (int64_t)b0 * max_blocks_per_seq;
        a.ctx_lens = ctx_lens + b0;
        a.row_starts = row_starts + b0;
        a.s.prefix_lens = prefix ? prefix + b0 : nullptr;
        auto launch = [&](auto d, auto code, auto m) {
            constexpr int D = decltype(d)::value, CODE = decltype(code)::value;
            constexpr bool MODS = decltype(m)::value;
            hipLaunchKernelGGL((kv8_prefill_kernel<D, CODE, MODS, 1>), dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
        };
        auto by_mods = [&](auto d, auto code) {
            if (mods)
                launch(d, code, std::true_type{});
            else
                launch(d, code, std::false_type{});
        };
        auto by_code = [&](auto d) {
            if (cache->code == NYION_KV8_E4M3)
                by_mods(d, std::integral_constant<int, NYION_KV8_E4M3>{});
            else
                by_mods(d, std::integral_constant<int, NYION_KV8_INT8>{});
        };
        if (a.c.head_dim == 64)
            by_code(std::integral_constant<int, 64>{});
        else
            by_code(std::integral_constant<int, 128>{});
        if ((rc = check_launch(what)) != NYION_OK) return rc;
    }
    return NYION_OK;
}

}  // extern "C"
