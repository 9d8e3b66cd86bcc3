// kv8_prefill.hip — attention of a ragged batch over the 8-bit cache (gfx950).
//
// Sequence b brings rows_b query rows, the last tokens of its context, and
// each kv head is read by `group` q heads.  The rows_b * group (row, head)
// pairs of a kv head are numbered row-major, whatever the group's size, and cut
// into tiles; a workgroup takes one tile, 32 pairs for each of its four or
// eight wavefronts, through the keys that its rows see, 64 at a time:
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
// Eight wavefronts work in two halves, a phase apart: while one half's products
// keep the matrix unit busy, the other takes exponentials and stages the next
// tile, one wavefront of each half on a SIMD.  Four have no phases; two
// workgroups (three at head_dim 64) on a CU overlap as they happen to.
//
// Pages: a table of 128 tiles (512 subtiles of 16 tokens, each in one block)
// is kept in LDS, the place and the scales of each subtile, so that the loads
// of a tile wait for nothing but LDS; longer ranges refill it.
//
// Weights are binary16 against a running maximum that moves only when a sum
// of 32 weights passes 2^14; q is binary16 relative to its row's largest value.
//
// Few tiles: their keys are cut into pieces as well, joined through the
// workspace by the last piece to arrive, in the order of the pieces.  Few rows a
// sequence (up to 16 pairs of a kv head, 64 in small launches): the decode's kernel
// takes them (kv8_few_rows).
//
// Bound: the matrix unit and the power that it may draw for large launches
// (8192 rows of 32/8 heads of 128: 534-565 us, 0.97-1.03 PFLOP/s, where a large
// library product reaches 1.21; 450 us with all data zero); with capped scores
// the exponentials (705 us); for smaller ones what a workgroup does besides its
// tiles, 7 us to find and fetch the first of them, and rounds that are not full.
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "kv8.hpp"

namespace nyion {

constexpr int kKeys = 64;          // per tile
constexpr int kWavePairs = 32;     // pairs per wavefront
constexpr int kTableTiles = 128;   // tiles of the page table in LDS
constexpr int kSeqsMax = 1024;     // sequences per launch
// Tiles of a kv head that are put in order of their lengths at most, and wavefronts
// of such a launch: about three rounds.
constexpr int kSorted = 512;
constexpr int kSortedItems = 6144;
constexpr int kPieceTiles = 4;     // fewest tiles of a piece
constexpr int kMaxPieces = 16;     // the join walks them one by one
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
    static constexpr int OFF = TILES;               // long long [SUBS]: bytes; 0 where absent
    static constexpr int KS = OFF + SUBS * 8;       // float [SUBS]
    static constexpr int VS = KS + SUBS * 4;        // float [SUBS]
    static constexpr int GONE = VS + SUBS * 4;      // uint32 [SUBS / 32]: bits of absent subtiles
    static constexpr int MISC = GONE + SUBS / 8;    // int [16]
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

// The keys that a tile of pairs sees, as tiles of kKeys.
struct PairSpan {
    int tile0, tiles;
};
__device__ __forceinline__ PairSpan pair_span(const Kv8PrefillArgs& a, const Kv8Rows& s, int tile, int tm) {
    PairSpan r;
    const int last_pair = min(tile * tm + tm, s.rows * a.group) - 1;
    const int first = s.pos0 + tile * tm / a.group, last = s.pos0 + last_pair / a.group;
    const int end = last < 0 ? 0 : min(max(last + 1, s.prefix), s.live);
    const int begin = a.s.window > 0 ? min(max(first - a.s.window + 1, 0), end) : 0;
    r.tile0 = begin / kKeys;
    r.tiles = (end + kKeys - 1) / kKeys - r.tile0;
    return r;
}

template <int D, int CODE, bool CAP, bool BIAS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 ? 1 : D == 128 ? 2 : 3) void
kv8_prefill_kernel(Kv8PrefillArgs a) {
    using L = Kv8Lds<D>;
    constexpr int DT = D / 32;       // 32-dim tiles of O^T
    constexpr int KS = D / 16;       // k-steps of the S product
    constexpr int NT = 64 * WAVES;
    constexpr bool PHASES = WAVES == 8;
    constexpr int TM = kWavePairs * WAVES;  // (row, head) pairs per workgroup
    // per thread, of a tile's D * 4 K chunks of 16 bytes and V units of 4 tokens by 4 dims
    constexpr int KL = 4 * D / NT, VL = KL;
    static_assert((kSeqsMax * (1 + sizeof(Kv8Rows) / 4) + kSorted) * 4 <= L::TILES, "the selection's lists");
    static_assert(KL * NT == 4 * D, "every thread stages the same");
    __shared__ __attribute__((aligned(16))) unsigned char lds[L::BYTES];
    long long* const sub_off = (long long*)(lds + L::OFF);
    float* const sub_ks = (float*)(lds + L::KS);
    float* const sub_vs = (float*)(lds + L::VS);
    uint32_t* const sub_gone = (uint32_t*)(lds + L::GONE);
    int* const misc = (int*)(lds + L::MISC);

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31;
    const int h = lane >> 5;
    const bool second = wave >= WAVES / 2;  // with phases: the half that is one behind

    // ---- this workgroup's sequence, kv head, tile of pairs and piece
    int b = 0, tile = 0, kvh = 0, piece = 0;
    int item;
    PairSpan sp;
    Kv8Rows seq;
    {
        int* const ends = (int*)lds;  // tiles up to and with each sequence
        Kv8Rows* const seqs = (Kv8Rows*)(ends + kSeqsMax);
        int before = 0;
        for (int b0 = 0; b0 < a.batch; b0 += NT) {
            const int s = b0 + tid;
            int x = 0;
            if (s < a.batch) {
                const Kv8Rows mine =
                    kv8_rows(a.row_starts, a.ctx_lens, a.s.prefix_lens, a.n_rows, a.span, s);
                seqs[s] = mine;
                x = (int)(((long long)mine.rows * a.group + TM - 1) / TM);
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
            for (int w = 0; w < WAVES; w++) {
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
        const uint32_t items = min((uint64_t)tiles * a.c.n_kv_heads, (uint64_t)a.max_items) * a.pieces;
        const uint32_t per = (items + 7) / 8, at = blockIdx.x >> 3;
        const uint32_t mine = (blockIdx.x & 7) * per + at;
        if (at >= per || mine >= items) return;
        // counters and partials go by (kv head, tile)
        item = (int)(mine / a.pieces);
        piece = (int)mine - item * a.pieces;
        kvh = item / tiles;
        const int place = item - kvh * tiles;
        const auto sequence_of = [&](int t) {
            int lo = 0, hi = a.batch - 1;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (ends[mid] > t)
                    hi = mid;
                else
                    lo = mid + 1;
            }
            return lo;
        };
        int t = tiles - 1 - place;  // later tiles of a sequence are longer: first
        if (a.batch > 1 && tiles <= kSorted && tiles * a.c.n_kv_heads <= kSortedItems / WAVES) {
            // several sequences: the longest of all first (a batch of nine, 1-900 rows
            // behind up to 2000 tokens: 134 -> 127 us, one of 40, 4-200 rows: 136 -> 126;
            // what it costs shows where all lengths are the same, 16 of 300 rows: 95 -> 103,
            // and where many rounds even the lengths out, 128 of 1-100: 192 -> 201)
            int* const length = (int*)(seqs + kSeqsMax);  // [tiles], zeros to a multiple of 16
            const int n16 = (tiles + 15) & ~15;
            for (int i = tid; i < n16; i += NT) {
                int n = 0;
                if (i < tiles) {
                    const int s = sequence_of(i);
                    n = pair_span(a, seqs[s], i - (s > 0 ? ends[s - 1] : 0), TM).tiles + 1;
                }
                length[i] = n;
            }
            __syncthreads();
            // four lanes count a tile's rank
            for (int i = tid >> 2; i < n16; i += NT / 4) {
                const int mine = length[i];
                int rank = 0;
#pragma unroll 4
                for (int k = 4 * (tid & 3); k < n16; k += 16) {
                    const int4 n = *(const int4*)(length + k);
                    rank += (n.x > mine || (n.x == mine && k < i)) + (n.y > mine || (n.y == mine && k + 1 < i)) +
                            (n.z > mine || (n.z == mine && k + 2 < i)) + (n.w > mine || (n.w == mine && k + 3 < i));
                }
                rank += __shfl_xor(rank, 1);
                rank += __shfl_xor(rank, 2);
                if (rank == place) misc[9] = i;
            }
            __syncthreads();
            t = misc[9];
        }
        b = __builtin_amdgcn_readfirstlane(sequence_of(t));
        tile = __builtin_amdgcn_readfirstlane(t - (b > 0 ? ends[b - 1] : 0));
        seq.row0 = __builtin_amdgcn_readfirstlane(seqs[b].row0);
        seq.rows = __builtin_amdgcn_readfirstlane(seqs[b].rows);
        seq.pos0 = __builtin_amdgcn_readfirstlane(seqs[b].pos0);
        seq.live = __builtin_amdgcn_readfirstlane(seqs[b].live);
        seq.prefix = __builtin_amdgcn_readfirstlane(seqs[b].prefix);
        sp = pair_span(a, seq, tile, TM);
        __syncthreads();
    }
    const int row0 = seq.row0, rows = seq.rows, live = seq.live, pos0 = seq.pos0, prefix = seq.prefix;
    const int pairs = rows * a.group;
    const int32_t* table = a.tables + (long long)b * a.max_blocks;
    const int n_pieces = max(min(a.pieces, sp.tiles / kPieceTiles), 1);
    if (piece >= n_pieces) return;
    // pieces of tiles / n_pieces, the first ones one more
    const int part = sp.tiles / n_pieces, more = sp.tiles - part * n_pieces;
    const int t_first = sp.tile0 + part * piece + min(piece, more);
    const int n_tiles = part + (piece < more ? 1 : 0);

    // ---- the pair of this lane: q, bounds
    half8_t qreg[KS];
    float crow, slope;
    int key_lo, key_hi, qpos;
    {
        const int x = min(tile * TM + wave * kWavePairs + j, pairs - 1);
        const int i = x / a.group;
        const int head = kvh * a.group + (x - i * a.group);
        qpos = pos0 + i;
        key_hi = qpos < 0 ? 0 : min(max(qpos + 1, prefix), live);  // exclusive
        key_lo = a.s.window > 0 ? max(qpos - a.s.window + 1, 0) : 0;
        slope = BIAS ? a.s.slopes[head] * 1.4426950408889634f : 0.f;
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
                qreg[s][2 * e] = (_Float16)__builtin_amdgcn_ldexpf(__uint_as_float(w[s][e] << 16), -ex);
                qreg[s][2 * e + 1] = (_Float16)__builtin_amdgcn_ldexpf(__uint_as_float(w[s][e] & 0xffff0000u), -ex);
            }
        crow = __builtin_amdgcn_ldexpf(a.s.scale_log2, ex);
    }
    // bounds of the wavefront's pairs together, for whole tiles
    int w_lo = 0, w_hi = 0;
    int q_lo, q_hi;  // first and last position of the wavefront's rows
    {
        const int x0 = min(tile * TM + wave * kWavePairs, pairs - 1) / a.group;
        const int x1 = min(tile * TM + wave * kWavePairs + kWavePairs - 1, pairs - 1) / a.group;
        q_lo = pos0 + x0;
        q_hi = pos0 + x1;
        w_hi = q_lo < 0 ? 0 : min(max(q_lo + 1, prefix), live);      // smallest end
        w_lo = a.s.window > 0 ? max(q_hi - a.s.window + 1, 0) : 0;   // largest begin
    }

    float16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = float16_t{};
    float mrun = -1e30f;  // finite: exp2(-inf - mrun) is 0, never NaN
    float lrun = 0.f;

    // ---- the page table of nt tiles from tile t0 on; returns the largest V scale
    auto fill = [&](int t0, int nt) __attribute__((always_inline)) {
        float top = 0.f;
#pragma unroll
        for (int x = tid; x < L::SUBS; x += NT) {
            const int tok = t0 * kKeys + 16 * x;
            int block = -1;
            if (x < 4 * nt && tok < live) block = kv8_block(a.c, table, a.max_blocks, tok);
            float ks = 0.f, vs = 0.f;
            long long off = 0;
            if (block >= 0) {
                off = kv8_offset(a.c, block, kvh) + (long long)(tok & ((1 << a.c.bt_log2) - 1)) * D;
                ks = a.c.k_scales[(long long)block * a.c.n_kv_heads + kvh];
                vs = a.c.v_scales[(long long)block * a.c.n_kv_heads + kvh];
            }
            const unsigned long long gone = __ballot(block < 0 && x < 4 * nt && tok < live);
            if (lane < 2) sub_gone[(x >> 5) + lane] = (uint32_t)(lane ? gone >> 32 : gone);
            sub_off[x] = off;
            sub_ks[x] = ks;
            sub_vs[x] = vs;
            top = fmaxf(top, fabsf(vs));
        }
        top = wave_reduce_dpp<true>(top);
        if (lane == 0) misc[wave] = __float_as_int(top);
        __syncthreads();
        top = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) top = fmaxf(top, __int_as_float(misc[w]));
        return top;
    };

    // ---- staging: codes in registers between their loads and the LDS
    u32x4_t kst[KL];
    uint32_t vst[VL][4];
    float vsc = 0.f;  // V scale of this thread's tokens
    unsigned char* const kslot0 = lds;
    unsigned char* const vslot0 = lds + 2 * L::KBYTES;
    // K chunk u: token (tid + NT u) / (D / 16), 16 bytes at (tid % (D / 16))
    constexpr int CPR = D / 16;
    // V unit u: four tokens from 4 tg on, four dims from 4 (vc + 8 u) on.  Of a
    // wavefront's stores to V^T, 8 bytes a lane, 32 lanes then cover every bank twice.
    const int tg = ((lane >> 2) & 7) + 8 * (wave & 1);
    const int vc = (lane & 3) + 4 * (lane >> 5) + 8 * VL * (wave >> 1);
    // what the next loads and weights need of the table, read ahead of them
    long long koff[KL], voff = 0;
    float vnext = 0.f;
    float4_t ks4;
    auto look_k = [&](int x) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < KL; u++) koff[u] = sub_off[4 * x + ((tid + NT * u) / CPR >> 4)];
    };
    auto look_v = [&](int x) __attribute__((always_inline)) {
        voff = sub_off[4 * x + (tg >> 2)];
        vnext = sub_vs[4 * x + (tg >> 2)];
    };
    auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < KL; u++) {
            const int tk = (tid + NT * u) / CPR;
            kst[u] = *(const u32x4_t*)(a.c.k + koff[u] + (tk & 15) * D + 16 * (tid % CPR));
        }
    };
    auto load_v = [&]() __attribute__((always_inline)) {
        vsc = vnext;
        const uint8_t* vb = a.c.v + voff + (tg & 3) * 4 * D + 4 * vc;
#pragma unroll
        for (int u = 0; u < VL; u++)
#pragma unroll
            for (int i = 0; i < 4; i++) vst[u][i] = *(const uint32_t*)(vb + i * D + 32 * u);
    };
    auto store_k = [&](int it) __attribute__((always_inline)) {
        unsigned char* ks = kslot0 + (it & 1) * L::KBYTES;
#pragma unroll
        for (int u = 0; u < KL; u++) {
            const int tk = (tid + NT * u) / CPR;
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
    };
    // bits of a tile's absent subtiles; most tables have none
    bool any_gone = false;
    auto gone_of = [&](int x) __attribute__((always_inline)) {
        return any_gone ? __builtin_amdgcn_readfirstlane((int)((sub_gone[x >> 3] >> (4 * (x & 7))) & 15)) : 0;
    };
    auto store_v = [&](int t0, int it, int x, float unit) __attribute__((always_inline)) {
        const int key = (t0 + x) * kKeys;
        const int gone = gone_of(x);
        if (gone || key + kKeys > live) {
            asm volatile("");
            // tokens behind the end and absent ones may hold NaN codes: zeros
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int u = 0; u < VL; u++)
                    vst[u][i] = ((gone >> (tg >> 2)) & 1) || key + 4 * tg + i >= live ? 0u : vst[u][i];
        }
        unsigned char* vs = vslot0 + (it & 1) * L::VBYTES;
        const _Float16 f = (_Float16)(vsc * unit);
        const half2_t f2 = {f, f};
        const int col = (tg >> 2) * 16 + (tg & 1) * 8 + ((tg >> 1) & 1) * 4;
#pragma unroll
        for (int u = 0; u < VL; u++) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = kv8_bias<CODE>(vst[u][i]);
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
    auto read_k = [&](int it, int kb, half8_t (&kf)[KS]) __attribute__((always_inline)) {
        const unsigned char* kp = kslot0 + (it & 1) * L::KBYTES + (32 * kb + j) * L::KROW + 16 * h;
#pragma unroll
        for (int s = 0; s < KS; s++) kf[s] = __builtin_bit_cast(half8_t, *(const u32x4_t*)(kp + 32 * s));
    };
    auto scores = [&](const half8_t (&kf)[KS]) __attribute__((always_inline)) {
        float16_t st = float16_t{};
#pragma unroll
        for (int s = 0; s < KS; s++) st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[s], qreg[s], st, 0, 0, 0);
        return st;
    };
    auto read_v = [&](int it, int kb, half8_t (&vf)[2][DT]) __attribute__((always_inline)) {
        const unsigned char* vp = vslot0 + (it & 1) * L::VBYTES + j * L::VROW + 16 * h + 64 * kb;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int d = 0; d < DT; d++)
                vf[t][d] = __builtin_bit_cast(half8_t, *(const u32x4_t*)(vp + 32 * d * L::VROW + 32 * t));
    };
    auto values = [&](const half8_t (&vf)[2][DT], const half8_t (&pa)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int d = 0; d < DT; d++)
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[t][d], pa[t], o[d], 0, 0, 0);
    };
    // The weights of a half.  A lane's score r is that of key k0 + c(r), c(r) =
    // 8 (r / 4) + r % 4, which lies in subtile 2 kb + r / 8.  In log2 units it
    // is st[r] * f[r / 8] + sb + sl * c(r); `ready` applies what is not linear and
    // the mask, in branches, so that `weigh` is one block with the products around it.
    struct Factors {
        float f[2], sb, sl;
    };
    auto ready = [&](float16_t& st, Factors& w, int t0, int x, int kb, bool edge) __attribute__((always_inline)) {
        const int k0 = (t0 + x) * kKeys + 32 * kb + 4 * h;
        w.sb = CAP ? a.s.cap_log2 : 0.f;
        w.sl = 0.f;
#pragma unroll
        for (int u = 0; u < 2; u++) w.f[u] = ks4[2 * kb + u] * crow;
        if constexpr (CAP) {
            // cap tanh(x) = cap - 2 cap / (e^2x + 1), linear in what is kept of it
#pragma unroll
            for (int r = 0; r < 16; r++)
                st[r] = __builtin_amdgcn_rcpf(
                    __builtin_amdgcn_exp2f(st[r] * (w.f[r >> 3] * 2.885390081777927f)) + 1.f);
            w.f[0] = w.f[1] = -2.f * a.s.cap_log2;
        }
        if constexpr (BIAS) {
            // keys in front of all rows, behind all of them (a prefix's), or some on
            // either side (a batch of nine, 1-900 rows behind prefixes: 149 us with
            // every tile by the last way, 133 with the three)
            w.sl = slope;
            w.sb = __builtin_fmaf(slope, (float)(k0 - qpos), w.sb);
            const int kt = (t0 + x) * kKeys;
            if (prefix > q_lo && kt + kKeys - 1 > q_lo) {
                asm volatile("");
                if (kt >= q_hi) {
                    w.sl = -slope;
                    w.sb = __builtin_fmaf(-slope, (float)(k0 - qpos), CAP ? a.s.cap_log2 : 0.f);
                } else {
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        st[r] = __builtin_fmaf(-slope, fabsf((float)(k0 - qpos) + (float)(8 * (r >> 2) + (r & 3))),
                                               st[r] * w.f[r >> 3]);
                    w.f[0] = w.f[1] = 1.f;
                    w.sl = 0.f;
                    w.sb = CAP ? a.s.cap_log2 : 0.f;
                }
            }
        }
        if (edge) {
            asm volatile("");  // a branch: few tiles are
            const int lo = key_lo - k0, hi = key_hi - k0;
            const int bits = gone_of(x) >> (2 * kb);
            const bool gone[2] = {(bits & 1) != 0, (bits & 2) != 0};
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int c = 8 * (r >> 2) + (r & 3);
                st[r] = c >= lo && c < hi && !gone[r >> 3] ? st[r] * w.f[r >> 3] : -INFINITY;
            }
            w.f[0] = w.f[1] = 1.f;
        }
    };
    // N halves against one maximum: it may move only while no weights wait for
    // their product.
    auto weigh = [&](auto n, const float16_t* st, const Factors* w, half8_t (*pa)[2]) __attribute__((always_inline)) {
        constexpr int N = decltype(n)::value;
        float psum;
        auto exps = [&]() __attribute__((always_inline)) {
            float sa = 0.f, sc = 0.f;
#pragma unroll
            for (int kb = 0; kb < N; kb++) {
                const float base = w[kb].sb - mrun;
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const int c = 8 * (r >> 2) + (r & 3);
                    const float b0 = BIAS ? __builtin_fmaf(w[kb].sl, (float)c, base) : base;
                    const float b1 = BIAS ? __builtin_fmaf(w[kb].sl, (float)(c + 1), base) : base;
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kb][r], w[kb].f[r >> 3], b0));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kb][r + 1], w[kb].f[r >> 3], b1));
                    sa += p0;
                    sc += p1;
                    pa[kb][r >> 3][r & 7] = (_Float16)p0;
                    pa[kb][r >> 3][(r & 7) + 1] = (_Float16)p1;
                }
            }
            psum = sa + sc;
        };
        exps();
        if (__any(psum > kSumLimit)) {
            float top = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < N; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const float bias =
                        BIAS ? __builtin_fmaf(w[kb].sl, (float)(8 * (r >> 2) + (r & 3)), w[kb].sb) : w[kb].sb;
                    top = fmaxf(top, __builtin_fmaf(st[kb][r], w[kb].f[r >> 3], bias));
                }
            // only this pair's own sum moves it: a pair's result is its own, whatever
            // pairs share the wavefront
            const float mnew = max_half(psum) > kSumLimit ? fmaxf(mrun, max_half(top)) : mrun;
            const float down = __builtin_amdgcn_exp2f(mrun - mnew);
            mrun = mnew;
            lrun *= down;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= down;
            exps();
        }
        lrun += psum;
    };

    float unit = 0.f;  // the largest V scale so far: what O is measured in
    // From the last keys to the first: those next to a row have its largest scores
    // where they are biased by distance, and its maximum then hardly moves (8192 rows
    // with slopes of 2^-8 to 2^-1/4: 870 -> 557 us).
    for (int base = (n_tiles - 1) / kTableTiles * kTableTiles; base >= 0 && n_tiles > 0; base -= kTableTiles) {
        const int t0 = t_first + base;
        const int nt = min(kTableTiles, n_tiles - base);
        if (unit > 0.f) __syncthreads();  // the table and the tiles are still read
        const float top = fmaxf(fill(t0, nt), kVLeast);
        if (top > unit) {
            const float down = unit / top;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= down;
            unit = top;
        }
        const float vunit = kVUnit / unit;
        any_gone = __any(lane < L::SUBS / 32 && sub_gone[lane & (L::SUBS / 32 - 1)] != 0);
        // whether a tile has keys that some row of the wavefront does not see
        const int last = nt - 1;
        // the table's tile of a step, the last one's past the end
        const auto tile_of = [&](int it) { return max(last - it, 0); };
        auto at_edge = [&](int it) {
            const int kt = (t0 + tile_of(it)) * kKeys;
            return gone_of(tile_of(it)) || kt + kKeys > w_hi || kt < w_lo;
        };
        constexpr std::integral_constant<int, 1> one{};
        constexpr std::integral_constant<int, 2> two{};
        if constexpr (PHASES) {
            // Before the phases: K of tile 0, and the second half's part of K of
            // tile 1 and V of tile 0 (the first half's follow in its first phase).
            const int ahead = second ? 1 : 0;
            look_k(last);
            load_k();
            store_k(0);
            look_k(tile_of(1));
            look_v(last);
            load_k();
            load_v();
            if (second) {
                store_k(1);
                store_v(t0, 0, tile_of(0), vunit);
                look_k(tile_of(2));
                look_v(tile_of(1));
                load_k();
                load_v();
            }
            __syncthreads();
            float16_t st[2];
            {
                half8_t kf[KS];
                read_k(0, 0, kf);
                st[0] = scores(kf);
                read_k(0, 1, kf);
                st[1] = scores(kf);
            }
            ks4 = *(const float4_t*)(sub_ks + 4 * last);
            look_k(tile_of(ahead + 2));
            look_v(tile_of(ahead + 1));
            if (second) __syncthreads();
            for (int it = 0; it < nt; it++) {
                half8_t pa[2][2];
                {
                    const bool edge = at_edge(it);
                    Factors w[2];
                    ready(st[0], w[0], t0, tile_of(it), 0, edge);
                    ready(st[1], w[1], t0, tile_of(it), 1, edge);
                    weigh(two, st, w, pa);
                    store_k(it + ahead + 1);
                    store_v(t0, it + ahead, tile_of(it + ahead), vunit);
                    load_k();
                    load_v();
                }
                __syncthreads();
                __builtin_amdgcn_s_setprio(1);
                {
                    half8_t kf[2][KS], vf[2][2][DT];
                    st[0] = st[1] = float16_t{};
                    read_k(it + 1, 0, kf[0]);
                    read_k(it + 1, 1, kf[1]);
#pragma unroll
                    for (int s = 0; s < KS; s++)
#pragma unroll
                        for (int kb = 0; kb < 2; kb++)
                            st[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[kb][s], qreg[s], st[kb], 0, 0, 0);
                    read_v(it, 0, vf[0]);
                    read_v(it, 1, vf[1]);
                    values(vf[0], pa[0]);
                    values(vf[1], pa[1]);
                    ks4 = *(const float4_t*)(sub_ks + 4 * tile_of(it + 1));
                    look_k(tile_of(it + ahead + 3));
                    look_v(tile_of(it + ahead + 2));
                    // reads run AHEAD products in front: an LDS round trip is four of them
                    constexpr int READS = 2 * KS + 4 * DT, AHEAD = 10;
                    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
                    for (int i = 0; i < READS - AHEAD; i++) {
                        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(0x8, AHEAD, 0);
                }
                __builtin_amdgcn_s_setprio(0);
                __syncthreads();
            }
            if (!second) __syncthreads();
        } else {
            // One barrier a step, behind the last use of its K: in front of it K and
            // V slots it & 1 hold tile it and K slot it + 1 & 1 is complete behind it;
            // the step writes K of tile it + 2 and V of tile it + 1 from registers and
            // requests the next (past the last tile it repeats that one, into slots
            // that nobody reads).  Operands are read well ahead of their products.
            look_k(last);
            look_v(last);
            load_k();
            load_v();
            store_k(0);
            store_v(t0, 0, tile_of(0), vunit);
            look_k(tile_of(1));
            look_v(tile_of(1));
            load_k();
            load_v();
            store_k(1);
            look_k(tile_of(2));
            load_k();
            __syncthreads();
            half8_t kf[KS], vf[2][DT];
            read_k(0, 0, kf);
            float16_t st0 = scores(kf);
            for (int it = 0; it < nt; it++) {
                const bool edge = at_edge(it);
                half8_t pa[2][2];
                Factors w;
                ks4 = *(const float4_t*)(sub_ks + 4 * tile_of(it));
                read_k(it, 1, kf);
                __builtin_amdgcn_sched_barrier(0);
                ready(st0, w, t0, tile_of(it), 0, edge);
                float16_t st1 = scores(kf);
                weigh(one, &st0, &w, pa);
                __syncthreads();
                read_v(it, 0, vf);
                look_v(tile_of(it + 2));
                look_k(tile_of(it + 3));
                __builtin_amdgcn_sched_barrier(0);
                ready(st1, w, t0, tile_of(it), 1, edge);
                values(vf, pa[0]);  // ahead of the next weights, which may move the maximum
                read_k(it + 1, 0, kf);
                weigh(one, &st1, &w, pa + 1);
                store_v(t0, it + 1, tile_of(it + 1), vunit);
                store_k(it + 2);
                load_v();
                load_k();
                read_v(it, 1, vf);
                __builtin_amdgcn_sched_barrier(0);
                st0 = scores(kf);
                values(vf, pa[1]);
            }
        }
    }

    // ---- results
    float l = sum_half(lrun), m = mrun;
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] *= unit / kVUnit;
    if (n_pieces > 1) {
        // [piece][wavefront][dim tile][4 registers][lane]
        const long long slot0 = (long long)item * a.pieces;
        const bool holds = tile * TM + wave * kWavePairs < pairs;  // pairs of the wavefront
        constexpr int PART = TM * D;
        const auto acc_at = [&](int p) {
            return partial_rsrc(a.ws_o + (slot0 + p) * PART + wave * (PART / WAVES), PART / WAVES * 4);
        };
        const auto ml_at = [&](int p) {
            return partial_rsrc(a.ws_ml + ((slot0 + p) * WAVES + wave) * 64, 64 * 8);
        };
        if (holds) {
            const __amdgpu_buffer_rsrc_t ro = acc_at(piece), rm = ml_at(piece);
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    __builtin_amdgcn_raw_buffer_store_b128(
                            u32x4_t{__float_as_uint(o[d][4 * r]), __float_as_uint(o[d][4 * r + 1]),
                                    __float_as_uint(o[d][4 * r + 2]), __float_as_uint(o[d][4 * r + 3])},
                            ro, ((d * 4 + r) * 64 + lane) * 16, 0, kSc1);
                __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(m), __float_as_uint(l)}, rm, lane * 8, 0,
                                                  kSc1);
        }
        // every wavefront's stores have completed before the arrival is counted
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (tid == 0)
            misc[8] = __hip_atomic_fetch_add(a.counters + item, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (misc[8] != n_pieces - 1) return;
        m = -1e30f;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = float16_t{};
        // a piece's loads are on their way while the one before is joined
        struct Part {
            u32x2_t ml;
            u32x4_t w[DT][4];
        } x, y;
        const auto fetch = [&](Part& q, int p) __attribute__((always_inline)) {
            const __amdgpu_buffer_rsrc_t ro = acc_at(p), rm = ml_at(p);
            q.ml = __builtin_amdgcn_raw_buffer_load_b64(rm, lane * 8, 0, kSc1);
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    q.w[d][r] = __builtin_amdgcn_raw_buffer_load_b128(ro, ((d * 4 + r) * 64 + lane) * 16, 0, kSc1);
        };
        const auto join = [&](const Part& q) __attribute__((always_inline)) {
            const float mp = __uint_as_float(q.ml[0]);
            const float mnew = fmaxf(m, mp);
            const float f0 = __builtin_amdgcn_exp2f(m - mnew), f1 = __builtin_amdgcn_exp2f(mp - mnew);
            m = mnew;
            l = __builtin_fmaf(__uint_as_float(q.ml[1]), f1, l * f0);
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    o[d][r] = __builtin_fmaf(__uint_as_float(q.w[d][r >> 2][r & 3]), f1, o[d][r] * f0);
        };
        if (holds) {
            fetch(x, 0);
            for (int p = 0; p < n_pieces; p += 2) {
                if (p + 1 < n_pieces) fetch(y, p + 1);
                join(x);
                if (p + 1 >= n_pieces) break;
                if (p + 2 < n_pieces) fetch(x, p + 2);
                join(y);
            }
        }
        if (tid == 0) __hip_atomic_store(a.counters + item, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    {
        const int x = tile * TM + wave * kWavePairs + j;
        if (x >= pairs) return;
        const int i = x / a.group;
        const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing seen: zeros
        uint16_t* orow = a.out + ((long long)(row0 + i) * a.n_heads + kvh * a.group + (x - i * a.group)) * D + 4 * h;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
                *(bf16x4_t*)(orow + 32 * d + 8 * r) =
                    bf16x4_t{(__bf16)(o[d][4 * r] * inv), (__bf16)(o[d][4 * r + 1] * inv),
                             (__bf16)(o[d][4 * r + 2] * inv), (__bf16)(o[d][4 * r + 3] * inv)};
            }
    }
}

// ------------------------------------------------------------- host side

struct Kv8PrefillPlan {
    int chunk, waves, pieces;
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
    // tiles of a launch at most: the whole ones, and a partial one per sequence
    const auto items = [&](int waves) {
        return ((long long)n_rows * group / (kWavePairs * waves) + std::min(p.chunk, n_rows)) * c.n_kv_heads;
    };
    const long long cus = device_cu_count();
    // Eight wavefronts in two phases at head_dim 128 where they give every CU two
    // workgroups or more in turn, in rounds that are nearly full and tiles that are not
    // much emptier than those of four; four without phases elsewhere.  Counted as for
    // sequences of equal rows.  Measured (us, four / eight; 32/8 heads of 128): 8192 rows
    // (1024 workgroups of eight) 608 / 555, 4096 (512) 171 / 154, four sequences of 1500
    // behind 500 (768) 187 / 172; 3000 rows (375) 108 / 127; nine of 1-900 (576: two rounds
    // and a quarter) 127 / 134; 64 of 16 behind 2000 (512, a quarter full) 94 / 154, of 40
    // behind 1000 (512) 109 / 100; 32/4 heads of 64, whose products are too short to hide
    // the other phase, 8192 rows 443 / 537.
    const auto tiles_of = [&](int waves) {
        const long long each = ((long long)n_rows * group + batch - 1) / batch, tm = kWavePairs * waves;
        return (each + tm - 1) / tm * p.chunk * c.n_kv_heads;
    };
    const long long n8 = tiles_of(8), rounds = (n8 + cus - 1) / cus;
    const bool full = 8 * n8 >= 7 * rounds * cus && 20 * n8 <= 11 * tiles_of(4);
    p.waves = c.head_dim == 128 && n8 >= 2 * cus && full ? 8 : 4;
    const int tm = kWavePairs * p.waves;
    p.items = items(p.waves);
    if (p.items >= (1 << 24)) return set_error(NYION_ERR_UNSUPPORTED, "%s: %lld tiles", what, p.items);
    const long long keys = window > 0 ? std::min((long long)window + max_rows, (long long)max_ctx) : max_ctx;
    const long long tiles = (keys + kKeys - 1) / kKeys;
    // Keys are cut only where all pieces are resident at once: a piece's partial result
    // is 64 KB at head_dim 128, written and read again past L2.  (Cutting the long tiles
    // of launches that fill the chip, to even out the causal triangle, measured 158 us
    // against 105 for 3000 rows of 32/8 heads of 128.)
    const long long resident = cus * (p.waves == 8 ? 1 : c.head_dim == 128 ? 2 : 3);
    const long long fill = p.items > 0 && p.items <= kKv8Counters ? resident / p.items : 1;
    p.pieces = (int)std::max(1LL, std::min({fill, tiles / kPieceTiles, (long long)kMaxPieces}));
    p.o = p.ml = p.bytes = 0;
    if (p.pieces > 1) {
        const size_t slots = (size_t)p.items * p.pieces;
        p.o = slots * tm * c.head_dim * sizeof(float);
        p.ml = slots * p.waves * 64 * sizeof(float2);
        p.bytes = kKv8CounterBytes + p.o + p.ml;
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
    if (kv8_few_rows(c, batch, n_heads, n_rows, max_rows)) {
        size_t bytes;
        return kv8_few_rows_size(bytes, c, batch, n_heads, max_rows, max_ctx, window, what) == NYION_OK ? bytes : 0;
    }
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
    if (kv8_few_rows(a.c, batch, n_heads, n_rows, max_rows))
        return kv8_few_rows_attention({a.c, a.s, cache->code, block_tables, max_blocks_per_seq, ctx_lens, row_starts,
                                       batch, n_rows, max_rows, max_ctx, q, q_stride, out, n_heads, d_workspace,
                                       workspace_bytes, (hipStream_t)stream},
                                      what);
    if (p.bytes) {
        if (!d_workspace || workspace_bytes < p.bytes)
            return set_error(NYION_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu", what,
                             d_workspace ? workspace_bytes : (size_t)0, p.bytes);
        if (!aligned(d_workspace, 256))
            return set_error(NYION_ERR_INVALID, "%s: workspace not 256-byte aligned", what);
    }
    a.counters = (int*)d_workspace;
    a.ws_o = (float*)((char*)d_workspace + kKv8CounterBytes);
    a.ws_ml = (float2*)((char*)a.ws_o + p.o);
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.max_blocks = max_blocks_per_seq;
    a.span = (int)std::min((long long)max_blocks_per_seq << a.c.bt_log2, (long long)INT_MAX - (1 << 16));
    a.n_rows = n_rows;
    a.n_heads = n_heads;
    a.group = n_heads / a.c.n_kv_heads;
    a.pieces = p.pieces;
    a.max_items = (int)p.items;
    const int grid = (int)((p.items * p.pieces + 7) / 8 * 8);
    const int32_t* prefix = a.s.prefix_lens;
    for (int b0 = 0; b0 < batch; b0 += p.chunk) {
        a.batch = std::min(p.chunk, batch - b0);
        a.tables = block_tables + (int64_t)b0 * max_blocks_per_seq;
        a.ctx_lens = ctx_lens + b0;
        a.row_starts = row_starts + b0;
        a.s.prefix_lens = prefix ? prefix + b0 : nullptr;
        auto launch = [&](auto d, auto code, auto cap, auto bias) {
            constexpr int D = decltype(d)::value, CODE = decltype(code)::value;
            constexpr bool CAP = decltype(cap)::value, BIAS = decltype(bias)::value;
            if constexpr (D == 128)
                if (p.waves == 8) {
                    hipLaunchKernelGGL((kv8_prefill_kernel<D, CODE, CAP, BIAS, 8>), dim3(grid), dim3(512), 0,
                                       (hipStream_t)stream, a);
                    return;
                }
            hipLaunchKernelGGL((kv8_prefill_kernel<D, CODE, CAP, BIAS, 4>), dim3(grid), dim3(256), 0,
                               (hipStream_t)stream, a);
        };
        auto by_options = [&](auto d, auto code) {
            if (a.s.cap_log2 > 0.f && a.s.slopes)
                launch(d, code, std::true_type{}, std::true_type{});
            else if (a.s.cap_log2 > 0.f)
                launch(d, code, std::true_type{}, std::false_type{});
            else if (a.s.slopes)
                launch(d, code, std::false_type{}, std::true_type{});
            else
                launch(d, code, std::false_type{}, std::false_type{});
        };
        auto by_code = [&](auto d) {
            if (cache->code == NYION_KV8_E4M3)
                by_options(d, std::integral_constant<int, NYION_KV8_E4M3>{});
            else
                by_options(d, std::integral_constant<int, NYION_KV8_INT8>{});
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
