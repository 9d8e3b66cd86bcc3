// kv8_cache.hip — the batch map (block tables and slots from request lengths)
// and the write into the 8-bit cache.
#include <limits.h>

#include <algorithm>

#include "kv8.hpp"

namespace nyion {

// ------------------------------------------------------------- batch map
//
// Row r's slot needs the sequence it belongs to (a search in the running sum
// of the new lengths) and, for a page that the call itself adds, its place in
// the free list (the running sum of the new pages).  Both sums are over the
// batch only, at most 4096 entries, so every workgroup takes them itself into
// LDS: one launch and no wait between workgroups.  A row of a new page reads
// the free list and not the table, which another workgroup is writing.
//
// Bound: latency, a chain of lengths -> sums -> search -> table or free list
// (64 sequences of one token each 3.8 us, 250 with 62,000 rows 5.2 us).

constexpr int kMapThreads = 512;
constexpr int kMapMaxBatch = 4096;

struct MapArgs {
    const int32_t* cached;
    const int32_t* fresh;  // new tokens
    const int32_t* free_blocks;
    int32_t* tables;
    int32_t* ctx_lens;
    int32_t* row_starts;
    int64_t* slots;
    int32_t* positions;
    int32_t* counts;
    int batch, n_free, max_blocks, n_rows, num_blocks, bt_log2;
};

// Sum of numbers that are not negative, INT_MAX at most.
__device__ __forceinline__ int sat_add(int a, int b) {
    return (int)min((unsigned)a + (unsigned)b, (unsigned)INT_MAX);
}

struct MapSeq {
    int cached, ctx;  // lengths before and after
    int first, last;  // the new pages
};
__device__ __forceinline__ MapSeq map_seq(const MapArgs& a, int b) {
    MapSeq s;
    s.cached = max(a.cached[b], 0);
    s.ctx = sat_add(s.cached, max(a.fresh[b], 0));
    // pages of n tokens: (n + bt - 1) >> log2, without leaving 32 bits
    const int up = (1 << a.bt_log2) - 1;
    s.last = min((s.ctx >> a.bt_log2) + ((s.ctx & up) != 0), a.max_blocks);
    s.first = min((s.cached >> a.bt_log2) + ((s.cached & up) != 0), s.last);
    return s;
}

// First entry of the rising list ends[n] that is greater than i (n: none).
__device__ __forceinline__ int first_above(const int* ends, int n, int i) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > i)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

__global__ __launch_bounds__(kMapThreads) void batch_map_kernel(MapArgs a) {
    extern __shared__ int map_lds[];
    int* row_ends = map_lds;            // [batch]
    int* page_ends = map_lds + a.batch;  // [batch]
    constexpr int kWaves = kMapThreads / 64;
    __shared__ int wave_rows[kWaves], wave_pages[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int rows_before = 0, pages_before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kMapThreads) {
        const int b = b0 + tid;
        int rows = 0, pages = 0;
        if (b < a.batch) {
            const MapSeq s = map_seq(a, b);
            rows = max(a.fresh[b], 0);
            pages = s.last - s.first;
            if (blockIdx.x == 0) a.ctx_lens[b] = s.ctx;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int r = __shfl_up(rows, d), p = __shfl_up(pages, d);
            if (lane >= d) {
                rows = sat_add(rows, r);
                pages = sat_add(pages, p);
            }
        }
        if (lane == 63) {
            wave_rows[wave] = rows;
            wave_pages[wave] = pages;
        }
        __syncthreads();
        int rb = rows_before, pb = pages_before;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            if (w < wave) {
                rb = sat_add(rb, wave_rows[w]);
                pb = sat_add(pb, wave_pages[w]);
            }
            rows_before = sat_add(rows_before, wave_rows[w]);
            pages_before = sat_add(pages_before, wave_pages[w]);
        }
        rows = sat_add(rows, rb);
        pages = sat_add(pages, pb);
        if (b < a.batch) {
            row_ends[b] = rows;
            page_ends[b] = pages;
            if (blockIdx.x == 0) a.row_starts[b + 1] = rows;
        }
        __syncthreads();
    }
    const int id = blockIdx.x * kMapThreads + tid;
    const int step = gridDim.x * kMapThreads;
    if (id == 0) {
        a.row_starts[0] = 0;
        a.counts[0] = pages_before;
        a.counts[1] = rows_before;
    }
    const int bt = 1 << a.bt_log2;
    for (int r = id; r < a.n_rows; r += step) {
        const int b = first_above(row_ends, a.batch, r);
        int pos = -1;
        long long slot = -1;
        if (b < a.batch) {
            const MapSeq s = map_seq(a, b);
            const long long p = (long long)s.cached + (r - (b > 0 ? row_ends[b - 1] : 0));
            pos = (int)min(p, (long long)INT_MAX);
            const int page = pos >> a.bt_log2;
            int block = -1;
            if (page >= s.first && page < s.last) {
                const int at = (b > 0 ? page_ends[b - 1] : 0) + (page - s.first);
                if (at < a.n_free) block = a.free_blocks[at];
            } else if (page < s.first) {
                block = a.tables[(long long)b * a.max_blocks + page];
            }
            if ((unsigned)block < (unsigned)a.num_blocks)
                slot = (long long)block * bt + (pos & (bt - 1));
        }
        a.slots[r] = slot;
        a.positions[r] = pos;
    }
    for (long long i = id; i < pages_before; i += step) {
        const int p = (int)i;
        const int b = first_above(page_ends, a.batch, p);
        const MapSeq s = map_seq(a, b);
        const int page = s.first + (p - (b > 0 ? page_ends[b - 1] : 0));
        if (page >= s.last) continue;  // a sum that saturated
        a.tables[(long long)b * a.max_blocks + page] = p < a.n_free ? a.free_blocks[p] : -1;
    }
}

// ------------------------------------------------------------- the write
//
// One team of wavefronts per (block, kv head, K or V): a run's largest
// magnitude decides the scale before any code is known, so the values are held
// in registers between the two (a run that does not fit is read a second
// time, from L2).  The rows of a block are found from the slots alone: the
// first is one whose predecessor (the last row before it that is not skipped,
// 63 rows back at most) goes to another block.  A team takes the block's runs
// one after the other, so what order they have decides the result and nothing
// else does.
//
// Bound: the rows' bytes for prompts (8192 rows of 8 heads of 128, bf16: 12.8 us,
// 3.9 TB/s); latency (slot -> scale and rows -> store) for one token per sequence
// (64 of 4 heads of 64: 4.3 us).

struct Kv8WriteArgs {
    Kv8 c;
    const int64_t* slots;
    const void* x[2];  // k, v
    long long stride[2];
    int n_rows;
    int span;   // rows that a team looks through for the first rows of runs
    unsigned* status;
};

constexpr int kWriteVec = 8;  // values per lane and step

template <int CODE>
__device__ __forceinline__ float kv8_scale_of(float amax) {
    // 448 = 1.75 * 2^8 and 127 = 1.984375 * 2^6: the exponent of amax less 8
    // or 6, one more when its mantissa is above the format's
    constexpr uint32_t kTopFrac = CODE == NYION_KV8_E4M3 ? 0x600000u : 0x7e0000u;
    constexpr int kTopExp = CODE == NYION_KV8_E4M3 ? 8 : 6;
    const uint32_t bits = __float_as_uint(amax);
    const int e = (int)(bits >> 23) - kTopExp + ((bits & 0x7fffffu) > kTopFrac ? 1 : 0);
    return __uint_as_float((uint32_t)max(e, 1) << 23);  // 2^-126 at least
}

// Four values within the format's range -> four codes.
template <int CODE>
__device__ __forceinline__ uint32_t kv8_encode4(const float* y) {
    if constexpr (CODE == NYION_KV8_E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) w |= ((uint32_t)(int)rintf(y[i]) & 0xffu) << (8 * i);
        return w;
    }
}

// Four codes -> their values.
template <int CODE>
__device__ __forceinline__ void kv8_decode4(uint32_t w, float* y) {
    if constexpr (CODE == NYION_KV8_E4M3) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        y[0] = lo[0], y[1] = lo[1], y[2] = hi[0], y[3] = hi[1];
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = (float)(int8_t)(w >> (8 * i));
    }
}

template <bool BF16>
__device__ __forceinline__ void load_vec(const void* x, long long at, float* y) {
    if constexpr (BF16) {
        const u32x4_t w = *(const u32x4_t*)((const uint16_t*)x + at);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            y[2 * i] = __uint_as_float(w[i] << 16);
            y[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const float4_t a = *(const float4_t*)((const float*)x + at);
        const float4_t b = *(const float4_t*)((const float*)x + at + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = a[i], y[4 + i] = b[i];
    }
}

// TEAM wavefronts per unit; HELD steps of 8 values per lane stay in registers.
template <int CODE, bool BF16, int TEAM>
__global__ __launch_bounds__(256) void kv8_write_kernel(Kv8WriteArgs a) {
    constexpr int HELD = 4;
    constexpr int LANES = 64 * TEAM;
    constexpr float kTop = CODE == NYION_KV8_E4M3 ? 448.f : 127.f;
    __shared__ float team_max[4];
    const int lane = threadIdx.x & 63;
    const int at = threadIdx.x & (LANES - 1);  // within the team
    const int unit = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * (256 / LANES) + threadIdx.x / LANES));
    const int per = 2 * a.c.n_kv_heads;
    const int part = unit / per;  // which span of rows
    const int h = (unit - part * per) >> 1, kv = unit & 1;
    const long long r0 = (long long)part * a.span;
    const int bt = 1 << a.c.bt_log2;
    const int cpr = a.c.head_dim / kWriteVec;  // vectors per row: 8 or 16
    const int cpr_log2 = cpr == 16 ? 4 : 3;
    const long long end = (long long)a.c.num_blocks << a.c.bt_log2;
    const long long r1 = min(r0 + a.span, (long long)a.n_rows);
    bool bad = false;
    const auto inside = [&](long long slot) { return slot >= 0 && slot < end; };
    // the first rows of blocks among the span's, all at once: a lane looks at
    // one row and at the last row before it that is not skipped
    const long long cur = r0 + lane < a.n_rows ? a.slots[r0 + lane] : -1;
    const long long prev = r0 - 64 + lane >= 0 ? a.slots[r0 - 64 + lane] : -1;
    unsigned long long firsts;
    {
        const unsigned long long on = __ballot(inside(cur)), before = __ballot(inside(prev));
        const unsigned long long below = on & ((1ull << lane) - 1);
        const int mine = (int)(cur >> a.c.bt_log2);
        const int last = before ? 63 - (int)__builtin_clzll(before) : 0;
        const int last_block = __builtin_amdgcn_readlane((int)(prev >> a.c.bt_log2), last);
        const int near_block = __shfl(mine, below ? 63 - (int)__builtin_clzll(below) : 0);
        const bool follows = below ? near_block == mine : before && lane + 64 - last < 64 && last_block == mine;
        firsts = __ballot(inside(cur) && lane < r1 - r0 && !follows);
    }
    for (; firsts; firsts &= firsts - 1) {
        const int i0 = (int)__builtin_ctzll(firsts);
        long long r = r0 + i0;
        bool in_window = true;
        for (bool more = true; more; in_window = false) {
            long long slot;
            if (in_window) {
                const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)cur, i0);
                const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(cur >> 32), i0);
                slot = (long long)(((unsigned long long)hi << 32) | lo);
            } else {
                slot = a.slots[r];
            }
            const int place = (int)(slot & (bt - 1));
            // the run's length
            const int most = (int)min((long long)(bt - place), a.n_rows - r);
            int n = 0;
            if (in_window) {  // from the rows that are here already
                const unsigned long long on = __ballot(lane >= i0 && cur == slot + (lane - i0)) >> i0;
                n = min(~on ? (int)__builtin_ctzll(~on) : 64, most);
            }
            if (!in_window || (i0 + n == 64 && n < most)) {
                for (int i = n; i < most; i += 64) {
                    const bool on = i + lane < most && a.slots[r + i + lane] == slot + i + lane;
                    const unsigned long long off = ~__ballot(on);
                    n = i + (off ? (int)__builtin_ctzll(off) : 64);
                    if (off) break;
                }
            }
            // what follows it, requested ahead of the rows
            const long long next = r + n + lane < a.n_rows ? a.slots[r + n + lane] : -1;
            const int block = (int)(slot >> a.c.bt_log2);
            uint8_t* codes = (kv ? a.c.v : a.c.k) + kv8_offset(a.c, block, h);
            float* scale_at = (kv ? a.c.v_scales : a.c.k_scales) + (long long)block * a.c.n_kv_heads + h;
            const float before = place > 0 ? fmaxf(*scale_at, 0.f) : 0.f;
            const void* x = a.x[kv];
            const long long x0 = r * a.stride[kv] + (long long)h * a.c.head_dim;
            const int vecs = n << cpr_log2;
            float y[HELD][kWriteVec];
            auto load = [&](int i, float* to) __attribute__((always_inline)) {
                load_vec<BF16>(x, x0 + (long long)(i >> cpr_log2) * a.stride[kv] + kWriteVec * (i & (cpr - 1)), to);
            };
            float amax = 0.f;
            auto take = [&](const float* v) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < kWriteVec; e++) {
                    const float m = fabsf(v[e]);
                    const bool fine = m <= 3.402823466e38f;
                    bad |= !fine;
                    amax = fmaxf(amax, fine ? m : 0.f);
                }
            };
#pragma unroll
            for (int s = 0; s < HELD; s++) {
                const int i = s * LANES + at;
                if (i < vecs)
                    load(i, y[s]);
                else
#pragma unroll
                    for (int e = 0; e < kWriteVec; e++) y[s][e] = 0.f;
            }
#pragma unroll
            for (int s = 0; s < HELD; s++) take(y[s]);
            for (int i = HELD * LANES + at; i < vecs; i += LANES) {
                float z[kWriteVec];
                load(i, z);
                take(z);
            }
            amax = wave_reduce_dpp<true>(amax);
            if constexpr (TEAM > 1) {
                if (lane == 0) team_max[threadIdx.x >> 6] = amax;
                __syncthreads();
                amax = fmaxf(fmaxf(team_max[0], team_max[1]), fmaxf(team_max[2], team_max[3]));
                __syncthreads();  // every wavefront has read `before`, and team_max may be written again
            }
            const float scale = fmaxf(kv8_scale_of<CODE>(amax), before);
            if (place > 0 && scale > before) {
                const float ratio = before / scale;
                for (int i = at; i < (place << cpr_log2); i += LANES) {
                    uint2* p = (uint2*)(codes + kWriteVec * i);
                    const uint2 w = *p;
                    float z[kWriteVec];
                    kv8_decode4<CODE>(w.x, z);
                    kv8_decode4<CODE>(w.y, z + 4);
#pragma unroll
                    for (int e = 0; e < kWriteVec; e++) z[e] *= ratio;
                    *p = uint2{kv8_encode4<CODE>(z), kv8_encode4<CODE>(z + 4)};
                }
            }
            const float inv = 1.0f / scale;  // exact: a power of two
            auto store = [&](int i, const float* v) __attribute__((always_inline)) {
                float z[kWriteVec];
#pragma unroll
                for (int e = 0; e < kWriteVec; e++) {
                    z[e] = v[e] * inv;
                    z[e] = v[e] == v[e] ? fminf(fmaxf(z[e], -kTop), kTop) : 0.f;
                }
                *(uint2*)(codes + (((long long)place << cpr_log2) + i) * kWriteVec) =
                    uint2{kv8_encode4<CODE>(z), kv8_encode4<CODE>(z + 4)};
            };
#pragma unroll
            for (int s = 0; s < HELD; s++) {
                const int i = s * LANES + at;
                if (i < vecs) store(i, y[s]);
            }
            for (int i = HELD * LANES + at; i < vecs; i += LANES) {
                float z[kWriteVec];
                load(i, z);
                store(i, z);
            }
            if (at == 0) *scale_at = scale;
            // another run of this block
            const unsigned long long any = __ballot(inside(next));
            const int skip = any ? (int)__builtin_ctzll(any) : 0;
            more = any && __builtin_amdgcn_readlane((int)(next >> a.c.bt_log2), skip) == block;
            r += n - 1;
            if (more) {
                r += 1 + skip;
                // its scale and live codes are what the team has just stored
                if constexpr (TEAM > 1)
                    __syncthreads();
                else
                    __threadfence_block();
            }
        }
    }
    report_range(a.status, bad, kRangeKv8Write);
}

// ------------------------------------------------------------- host side

int kv8_cache_args(Kv8& c, const nyion_kv8_cache* cache, const char* what) {
    if (!cache) return set_error(NYION_ERR_INVALID, "%s: null cache", what);
    if (!cache->k_codes || !cache->v_codes || !cache->k_scales || !cache->v_scales)
        return set_error(NYION_ERR_INVALID, "%s: null pointer in the cache", what);
    if (cache->num_blocks <= 0 || cache->n_kv_heads <= 0)
        return set_error(NYION_ERR_INVALID, "%s: num_blocks and n_kv_heads must be positive", what);
    if (cache->code != NYION_KV8_E4M3 && cache->code != NYION_KV8_INT8)
        return set_error(NYION_ERR_INVALID, "%s: code %d", what, cache->code);
    if (cache->reserved) return set_error(NYION_ERR_INVALID, "%s: reserved field of the cache is not 0", what);
    const int bt = cache->block_tokens;
    if (!is_pow2(bt) || bt < 16 || bt > 256)
        return set_error(NYION_ERR_UNSUPPORTED, "%s: block_tokens %d (supported: 16, 32, 64, 128, 256)", what, bt);
    if (cache->head_dim != 64 && cache->head_dim != 128)
        return set_error(NYION_ERR_UNSUPPORTED, "%s: head_dim %d (supported: 64, 128)", what, cache->head_dim);
    if (cache->n_kv_heads > 1024)
        return set_error(NYION_ERR_UNSUPPORTED, "%s: n_kv_heads %d (at most 1024)", what, cache->n_kv_heads);
    if (!aligned(cache->k_codes, 16) || !aligned(cache->v_codes, 16) || !aligned(cache->k_scales, 4) ||
        !aligned(cache->v_scales, 4))
        return set_error(NYION_ERR_INVALID, "%s: codes must be 16-byte and scales 4-byte aligned", what);
    c.k = cache->k_codes;
    c.v = cache->v_codes;
    c.k_scales = cache->k_scales;
    c.v_scales = cache->v_scales;
    c.num_blocks = cache->num_blocks;
    c.n_kv_heads = cache->n_kv_heads;
    c.head_dim = cache->head_dim;
    c.bt_log2 = ilog2(bt);
    return NYION_OK;
}

int kv8_score_args(ScoreArgs& s, const nyion_score_options* o, int head_dim, bool prefix_ok,
                   const char* what) {
    const nyion_score_options none = {};
    if (!o) o = &none;
    if (o->reserved) return set_error(NYION_ERR_INVALID, "%s: reserved field of the options is not 0", what);
    if (!isfinite(o->scale) || !isfinite(o->softcap))
        return set_error(NYION_ERR_INVALID, "%s: scale and softcap must be finite", what);
    if (o->softcap < 0.f) return set_error(NYION_ERR_INVALID, "%s: softcap %g", what, (double)o->softcap);
    if (o->prefix_lens && !prefix_ok)
        return set_error(NYION_ERR_INVALID, "%s: prefix_lens is an option of the prefill", what);
    if (!aligned(o->slopes, 4) || !aligned(o->prefix_lens, 4))
        return set_error(NYION_ERR_INVALID, "%s: slopes and prefix_lens must be 4-byte aligned", what);
    const double scale = o->scale > 0.f ? (double)o->scale : 1.0 / sqrt((double)head_dim);
    const double log2e = 1.4426950408889634;
    s.scale_log2 = (float)(o->softcap > 0.f ? scale / o->softcap : scale * log2e);
    s.cap_log2 = (float)(o->softcap * log2e);
    if (!isfinite(s.scale_log2) || !isfinite(s.cap_log2))
        return set_error(NYION_ERR_INVALID, "%s: scale %g with softcap %g leaves f32's range", what, scale,
                         (double)o->softcap);
    s.window = o->window > 0 ? std::min(o->window, 1 << 30) : 0;  // sums with a position stay in 32 bits
    s.slopes = o->slopes;
    s.prefix_lens = o->prefix_lens;
    return NYION_OK;
}

}  // namespace nyion

using namespace nyion;

extern "C" {

int nyion_batch_map(const int32_t* cached_lens, const int32_t* new_lens, int batch,
                    const int32_t* free_blocks, int n_free, int block_tokens, int num_blocks,
                    int32_t* block_tables, int max_blocks_per_seq, int32_t* ctx_lens,
                    int32_t* row_starts, int64_t* slots, int32_t* positions, int n_rows,
                    int32_t* counts, nyion_stream_t stream) {
    clear_error();
    int rc;
    if ((rc = require_device()) != NYION_OK) return rc;
    const char* what = "batch_map";
    if (batch <= 0 || n_free < 0 || num_blocks <= 0 || max_blocks_per_seq <= 0 || n_rows < 0)
        return set_error(NYION_ERR_INVALID, "%s: batch, num_blocks and max_blocks_per_seq must be positive, "
                         "n_free and n_rows not negative", what);
    if (batch > kMapMaxBatch)
        return set_error(NYION_ERR_UNSUPPORTED, "%s: batch %d (at most %d)", what, batch, kMapMaxBatch);
    if (!is_pow2(block_tokens))
        return set_error(NYION_ERR_INVALID, "%s: block_tokens %d is not a power of two", what, block_tokens);
    if (n_rows > (1 << 28)) return set_error(NYION_ERR_UNSUPPORTED, "%s: n_rows %d", what, n_rows);
    if (!cached_lens || !new_lens || !block_tables || !ctx_lens || !row_starts || !counts ||
        (n_free > 0 && !free_blocks) || (n_rows > 0 && (!slots || !positions)))
        return set_error(NYION_ERR_INVALID, "%s: null pointer", what);
    if (ctx_lens == cached_lens || ctx_lens == new_lens)
        return set_error(NYION_ERR_INVALID, "%s: ctx_lens is one of the inputs", what);
    MapArgs a;
    a.cached = cached_lens;
    a.fresh = new_lens;
    a.free_blocks = free_blocks;
    a.tables = block_tables;
    a.ctx_lens = ctx_lens;
    a.row_starts = row_starts;
    a.slots = slots;
    a.positions = positions;
    a.counts = counts;
    a.batch = batch;
    a.n_free = n_free;
    a.max_blocks = max_blocks_per_seq;
    a.n_rows = n_rows;
    a.num_blocks = num_blocks;
    a.bt_log2 = ilog2(block_tokens);
    // one row a thread; the loops take what is more
    const int grid = std::min(std::max((n_rows + kMapThreads - 1) / kMapThreads, 1), 2048);
    hipLaunchKernelGGL(batch_map_kernel, dim3(grid), dim3(kMapThreads), (size_t)batch * 8, (hipStream_t)stream, a);
    return check_launch(what);
}

int nyion_kv8_write(const nyion_kv8_cache* cache, const int64_t* slots, int n_rows, const void* k,
                    int64_t k_stride, const void* v, int64_t v_stride, int io_dtype,
                    nyion_stream_t stream) {
    clear_error();
    int rc;
    if ((rc = require_device()) != NYION_OK) return rc;
    const char* what = "kv8_write";
    Kv8WriteArgs a;
    if ((rc = kv8_cache_args(a.c, cache, what)) != NYION_OK) return rc;
    if (n_rows < 0) return set_error(NYION_ERR_INVALID, "%s: n_rows %d", what, n_rows);
    if (io_dtype != NYION_IO_F32 && io_dtype != NYION_IO_BF16)
        return set_error(NYION_ERR_INVALID, "%s: io_dtype %d", what, io_dtype);
    if (n_rows == 0) return NYION_OK;
    if (!slots || !k || !v) return set_error(NYION_ERR_INVALID, "%s: null pointer", what);
    const int64_t size = io_dtype == NYION_IO_F32 ? 4 : 2, row = (int64_t)a.c.n_kv_heads * a.c.head_dim;
    if (k_stride < row || v_stride < row)
        return set_error(NYION_ERR_INVALID, "%s: strides %lld, %lld below n_kv_heads * head_dim", what,
                         (long long)k_stride, (long long)v_stride);
    if (!aligned(k, 16) || !aligned(v, 16) || k_stride * size % 16 || v_stride * size % 16 || !aligned(slots, 8))
        return set_error(NYION_ERR_INVALID, "%s: rows must be 16-byte and slots 8-byte aligned", what);
    a.slots = slots;
    a.x[0] = k;
    a.x[1] = v;
    a.stride[0] = k_stride;
    a.stride[1] = v_stride;
    a.n_rows = n_rows;
    a.status = device_status_word();
    const int bt = cache->block_tokens, per = 2 * a.c.n_kv_heads;
    a.span = 1;
    const bool wide = bt > 16;
    const int teams = wide ? 1 : 4;  // per workgroup
    if ((long long)n_rows * per > 16384) a.span = std::min(bt, 64);
    const long long units = (long long)((n_rows + a.span - 1) / a.span) * per;
    const long long grid = (units + teams - 1) / teams;
    if (units > INT_MAX) return set_error(NYION_ERR_UNSUPPORTED, "%s: n_rows %d", what, n_rows);
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
    };
    auto pick = [&](auto code, auto bf16) {
        constexpr int CODE = decltype(code)::value;
        constexpr bool BF = decltype(bf16)::value;
        if (wide)
            launch(kv8_write_kernel<CODE, BF, 4>);
        else
            launch(kv8_write_kernel<CODE, BF, 1>);
    };
    auto by_code = [&](auto code) {
        if (io_dtype == NYION_IO_BF16)
            pick(code, std::true_type{});
        else
            pick(code, std::false_type{});
    };
    if (cache->code == NYION_KV8_E4M3)
        by_code(std::integral_constant<int, NYION_KV8_E4M3>{});
    else
        by_code(std::integral_constant<int, NYION_KV8_INT8>{});
    return check_launch(what);
}

}  // extern "C"
