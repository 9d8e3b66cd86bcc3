// kv8.hpp — what the kernels of the 8-bit cache share: its geometry on the
// device, the host-side checks of the structs that callers pass, and the
// codes' way into binary16.
#pragma once

#include <math.h>

#include "common.hpp"

namespace nyion {

struct Kv8 {
    uint8_t* k;
    uint8_t* v;
    float* k_scales;
    float* v_scales;
    int num_blocks;
    int n_kv_heads;
    int head_dim;
    int bt_log2;  // log2(block_tokens)
};

// Score options with every default resolved (log2 units where noted).
struct ScoreArgs {
    float scale_log2;  // scale * log2(e); with a cap: scale / softcap
    float cap_log2;    // softcap * log2(e), 0: none
    int window;        // 0: none
    const float* slopes;
    const int32_t* prefix_lens;
};

// Workspaces of both attentions begin with their arrival counters, in a place
// that no argument moves: one workspace then serves calls of any shapes.
constexpr int kKv8Counters = 4096;
constexpr size_t kKv8CounterBytes = kKv8Counters * sizeof(int);

// Host: checks a caller's cache struct and fills `c`.
int kv8_cache_args(Kv8& c, const nyion_kv8_cache* cache, const char* what);
// Host: checks a caller's options (nullptr: none) and fills `s`.
int kv8_score_args(ScoreArgs& s, const nyion_score_options* o, int head_dim, bool prefix_ok,
                   const char* what);

// A ragged batch of few rows a sequence, as the decode takes it from the prefill
// (kv8_decode.hip): q and out bf16.
struct Kv8FewRows {
    Kv8 c;
    ScoreArgs s;
    int code;
    const int32_t* tables;
    int max_blocks;
    const int32_t* ctx_lens;
    const int32_t* row_starts;
    int batch, n_rows, max_rows, max_ctx;
    const uint16_t* q;
    long long q_stride;
    uint16_t* out;
    int n_heads;
    void* workspace;
    size_t workspace_bytes;
    hipStream_t stream;
};
bool kv8_few_rows(const Kv8& c, int batch, int n_heads, int n_rows, int max_rows);
int kv8_few_rows_size(size_t& bytes, const Kv8& c, int batch, int n_heads, int max_rows, int max_ctx, int window,
                      const char* what);
int kv8_few_rows_attention(const Kv8FewRows& x, const char* what);

// Token t's block in a sequence's table, or -1: past the table (or t
// negative), or not a block of the cache.
__device__ __forceinline__ int kv8_block(const Kv8& c, const int32_t* table, int max_blocks, int t) {
    const int page = t >> c.bt_log2;
    if ((unsigned)page >= (unsigned)max_blocks) return -1;
    const int b = table[page];
    return (unsigned)b < (unsigned)c.num_blocks ? b : -1;
}

// The rows of sequence b of a ragged batch, and how far its keys go.
struct Kv8Rows {
    int row0, rows;  // of those that q holds
    int pos0;        // position of row0
    int live;        // its keys that can be read
    int prefix;
    __device__ __forceinline__ int key_end(int pos) const {  // of a row at pos, exclusive
        return pos < 0 ? 0 : min(max(pos + 1, prefix), live);
    }
};
__device__ __forceinline__ Kv8Rows kv8_rows(const int32_t* row_starts, const int32_t* ctx_lens,
                                            const int32_t* prefix_lens, int n_rows, int span, int b) {
    Kv8Rows s;
    const int end = row_starts[b + 1], ctx = ctx_lens[b];
    s.row0 = min(max(row_starts[b], 0), n_rows);
    s.rows = min(max(end, s.row0), n_rows) - s.row0;
    s.pos0 = (int)((unsigned)ctx - (unsigned)end + (unsigned)s.row0);
    s.live = max(min(ctx, span), 0);
    s.prefix = prefix_lens ? prefix_lens[b] : 0;
    return s;
}

// Byte offset of kv head h of a block: 64 bits, a cache may pass 4 GiB.
__device__ __forceinline__ long long kv8_offset(const Kv8& c, int block, int h) {
    return ((long long)block * c.n_kv_heads + h) * ((long long)c.head_dim << c.bt_log2);
}

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Two neighbouring codes of a word (the high two if HI) as binary16 pairs;
// both formats' values are exact there.  Integers: a byte b + 128 under the
// exponent byte 0x64 is 1024 + 128 + b, from which 1152 is taken.  `w` holds
// the integers with their top bits flipped (kv8_bias).
template <int CODE, bool HI>
__device__ __forceinline__ uint32_t kv8_pair(uint32_t w) {
    if constexpr (CODE == NYION_KV8_E4M3) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
    } else {
        const uint32_t x = __builtin_amdgcn_perm(0x64646464u, w, HI ? 0x04030402u : 0x04010400u);
        const half2_t y = __builtin_bit_cast(half2_t, x) - half2_t{(_Float16)1152.f, (_Float16)1152.f};
        return __builtin_bit_cast(uint32_t, y);
    }
}
template <int CODE>
__device__ __forceinline__ uint32_t kv8_bias(uint32_t w) {
    return CODE == NYION_KV8_INT8 ? w ^ 0x80808080u : w;
}

}  // namespace nyion
