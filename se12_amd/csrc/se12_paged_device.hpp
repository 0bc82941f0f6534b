// What the paged-cache kernels (se12_paged.hip, se12_paged_attention.hip) share:
// the cache and the new tokens of a call as the kernels see them, and the checks
// of both at the C entries.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "se12_step.h"
#include "se12_step_math.hpp"

namespace se12step {

struct Batch {
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    const int32_t* starts;
    int width, seqs, tokens, max_new;
};

// one sequence of a call: its new tokens are rows start .. start + n - 1, at
// positions len ..; what the device memory says is kept inside the call's rows
// and the table
struct Seq {
    int start, n, len;
};

__device__ __forceinline__ Seq load_seq(const Batch& b, int s, int capacity) {
    const int a = min(max(b.starts[s], 0), b.tokens);
    const int e = min(max(b.starts[s + 1], a), b.tokens);
    return {a, min(e - a, b.max_new), min(max(b.lengths[s], 0), capacity)};
}

// the page holding column `c` of sequence s's table row, or -1
__device__ __forceinline__ int page_of(const Batch& b, int s, int c, int pages) {
    if (c < 0 || c >= b.width) return -1;
    const int id = b.table[s * b.table_stride + c];
    return (uint32_t)id < (uint32_t)pages ? id : -1;
}

// host: the first thing wrong with a cache and the new tokens of a call, or NULL
inline const char* paged_error(const se12_step_pages* p, const se12_step_batch* b, int32_t heads) {
    if (!p || !b) return "NULL argument";
    if (!p->k || !p->v) return "NULL cache";
    if (p->dtype != SE12_STEP_BF16 && p->dtype != SE12_STEP_E4M3) return "the cache must be BF16 or E4M3";
    if (p->dtype == SE12_STEP_E4M3 && (!p->k_scale || !p->v_scale)) return "an E4M3 cache needs scales";
    if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128)
        return "page_size must be 16, 32, 64 or 128";
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return "head_dim must be 64, 128 or 256";
    if (p->pages < 1 || p->kv_heads < 1 || p->kv_heads > 1024) return "bad cache shape";
    if (heads < 1 || heads > 65535 || heads % p->kv_heads) return "heads must be a multiple of kv_heads";
    if (!b->page_table || !b->lengths || !b->starts) return "NULL batch tensor";
    if (b->sequences < 1 || b->sequences > 65536 || b->tokens < 0 || b->max_new < 1 || b->table_width < 1 ||
        b->table_stride < b->table_width)
        return "bad batch shape";
    if ((int64_t)b->table_width * p->page_size > ((int64_t)1 << 30) || b->tokens > (1 << 30)) return "sequences above 2^30 tokens";
    if (reinterpret_cast<uintptr_t>(p->k) % 16 || reinterpret_cast<uintptr_t>(p->v) % 16) return "cache not 16-byte aligned";
    if (reinterpret_cast<uintptr_t>(b->page_table) % 4 || reinterpret_cast<uintptr_t>(b->lengths) % 4 ||
        reinterpret_cast<uintptr_t>(b->starts) % 4 || reinterpret_cast<uintptr_t>(p->k_scale) % 4 ||
        reinterpret_cast<uintptr_t>(p->v_scale) % 4)
        return "misaligned tensor";
    return nullptr;
}

inline Batch device_batch(const se12_step_batch* b) {
    return {b->page_table, b->table_stride, b->lengths,  b->starts,
            b->table_width, b->sequences,   b->tokens, b->max_new < b->tokens ? b->max_new : b->tokens};
}

inline int log2_of(int n) { return 31 - __builtin_clz((unsigned)n); }

}  // namespace se12step
