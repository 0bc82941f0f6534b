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
// positions len ..; what the device memory says is kept inside the call's rows, and
// positions inside 31 bits (those behind the table's last column are held nowhere)
struct Seq {
    int start, n, len;
};

__device__ __forceinline__ Seq load_seq(const Batch& b, int s) {
    const int a = min(max(b.starts[s], 0), b.tokens);
    const int e = min(max(b.starts[s + 1], a), b.tokens);
    return {a, min(e - a, b.max_new), min(max(b.lengths[s], 0), (1 << 30) - 1)};
}

// the page holding column `c` of sequence s's table row, or -1
__device__ __forceinline__ int page_of(const Batch& b, int s, int c, int pages) {
    if (c < 0 || c >= b.width) return -1;
    const int id = b.table[s * b.table_stride + c];
    return (uint32_t)id < (uint32_t)pages ? id : -1;
}

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));

constexpr float kSlack = 16.0f;       // how far a score may pass the maximum it is taken from, base 2

struct AttendArgs {
    const uint16_t* q;
    int64_t q_stride;
    uint16_t* out;
    const void* kc;
    const void* vc;
    const float* k_scale;
    const float* v_scale;
    Batch b;
    int heads, kvh, group, pages, page_log2, window;
    float c1, cap;       // scores: c1 x (no cap), or cap - 2 cap / (1 + 2^(c1 x)), base 2
    // BF16 pages: weights are 2^-shift of what they are, so that they add up to less than
    // one and sums of any finite values stay finite (the largest weight is 2^-47 at least).
    // An E4M3 page's scale takes that range: with weights up to 2^kSlack, values of up to
    // 2^112 / keys are safe, and pages of the least scale, 2^-100, keep weights of 2^-26.
    float shift;
    float* part;         // sums of a part of a unit's keys, then their (m, l)
    int workers, columns;
    // sequences of more than kFewColumns columns are se12_paged_prompt.hip's: what its
    // blocks are to do, and the blocks that join parts (se12_paged_units.hpp)
    struct UnitWork* units;
    int unit_count, join_count;
    int parts;           // blocks of a KV head that may hold parts of a unit's keys, 0 for none
    int most;            // parts of a unit, at most
};

// What a lane holds of a tile, by the cache's type: 16 bytes of each key row's
// 64-byte part, and the lane's keys of a value column, 16 bytes as well.
template <int CT>
struct Form {
    static constexpr int kPer = CT == SE12_STEP_E4M3 ? 16 : 8;   // values of 16 bytes, and keys of a lane
    static constexpr int kTile = 4 * kPer;                        // keys of a tile
    static constexpr int kHalves = kPer / 8;                      // matrix operands of a piece
    static constexpr int kWord = kPer / 4;                        // values of a 32-bit word
};

template <int CT>
__device__ __forceinline__ uint4 load_piece(const void* p, int64_t i) {
    return *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + i * (16 / Form<CT>::kPer));
}

// values 8 h .. 8 h + 7 of a piece in BF16 (every E4M3 value is one)
template <int CT>
__device__ __forceinline__ bf16x8_t operand(const uint4 v, int h) {
    if constexpr (CT == SE12_STEP_E4M3) {
        const uint32_t a = h ? v.z : v.x, b = h ? v.w : v.y;
        const bf16x2_t w0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
        const bf16x2_t w1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
        const bf16x2_t w2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
        const bf16x2_t w3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
        return bf16x8_t{w0.x, w0.y, w1.x, w1.y, w2.x, w2.y, w3.x, w3.y};
    } else {
        return __builtin_bit_cast(bf16x8_t, v);
    }
}

// the bits of values from .. to - 1 of the kWord values of a word
template <int CT>
__device__ __forceinline__ uint32_t word_mask(int from, int to) {
    constexpr int per = Form<CT>::kWord, bits = 32 / per;
    const uint32_t below_to = to <= 0 ? 0u : to >= per ? ~0u : (1u << (bits * to)) - 1u;
    const uint32_t below_from = from <= 0 ? 0u : from >= per ? ~0u : (1u << (bits * from)) - 1u;
    return below_to & ~below_from;
}

template <int CT>
__device__ __forceinline__ uint4 piece_mask(int from, int to) {
    constexpr int per = Form<CT>::kWord;
    return make_uint4(word_mask<CT>(from, to), word_mask<CT>(from - per, to - per), word_mask<CT>(from - 2 * per, to - 2 * per),
                      word_mask<CT>(from - 3 * per, to - 3 * per));
}

__device__ __forceinline__ uint4 masked(const uint4 v, const uint4 m) { return make_uint4(v.x & m.x, v.y & m.y, v.z & m.z, v.w & m.w); }

// bit 7 of every value (bit 15 of a BF16 one) that is a NaN or an infinity:
// exponent all ones; E4M3: all ones but the sign
template <int CT>
__device__ __forceinline__ uint32_t no_numbers(uint32_t w) {
    return CT == SE12_STEP_E4M3 ? ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u : ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
}

template <int CT>
__device__ __forceinline__ bool has_no_number(const uint4 v) {
    return (no_numbers<CT>(v.x) | no_numbers<CT>(v.y) | no_numbers<CT>(v.z) | no_numbers<CT>(v.w)) != 0;
}

template <int CT>
__device__ __forceinline__ uint32_t numbers_only(uint32_t w) {
    return CT == SE12_STEP_E4M3 ? w & ~((no_numbers<CT>(w) >> 7) * 0xFFu) : w & ~((no_numbers<CT>(w) >> 15) * 0xFFFFu);
}

// BF16 values: 1 where a value is a NaN (kind 0), +inf (1) or -inf (2), else 0
__device__ __forceinline__ uint32_t where_no_number(uint32_t w, int kind) {
    const uint32_t all = no_numbers<SE12_STEP_BF16>(w) >> 8, fraction = ((w & 0x007F007Fu) + 0x007F007Fu) & 0x00800080u;
    const uint32_t is = kind == 0 ? all & fraction : kind == 1 ? all & ~fraction & ~(w >> 8) : all & ~fraction & (w >> 8);
    return is * 0x7Fu;
}

__device__ __forceinline__ void store4(uint16_t* p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(p) = make_uint2(f_to_bf16x2(a, b), f_to_bf16x2(c, d));
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

// host: whether `a_bytes` from a and `b_bytes` from b have a byte in common
inline bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}

// host: caps whose factors FP32 holds (the cap's form holds a score to 2^-22 of the cap)
inline bool softcap_fits(float cap) { return cap == 0.0f || (cap >= 0x1p-60f && cap <= 1024.0f); }

// se12_paged_prompt.hip: what a call can have of it
struct PromptPlan {
    int64_t slots;               // units of a KV head, at most
    int parts, most;             // as AttendArgs
    int64_t records, record_bytes, part_bytes;
};
PromptPlan prompt_plan(const Batch& b, int kvh, int group, int page_size, int d, bool e4m3);
void launch_prompt(const AttendArgs& a, bool e4m3, int d, hipStream_t st);

inline int log2_of(int n) { return 31 - __builtin_clz((unsigned)n); }

}  // namespace se12step
