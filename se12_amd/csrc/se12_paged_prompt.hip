// Attention over a paged cache for sequences with many new tokens (prompts, or
// parts of one behind what is held): the mathematics and the roundings of
// se12_paged_attention.hip, laid out for many columns ((token, query head) pairs of
// a KV head) that read the same keys.
//
// A block takes 128 columns, 32 a wave, and walks the key tiles they see. A tile's
// keys and values go from their pages into LDS as they are held (8 bits stay 8
// bits), one tile ahead, without passing registers, and each wave turns them into
// BF16 operands of v_mfma_f32_32x32x16_bf16 as it reads them (A: lane l holds row l %
// 32, inner positions 8 (l / 32) ..; B: the same of column l % 32; D: column l % 32,
// rows (i % 4) + 8 (i / 4) + 4 (l / 32)). Rows of the first product are keys in the
// order that leaves a lane's scores those of 16 keys in a row of its column, so they
// are the second product's operand where they are. The 16-byte pieces of a row lie in
// LDS in an order of its own, row by row, so that the 16 lanes that read the same
// piece of 16 rows take all banks once.
//
// Bound by the instructions of the one wave a SIMD has room for at head dim 256 (128
// sums, 64 registers of Q): of 3,190 cycles to 32 keys it issues for 2,230, 1,830 of them
// 374 vector and 32 matrix instructions (a third of the vector ones convert 8 bits), and
// waits for 680; the matrix unit is busy for 1,030, beside other instructions for the most
// part. 6,194 tokens of 5 prompts behind up to 1,500 keys, 8 / 4 heads of 256, E4M3, cap:
// 159 us, 0.53 PFLOP/s. BF16 pages: 5,040 cycles, 1,780 of them waits (tiles of 32 keys,
// so twice the barriers, and twice the bytes): 64 x 64 tokens behind 2,048 160 us, 113 from E4M3.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "se12_device.hpp"
#include "se12_paged_units.hpp"

namespace se12step {

constexpr int kPromptThreads = 256;
constexpr int kPromptWaves = kPromptThreads / 64;
constexpr int kWaveColumns = 32;
static_assert(kBlockColumns == kPromptWaves * kWaveColumns, "");
constexpr int kSubTile = 32;              // keys of a first product
constexpr int kSharedUnits = 1024;        // with more, blocks end close enough to each other as they are

// se12::lds_load16 from a uniform address and the lane's offset
__device__ __forceinline__ void lds_load16(const void* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}

// x by and x + y of a sum. At D = 256 in an accumulation register, where it is kept,
// written with the register's class: as ordinary arithmetic it makes the compiler keep
// all sums in vector registers as well, over the whole walk, and spill. The wait states
// it puts between matrix instructions and others do not cover these, so
// settle_products() stands on both sides: no matrix instruction is in flight for longer.
template <int D>
__device__ __forceinline__ float times(float x, float by) {
    if constexpr (D < 256) return x * by;
    float t;
    asm volatile("v_accvgpr_read_b32 %1, %0\n\ts_nop 1\n\tv_mul_f32 %1, %1, %2\n\ts_nop 1\n\tv_accvgpr_write_b32 %0, %1"
                 : "+a"(x), "=&v"(t) : "v"(by));
    return x;
}
template <int D>
__device__ __forceinline__ float plus(float x, float y) {
    if constexpr (D < 256) return x + y;
    float t;
    asm volatile("v_accvgpr_read_b32 %1, %0\n\ts_nop 1\n\tv_add_f32 %1, %1, %2\n\ts_nop 1\n\tv_accvgpr_write_b32 %0, %1"
                 : "+a"(x), "=&v"(t) : "v"(y));
    return x;
}
template <int D>
__device__ __forceinline__ void settle_products() {
    if constexpr (D == 256) asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15");
}

template <int CT, int D, bool kCapped>
__global__ __launch_bounds__(kPromptThreads, D == 64 || (D == 128 && CT == SE12_STEP_E4M3) ? 2 : 1) void paged_prompt_kernel(AttendArgs a) {
    using F = Form<CT>;
    constexpr int kTile = F::kTile, kSubs = kTile / kSubTile;
    constexpr int kKeyPieces = D / F::kPer;           // 16-byte pieces of a key
    constexpr int kValuePieces = kTile / F::kPer;     // and of a value column: 4
    constexpr int kHalfTile = 64 * D;                 // bytes of a tile's keys, or values
    constexpr int kLoads = kHalfTile / 1024 / kPromptWaves;   // of a wave, 64 pieces each
    constexpr int kRows = D / 32;
    static_assert(kValuePieces == 4 && kLoads >= 1, "");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];     // [2][keys, values]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int kh = blockIdx.x % a.kvh;
    const UnitWork u = unit_work(a, blockIdx.x / a.kvh);
    if (u.s < 0) return;
    const int t0 = u.t0, t1 = u.t1;

    const int col = lane & 31, half = lane >> 5;
    const int c0 = u.first + wave * kWaveColumns, mine = min(kWaveColumns, u.columns - c0);   // (may be none)
    const bool live = col < mine;
    const int c = live ? c0 + col : u.first, token = c / a.group;
    const int pos = live ? u.len + token : -1;
    const int pos_min = u.len + c0 / a.group, pos_max = mine > 0 ? u.len + (c0 + mine - 1) / a.group : -1;
    const int reach = a.window > 0 ? a.window : INT32_MAX;
    const int low = max(0, pos_min - reach + 1), high = min(u.keys, pos_max + 1);      // keys some column of the wave sees

    // Q: inner positions as the pieces of a key bring them
    constexpr int kQSteps = D / 16;
    bf16x8_t qf[kQSteps];
    floatx16_t o[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // Loads of a tile. Piece p of a row lies at place p ^ f(row): f of a key from the
    // four bits that tell the rows of 16 lanes apart, of a value column from two. A
    // wave's keys lie in one page (16 of a tile, or 8); a lane's values in the page of
    // its piece.
    const int P = 1 << a.page_log2;
    constexpr int kElem = 16 / F::kPer;
    const int32_t* table = a.b.table + u.s * a.b.table_stride;
    auto entry = [&](int key) { return table[min(key >> a.page_log2, a.b.width - 1)]; };
    auto in_pool = [&](int e) { return (uint32_t)e < (uint32_t)a.pages ? e : 0; };
    auto key_twist = [](int r) {
        const int b = (r & 7) | ((r & 16) >> 1);
        return kKeyPieces >= 16 ? b : b >> (kKeyPieces == 8 ? 1 : 2);
    };
    constexpr int kWaveKeys = kTile / kPromptWaves, kRowsPerLoad = 64 / kKeyPieces;
    static_assert(kLoads * kRowsPerLoad == kWaveKeys, "");
    const int vpiece = (lane & 3) ^ ((lane >> 4) & 3);
    const uint32_t lds0 = se12::lds_address(lds);
    uint32_t key_at[kLoads];      // the lane's bytes of a load, from the wave's first key
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int r = i * kRowsPerLoad + lane / kKeyPieces;
        key_at[i] = r * (D * kElem) + 16 * ((lane % kKeyPieces) ^ key_twist(wave * kWaveKeys + r));
    }
    struct Source {
        const uint8_t* from;
        uint32_t to;
    };
    auto keys_of = [&](int t, int buffer, int key_entry) {
        const int page = in_pool(__builtin_amdgcn_readfirstlane(key_entry)), first = (t * kTile + wave * kWaveKeys) & (P - 1);
        return Source{static_cast<const uint8_t*>(a.kc) + (((int64_t)page * a.kvh + kh) * P + first) * (D * kElem),
                      (uint32_t)(__builtin_amdgcn_readfirstlane(lds0 + buffer * 2 * kHalfTile) + wave * kLoads * 1024)};
    };
    auto values_of = [&](int t, int buffer, int value_entry) {
        return Source{static_cast<const uint8_t*>(a.vc) +
                          (((int64_t)in_pool(value_entry) * a.kvh + kh) * D + wave * kLoads * 16 + (lane >> 2)) * (int64_t)(P * kElem) +
                          ((t * kTile + vpiece * F::kPer) & (P - 1)) * kElem,
                      (uint32_t)(__builtin_amdgcn_readfirstlane(lds0 + buffer * 2 * kHalfTile) + kHalfTile + wave * kLoads * 1024)};
    };
    auto load_key = [&](const Source& x, int i) { lds_load16(x.from, key_at[i], x.to + i * 1024); };
    auto load_value = [&](const Source& x, int i) { se12::lds_load16(x.from + i * 16 * P * kElem, x.to + i * 1024); };
    auto load_keys = [&](int t, int buffer, int key_entry) {
        const Source x = keys_of(t, buffer, key_entry);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load_key(x, i);
    };
    auto load_values = [&](int t, int buffer, int value_entry) {
        const Source x = values_of(t, buffer, value_entry);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load_value(x, i);
    };
    auto key_entry_of = [&](int t) { return entry(t * kTile + wave * kWaveKeys); };
    auto value_entry_of = [&](int t) { return entry(t * kTile + vpiece * F::kPer); };
    // scales of the lane's 16 keys of each sub-tile, and whether a page holds them
    struct Lane {
        float ks0 = 1.0f, vs0 = 1.0f, ks1 = 1.0f, vs1 = 1.0f;
        int held0 = 0, held1 = 0;
    };
    auto lane_of = [&](int2 e) {
        Lane x;
        x.held0 = (uint32_t)e.x < (uint32_t)a.pages;
        x.held1 = (uint32_t)e.y < (uint32_t)a.pages;
        if constexpr (CT == SE12_STEP_E4M3) {
            const int64_t at0 = (int64_t)in_pool(e.x) * a.kvh + kh, at1 = (int64_t)in_pool(e.y) * a.kvh + kh;
            x.ks0 = a.k_scale[at0];
            x.vs0 = a.v_scale[at0];
            x.ks1 = a.k_scale[at1];
            x.vs1 = a.v_scale[at1];
        }
        return x;
    };
    auto lane_entries_of = [&](int t) {
        return make_int2(entry(t * kTile + 16 * half), entry(t * kTile + (kSubs - 1) * kSubTile + 16 * half));
    };
    auto arrived = [](Lane& x) {     // (loaded with what is waited for here)
        asm volatile("" : "+v"(x.ks0), "+v"(x.vs0), "+v"(x.ks1), "+v"(x.vs1), "+v"(x.held0), "+v"(x.held1));
    };
    // What the wave holds of a sub-tile of 32 keys: keys' pieces, value columns' pieces.
    constexpr int kKeyReads = kKeyPieces / 2, kValueReads = 2 / F::kHalves;
    uint4 kf[kKeyReads], vf[kRows];
    // (pieces 2 i + half of the lane's row: the place's bits and those of i meet in an
    // exclusive or, so one address gives all of them)
    const int key_row0 = key_of_row(col), key_off0 = key_row0 * (kKeyPieces * 16) + 16 * (half ^ key_twist(key_row0));
    auto read_keys = [&](int t, int j) {
        const int at = key_off0 + ((t - t0) & 1) * 2 * kHalfTile + j * kSubTile * kKeyPieces * 16;
#pragma unroll
        for (int i = 0; i < kKeyReads; ++i) kf[i] = *reinterpret_cast<const uint4*>(lds + (at ^ (32 * (i & 7))) + 256 * (i >> 3));
    };
    // (the n-th of the lane's pieces of each row)
    auto read_values = [&](int t, int j, int n) {
        const uint8_t* p = lds + (((t - t0) & 1) * 2 + 1) * kHalfTile;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int r = 32 * i + col, piece = CT == SE12_STEP_E4M3 ? 2 * j + half : 2 * half + n;
            vf[i] = *reinterpret_cast<const uint4*>(p + r * 64 + 16 * (piece ^ ((r >> 2) & 3)));
        }
    };
    auto mask_values = [&](int key0, bool held, int n) {
        const uint4 mask = piece_mask<CT>(low - key0 - n * F::kPer, held ? high - key0 - n * F::kPer : 0);
#pragma unroll
        for (int i = 0; i < kRows; ++i) vf[i] = masked(vf[i], mask);
    };
    auto numbers_of_values = [&]() {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            vf[i] = make_uint4(numbers_only<CT>(vf[i].x), numbers_only<CT>(vf[i].y), numbers_only<CT>(vf[i].z), numbers_only<CT>(vf[i].w));
    };
    auto any_no_number = [&]() {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kRows; ++i) bad |= has_no_number<CT>(vf[i]);
        return __builtin_amdgcn_ballot_w64(bad) != 0;
    };
    float sc[16], top = 0.0f;      // scores, or r of cap - 2 cap r
    // the values' scale, in the weights' exponent: log2, and its inverse
    float lv = CT == SE12_STEP_BF16 ? -a.shift : 0.0f, iv = 1.0f;
    bf16x8_t pf[2];
    auto weights = [&]() {
        const float base = (m == -INFINITY ? 0.0f : m) - lv;
        float sum = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float p0, p1;
                if constexpr (kCapped) {
                    p0 = __builtin_amdgcn_exp2f((a.cap - base) - 2.0f * a.cap * sc[8 * h + 2 * k]);
                    p1 = __builtin_amdgcn_exp2f((a.cap - base) - 2.0f * a.cap * sc[8 * h + 2 * k + 1]);
                } else {
                    p0 = __builtin_amdgcn_exp2f(sc[8 * h + 2 * k] - base);
                    p1 = __builtin_amdgcn_exp2f(sc[8 * h + 2 * k + 1] - base);
                }
                w[k] = f_to_bf16x2(p0, p1);
                // (the sum of what the product takes: two at once, times 1)
                sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w[k]), __builtin_bit_cast(bf16x2_t, 0x3F803F80u), sum, false);
            }
            pf[h] = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
        }
        l += sum * iv;
    };

    // The walk, sub-tile by sub-tile: scores of the next while the weights of this one are
    // worked out, then the product of its weights and values while the scores of the
    // next are capped; keys are in registers two sub-tiles ahead of the
    // values. At the start of a tile a barrier: its values and the keys kLead tiles on
    // have come (their loads were sent a tile ago), and every wave is done with what
    // the next loads overwrite.
    constexpr int kLead = 2 / kSubs;
    // `ke`, `ve`: table entries of the tiles whose keys and values are loaded next; `se`:
    // of the lane's keys two tiles on, for their scales. Behind the last tile it is loaded
    // again: nothing reads those places.
    auto to_last = [&](int t) { return min(t, t1 - 1); };
    int ke = key_entry_of(t0);
    load_keys(t0, 0, ke);
    Lane now = lane_of(lane_entries_of(t0)), next = lane_of(lane_entries_of(to_last(t0 + 1))), after = next;
    if constexpr (kLead == 2) {
        ke = key_entry_of(to_last(t0 + 1));
        asm volatile("" : "+v"(ke));
        load_keys(to_last(t0 + 1), 1, ke);
    }
    {
        const uint16_t* qp = a.q + (u.start + token) * a.q_stride + (int64_t)(kh * a.group + c % a.group) * D;
#pragma unroll
        for (int i = 0; i < kQSteps; ++i)
            qf[i] = *reinterpret_cast<const bf16x8_t*>(qp + (i / F::kHalves) * 2 * F::kPer + half * F::kPer + 8 * (i % F::kHalves));
    }
    // (in accumulation registers, which the products read as well)
    if constexpr (D == 256) {
#pragma unroll
        for (int i = 0; i < kQSteps; ++i) asm volatile("" : "+a"(qf[i]));
    }
    se12::wait_vector_loads();
    arrived(now);
    arrived(next);
    __syncthreads();
    floatx16_t d;
    auto scores = [&](auto beside) {
#pragma unroll
        for (int e = 0; e < 16; ++e) d[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < kKeyReads; ++i) {
            beside(i);
#pragma unroll
            for (int h = 0; h < F::kHalves; ++h)
                d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand<CT>(kf[i], h), qf[i * F::kHalves + h], d, 0, 0, 0);
        }
    };
    auto cap_scores = [&](float ks) {
        const float by = a.c1 * ks;
#pragma unroll
        for (int e = 0; e < 16; ++e)
            sc[e] = kCapped ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(d[e] * by)) : d[e] * by;
    };
    auto find_top = [&]() {
        top = sc[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = kCapped ? fminf(top, sc[e]) : fmaxf(top, sc[e]);
        if constexpr (kCapped) top = a.cap - 2.0f * a.cap * top;
    };
    read_keys(t0, 0);
    scores([](int) {});
    read_keys(t0 + 1 / kSubs, 1 % kSubs);
    cap_scores(now.ks0);
    find_top();
    // (a buffer is written again only behind a barrier that every wave reaches after its
    // reads: with kLead 2 the next keys go over those of t0, which all waves read above)
    if constexpr (kLead == 2) __syncthreads();
    ke = key_entry_of(to_last(t0 + kLead));
    int ve = value_entry_of(t0);
    asm volatile("" : "+v"(ke), "+v"(ve));
    load_keys(to_last(t0 + kLead), kLead & 1, ke);
    load_values(t0, 0, ve);
    ke = key_entry_of(to_last(t0 + kLead + 1));
    ve = value_entry_of(to_last(t0 + 1));
    int2 se = lane_entries_of(to_last(t0 + 2));

    auto move_maximum = [&]() {
        const float to = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
        const float scale = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= scale;
        settle_products<D>();
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] = times<D>(o[i][e], scale);
        settle_products<D>();
    };
    // 0 x NaN is NaN: what is no number comes in the columns that give it a weight (and
    // leaves the product)
    auto bring_no_numbers = [&](int t, int j, int key0, bool held) {
#pragma unroll
        for (int n = 0; n < kValueReads; ++n) {
            read_values(t, j, n);
            mask_values(key0, held, n);
#pragma unroll
            for (int i = 0; i < kRows; ++i)
#pragma unroll
                for (int kind = 0; kind < (CT == SE12_STEP_E4M3 ? 1 : 3); ++kind) {
                    __builtin_amdgcn_sched_barrier(0);
                    settle_products<D>();
                    floatx16_t x;
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = 0.0f;
#pragma unroll
                    for (int h = 0; h < F::kHalves; ++h) {
                        const uint4 w = __builtin_bit_cast(uint4, operand<CT>(vf[i], h));
                        const uint4 is = make_uint4(where_no_number(w.x, kind), where_no_number(w.y, kind),
                                                    where_no_number(w.z, kind), where_no_number(w.w, kind));
                        x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, is), pf[n + h], x, 0, 0, 0);
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        o[i][e] = plus<D>(o[i][e], x[e] == 0.0f ? 0.0f : kind == 0 ? __builtin_nanf("") : kind == 1 ? INFINITY : -INFINITY);
                }
        }
        settle_products<D>();
    };
    auto edge = []() { asm volatile(""); };
    for (int t = t0; t < t1; ++t) {
        se12::wait_vector_loads();
        if (t > t0) {
            now = next;
            next = after;
        }
        arrived(next);
        asm volatile("" : "+v"(ke), "+v"(ve), "+v"(se.x), "+v"(se.y));
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kSubs; ++j) {
            const int k0 = (t * kSubs + j) * kSubTile, key0 = k0 + 16 * half;
            const bool held = ((j ? now.held1 : now.held0) != 0) & (key0 < high) & (key0 + 16 > low);
            const bool inside = (k0 + kSubTile - 1 <= pos_min) & (k0 + kSubTile <= u.keys) & (pos_max - k0 < reach) &
                                (__builtin_amdgcn_ballot_w64(!held) == 0);
            if constexpr (CT == SE12_STEP_E4M3) {
                const float vs = j ? now.vs1 : now.vs0;
                lv = __builtin_amdgcn_logf(vs);
                iv = __builtin_amdgcn_rcpf(vs);
            }
            bool apart = false;      // a value that is no number may be hidden from some of the columns
            // (edge(): what follows is left to the sub-tiles that need it, not worked out for
            // all and chosen from)
            if (!inside) {
                edge();
                if constexpr (CT == SE12_STEP_E4M3) {
                    // (what no page holds, or nobody sees, has any scale; its weights are 0)
                    lv = held ? lv : 0.0f;
                    iv = held ? iv : 0.0f;
                }
                const int since = max(pos - reach + 1, 0) - key0, to = held ? min(pos + 1, u.keys) - key0 : 0;
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[e] = (e < since || e >= to) ? (kCapped ? INFINITY : -INFINITY) : sc[e];
                find_top();
#pragma unroll
                for (int n = 1; n < kValueReads; ++n) {
                    read_values(t, j, n);
                    mask_values(key0, held, n);
                    apart |= any_no_number();
                }
            }
            read_values(t, j, 0);
            if (!inside) {
                edge();
                mask_values(key0, held, 0);
                apart |= any_no_number();
            }
            if (__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0) move_maximum();
            // The loads of the tiles to come, one beside every other row's products, the values'
            // here and the keys' below: a wave waits for as long as a load is not taken.
            // (Both below, 64 x 64 tokens behind 2,048, heads of 256: 133 us as well from E4M3
            // pages, 194 for 170 from BF16; the values' a sub-tile later: 139 and 184.)
            const Source vs = values_of(to_last(t + 1), (t + 1 - t0) & 1, ve);
            if (j == 0) {
                ve = value_entry_of(to_last(t + 2));
                after = lane_of(se);
                se = lane_entries_of(to_last(t + 3));
            }
            scores([&](int i) {
                if (j == 0 && i % (kKeyReads / kLoads) == 0) load_value(vs, i / (kKeyReads / kLoads));
            });
            weights();
            if (apart) {
                bring_no_numbers(t, j, key0, held);
                read_values(t, j, 0);
                mask_values(key0, held, 0);
                numbers_of_values();
            }
            static_assert(kRows == 2 * kLoads && kKeyReads % kLoads == 0, "");
            const Source ks = keys_of(to_last(t + kLead + 1), (t + kLead + 1 - t0) & 1, ke);
            if (j == 0) ke = key_entry_of(to_last(t + kLead + 2));
            __builtin_amdgcn_sched_barrier(0);
            read_keys(t + (j + 2) / kSubs, (j + 2) % kSubs);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < kValueReads; ++n) {
                if (n > 0) {
                    read_values(t, j, n);
                    if (!inside) {
                        edge();
                        mask_values(key0, held, n);
                        if (apart) numbers_of_values();
                    }
                }
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    if (n == 0 && j == 0 && i % 2 == 0) load_key(ks, i / 2);
#pragma unroll
                    for (int h = 0; h < F::kHalves; ++h)
                        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand<CT>(vf[i], h), pf[n + h], o[i], 0, 0, 0);
                }
            }
            cap_scores(j + 1 < kSubs ? now.ks1 : next.ks0);
            find_top();
        }
    }
    se12::wait_vector_loads();      // (before this block's LDS is another's)
    l += __shfl_xor(l, 32, 64);
    if (u.parts > 1) {
        // the part, as the lanes hold it
        const int64_t p = part_place(a, u, kh);
        float4* to = reinterpret_cast<float4*>(a.part + p * kBlockColumns * D) + wave * (D / 8) * 64 + lane;
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                to[(4 * i + g) * 64] = make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
        if (half == 0)
            reinterpret_cast<float2*>(a.part + (int64_t)a.parts * a.kvh * kBlockColumns * D)[p * kBlockColumns + wave * kWaveColumns + col] =
                make_float2(m, l);
        return;
    }
    // Through LDS to whole rows (a lane holds four values of a row in a row; written from
    // there, 8 bytes of 64 rows at once, they took 11,000 cycles of a block). The 16-byte
    // pieces of a row in an order of its own, as those of the keys.
    __syncthreads();
    constexpr int kOutPieces = D / 8, kTwist = kOutPieces < 16 ? kOutPieces - 1 : 15, kRowsAtOnce = 64 / kOutPieces;
    uint8_t* own = lds + wave * kWaveColumns * 2 * D;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            store4(reinterpret_cast<uint16_t*>(own + col * 2 * D + 16 * ((4 * i + g) ^ (col & kTwist)) + 8 * half), o[i][4 * g] * inv,
                   o[i][4 * g + 1] * inv, o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int k = 0; k < kWaveColumns / kRowsAtOnce; ++k) {
        const int r = k * kRowsAtOnce + lane / kOutPieces, piece = lane % kOutPieces, x = c0 + r;
        if (r >= mine) continue;
        const uint4 v = *reinterpret_cast<const uint4*>(own + r * 2 * D + 16 * (piece ^ (r & kTwist)));
        *reinterpret_cast<uint2*>(a.out + ((int64_t)(u.start + x / a.group) * a.heads + kh * a.group + x % a.group) * D + 8 * piece) =
            make_uint2(v.x, v.y);
        *reinterpret_cast<uint2*>(a.out + ((int64_t)(u.start + x / a.group) * a.heads + kh * a.group + x % a.group) * D + 8 * piece + 4) =
            make_uint2(v.z, v.w);
    }
}

namespace {

template <int CT, int D>
void launch(const AttendArgs& a, hipStream_t st) {
    const int grid = a.unit_count * a.kvh;
    if (a.cap > 0.0f)
        hipLaunchKernelGGL((paged_prompt_kernel<CT, D, true>), dim3(grid), dim3(kPromptThreads), 4 * 64 * D, st, a);
    else
        hipLaunchKernelGGL((paged_prompt_kernel<CT, D, false>), dim3(grid), dim3(kPromptThreads), 4 * 64 * D, st, a);
}

}  // namespace

// A sequence has units only with more than kFewColumns columns, so at most one of so many
// of all columns does, and its last unit holds one column at least. Parts: twice a round's
// blocks (Sharing), or where few units can be as many as the rule for `splits` asks for.
// Where there are many units none is shared, but the memory stays: no call takes less than
// one of fewer tokens.
PromptPlan prompt_plan(const Batch& b, int kvh, int group, int page_size, int d, int dtype) {
    const int64_t columns = (int64_t)b.tokens * group, many = std::min<int64_t>(b.seqs, columns / (kFewColumns + 1));
    const int64_t resident = resident_blocks(dtype, d);
    PromptPlan x;
    x.slots = (columns + (kBlockColumns - 1) * many) / kBlockColumns;
    x.most = (int)(((int64_t)b.width * page_size + 32 * kLeastTiles - 1) / (32 * kLeastTiles));
    int64_t parts = std::min(std::min(2 * resident, std::max(resident, 2 * x.slots * kvh)) / kvh, x.slots * x.most);
    if (x.most < 2 || parts < 2) parts = 0;
    x.parts = columns / kBlockColumns * kvh > kSharedUnits ? 0 : (int)parts;
    x.records = x.slots + parts + parts / 2;
    x.record_bytes = (x.records * (int64_t)sizeof(UnitWork) + 255) / 256 * 256;
    x.part_bytes = parts * kvh * kBlockColumns * (d + 2) * (int64_t)sizeof(float);
    return x;
}

void launch_prompt(const AttendArgs& a, int dtype, int d, hipStream_t st) {
    if (dtype == SE12_STEP_E2M1) return launch_prompt4(a, d, st);
    const bool e4m3 = dtype == SE12_STEP_E4M3;
    switch (d) {
        case 64: e4m3 ? launch<SE12_STEP_E4M3, 64>(a, st) : launch<SE12_STEP_BF16, 64>(a, st); break;
        case 128: e4m3 ? launch<SE12_STEP_E4M3, 128>(a, st) : launch<SE12_STEP_BF16, 128>(a, st); break;
        default: e4m3 ? launch<SE12_STEP_E4M3, 256>(a, st) : launch<SE12_STEP_BF16, 256>(a, st);
    }
}

}  // namespace se12step
