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
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "se12_device.hpp"
#include "se12_paged_device.hpp"

namespace se12step {

typedef float floatx16_t __attribute__((ext_vector_type(16)));

constexpr int kPromptThreads = 256;
constexpr int kPromptWaves = kPromptThreads / 64;
constexpr int kWaveColumns = 32;
constexpr int kBlockColumns = kPromptWaves * kWaveColumns;
constexpr int kSubTile = 32;              // keys of a first product
constexpr int kLeastTiles = 8;            // of a block, where a unit's keys are split

// the key (of 32) of row m of the first product's A operand: lane half h = bit 2 of
// m takes keys 16 h ..
__device__ __forceinline__ int key_of_row(int m) { return (m & 3) | ((m & 8) >> 1) | ((m & 16) >> 1) | ((m & 4) << 2); }

// one unit: 128 columns of a sequence and KV head
struct Unit {
    int s, first;          // sequence, its first column of the unit
    Seq seq;
    int keys, columns;     // of the sequence
};

// Unit slots: sequence s has slots starts[s] * group / 128 + s onwards, enough for
// its ceil(n group / 128) units.
__device__ __forceinline__ bool find_unit(const AttendArgs& a, int slot, Unit& u) {
    auto base = [&](int s) { return (int)((int64_t)min(max(a.b.starts[s], 0), a.b.tokens) * a.group / kBlockColumns) + s; };
    int lo = 0, hi = a.b.seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (base(mid) <= slot)
            lo = mid;
        else
            hi = mid;
    }
    // (the same for all lanes, and kept in scalar registers)
    lo = __builtin_amdgcn_readfirstlane(lo);
    u.s = lo;
    const int capacity = a.b.width << a.page_log2;
    const Seq seq = load_seq(a.b, lo, capacity);
    u.seq = {__builtin_amdgcn_readfirstlane(seq.start), __builtin_amdgcn_readfirstlane(seq.n), __builtin_amdgcn_readfirstlane(seq.len)};
    u.keys = min(u.seq.len + u.seq.n, capacity);
    u.columns = u.seq.n * a.group;
    const int64_t first = (int64_t)(slot - __builtin_amdgcn_readfirstlane(base(lo))) * kBlockColumns;
    u.first = (int)first;
    return first >= 0 && first < u.columns && u.columns > a.few;
}

// the key tiles the unit's columns see
template <int kTile>
__device__ __forceinline__ void unit_tiles(const AttendArgs& a, const Unit& u, int& t0, int& t1) {
    const int pos0 = u.seq.len + u.first / a.group;
    const int pos1 = u.seq.len + (min(u.first + kBlockColumns, u.columns) - 1) / a.group;
    t0 = (a.window > 0 ? max(0, pos0 - a.window + 1) : 0) / kTile;
    t1 = max((min(u.keys, pos1 + 1) + kTile - 1) / kTile, t0 + 1);
}

template <int CT, int D, bool kCapped>
__global__ __launch_bounds__(kPromptThreads, 1) void paged_prompt_kernel(AttendArgs a) {
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
    const int kh = blockIdx.x % a.kvh, rest = blockIdx.x / a.kvh, split = rest % a.splits;
    const int slot = (int)(gridDim.x / a.kvh / a.splits) - 1 - rest / a.splits;   // the last columns, with the most keys, first
    Unit u;
    if (!find_unit(a, slot, u)) return;
    int t0, t1;
    unit_tiles<kTile>(a, u, t0, t1);
    const int length = max((t1 - t0 + a.splits - 1) / a.splits, kLeastTiles);
    const bool whole = t1 - t0 <= length;
    t0 += split * length;
    t1 = min(t1, t0 + length);
    if (t0 >= t1) return;

    const int col = lane & 31, half = lane >> 5;
    const int c0 = u.first + wave * kWaveColumns, mine = min(kWaveColumns, u.columns - c0);   // (may be none)
    const bool live = col < mine;
    const int c = live ? c0 + col : u.first, token = c / a.group;
    const int pos = live ? u.seq.len + token : -1;
    const int pos_min = u.seq.len + c0 / a.group, pos_max = mine > 0 ? u.seq.len + (c0 + mine - 1) / a.group : -1;
    const int reach = a.window > 0 ? a.window : INT32_MAX;
    const int low = max(0, pos_min - reach + 1), high = min(u.keys, pos_max + 1);      // keys some column of the wave sees

    // Q: inner positions as the pieces of a key bring them
    constexpr int kQSteps = D / 16;
    bf16x8_t qf[kQSteps];
    {
        const uint16_t* qp = a.q + (u.seq.start + token) * a.q_stride + (int64_t)(kh * a.group + c % a.group) * D;
#pragma unroll
        for (int i = 0; i < kQSteps; ++i)
            qf[i] = *reinterpret_cast<const bf16x8_t*>(qp + (i / F::kHalves) * 2 * F::kPer + half * F::kPer + 8 * (i % F::kHalves));
    }
    floatx16_t o[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // Loads of a tile. Piece p of a row lies at place p ^ f(row): f of a key from the
    // four bits that tell the rows of 16 lanes apart, of a value column from two.
    const int P = 1 << a.page_log2;
    constexpr int kElem = 16 / F::kPer;
    const int32_t* table = a.b.table + u.s * a.b.table_stride;
    auto entry = [&](int key) { return table[min(key >> a.page_log2, a.b.width - 1)]; };
    auto in_pool = [&](int e) { return (uint32_t)e < (uint32_t)a.pages ? e : 0; };
    auto key_twist = [](int r) {
        const int b = (r & 7) | ((r & 16) >> 1);
        return kKeyPieces >= 16 ? b : b >> (kKeyPieces == 8 ? 1 : 2);
    };
    constexpr int kRowsPerLoad = 64 / kKeyPieces;     // keys of one load, of one group of 16
    const int vpiece = (lane & 3) ^ ((lane >> 4) & 3);
    const uint32_t lds0 = se12::lds_address(lds);
    auto load_tile = [&](int t, int buffer, int key_entry, int value_entry) {
        const int k0 = t * kTile;
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + buffer * 2 * kHalfTile);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int n = wave * kLoads + i;
            const int r = n * kRowsPerLoad + lane / kKeyPieces, g = n * kRowsPerLoad / 16;
            const int page = in_pool(__builtin_amdgcn_readlane(key_entry, g));
            const int piece = (lane % kKeyPieces) ^ key_twist(r);
            const int64_t at = (((int64_t)page * a.kvh + kh) * P + ((k0 + r) & (P - 1))) * (D * kElem) + 16 * piece;
            se12::lds_load16(static_cast<const uint8_t*>(a.kc) + at, to + n * 1024);
        }
        const int64_t vbase = (((int64_t)in_pool(value_entry) * a.kvh + kh) * D + (lane >> 2)) * (int64_t)(P * kElem) +
                              ((k0 + vpiece * F::kPer) & (P - 1)) * kElem;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int n = wave * kLoads + i;
            se12::lds_load16(static_cast<const uint8_t*>(a.vc) + vbase + (int64_t)n * 16 * P * kElem, to + kHalfTile + n * 1024);
        }
    };
    auto key_entry_of = [&](int t) { return entry(t * kTile + 16 * (lane & (kTile / 16 - 1))); };
    auto value_entry_of = [&](int t) { return entry(t * kTile + vpiece * F::kPer); };
    // scales of the lane's 16 keys of each sub-tile, and whether a page holds them
    struct Lane {
        float ks[kSubs], vs[kSubs];
        int held[kSubs];
    };
    auto lane_of = [&](int key_entry) {
        Lane x;
#pragma unroll
        for (int j = 0; j < kSubs; ++j) {
            const int e = __shfl(key_entry, 2 * j + half, 64);
            x.held[j] = (uint32_t)e < (uint32_t)a.pages;
            x.ks[j] = x.vs[j] = 1.0f;
            if constexpr (CT == SE12_STEP_E4M3) {
                const int64_t at = (int64_t)in_pool(e) * a.kvh + kh;
                x.ks[j] = a.k_scale[at];
                x.vs[j] = a.v_scale[at];
            }
        }
        return x;
    };
    // What the wave holds of a sub-tile of 32 keys: keys' pieces, value columns' pieces.
    constexpr int kKeyReads = kKeyPieces / 2, kValueReads = 2 / F::kHalves;
    // (of a key no more than 8 pieces at once)
    constexpr int kAhead = kKeyReads < 8 ? kKeyReads : 8;
    uint4 kf[kAhead], vf[kRows][kValueReads];
    auto key_piece = [&](int t, int j, int i) {
        const int row = j * kSubTile + key_of_row(col), twist = key_twist(row);
        const uint8_t* p = lds + ((t - t0) & 1) * 2 * kHalfTile + row * (kKeyPieces * 16);
        return *reinterpret_cast<const uint4*>(p + 16 * ((2 * i + half) ^ twist));
    };
    auto read_keys = [&](int t, int j) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) kf[i] = key_piece(t, j, i);
    };
    auto read_values = [&](int t, int j) {
        const uint8_t* p = lds + (((t - t0) & 1) * 2 + 1) * kHalfTile;
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int n = 0; n < kValueReads; ++n) {
                const int r = 32 * i + col, piece = CT == SE12_STEP_E4M3 ? 2 * j + half : 2 * half + n;
                vf[i][n] = *reinterpret_cast<const uint4*>(p + r * 64 + 16 * (piece ^ ((r >> 2) & 3)));
            }
    };
    float sc[16], top = 0.0f, vs = 1.0f;    // sc: scores, or r of cap - 2 cap r
    bf16x8_t pf[2];
    auto weights = [&]() {
        const float base = m == -INFINITY ? 0.0f : m;
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
                l += p0 + p1;
                if constexpr (CT == SE12_STEP_E4M3)
                    w[k] = f_to_bf16x2(p0 * vs, p1 * vs);
                else
                    w[k] = f_to_bf16x2(p0, p1);
            }
            pf[h] = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
        }
    };

    int ke = key_entry_of(t0), ve = value_entry_of(t0);
    Lane now, next = lane_of(ke);
    load_tile(t0, 0, ke, ve);
    ke = key_entry_of(min(t0 + 1, t1 - 1));
    ve = value_entry_of(min(t0 + 1, t1 - 1));
    // Tile t + 1 (its loads were sent a tile ago) takes over: after the barrier it is
    // whole, and every wave is done with tile t, whose place tile t + 2 may take.
    auto next_tile = [&](int t) {
        se12::wait_vector_loads();
        now = next;
#pragma unroll
        for (int j = 0; j < kSubs; ++j) asm volatile("" : "+v"(now.ks[j]), "+v"(now.vs[j]), "+v"(now.held[j]));
        asm volatile("" : "+v"(ke), "+v"(ve));
        __syncthreads();
        if (t + 2 < t1) {
            next = lane_of(ke);
            load_tile(t + 2, (t - t0) & 1, ke, ve);
            ke = key_entry_of(min(t + 3, t1 - 1));
            ve = value_entry_of(min(t + 3, t1 - 1));
        }
    };
    next_tile(t0 - 1);
    read_keys(t0, 0);
    bool known = false;      // what is no number in the sub-tile's values has been dealt with
    for (int n32 = t0 * kSubs; n32 < t1 * kSubs;) {
        bool apart = false;
        for (; n32 < t1 * kSubs; ++n32) {
            const int t = n32 / kSubs, j = n32 % kSubs, k0 = n32 * kSubTile, key0 = k0 + 16 * half;
            floatx16_t d;
#pragma unroll
            for (int e = 0; e < 16; ++e) d[e] = 0.0f;
#pragma unroll
            for (int i = 0; i < kKeyReads; ++i) {
#pragma unroll
                for (int h = 0; h < F::kHalves; ++h)
                    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand<CT>(kf[i % kAhead], h), qf[i * F::kHalves + h], d, 0, 0, 0);
                if (i + kAhead < kKeyReads) kf[i % kAhead] = key_piece(t, j, i + kAhead);
            }
            __builtin_amdgcn_sched_barrier(0);
            read_values(t, j);
            __builtin_amdgcn_sched_barrier(0);
            const float by = a.c1 * (j ? now.ks[kSubs - 1] : now.ks[0]);
#pragma unroll
            for (int e = 0; e < 16; ++e)
                sc[e] = kCapped ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(d[e] * by)) : d[e] * by;
            const bool held = (j ? now.held[kSubs - 1] : now.held[0]) != 0 && key0 < high && key0 + 16 > low;
            const bool inside = k0 + kSubTile - 1 <= pos_min && k0 + kSubTile <= u.keys && pos_max - k0 < reach &&
                                __builtin_amdgcn_ballot_w64(!held) == 0;
            vs = j ? now.vs[kSubs - 1] : now.vs[0];
            if (!inside) {
                vs = held ? vs : 0.0f;
                const int since = max(pos - reach + 1, 0) - key0, to = held ? min(pos + 1, u.keys) - key0 : 0;
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[e] = (e < since || e >= to) ? (kCapped ? INFINITY : -INFINITY) : sc[e];
                bool bad = false;
#pragma unroll
                for (int n = 0; n < kValueReads; ++n) {
                    const uint4 mask = piece_mask<CT>(low - key0 - n * F::kPer, held ? high - key0 - n * F::kPer : 0);
#pragma unroll
                    for (int i = 0; i < kRows; ++i) {
                        vf[i][n] = masked(vf[i][n], mask);
                        bad |= has_no_number<CT>(vf[i][n]);
                        if (known)
                            vf[i][n] = make_uint4(numbers_only<CT>(vf[i][n].x), numbers_only<CT>(vf[i][n].y),
                                                  numbers_only<CT>(vf[i][n].z), numbers_only<CT>(vf[i][n].w));
                    }
                }
                apart = !known && __builtin_amdgcn_ballot_w64(bad) != 0;
            }
            top = sc[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) top = kCapped ? fminf(top, sc[e]) : fmaxf(top, sc[e]);
            if constexpr (kCapped) top = a.cap - 2.0f * a.cap * top;
            if (n32 == t0 * kSubs) m = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0 || apart) break;
            weights();
            known = false;
            // (after the last sub-tile its own keys again: on every path as many reads,
            // so that the waits below count exactly)
            if (j == kSubs - 1 && t + 1 < t1) next_tile(t);
            const int n = min(n32 + 1, t1 * kSubs - 1);
            read_keys(n / kSubs, n % kSubs);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kRows; ++i)
#pragma unroll
                for (int n = 0; n < kValueReads; ++n)
#pragma unroll
                    for (int h = 0; h < F::kHalves; ++h)
                        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand<CT>(vf[i][n], h), pf[n + h], o[i], 0, 0, 0);
        }
        if (n32 >= t1 * kSubs) break;
        // The rare sub-tile, outside the loop, where the sums may stay in accumulation
        // registers: the maximum moves, and what is summed with it; 0 x NaN is NaN, so
        // a value that is no number comes in the columns that give it a weight, and
        // leaves the product. Then the sub-tile starts again.
        const float to = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
        const float scale = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= scale;
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] *= scale;
        if (apart) {
            const float sum = l;
            weights();
            l = sum;
#pragma unroll
            for (int i = 0; i < kRows; ++i)
#pragma unroll
                for (int n = 0; n < kValueReads; ++n) {
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int kind = 0; kind < (CT == SE12_STEP_E4M3 ? 1 : 3); ++kind) {
                        floatx16_t x;
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[e] = 0.0f;
#pragma unroll
                        for (int h = 0; h < F::kHalves; ++h) {
                            const uint4 w = __builtin_bit_cast(uint4, operand<CT>(vf[i][n], h));
                            const uint4 is = make_uint4(where_no_number(w.x, kind), where_no_number(w.y, kind),
                                                        where_no_number(w.z, kind), where_no_number(w.w, kind));
                            x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, is), pf[n + h], x, 0, 0, 0);
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            o[i][e] += x[e] == 0.0f ? 0.0f : kind == 0 ? __builtin_nanf("") : kind == 1 ? INFINITY : -INFINITY;
                    }
                }
            known = true;
        }
        read_keys(n32 / kSubs, n32 % kSubs);
    }
    l += __shfl_xor(l, 32, 64);
    if (!live) return;
    if (whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* out = a.out + ((int64_t)(u.seq.start + token) * a.heads + kh * a.group + c % a.group) * D + 4 * half;
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                store4(out + 32 * i + 8 * g, o[i][4 * g] * inv, o[i][4 * g + 1] * inv, o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv);
        return;
    }
    // the part of (slot, head, split)
    const int64_t p = (((int64_t)slot * a.kvh + kh) * a.splits + split) * kBlockColumns + wave * kWaveColumns + col;
    float* to = a.part + p * D + 4 * half;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4*>(to + 32 * i + 8 * g) = make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
    if (half == 0) {
        float* ml = a.part + (int64_t)(gridDim.x) * kBlockColumns * D + 2 * p;
        ml[0] = m;
        ml[1] = l;
    }
}

// Units whose keys were split, from their parts in order: a wave per column.
template <int CT, int D>
__global__ __launch_bounds__(kPromptThreads) void paged_prompt_join_kernel(AttendArgs a, int64_t parts) {
    constexpr int kTile = Form<CT>::kTile, kPerLane = D / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int kh = blockIdx.x % a.kvh, slot = blockIdx.x / a.kvh;
    Unit u;
    if (!find_unit(a, slot, u)) return;
    int t0, t1;
    unit_tiles<kTile>(a, u, t0, t1);
    const int length = max((t1 - t0 + a.splits - 1) / a.splits, kLeastTiles), count = (t1 - t0 + length - 1) / length;
    const int c = blockIdx.y * kPromptWaves + wave;
    if (count <= 1 || u.first + c >= u.columns) return;
    const int64_t p0 = ((int64_t)slot * a.kvh + kh) * a.splits * kBlockColumns + c;
    const float* ml = a.part + parts * kBlockColumns * D;
    float m = -INFINITY;
    for (int k = 0; k < count; ++k) m = fmaxf(m, ml[2 * (p0 + (int64_t)k * kBlockColumns)]);
    const float top = m == -INFINITY ? 0.0f : m;
    float o[kPerLane] = {}, l = 0.0f;
    for (int k = 0; k < count; ++k) {
        const int64_t p = p0 + (int64_t)k * kBlockColumns;
        const float by = __builtin_amdgcn_exp2f(ml[2 * p] - top);
        l += by * ml[2 * p + 1];
#pragma unroll
        for (int e = 0; e < kPerLane; ++e) o[e] += by * a.part[p * D + 64 * e + lane];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int col = u.first + c;
    uint16_t* out = a.out + ((int64_t)(u.seq.start + col / a.group) * a.heads + kh * a.group + col % a.group) * D + lane;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) out[64 * e] = f_to_bf16(o[e] * inv);
}

namespace {

template <int CT, int D>
void launch(const AttendArgs& a, int slots, hipStream_t st) {
    const int grid = slots * a.splits * a.kvh;
    if (a.cap > 0.0f)
        hipLaunchKernelGGL((paged_prompt_kernel<CT, D, true>), dim3(grid), dim3(kPromptThreads), 4 * 64 * D, st, a);
    else
        hipLaunchKernelGGL((paged_prompt_kernel<CT, D, false>), dim3(grid), dim3(kPromptThreads), 4 * 64 * D, st, a);
    if (a.splits > 1)
        hipLaunchKernelGGL((paged_prompt_join_kernel<CT, D>), dim3(slots * a.kvh, kBlockColumns / kPromptWaves), dim3(kPromptThreads), 0,
                           st, a, (int64_t)grid);
}

int unit_slots(const Batch& b, int group) { return (int)((int64_t)b.tokens * group / kBlockColumns) + b.seqs; }

}  // namespace

// Blocks that share a unit's keys: as many as it takes to fill the card.
int prompt_splits(const Batch& b, int kvh, int group, int page_size) {
    const int64_t units = std::max<int64_t>((int64_t)b.tokens * group / kBlockColumns, 1) * kvh;
    const int64_t most = ((int64_t)b.width * page_size + 32 * kLeastTiles - 1) / (32 * kLeastTiles);
    return (int)std::max<int64_t>(1, std::min<int64_t>(512 / units, most));
}

bool prompt_fits(const Batch& b, int kvh, int group, int page_size) {
    return (int64_t)unit_slots(b, group) * kvh * prompt_splits(b, kvh, group, page_size) <= INT32_MAX &&
           (int64_t)b.tokens * group <= INT32_MAX;
}

int64_t prompt_part_bytes(const Batch& b, int kvh, int group, int page_size, int d) {
    const int splits = prompt_splits(b, kvh, group, page_size);
    return splits == 1 ? 0 : (int64_t)unit_slots(b, group) * splits * kvh * kBlockColumns * (d + 2) * (int64_t)sizeof(float);
}

void launch_prompt(const AttendArgs& a, bool e4m3, int d, hipStream_t st) {
    const int slots = unit_slots(a.b, a.group);
    switch (d) {
        case 64: e4m3 ? launch<SE12_STEP_E4M3, 64>(a, slots, st) : launch<SE12_STEP_BF16, 64>(a, slots, st); break;
        case 128: e4m3 ? launch<SE12_STEP_E4M3, 128>(a, slots, st) : launch<SE12_STEP_BF16, 128>(a, slots, st); break;
        default: e4m3 ? launch<SE12_STEP_E4M3, 256>(a, slots, st) : launch<SE12_STEP_BF16, 256>(a, slots, st);
    }
}

}  // namespace se12step
