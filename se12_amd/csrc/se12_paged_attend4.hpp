// Attention over pages of E2M1 for few columns: Attend (se12_paged_attention.hip) for a
// cache of 4 bits. The same mathematics, tiles of 64 keys and order of the keys; what is
// its own:
//
// Operands are FP16. A code times its scale has 6 significant bits, so keys and values
// are exact (a conversion and a packed product to two of them); a weight is off by 2^-11
// of itself. FP16 spans 40 powers of two, so a query is taken times a power of two that
// brings its largest value to 2^14 (its scores are taken back by their factor), and a
// weight times 2^7, with maxima that a score may pass by 2^8: from 2^15 down to 2^-31 of
// the largest.
//
// A lane's 16 bytes of a key row are 32 columns, so one scale; its 16 bytes of a block of
// values are 16 tokens of two columns side by side, which become rows of two products.
// The scales of 16 tokens and 32 columns are 16 bytes: of each 16 lanes (which share the
// tokens) lane g takes those of group g, and they go from there to the others by DPP.
//
// Bound by the bytes of the pages: 32 sequences to 8,191 keys, 16 / 8 heads of 256, 328 MB in 64 to 67 us
// and 5 of the join (4.9 to 5.1 TB/s, a copy's rate); 3 to 130,000, 28 / 4 heads of 128, 159 MB in 33 to 34
// (4.7 to 4.8) and 6.5. 1,024 waves as for the other types: with 2,048 the calls took 75 and 44 for 68 and
// 40, in 256 registers 91; where a wave has four tiles, 31 tokens of 12 sequences to 5,000 under a window of
// 4,096, heads of 64, 128 and 256 17.7, 21.0 and 32.3 for 16.9, 19.3 and 25.4. (8 to 2,000, 16 / 8 heads of
// 128, two tiles to a wave: 12.2 for 13.6.)
#pragma once

#include "se12_paged_device.hpp"

namespace se12step {

constexpr float kSlack4 = 8.0f;
constexpr float kLift4 = 7.0f;

// What the scores of a query times 2^lift are to be multiplied by, 2^80 at most: sums of products are
// multiples of 2^-42 (a query's and a key's least steps) below 2^39, so those that differ do by 2^38
// all the same, the largest stay finite, and those of 0 are 0.
__device__ __forceinline__ float score_factor(float c1, int lift) { return fminf(fmaxf(ldexpf(c1, -lift), -0x1p80f), 0x1p80f); }

template <int CT, int D>
struct Attend;

// lane `kFrom` of every 16 lanes, to all of them
template <int kFrom>
__device__ __forceinline__ uint32_t of_row16(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x150 + kFrom, 0xF, 0xF, true);
}

template <int N, typename F>
__device__ __forceinline__ void each_of(F f) {
    if constexpr (N > 0) {
        each_of<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}

template <int D>
struct Attend<SE12_STEP_E2M1, D> {
    static constexpr int kTile = 64;
    static constexpr int kWords = D >= 128 ? 4 : 2;          // of a lane's part of a key row: 8 codes each
    static constexpr int kChunks = D / (32 * kWords);
    static constexpr int kGroups = D / 32;
    struct Piece {
        uint32_t w[kWords];
    };
    floatx4_t o[D / 16];      // 2 i and 2 i + 1: the even and the odd columns of group i
    float m, l;

    // o of part i of 8 columns: those from 32 i + 8 (lane / 16)
    template <typename Store>
    __device__ __forceinline__ void each_part(Store store) const {
        const int quarter = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
            store(32 * i + 8 * quarter, floatx4_t{o[2 * i][0], o[2 * i + 1][0], o[2 * i][1], o[2 * i + 1][1]});
            store(32 * i + 8 * quarter + 4, floatx4_t{o[2 * i][2], o[2 * i + 1][2], o[2 * i][3], o[2 * i + 1][3]});
        }
    }

    // one run of tiles of a unit
    template <typename Work>
    __device__ __forceinline__ void run(const AttendArgs& a, int s, const Work& w, int kh, int unit, int tile, int tiles) {
        constexpr int kColumns = 16;
        const int lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
        const int columns = min(kColumns, w.seq.n * a.group - unit * kColumns);
        const bool live = col < columns;
        const int c = unit * kColumns + (live ? col : 0), token = c / a.group;
        const int pos = live ? w.seq.len + token : -1;                       // -1 sees nothing
        const int pos_min = w.seq.len + unit * kColumns / a.group;
        const int pos_max = w.seq.len + (unit * kColumns + columns - 1) / a.group;
        const int reach = a.window > 0 ? a.window : INT32_MAX;
        const int low = max(0, pos_min - reach + 1), high = min(w.keys, pos_max + 1);   // keys some column sees
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
        m = -INFINITY;
        l = 0.0f;
        const int t0 = max(w.tile0 + tile, low / kTile), t1 = min(w.tile0 + tile + tiles, (high + kTile - 1) / kTile);
        if (t0 >= t1) return;
        const int P = 1 << a.page_log2;
        // the keys a lane takes: K rows krow + 4 step of a tile, V keys vkey .. + 15
        const int kgroup = 16 * (col >> 2), krow = kgroup + (col & 3), vkey = 16 * quarter;
        const int kscale_group = D >= 128 ? quarter : quarter >> 1;
        const uint32_t kscale_pick = 0x0C000C00u | (uint32_t)(col & 3) * 0x00010001u;       // its byte of a word, twice
        const int32_t* table = a.b.table + s * a.b.table_stride;
        auto entry = [&](int key) { return table[min(key >> a.page_log2, a.b.width - 1)]; };
        auto held_page = [&](int e) { return (uint32_t)e < (uint32_t)a.pages ? e : 0; };
        const uint8_t* const kc = static_cast<const uint8_t*>(a.kc);
        const uint8_t* const vc = static_cast<const uint8_t*>(a.vc);
        const uint8_t* const k_scale = reinterpret_cast<const uint8_t*>(a.k_scale);
        const uint8_t* const v_scale = reinterpret_cast<const uint8_t*>(a.v_scale);
        Piece kf[4][kChunks];
        uint4 ks[kChunks];
        auto load_k = [&](int t, int page) {
            const int64_t head_page = (int64_t)held_page(page) * a.kvh + kh;
            const uint8_t* p = kc + (head_page * P + ((t * kTile + krow) & (P - 1))) * (D / 2) + 4 * kWords * quarter;
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int i = 0; i < kChunks; ++i) {
                    if constexpr (kWords == 4)
                        kf[g][i] = __builtin_bit_cast(Piece, *reinterpret_cast<const uint4*>(p + 4 * g * (D / 2) + 64 * i));
                    else
                        kf[g][i] = __builtin_bit_cast(Piece, *reinterpret_cast<const uint2*>(p + 4 * g * (D / 2)));
                }
            const uint8_t* q = k_scale + (head_page * kGroups + kscale_group) * P + ((t * kTile + kgroup) & (P - 1));
#pragma unroll
            for (int i = 0; i < kChunks; ++i) ks[i] = *reinterpret_cast<const uint4*>(q + 4 * i * P);
        };
        int vpage = entry(t0 * kTile + vkey), vpage_next = entry(min(t0 + 1, t1 - 1) * kTile + vkey);
        int kpage_next = entry(min(t0 + 1, t1 - 1) * kTile + kgroup);
        load_k(t0, entry(t0 * kTile + kgroup));

        // the queries, times 2^lift
        halfx8_t qf[kChunks][kWords];
        float by;
        {
            const uint16_t* qp = a.q + (w.seq.start + token) * a.q_stride + (int64_t)(kh * a.group + c % a.group) * D + 8 * kWords * quarter;
            uint4 u[kChunks][kWords];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
#pragma unroll
                for (int h = 0; h < kWords; ++h) {
                    u[i][h] = *reinterpret_cast<const uint4*>(qp + 128 * i + 8 * h);
                    for (const uint32_t x : {u[i][h].x, u[i][h].y, u[i][h].z, u[i][h].w})
                        top = max(top, max((x << 16) & 0x7FFF0000u, x & 0x7FFF0000u));
                }
            top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
            const int lift = 14 + 127 - (int)(top >> 23);
            by = score_factor(a.c1, lift);
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
#pragma unroll
                for (int h = 0; h < kWords; ++h) {
                    const uint32_t x[4] = {u[i][h].x, u[i][h].y, u[i][h].z, u[i][h].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        qf[i][h][2 * k] = (_Float16)ldexpf(__uint_as_float(x[k] << 16), lift);
                        qf[i][h][2 * k + 1] = (_Float16)ldexpf(__uint_as_float(x[k] & 0xFFFF0000u), lift);
                    }
                }
        }
        uint4 vf[kGroups];
        uint32_t vs[4];
        float sc[16], top = 0.0f;
        halfx8_t pf[2];
        auto weights = [&]() {
            const float base = (m == -INFINITY ? 0.0f : m) - kLift4;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = __builtin_amdgcn_exp2f(sc[e] - base);
                l += p;
                pf[e / 8][e % 8] = (_Float16)p;
            }
        };
        auto add_values = [&]() {
            halfx2_t pair[8];      // the scales of the lane's own group, two tokens each
#pragma unroll
            for (int k = 0; k < 8; ++k)
                pair[k] = __builtin_bit_cast(halfx2_t, __builtin_amdgcn_perm(0u, vs[k / 2], k & 1 ? 0x0C030C02u : 0x0C010C00u) << 7);
            each_of<kGroups>([&](auto group) {
                constexpr int i = group.value;
                halfx2_t by2[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) by2[k] = __builtin_bit_cast(halfx2_t, of_row16<i>(__builtin_bit_cast(uint32_t, pair[k])));
                const uint32_t v[4] = {vf[i].x, vf[i].y, vf[i].z, vf[i].w};
#pragma unroll
                for (int odd = 0; odd < 2; ++odd)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        o[2 * i + odd] = __builtin_amdgcn_mfma_f32_16x16x32_f16(e2m1_operand(v[2 * odd + h], by2 + 4 * h), pf[h], o[2 * i + odd], 0, 0, 0);
            });
        };
        auto column_max = [&](float v) {
            v = fmaxf(v, __shfl_xor(v, 16, 64));
            return fmaxf(v, __shfl_xor(v, 32, 64));
        };
        for (int t = t0;; ++t) {
            bool apart = false;     // a value that is no number may be hidden from some of the columns
            for (; t < t1; ++t) {
                const int k0 = t * kTile, key0 = k0 + vkey;
                const int64_t head_page = (int64_t)held_page(vpage) * a.kvh + kh;
                // (what the page of unseen keys holds, its scales too, may be anything)
                const bool held = (uint32_t)vpage < (uint32_t)a.pages && key0 < high && key0 + 16 > low;
                const int next = min(t + 1, t1 - 1), after = min(t + 2, t1 - 1);
                const int kpage_after = entry(after * kTile + kgroup), vpage_after = entry(after * kTile + vkey);
                {
                    const uint8_t* p = vc + ((head_page << (a.page_log2 - 4)) + ((key0 & (P - 1)) >> 4)) * (8 * D) + 16 * col;
#pragma unroll
                    for (int i = 0; i < kGroups; ++i) vf[i] = *reinterpret_cast<const uint4*>(p + 256 * i);
                    const uint4 x = *reinterpret_cast<const uint4*>(v_scale + (head_page * kGroups + col % kGroups) * P + (key0 & (P - 1)));
                    vs[0] = x.x, vs[1] = x.y, vs[2] = x.z, vs[3] = x.w;
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    floatx4_t d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < kChunks; ++i) {
                        const uint32_t sw = g == 0 ? ks[i].x : g == 1 ? ks[i].y : g == 2 ? ks[i].z : ks[i].w;
                        const halfx2_t s2 = __builtin_bit_cast(halfx2_t, __builtin_amdgcn_perm(0u, sw, kscale_pick) << 7);
                        const halfx2_t by2[4] = {s2, s2, s2, s2};
#pragma unroll
                        for (int h = 0; h < kWords; ++h)
                            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(e2m1_operand(kf[g][i].w[h], by2), qf[i][h], d, 0, 0, 0);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[4 * g + e] = d[e];
                }
                __builtin_amdgcn_sched_barrier(0);
                load_k(next, kpage_next);
                __builtin_amdgcn_sched_barrier(0);
                if (a.cap > 0.0f) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        sc[e] = a.cap - 2.0f * a.cap * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(sc[e] * by));
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[e] *= by;
                }
                const bool inside = k0 + kTile - 1 <= pos_min && k0 + kTile <= w.keys && pos_max - k0 < reach &&
                                    __builtin_amdgcn_ballot_w64(!held) == 0;
                if (!inside) {
                    const int from = max(pos - reach + 1, 0) - key0, to = held ? min(pos + 1, w.keys) - key0 : 0;
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[e] = (e < from || e >= to) ? -INFINITY : sc[e];
                    const uint4 mask = piece_mask<SE12_STEP_E4M3>(low - key0, held ? high - key0 : 0);      // a byte to a key
                    vs[0] &= mask.x, vs[1] &= mask.y, vs[2] &= mask.z, vs[3] &= mask.w;
                    apart = __builtin_amdgcn_ballot_w64((no_scales(vs[0]) | no_scales(vs[1]) | no_scales(vs[2]) | no_scales(vs[3])) != 0) != 0;
                }
                top = sc[0];
#pragma unroll
                for (int e = 1; e < 16; ++e) top = fmaxf(top, sc[e]);
                if (t == t0) m = column_max(top);
                const bool higher = __builtin_amdgcn_ballot_w64(top > m + kSlack4) != 0;      // than may be taken from m
                vpage = vpage_next;
                vpage_next = vpage_after;
                kpage_next = kpage_after;
                if (higher || apart) break;
                weights();
                add_values();
            }
            if (t >= t1) break;
            // The rare tile, outside the loop: the maximum moves, and what is summed with it;
            // 0 x NaN is NaN, so a scale that is no number leaves the product, and what it
            // scales comes back as a NaN in the columns that see its key, whatever its weight.
            const float to = fmaxf(m, column_max(top));
            const float scale = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= scale;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[i] *= scale;
            weights();
            if (apart) {
                uint32_t bad[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    bad[k] = no_scales(vs[k]) >> 7;
                    vs[k] &= ~(bad[k] * 255u);
                }
                each_of<kGroups>([&](auto group) {
                    constexpr int i = group.value;
                    int seen = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t x = of_row16<i>(bad[k]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) seen |= ((x >> (8 * e)) & 1u) != 0 && sc[4 * k + e] != -INFINITY;
                    }
                    seen |= __shfl_xor(seen, 16, 64);
                    seen |= __shfl_xor(seen, 32, 64);
#pragma unroll
                    for (int odd = 0; odd < 2; ++odd)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[2 * i + odd][e] += seen ? __builtin_nanf("") : 0.0f;
                });
            }
            add_values();
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
    }
};

}  // namespace se12step
