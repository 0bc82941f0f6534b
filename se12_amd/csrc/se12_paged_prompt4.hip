// Attention over pages of E2M1 for sequences with many new tokens: the units, columns and
// parts of se12_paged_prompt.hip, the operands of se12_paged_attend4.hpp, tiles of 64 keys.
//
// Each value of a tile is turned into FP16 once a block of 128 columns, on its way into LDS
// (se12_paged_tile4.hpp), not once a wave as it is read: 4 bits take a conversion and a packed
// product to two values, and all waves read each. Two tiles stand in LDS, the one after is
// on its way. Scores of keys to come are worked out beside the weights of those before, and the
// product of weights and values beside what becomes of the next scores.
//
// Head dim 64 and 128: four waves of 32 columns (v_mfma_f32_32x32x16_f16), two blocks to a CU.
// Head dim 256: a wave's sums and queries for 32 columns leave room for one wave to a SIMD, which
// waits for each of its own instructions; eight waves of 16 columns (v_mfma_f32_16x16x32_f16)
// read each operand twice as often from LDS, but two share a SIMD. (6,194 tokens of 5 prompts
// behind up to 1,500 keys, 84.7 GFLOP, calls: 8 / 4 heads of 256, capped, 135 us, 0.63 PFLOP/s, 173 the
// other way; 16 / 8 heads of 128 139, 173 the other way, capped 149; 32 / 16 of 64 173, capped 215.)
//
// Nothing is full: a SIMD's two waves overlap vector instructions and products in part, and wait for
// each other's at a tile's barrier. Capped, as above, vector instructions / the matrix unit / LDS: at 256, of
// 257,000 cycles 56 / 34 / 45% (48 of 309 vector instructions to 64 keys of 16 columns are exponentials
// and inverses, at half the rate), at 128 of 281,000 72 / 31 / 26%, at 64, with four times the
// exponentials to a product, of 464,000 78 / 19 / 19%.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "se12_paged_tile4.hpp"

namespace se12step {

// a wave's columns of a unit and what they see
struct Columns4 {
    int c0, mine, pos, pos_min, pos_max, reach;      // (mine: may be none; pos -1 sees nothing)
    const uint16_t* q;
};

template <int D>
__device__ __forceinline__ Columns4 columns_of(const AttendArgs& a, const UnitWork& u, int kh, int first, int most, int col) {
    Columns4 x;
    x.c0 = u.first + first;
    x.mine = min(most, u.columns - x.c0);
    const bool live = col < x.mine;
    const int c = live ? x.c0 + col : u.first, token = c / a.group;
    x.pos = live ? u.len + token : -1;
    x.pos_min = u.len + x.c0 / a.group;
    x.pos_max = x.mine > 0 ? u.len + (x.c0 + x.mine - 1) / a.group : -1;
    x.reach = a.window > 0 ? a.window : INT32_MAX;
    x.q = a.q + (u.start + token) * a.q_stride + (int64_t)(kh * a.group + c % a.group) * D;
    return x;
}

// of two weights, in FP16: into place `at` of the product's operands, their sum added to l
template <int kAt>
__device__ __forceinline__ void put_weights(halfx8_t (&pf)[2], float& l, float p0, float p1) {
    const halfx2_t w = {(_Float16)p0, (_Float16)p1};
    pf[kAt / 8][kAt % 8] = w.x;
    pf[kAt / 8][kAt % 8 + 1] = w.y;
    // (the sum of what the product takes: two at once, times 1)
    l = __builtin_amdgcn_fdot2(w, halfx2_t{(_Float16)1.0f, (_Float16)1.0f}, l, false);
}

// a wave's rows of the output, kCols of D / 8 pieces each, from `own` in LDS
template <int D, int kCols>
__device__ __forceinline__ void write_rows(const AttendArgs& a, const UnitWork& u, int kh, const Columns4& x, const uint8_t* own) {
    constexpr int kPieces = D / 8, kTwist = kPieces < 16 ? kPieces - 1 : 15, kAtOnce = 64 / kPieces;
    const int lane = threadIdx.x & 63;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int k = 0; k < kCols / kAtOnce; ++k) {
        const int r = k * kAtOnce + lane / kPieces, piece = lane % kPieces, c = x.c0 + r;
        if (r >= x.mine) continue;
        const uint4 v = *reinterpret_cast<const uint4*>(own + r * 2 * D + 16 * (piece ^ (r & kTwist)));
        uint2* to = reinterpret_cast<uint2*>(a.out + ((int64_t)(u.start + c / a.group) * a.heads + kh * a.group + c % a.group) * D + 8 * piece);
        to[0] = make_uint2(v.x, v.y);
        to[1] = make_uint2(v.z, v.w);
    }
}

template <int D, bool kCapped>
__global__ __launch_bounds__(256, 2) void paged_prompt4_kernel(AttendArgs a) {
    using Tile = Tile4<D, 256, false>;
    constexpr int kRows = D / 32, kN = D / 16;                // rows of 32 columns of the output; steps of either product
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kh = blockIdx.x % a.kvh;
    const UnitWork u = unit_work(a, blockIdx.x / a.kvh);
    if (u.s < 0) return;
    const int t0 = u.t0, t1 = u.t1, col = lane & 31, half = lane >> 5;
    const Columns4 x = columns_of<D>(a, u, kh, 32 * wave, 32, col);
    auto to_last = [&](int t) { return min(t, t1 - 1); };

    // The walk, in halves of 32 keys. Operands are read from LDS half a half ahead, so keys are
    // two tiles ahead of the products in LDS, values one, and a barrier a tile is enough: what is
    // written in a tile's time goes over what every wave had read before its start.
    Tile tile(a, u, kh, lds);
    int ke = tile.key_entry(t0), ve = tile.value_entry(t0);
    auto page_entries = [&](int t) { return make_int2(tile.entry(t * kTile4 + 16 * half), tile.entry(t * kTile4 + 32 + 16 * half)); };
    int2 pages = page_entries(t0);
    tile.load_keys(t0, ke);
    tile.load_values(t0, ve);
    ke = tile.key_entry(to_last(t0 + 1));
    ve = tile.value_entry(to_last(t0 + 1));
    if (tid < 64) tile.bad[tid] = 0;
    halfx8_t qf[kN];
    const float by = load_query<kN, 16, 32>(qf, x.q + 8 * half, a.c1);
    __syncthreads();
    tile.put_keys(0);
    tile.note_none(0);
    tile.put_values(0);
    tile.load_keys(to_last(t0 + 1), ke);
    tile.load_values(to_last(t0 + 1), ve);
    ke = tile.key_entry(to_last(t0 + 2));
    ve = tile.value_entry(to_last(t0 + 2));
    tile.put_keys(1);
    tile.load_keys(to_last(t0 + 2), ke);
    ke = tile.key_entry(to_last(t0 + 3));
    __syncthreads();

    floatx16_t o[kRows], d;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    uint32_t none_seen = 0;       // groups of which the column sees what is no number
    halfx8_t kf[kN], vf[kRows][2];
    const int lds0 = (int)se12::lds_address(lds);
    const int key_at0 = lds0 + Tile::key_place(key_of_row(col), half), value_at0 = lds0 + Tile::value_place(col, 2 * half);
    // (order(p) of piece p = 2 i + half is order(2 i) ^ half)
    auto read_key = [&](int at, int i, int j) { return lds_get((at ^ (16 * Tile::key_order(2 * i))) + j * 32 * 16 * Tile::kKeyPieces); };
    float sc[16], top, p[2];      // scores, or r of cap - 2 cap r; two weights
    auto cap_score = [&](int e) { sc[e] = kCapped ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(d[e] * by)) : d[e] * by; };
    auto find_top = [&]() {
        top = sc[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = kCapped ? fminf(top, sc[e]) : fmaxf(top, sc[e]);
        if constexpr (kCapped) top = a.cap - 2.0f * a.cap * top;
    };
    auto no_scores = [&]() {
#pragma unroll
        for (int e = 0; e < 16; ++e) d[e] = 0.0f;
    };
    no_scores();
#pragma unroll
    for (int i = 0; i < kN; ++i) d = __builtin_amdgcn_mfma_f32_32x32x16_f16(read_key(key_at0, i, 0), qf[i], d, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kN; ++i) kf[i] = read_key(key_at0, i, 1);
#pragma unroll
    for (int e = 0; e < 16; ++e) cap_score(e);
    find_top();
    for (int t = t0; t < t1; ++t) {
        const int buffer = (t - t0) & 1;
        __syncthreads();
        const uint4 none0 = tile.none_of(buffer, half), none1 = tile.none_of(buffer, 2 + half);
        const uint32_t any_none = none0.x | none0.y | none0.z | none0.w | none1.x | none1.y | none1.z | none1.w;
        const int2 here = pages;
        pages = page_entries(to_last(t + 1));
        each_of<2>([&](auto j) {
            const int k0 = t * kTile4 + 32 * j.value, key0 = k0 + 16 * half;
            const bool held = (uint32_t)(j.value ? here.y : here.x) < (uint32_t)a.pages;
            const bool inside = (k0 + 31 <= x.pos_min) & (k0 + 32 <= u.keys) & (x.pos_max - k0 < x.reach) & (__builtin_amdgcn_ballot_w64(!held) == 0);
            if (!inside) {
                asm volatile("");      // (left to the halves that need it)
                const int since = max(x.pos - x.reach + 1, 0) - key0, to = held ? min(x.pos + 1, u.keys) - key0 : 0;
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[e] = (e < since || e >= to) ? (kCapped ? INFINITY : -INFINITY) : sc[e];
                find_top();
            }
            if (j.value == 1) tile.note_none(buffer ^ 1);
            if (j.value == 1 && __builtin_amdgcn_ballot_w64(any_none != 0) != 0) {
                asm volatile("");
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int first = t * kTile4 + 32 * i + 16 * half;
                    const bool there = (uint32_t)(i ? here.y : here.x) < (uint32_t)a.pages;
                    none_seen |= Tile::groups_of(tile.none_of(buffer, 2 * i + half), max(x.pos - x.reach + 1, 0) - first,
                                                 there ? min(x.pos + 1, u.keys) - first : 0);
                }
            }
            if (__builtin_amdgcn_ballot_w64(top > m + kSlack4) != 0) {
                const float to = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
                const float scale = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
                m = to;
                l *= scale;
#pragma unroll
                for (int i = 0; i < kRows; ++i) o[i] *= scale;
            }
            // Beside each matrix instruction as much of the rest as it takes time for, in this
            // order (left to itself the compiler puts reads, conversions and exponentials into runs of
            // their own, the matrix unit idle).
            constexpr int kEach = 16 / kN, kPuts = j.value == 0 ? Tile::kWords : 4, kLast = 2 * kN - 2;
            constexpr int kAhead = kN / 2 > 4 ? kN / 2 : 4;      // values' pieces read before their product
            const float base = (m == -INFINITY ? 0.0f : m) - kLift4;
            halfx8_t pf[2];
            int key_at = key_at0 + (buffer ^ 1) * Tile::kBuffer, value_at = value_at0 + buffer * Tile::kBuffer;
            asm volatile("" : "+v"(key_at), "+v"(value_at));      // (addresses, not one for every piece over the walk)
            auto read_value = [&](int i) { vf[i / 2][i % 2] = lds_get((value_at ^ (16 * (4 * j.value + i % 2))) + 4096 * (i / 2)); };
            auto put_beside = [&](auto step) {      // of 2 kN steps
                constexpr int at = (step.value * kPuts + kLast - 1) / kLast, end = ((step.value + 1) * kPuts + kLast - 1) / kLast;
                if constexpr (at < end && at < kPuts) {
                    if constexpr (j.value == 0)
                        tile.template put_key<at>(buffer);
                    else
                        tile.template put_value<at>(buffer ^ 1);
                }
                if constexpr (step.value == kLast) {
                    if constexpr (j.value == 0) {
                        tile.load_keys(to_last(t + 3), ke);
                        ke = tile.key_entry(to_last(t + 4));
                    } else {
                        tile.load_values(to_last(t + 2), ve);
                        ve = tile.value_entry(to_last(t + 3));
                    }
                }
            };
            no_scores();
            each_of<kN>([&](auto step) {
                constexpr int i = step.value;
                d = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i], qf[i], d, 0, 0, 0);
                if constexpr (i >= kN - kAhead) read_value(i - (kN - kAhead));
                each_of<kEach>([&](auto each) {
                    constexpr int e = i * kEach + each.value;
                    p[e & 1] = __builtin_amdgcn_exp2f(kCapped ? (a.cap - base) - 2.0f * a.cap * sc[e] : sc[e] - base);
                    if constexpr (e & 1) put_weights<e - 1>(pf, l, p[0], p[1]);
                });
                put_beside(std::integral_constant<int, i>{});
                __builtin_amdgcn_sched_barrier(0);
            });
            each_of<kN>([&](auto step) {
                constexpr int i = step.value, lag = kN > 4 ? 2 : 0;
                o[i / 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[i / 2][i % 2], pf[i % 2], o[i / 2], 0, 0, 0);
                kf[i] = read_key(key_at, i, j.value);
                if constexpr (i + kAhead < kN) read_value(i + kAhead);
                put_beside(std::integral_constant<int, kN + i>{});
                // (the scores are there two products on)
#pragma unroll
                for (int e = max(i - lag, 0) * kEach; e < (i + 1 == kN ? 16 : max(i + 1 - lag, 0) * kEach); ++e) cap_score(e);
                __builtin_amdgcn_sched_barrier(0);
            });
            find_top();
        });
    }
    l += __shfl_xor(l, 32, 64);
    none_seen |= (uint32_t)__shfl_xor((int)none_seen, 32, 64);
    if (__builtin_amdgcn_ballot_w64(none_seen != 0) != 0) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) o[i] += (none_seen >> i & 1u) ? __builtin_nanf("") : 0.0f;
    }
    if (u.parts > 1) {
        // the part, as the lanes hold it
        const int64_t part = part_place(a, u, kh);
        float4* to = reinterpret_cast<float4*>(a.part + part * kBlockColumns * D) + wave * (D / 8) * 64 + lane;
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                to[(4 * i + g) * 64] = make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
        if (half == 0)
            reinterpret_cast<float2*>(a.part + (int64_t)a.parts * a.kvh * kBlockColumns * D)[part * kBlockColumns + 32 * wave + col] = make_float2(m, l);
        return;
    }
    // through LDS to whole rows
    __syncthreads();
    constexpr int kTwist = D / 8 < 16 ? D / 8 - 1 : 15;
    uint8_t* own = lds + wave * 32 * 2 * D;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            store4(reinterpret_cast<uint16_t*>(own + col * 2 * D + 16 * ((4 * i + g) ^ (col & kTwist)) + 8 * half), o[i][4 * g] * inv,
                   o[i][4 * g + 1] * inv, o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv);
    write_rows<D, 32>(a, u, kh, x, own);
}

// Eight waves of 16 columns. Row r of the first product's step g is key 16 (r / 4) + 4 g + r % 4,
// so a lane's scores are those of 16 keys in a row of its column.
template <int D, bool kCapped>
__global__ __launch_bounds__(512, 2) void paged_prompt4_wide_kernel(AttendArgs a) {
    using Tile = Tile4<D, 512, true>;
    constexpr int kRows = D / 16, kSteps = D / 32, kN = D / 8;      // kN: products of either kind
    constexpr int kAhead = 8;                                       // operands read ahead of theirs
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kh = blockIdx.x % a.kvh;
    const UnitWork u = unit_work(a, blockIdx.x / a.kvh);
    if (u.s < 0) return;
    const int t0 = u.t0, t1 = u.t1, col = lane & 15, quarter = lane >> 4;
    const Columns4 x = columns_of<D>(a, u, kh, 16 * wave, 16, col);
    auto to_last = [&](int t) { return min(t, t1 - 1); };

    // The walk: scores of the next tile beside the weights of this one, then the product of its
    // weights and values beside what becomes of the next scores. In LDS keys are two tiles ahead of
    // that product and values one, so a barrier a tile is enough: what is written in a tile's time
    // goes over what every wave had read before its start.
    Tile tile(a, u, kh, lds);
    int ke = tile.key_entry(t0), ve = tile.value_entry(t0), page_entry = tile.entry(t0 * kTile4 + 16 * quarter);
    tile.load_keys(t0, ke);
    tile.load_values(t0, ve);
    ke = tile.key_entry(to_last(t0 + 1));
    ve = tile.value_entry(to_last(t0 + 1));
    if (tid < 64) tile.bad[tid] = 0;
    halfx8_t qf[kSteps];
    const float by = load_query<kSteps, 32, 16>(qf, x.q + 8 * quarter, a.c1);
    __syncthreads();
    tile.put_keys(0);
    tile.note_none(0);
    tile.put_values(0);
    tile.load_keys(to_last(t0 + 1), ke);
    tile.load_values(to_last(t0 + 1), ve);
    ke = tile.key_entry(to_last(t0 + 2));
    ve = tile.value_entry(to_last(t0 + 2));
    tile.put_keys(1);
    tile.load_keys(to_last(t0 + 2), ke);
    ke = tile.key_entry(to_last(t0 + 3));
    __syncthreads();

    floatx4_t o[kRows], d[4];
#pragma unroll
    for (int i = 0; i < kRows; ++i) o[i] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    uint32_t none_seen = 0;       // groups of which the column sees what is no number
    const int lds0 = (int)se12::lds_address(lds);
    const int key_at0 = lds0 + Tile::key_place(16 * (col >> 2) + (col & 3), quarter), value_at0 = lds0 + Tile::value_place(col, 2 * quarter);
    float sc[16], top, p[2];      // scores, or r of cap - 2 cap r; two weights
    auto cap_score = [&](int e) {
        const float v = d[e / 4][e % 4] * by;
        sc[e] = kCapped ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v)) : v;
    };
    auto find_top = [&]() {
        top = sc[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = kCapped ? fminf(top, sc[e]) : fmaxf(top, sc[e]);
        if constexpr (kCapped) top = a.cap - 2.0f * a.cap * top;
    };
    // product n of the scores: step n / 4 of the inner dimension, of the rows step n % 4 (order(p)
    // of piece p = 4 s + quarter is order(4 s) ^ quarter)
    auto read_key = [&](int at, int n) { return lds_get((at ^ (16 * Tile::key_order(4 * (n / 4)))) + (n % 4) * 4 * 16 * Tile::kKeyPieces); };
    auto score_step = [&](int n, halfx8_t k) {
        d[n % 4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[n / 4], n < 4 ? floatx4_t{0.0f, 0.0f, 0.0f, 0.0f} : d[n % 4], 0, 0, 0);
    };
#pragma unroll
    for (int n = 0; n < kN; ++n) score_step(n, read_key(key_at0, n));
#pragma unroll
    for (int e = 0; e < 16; ++e) cap_score(e);
    find_top();
    for (int t = t0; t < t1; ++t) {
        const int buffer = (t - t0) & 1;
        __syncthreads();
        const uint4 none = tile.none_of(buffer, quarter);
        int key_at = key_at0 + (buffer ^ 1) * Tile::kBuffer, value_at = value_at0 + buffer * Tile::kBuffer;
        asm volatile("" : "+v"(key_at), "+v"(value_at));      // (addresses, not one for every piece over the walk)
        halfx8_t ring[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) ring[n] = read_key(key_at, n);
        const int k0 = t * kTile4, key0 = k0 + 16 * quarter;
        const bool held = (uint32_t)page_entry < (uint32_t)a.pages;
        page_entry = tile.entry(to_last(t + 1) * kTile4 + 16 * quarter);
        tile.note_none(buffer ^ 1);
        const bool inside = (k0 + kTile4 - 1 <= x.pos_min) & (k0 + kTile4 <= u.keys) & (x.pos_max - k0 < x.reach) & (__builtin_amdgcn_ballot_w64(!held) == 0);
        const int since = max(x.pos - x.reach + 1, 0) - key0, to = held ? min(x.pos + 1, u.keys) - key0 : 0;
        if (!inside) {
            asm volatile("");      // (left to the tiles that need it)
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[e] = (e < since || e >= to) ? (kCapped ? INFINITY : -INFINITY) : sc[e];
            find_top();
        }
        if (__builtin_amdgcn_ballot_w64((none.x | none.y | none.z | none.w) != 0) != 0) {
            asm volatile("");
            none_seen |= Tile::groups_of(none, since, to);
        }
        if (__builtin_amdgcn_ballot_w64(top > m + kSlack4) != 0) {
            asm volatile("");
            float next = fmaxf(top, __shfl_xor(top, 16, 64));
            next = fmaxf(m, fmaxf(next, __shfl_xor(next, 32, 64)));
            const float scale = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - next);
            m = next;
            l *= scale;
#pragma unroll
            for (int i = 0; i < kRows; ++i) o[i] *= scale;
        }
        const float base = (m == -INFINITY ? 0.0f : m) - kLift4;
        halfx8_t pf[2];
        auto read_value = [&](int n) { return lds_get((value_at ^ (16 * (n % 2))) + 2048 * (n / 2)); };
        each_of<kN>([&](auto step) {
            constexpr int n = step.value, from = 16 * n / kN, upto = 16 * (n + 1) / kN;
            score_step(n, ring[n % kAhead]);
            ring[n % kAhead] = n + kAhead < kN ? read_key(key_at, n + kAhead) : read_value(n + kAhead - kN);
            each_of<upto - from>([&](auto each) {
                constexpr int e = from + each.value;
                p[e & 1] = __builtin_amdgcn_exp2f(kCapped ? (a.cap - base) - 2.0f * a.cap * sc[e] : sc[e] - base);
                if constexpr (e & 1) put_weights<e - 1>(pf, l, p[0], p[1]);
            });
            if constexpr (n < 4) tile.template put_value<n>(buffer ^ 1);
            if constexpr (n == 4) {
                tile.load_values(to_last(t + 2), ve);
                ve = tile.value_entry(to_last(t + 3));
            }
        });
        each_of<kN>([&](auto step) {
            constexpr int n = step.value, from = 16 * n / kN, upto = 16 * (n + 1) / kN;
            o[n / 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[n % kAhead], pf[n % 2], o[n / 2], 0, 0, 0);
            if constexpr (n + kAhead < kN) ring[n % kAhead] = read_value(n + kAhead);
#pragma unroll
            for (int e = from; e < upto; ++e) cap_score(e);
            if constexpr (n < Tile::kWords) tile.template put_key<n>(buffer);
            if constexpr (n == Tile::kWords) {
                tile.load_keys(to_last(t + 3), ke);
                ke = tile.key_entry(to_last(t + 4));
            }
        });
        find_top();
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    none_seen |= (uint32_t)__shfl_xor((int)none_seen, 16, 64);
    none_seen |= (uint32_t)__shfl_xor((int)none_seen, 32, 64);
    if (__builtin_amdgcn_ballot_w64(none_seen != 0) != 0) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) o[i] += (none_seen >> (i / 2) & 1u) ? __builtin_nanf("") : 0.0f;
    }
    if (u.parts > 1) {
        // the part, where a lane of a wave of 32 columns would hold it
        const int64_t part = part_place(a, u, kh);
        const int column = 16 * wave + col;
        float4* to = reinterpret_cast<float4*>(a.part + part * kBlockColumns * D) + ((column / 32) * (D / 8) + (quarter >> 1)) * 64 + column % 32 + 32 * (quarter & 1);
#pragma unroll
        for (int i = 0; i < kRows; ++i) to[2 * i * 64] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
        if (quarter == 0)
            reinterpret_cast<float2*>(a.part + (int64_t)a.parts * a.kvh * kBlockColumns * D)[part * kBlockColumns + column] = make_float2(m, l);
        return;
    }
    // through LDS to whole rows
    __syncthreads();
    constexpr int kTwist = D / 8 < 16 ? D / 8 - 1 : 15;
    uint8_t* own = lds + wave * 16 * 2 * D;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
        store4(reinterpret_cast<uint16_t*>(own + col * 2 * D + 16 * ((2 * i + (quarter >> 1)) ^ (col & kTwist)) + 8 * (quarter & 1)), o[i][0] * inv,
               o[i][1] * inv, o[i][2] * inv, o[i][3] * inv);
    write_rows<D, 16>(a, u, kh, x, own);
}

namespace {

template <int D, bool kCapped>
void launch4(const AttendArgs& a, hipStream_t st) {
    const dim3 grid(a.unit_count * a.kvh);
    if constexpr (D == 256)
        hipLaunchKernelGGL((paged_prompt4_wide_kernel<D, kCapped>), grid, dim3(512), (Tile4<D, 512, true>::kBytes), st, a);
    else
        hipLaunchKernelGGL((paged_prompt4_kernel<D, kCapped>), grid, dim3(256), (Tile4<D, 256, false>::kBytes), st, a);
}

}  // namespace

void launch_prompt4(const AttendArgs& a, int d, hipStream_t st) {
    const bool capped = a.cap > 0.0f;
    switch (d) {
        case 64: capped ? launch4<64, true>(a, st) : launch4<64, false>(a, st); break;
        case 128: capped ? launch4<128, true>(a, st) : launch4<128, false>(a, st); break;
        default: capped ? launch4<256, true>(a, st) : launch4<256, false>(a, st);
    }
}

}  // namespace se12step
