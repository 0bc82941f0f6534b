// Attention over pages of E2M1 for sequences with many new tokens: the units, columns and
// order of keys of se12_paged_prompt.hip, the operands of se12_paged_attend4.hpp.
//
// A block takes 128 columns, 32 a wave, and walks the tiles of 64 keys they see. Each
// value of a tile is turned into FP16 once a block, on its way into LDS, not once a wave
// as it is read: 4 bits take a conversion and a product to two values, and four waves read
// each. The tile after next is asked for and the next one turned while the products of this one
// run; two tiles stand in LDS. v_mfma_f32_32x32x16_f16; keys' rows in the order that leaves a
// lane's scores the second product's operand. The 16-byte pieces of an LDS row lie in an
// order of its own, so that neither the lanes that read the same piece of 8 rows nor those
// that write 8 pieces of a row meet in a bank.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "se12_paged_attend4.hpp"
#include "se12_paged_units.hpp"

namespace se12step {

typedef float floatx16_t __attribute__((ext_vector_type(16)));

constexpr int kPrompt4Threads = 256, kWave4Columns = 32, kTile4 = 64;

// the key (of 32) of row m of the first product's A operand
__device__ __forceinline__ int key_of_row4(int m) { return (m & 3) | ((m & 8) >> 1) | ((m & 16) >> 1) | ((m & 4) << 2); }

template <int D, bool kCapped>
__global__ __launch_bounds__(kPrompt4Threads, D == 256 ? 1 : 2) void paged_prompt4_kernel(AttendArgs a) {
    constexpr int kGroups = D / 32, kRows = D / 32, kQSteps = D / 16;
    constexpr int kKeyPieces = D / 8;                        // 16-byte pieces of a key's row in LDS
    constexpr int kWords = D >= 128 ? 4 : 2;                 // of a thread's piece of a key as it is held
    constexpr int kKeyLoads = kTile4 * D / 8 / kWords / kPrompt4Threads;       // pieces of a thread
    constexpr int kHeldPieces = D / (8 * kWords);            // of a key
    constexpr int kValueLoads = kTile4 * D / 32 / kPrompt4Threads;             // pieces of 16 tokens of two columns
    constexpr int kValueThreads = kValueLoads > 0 ? kPrompt4Threads : kTile4 * D / 32;
    constexpr int kKeyBytes = kTile4 * D * 2, kBuffer = 2 * kKeyBytes;
    static_assert(kKeyLoads >= 1, "");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];     // [2][keys, values], then the values' scales that are none
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kh = blockIdx.x % a.kvh;
    const UnitWork u = unit_work(a, blockIdx.x / a.kvh);
    if (u.s < 0) return;
    const int t0 = u.t0, t1 = u.t1;
    uint16_t* const bad = reinterpret_cast<uint16_t*>(lds + 2 * kBuffer);      // [2][4 runs of 16 tokens][8 groups]

    const int col = lane & 31, half = lane >> 5;
    const int c0 = u.first + wave * kWave4Columns, mine = min(kWave4Columns, u.columns - c0);   // (may be none)
    const bool live = col < mine;
    const int c = live ? c0 + col : u.first, token = c / a.group;
    const int pos = live ? u.len + token : -1;
    const int pos_min = u.len + c0 / a.group, pos_max = mine > 0 ? u.len + (c0 + mine - 1) / a.group : -1;
    const int reach = a.window > 0 ? a.window : INT32_MAX;

    const int P = 1 << a.page_log2;
    const int32_t* table = a.b.table + u.s * a.b.table_stride;
    auto entry = [&](int key) { return table[min(key >> a.page_log2, a.b.width - 1)]; };
    auto in_pool = [&](int e) { return (uint32_t)e < (uint32_t)a.pages ? e : 0; };
    auto to_last = [&](int t) { return min(t, t1 - 1); };
    const uint8_t* const kc = static_cast<const uint8_t*>(a.kc);
    const uint8_t* const vc = static_cast<const uint8_t*>(a.vc);
    const uint8_t* const k_scale = reinterpret_cast<const uint8_t*>(a.k_scale);
    const uint8_t* const v_scale = reinterpret_cast<const uint8_t*>(a.v_scale);

    // What a thread brings of a tile. Keys: pieces of rows; values: columns 2 x, 2 x + 1 of a run.
    struct Held {
        uint32_t k[kKeyLoads][kWords];
        uint32_t ks[kKeyLoads];
        uint4 v[kValueLoads > 0 ? kValueLoads : 1], vs[kValueLoads > 0 ? kValueLoads : 1];
    } held;
    auto key_row = [&](int i) { return (tid + i * kPrompt4Threads) / kHeldPieces; };
    auto run_of = [&](int i) { return (tid + i * kPrompt4Threads) / (D / 2); };
    struct Entries {
        int k[kKeyLoads], v[kValueLoads > 0 ? kValueLoads : 1];
    } entries;
    auto load_entries = [&](int t) {
#pragma unroll
        for (int i = 0; i < kKeyLoads; ++i) entries.k[i] = entry(t * kTile4 + key_row(i));
#pragma unroll
        for (int i = 0; i < (kValueLoads > 0 ? kValueLoads : 1); ++i) entries.v[i] = entry(t * kTile4 + 16 * min(run_of(i), 3));
    };
    auto load_held = [&](int t) {
#pragma unroll
        for (int i = 0; i < kKeyLoads; ++i) {
            const int r = key_row(i), piece = (tid + i * kPrompt4Threads) % kHeldPieces, slot = (t * kTile4 + r) & (P - 1);
            const int64_t head_page = (int64_t)in_pool(entries.k[i]) * a.kvh + kh;
            const uint8_t* p = kc + (head_page * P + slot) * (D / 2) + 4 * kWords * piece;
            if constexpr (kWords == 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(p);
                held.k[i][0] = x.x, held.k[i][1] = x.y, held.k[i][2] = x.z, held.k[i][3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(p);
                held.k[i][0] = x.x, held.k[i][1] = x.y;
            }
            held.ks[i] = k_scale[(head_page * kGroups + piece * 8 * kWords / 32) * P + slot];
        }
#pragma unroll
        for (int i = 0; i < (kValueLoads > 0 ? kValueLoads : 1); ++i) {
            const int run = min(run_of(i), 3), x = (tid + i * kPrompt4Threads) % (D / 2), slot = (t * kTile4 + 16 * run) & (P - 1);
            const int64_t head_page = (int64_t)in_pool(entries.v[i]) * a.kvh + kh;
            held.v[i] = *reinterpret_cast<const uint4*>(vc + ((head_page << (a.page_log2 - 4)) + (slot >> 4)) * (8 * D) + 16 * x);
            held.vs[i] = *reinterpret_cast<const uint4*>(v_scale + (head_page * kGroups + x / 16) * P + slot);
        }
    };
    // where piece p of a key's row, or of a value column, lies
    auto key_place = [](int r, int p) {
        const int twist = kKeyPieces >= 16 ? (r & 7) | ((r & 16) >> 1) : ((r & 7) | ((r & 16) >> 1)) >> 1;
        const int q = p ^ ((p >> 2) & 7);
        return r * (kKeyPieces * 16) + 16 * (q ^ twist);
    };
    auto value_place = [](int r, int p) { return r * 128 + 16 * (p ^ (r & 7) ^ ((r >> 3) & 1)); };
    auto put_keys = [&](int buffer) {
        uint8_t* to = lds + buffer * kBuffer;
#pragma unroll
        for (int i = 0; i < kKeyLoads; ++i) {
            const int r = key_row(i), piece = (tid + i * kPrompt4Threads) % kHeldPieces;
            const halfx2_t s2 = __builtin_bit_cast(halfx2_t, held.ks[i] * 0x00800080u);
            const halfx2_t by[4] = {s2, s2, s2, s2};
#pragma unroll
            for (int h = 0; h < kWords; ++h)
                *reinterpret_cast<halfx8_t*>(to + key_place(r, kWords * piece + h)) = e2m1_operand(held.k[i][h], by);
        }
    };
    auto put_values = [&](int buffer) {
        uint8_t* to = lds + buffer * kBuffer + kKeyBytes;
        if (tid >= kValueThreads) return;
#pragma unroll
        for (int i = 0; i < (kValueLoads > 0 ? kValueLoads : 1); ++i) {
            const int run = run_of(i), x = (tid + i * kPrompt4Threads) % (D / 2);
            uint32_t s[4] = {held.vs[i].x, held.vs[i].y, held.vs[i].z, held.vs[i].w};
            // (a scale that is no number leaves the product: 0 x NaN is NaN)
            uint32_t none = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t b = no_scales(s[k]) >> 7;
                s[k] &= ~(b * 255u);
                none |= ((b * 0x01020408u) >> 24 & 15u) << (4 * k);
            }
            if (x % 16 == 0) bad[buffer * 32 + run * 8 + x / 16] = (uint16_t)none;
            halfx2_t pair[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                pair[k] = __builtin_bit_cast(halfx2_t, __builtin_amdgcn_perm(0u, s[k / 2], k & 1 ? 0x0C030C02u : 0x0C010C00u) << 7);
            const uint32_t w[4] = {held.v[i].x, held.v[i].y, held.v[i].z, held.v[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<halfx8_t*>(to + value_place(2 * x + j / 2, 2 * run + (j & 1))) = e2m1_operand(w[j], pair + 4 * (j & 1));
        }
    };

    load_entries(t0);
    load_held(t0);
    load_entries(to_last(t0 + 1));
    if (tid < 64) bad[tid] = 0;
    __syncthreads();
    halfx8_t qf[kQSteps];
    float by;
    {
        // the queries, times 2^lift
        const uint16_t* qp = a.q + (u.start + token) * a.q_stride + (int64_t)(kh * a.group + c % a.group) * D + 8 * half;
        uint4 x[kQSteps];
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < kQSteps; ++i) {
            x[i] = *reinterpret_cast<const uint4*>(qp + 16 * i);
            for (const uint32_t v : {x[i].x, x[i].y, x[i].z, x[i].w}) most = max(most, max((v << 16) & 0x7FFF0000u, v & 0x7FFF0000u));
        }
        most = max(most, (uint32_t)__shfl_xor((int)most, 32, 64));
        const int lift = 14 + 127 - (int)(most >> 23);
        by = ldexpf(a.c1, -lift);
#pragma unroll
        for (int i = 0; i < kQSteps; ++i) {
            const uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                qf[i][2 * k] = (_Float16)ldexpf(__uint_as_float(v[k] << 16), lift);
                qf[i][2 * k + 1] = (_Float16)ldexpf(__uint_as_float(v[k] & 0xFFFF0000u), lift);
            }
        }
    }
    put_keys(0);
    put_values(0);
    load_held(to_last(t0 + 1));
    load_entries(to_last(t0 + 2));

    floatx16_t o[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    uint32_t none_seen = 0;       // groups of which the column saw what is no number
    const int key_row0 = key_of_row4(col);
    for (int t = t0; t < t1; ++t) {
        const int buffer = (t - t0) & 1;
        __syncthreads();          // this tile has come, and every wave is done with the other buffer
        const uint8_t* const keys = lds + buffer * kBuffer;
        const uint8_t* const values = keys + kKeyBytes;
        floatx16_t d[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int e = 0; e < 16; ++e) d[j][e] = 0.0f;
#pragma unroll
            for (int i = 0; i < kQSteps; ++i) {
                const halfx8_t k = *reinterpret_cast<const halfx8_t*>(keys + key_place(32 * j + key_row0, 2 * i + half));
                d[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qf[i], d[j], 0, 0, 0);
            }
        }
        put_keys(buffer ^ 1);
        put_values(buffer ^ 1);
        load_held(to_last(t + 2));
        load_entries(to_last(t + 3));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int k0 = t * kTile4 + 32 * j, key0 = k0 + 16 * half;
            float sc[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
                sc[e] = kCapped ? a.cap - 2.0f * a.cap * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(d[j][e] * by)) : d[j][e] * by;
            const bool here = (uint32_t)entry(key0) < (uint32_t)a.pages;
            const bool inside = (k0 + 31 <= pos_min) & (k0 + 32 <= u.keys) & (pos_max - k0 < reach) & (__builtin_amdgcn_ballot_w64(!here) == 0);
            if (!inside) {
                const int since = max(pos - reach + 1, 0) - key0, to = here ? min(pos + 1, u.keys) - key0 : 0;
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[e] = (e < since || e >= to) ? -INFINITY : sc[e];
            }
            float top = sc[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) top = fmaxf(top, sc[e]);
            if (__builtin_amdgcn_ballot_w64(top > m + kSlack4) != 0) {
                const float to = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
                const float scale = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
                m = to;
                l *= scale;
#pragma unroll
                for (int i = 0; i < kRows; ++i) o[i] *= scale;
            }
            const float base = (m == -INFINITY ? 0.0f : m) - kLift4;
            halfx8_t pf[2];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = __builtin_amdgcn_exp2f(sc[e] - base);
                l += p;
                pf[e / 8][e % 8] = (_Float16)p;
            }
            const uint4 none = *reinterpret_cast<const uint4*>(bad + buffer * 32 + (2 * j + half) * 8);
            if (__builtin_amdgcn_ballot_w64((none.x | none.y | none.z | none.w) != 0) != 0) {
                const uint32_t w[4] = {none.x, none.y, none.z, none.w};
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool seen = !((float)pf[e / 8][e % 8] <= 0.0f);
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) none_seen |= seen && (w[g / 2] >> (16 * (g & 1) + e) & 1u) ? 1u << g : 0u;
                }
            }
#pragma unroll
            for (int i = 0; i < kRows; ++i)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const halfx8_t v = *reinterpret_cast<const halfx8_t*>(values + value_place(32 * i + col, 4 * j + 2 * half + n));
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pf[n], o[i], 0, 0, 0);
                }
        }
    }
    l += __shfl_xor(l, 32, 64);
    none_seen |= (uint32_t)__shfl_xor((int)none_seen, 32, 64);
    if (__builtin_amdgcn_ballot_w64(none_seen != 0) != 0) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) o[i] += (none_seen >> i & 1u) ? __builtin_nanf("") : 0.0f;
    }
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
            reinterpret_cast<float2*>(a.part + (int64_t)a.parts * a.kvh * kBlockColumns * D)[p * kBlockColumns + wave * kWave4Columns + col] =
                make_float2(m, l);
        return;
    }
    // through LDS to whole rows
    __syncthreads();
    constexpr int kOutPieces = D / 8, kTwist = kOutPieces < 16 ? kOutPieces - 1 : 15, kRowsAtOnce = 64 / kOutPieces;
    uint8_t* own = lds + wave * kWave4Columns * 2 * D;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            store4(reinterpret_cast<uint16_t*>(own + col * 2 * D + 16 * ((4 * i + g) ^ (col & kTwist)) + 8 * half), o[i][4 * g] * inv,
                   o[i][4 * g + 1] * inv, o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int k = 0; k < kWave4Columns / kRowsAtOnce; ++k) {
        const int r = k * kRowsAtOnce + lane / kOutPieces, piece = lane % kOutPieces, x = c0 + r;
        if (r >= mine) continue;
        const uint4 v = *reinterpret_cast<const uint4*>(own + r * 2 * D + 16 * (piece ^ (r & kTwist)));
        uint2* to = reinterpret_cast<uint2*>(a.out + ((int64_t)(u.start + x / a.group) * a.heads + kh * a.group + x % a.group) * D + 8 * piece);
        to[0] = make_uint2(v.x, v.y);
        to[1] = make_uint2(v.z, v.w);
    }
}

namespace {

template <int D>
void launch4(const AttendArgs& a, hipStream_t st) {
    const dim3 grid(a.unit_count * a.kvh);
    constexpr size_t kLds = 2 * 2 * kTile4 * D * 2 + 2 * 32 * sizeof(uint16_t);
    if (a.cap > 0.0f)
        hipLaunchKernelGGL((paged_prompt4_kernel<D, true>), grid, dim3(kPrompt4Threads), kLds, st, a);
    else
        hipLaunchKernelGGL((paged_prompt4_kernel<D, false>), grid, dim3(kPrompt4Threads), kLds, st, a);
}

}  // namespace

void launch_prompt4(const AttendArgs& a, int d, hipStream_t st) {
    switch (d) {
        case 64: launch4<64>(a, st); break;
        case 128: launch4<128>(a, st); break;
        default: launch4<256>(a, st);
    }
}

}  // namespace se12step
