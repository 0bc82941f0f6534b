// A tile of 64 keys of E2M1 pages on its way into LDS, in FP16 (se12_paged_prompt4.hip):
// every thread of the block brings a piece of the keys and one of the values, turns them
// a 16-byte piece at a time, and puts them where the products read them.
#pragma once

#include "se12_device.hpp"
#include "se12_paged_attend4.hpp"
#include "se12_paged_units.hpp"

namespace se12step {

constexpr int kTile4 = 64;

// 16 bytes of LDS by their address (a pointer to shared memory costs an addition of its base)
__device__ __forceinline__ halfx8_t lds_get(int at) { return *(const __attribute__((address_space(3))) halfx8_t*)(uint32_t)at; }
__device__ __forceinline__ void lds_put(int at, halfx8_t v) { *(__attribute__((address_space(3))) halfx8_t*)(uint32_t)at = v; }

// a column's query pieces, every kStep values from `from` on, in FP16 times 2^lift; what the
// scores are to be multiplied by. kSpread: lanes `kSpread` apart and so on hold the rest of it
template <int kPieces, int kStep, int kSpread>
__device__ __forceinline__ float load_query(halfx8_t (&q)[kPieces], const uint16_t* from, float c1) {
    uint4 w[kPieces];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        w[i] = *reinterpret_cast<const uint4*>(from + kStep * i);
        for (const uint32_t v : {w[i].x, w[i].y, w[i].z, w[i].w}) most = max(most, max((v << 16) & 0x7FFF0000u, v & 0x7FFF0000u));
    }
#pragma unroll
    for (int o = kSpread; o < 64; o <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
    const int lift = 14 + 127 - (int)(most >> 23);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            q[i][2 * k] = (_Float16)ldexpf(__uint_as_float(v[k] << 16), lift);
            q[i][2 * k + 1] = (_Float16)ldexpf(__uint_as_float(v[k] & 0xFFFF0000u), lift);
        }
    }
    return score_factor(c1, lift);
}

// kRows16: keys are read 16 rows at a time (16 r / 4 + r % 4), else 32 in key_of_row's order
template <int D, int kThreads, bool kRows16>
struct Tile4 {
    static constexpr int kGroups = D / 32;
    static constexpr int kKeyPieces = D / 8;                             // 16-byte pieces of a key's row in LDS
    static constexpr int kWords = kTile4 * D / 8 / kThreads;             // of a thread's piece of a key as it is held
    static constexpr int kHeldPieces = D / (8 * kWords), kWaveRows = 64 / kHeldPieces;
    static constexpr int kValueThreads = kTile4 * D / 32;                // each with 16 tokens of two columns
    static constexpr int kKeyBytes = kTile4 * D * 2, kBuffer = 2 * kKeyBytes;
    static constexpr int kBytes = 2 * kBuffer + 2 * 32 * (int)sizeof(uint16_t);      // [2][keys, values], then `bad`
    static_assert((kWords == 2 || kWords == 4) && kValueThreads <= kThreads && kWaveRows <= 16, "");

    const AttendArgs& a;
    const int32_t* table;
    uint16_t* bad;               // [2][4 runs of 16 tokens][8 groups]: scales that are no number, a bit to a token
    int kh, P, wave_row, run, x;
    uint32_t k_offset, ks_offset, ks_pick, vs_offset;
    int put_key_at, put_value_at;
    uint32_t k_held[kWords], ks_held;
    uint4 v_held, vs_held;
    halfx2_t pair[8];            // the values' scales, of two tokens each

    // Where piece p of row r lies: keys at row r, place order(p) ^ twist(r), values' columns at
    // place p ^ twist(r), so that neither the lanes that read one piece of many rows nor those that
    // write a row's pieces meet in a bank. All of it exclusive ors: a lane's other pieces lie at its
    // first one's address ^ a constant.
    static __device__ __forceinline__ int key_twist(int r) {
        const int b = kRows16 ? (r & 3) | ((r >> 2) & 12) : (r & 7) | ((r & 16) >> 1);
        return kKeyPieces >= 16 ? b : b >> 1;
    }
    static __device__ __forceinline__ constexpr int key_order(int p) { return p ^ ((p >> 2) & 7); }
    static __device__ __forceinline__ int value_twist(int r) { return (r & 7) ^ ((r >> 3) & 1); }
    static __device__ __forceinline__ int key_place(int r, int p) { return r * (16 * kKeyPieces) + 16 * (key_order(p) ^ key_twist(r)); }
    static __device__ __forceinline__ int value_place(int r, int p) { return kKeyBytes + r * 128 + 16 * (p ^ value_twist(r)); }

    // Keys: a piece of a row, a wave's in one run of 16 tokens; values: columns 2 x, 2 x + 1 of a
    // run (at D = 64 a wave has two of the runs, and half of the waves have none).
    __device__ __forceinline__ Tile4(const AttendArgs& args, const UnitWork& u, int head, uint8_t* lds)
        : a(args), table(args.b.table + u.s * args.b.table_stride), bad(reinterpret_cast<uint16_t*>(lds + 2 * kBuffer)), kh(head),
          P(1 << args.page_log2) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lds0 = (int)se12::lds_address(lds);
        const int row = lane / kHeldPieces, piece = tid % kHeldPieces;
        wave_row = wave * kWaveRows;
        x = tid % (D / 2);
        run = D == 64 ? min(tid / 32, 3) : wave * 64 / (D / 2);
        k_offset = row * (D / 2) + 4 * kWords * piece;
        ks_offset = (piece * kWords / 4) * P + row / 4 * 4;
        ks_pick = 0x0C000C00u | (uint32_t)(row % 4) * 0x00010001u;       // its byte of four tokens', twice
        vs_offset = (x / 16) * P;
        put_key_at = lds0 + key_place(wave_row + row, kWords * piece);
        put_value_at = lds0 + value_place(2 * x, 2 * run);
    }
    __device__ __forceinline__ bool has_values() const { return kValueThreads == kThreads || (int)threadIdx.x < kValueThreads; }
    __device__ __forceinline__ int entry(int key) const { return table[min(key >> a.page_log2, a.b.width - 1)]; }
    __device__ __forceinline__ int in_pool(int e) const { return (uint32_t)e < (uint32_t)a.pages ? e : 0; }
    __device__ __forceinline__ int key_entry(int t) const { return entry(t * kTile4 + wave_row); }
    __device__ __forceinline__ int value_entry(int t) const { return entry(t * kTile4 + 16 * run); }
    // tile t's, of the page of entry e
    __device__ __forceinline__ void load_keys(int t, int e) {
        const int slot = (t * kTile4 + wave_row) & (P - 1);
        const int64_t head_page = (int64_t)in_pool(__builtin_amdgcn_readfirstlane(e)) * a.kvh + kh;
        const uint8_t* p = static_cast<const uint8_t*>(a.kc) + (head_page * P + slot) * (D / 2) + k_offset;
        if constexpr (kWords == 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(p);
            k_held[0] = w.x, k_held[1] = w.y, k_held[2] = w.z, k_held[3] = w.w;
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(p);
            k_held[0] = w.x, k_held[1] = w.y;
        }
        // (as a word: a byte is cut to size, and so waited for, where it is loaded)
        ks_held = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(a.k_scale) + head_page * kGroups * P + slot + ks_offset);
    }
    __device__ __forceinline__ void load_values(int t, int e) {
        const int slot = (t * kTile4 + 16 * run) & (P - 1);
        const int64_t head_page = (int64_t)in_pool(D == 64 ? e : __builtin_amdgcn_readfirstlane(e)) * a.kvh + kh;
        const uint8_t* p = static_cast<const uint8_t*>(a.vc) + ((head_page << (a.page_log2 - 4)) + (slot >> 4)) * (8 * D);
        v_held = *reinterpret_cast<const uint4*>(p + 16 * (uint32_t)x);
        vs_held = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.v_scale) + head_page * kGroups * P + slot + vs_offset);
    }
    // piece kPut of the thread's (kWords of keys, four of values)
    template <int kPut>
    __device__ __forceinline__ void put_key(int buffer) {
        const halfx2_t s2 = __builtin_bit_cast(halfx2_t, __builtin_amdgcn_perm(0u, ks_held, ks_pick) << 7);
        const halfx2_t by[4] = {s2, s2, s2, s2};
        lds_put((put_key_at + buffer * kBuffer) ^ (16 * kPut), e2m1_operand(k_held[kPut], by));
    }
    template <int kPut>
    __device__ __forceinline__ void put_value(int buffer) {
        if (!has_values()) return;
        const uint32_t s[4] = {vs_held.x, vs_held.y, vs_held.z, vs_held.w};
        if constexpr (kPut < 2) {
#pragma unroll
            for (int k = 4 * kPut; k < 4 * kPut + 4; ++k)
                pair[k] = __builtin_bit_cast(halfx2_t, __builtin_amdgcn_perm(0u, s[k / 2], k & 1 ? 0x0C030C02u : 0x0C010C00u) << 7);
        }
        const uint32_t w = kPut == 0 ? v_held.x : kPut == 1 ? v_held.y : kPut == 2 ? v_held.z : v_held.w;
        // (the odd column's row has the even one's twist ^ 1)
        lds_put(((put_value_at + buffer * kBuffer) ^ (16 * ((kPut & 1) ^ (kPut / 2)))) + 128 * (kPut / 2), e2m1_operand(w, pair + 4 * (kPut & 1)));
    }
    __device__ __forceinline__ void put_keys(int buffer) {
        each_of<kWords>([&](auto put) { put_key<put.value>(buffer); });
    }
    __device__ __forceinline__ void put_values(int buffer) {
        each_of<4>([&](auto put) { put_value<put.value>(buffer); });
    }
    // A scale that is no number leaves the product (0 x NaN is NaN), and its place is noted: what a
    // column sees of it makes the group NaN at the walk's end.
    __device__ __forceinline__ void note_none(int buffer) {
        const uint32_t any = no_scales(vs_held.x) | no_scales(vs_held.y) | no_scales(vs_held.z) | no_scales(vs_held.w);
        uint32_t none = 0;
        if (__builtin_amdgcn_ballot_w64(any != 0) != 0) {
            asm volatile("");
            uint32_t s[4] = {vs_held.x, vs_held.y, vs_held.z, vs_held.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t b = no_scales(s[k]) >> 7;
                s[k] &= ~(b * 255u);
                none |= ((b * 0x01020408u) >> 24 & 15u) << (4 * k);
            }
            vs_held = make_uint4(s[0], s[1], s[2], s[3]);
        }
        if (x % 16 == 0 && has_values()) bad[buffer * 32 + run * 8 + x / 16] = (uint16_t)none;
    }
    // of 16 keys, run r of the tile in `buffer`: a bit to a key, 16 to a group
    __device__ __forceinline__ uint4 none_of(int buffer, int r) const { return *reinterpret_cast<const uint4*>(bad + buffer * 32 + 8 * r); }
    // the groups with any in keys since .. to - 1 of them
    static __device__ __forceinline__ uint32_t groups_of(uint4 none, int since, int to) {
        const uint32_t seen = ((1u << min(max(to, 0), 16)) - 1u) & ~((1u << min(max(since, 0), 16)) - 1u), w[4] = {none.x, none.y, none.z, none.w};
        uint32_t groups = 0;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) groups |= (w[g / 2] >> (16 * (g & 1)) & seen) != 0 ? 1u << g : 0u;
        return groups;
    }
};

}  // namespace se12step
