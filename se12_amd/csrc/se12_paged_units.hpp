// The units of attention over a paged cache for sequences with many new tokens (128
// columns of a sequence and KV head), in the order their blocks are started. Found by
// the waves of the launch before (se12_paged_attention.hip), which leave what a block
// of se12_paged_prompt.hip is to do in the workspace: a block that looked for its unit
// itself took 7,000 cycles to, and the join of parts as long (6,194 tokens of 5 prompts:
// 170 us that way, 164 this).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "se12_paged_device.hpp"

namespace se12step {

constexpr int kBlockColumns = 128;
constexpr int kLeastTiles = 8;            // of a block, where a unit's keys are split

// one unit: 128 columns of a sequence and KV head
struct Unit {
    int s, first;          // sequence, its first column of the unit
    Seq seq;
    int keys, columns;     // of the sequence
};

// The units in the order they are started: 64 sequences after the other, and among
// those by the last key they see, the most first, so that what is left for the last
// blocks is short. One lane holds one sequence: how many of its units see a key past
// 64 x is in closed form, so the x of a rank is found by halving.
struct UnitCounts {
    Seq seq;
    int keys, columns, units;
    // units that see past key x
    __device__ __forceinline__ int past(int x, int group) const {
        const int64_t c = (int64_t)max(x - seq.len, 0) * group;     // the first column that does
        return keys > x && c < columns ? units - (int)(c / kBlockColumns) : 0;
    }
};

// (within rows of 16 lanes by DPP, as the float sums of se12_step_math.hpp)
template <typename Op>
__device__ __forceinline__ int wave_all(int v, Op op) {
    v = op(v, __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true));
    v = op(v, __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true));
    v = op(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true));
    v = op(v, __builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, true));
    return op(op(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
              op(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ __forceinline__ int wave_total(int v) {
    return wave_all(v, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int wave_most(int v) {
    return wave_all(v, [](int a, int b) { return a > b ? a : b; });
}

__device__ __forceinline__ UnitCounts load_counts(const AttendArgs& a, int s0, int lane, int capacity) {
    UnitCounts c;
    c.seq = load_seq(a.b, min(s0 + lane, a.b.seqs - 1), capacity);
    c.keys = min(c.seq.len + c.seq.n, capacity);
    c.columns = s0 + lane < a.b.seqs ? c.seq.n * a.group : 0;
    c.units = c.columns > a.few ? (c.columns + kBlockColumns - 1) / kBlockColumns : 0;
    c.columns = c.units > 0 ? c.columns : 0;
    return c;
}

// Keys of a block where units are shared (splits > 1): about as many as make all units'
// keys one round of blocks, those of a sequence's units taken as a run from the first
// to the last.
template <int kTile>
__device__ __forceinline__ int shared_tiles(const AttendArgs& a, int lane, int resident) {
    const int capacity = a.b.width << a.page_log2;
    int64_t all = 0;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 64) {
        const UnitCounts c = load_counts(a, s0, lane, capacity);
        const int last = c.keys, first = min(c.seq.len + kBlockColumns / a.group, last), reach = a.window > 0 ? min(a.window, INT32_MAX - kTile) + kTile : INT32_MAX;
        // (a float holds it closely enough, and is the same for every block)
        all += wave_total((int)fminf((float)c.units * (float)(min(first, reach) / 2 + min(last, reach) / 2) / kTile, 1e7f));
    }
    return (int)min(all * a.kvh / resident + 1, (int64_t)INT32_MAX);
}

__device__ __forceinline__ bool find_unit(const AttendArgs& a, int rank, Unit& u) {
    const int lane = threadIdx.x & 63, capacity = a.b.width << a.page_log2;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 64) {
        const UnitCounts c = load_counts(a, s0, lane, capacity);
        const int all = wave_total(c.units);
        if (rank >= all) {
            rank -= all;
            continue;
        }
        const int most = wave_most(c.units > 0 ? c.keys : 0);
        // the largest x with more than `rank` units past 64 x (every unit is past -1)
        int lo = -1, hi = (most + 63) / 64;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (wave_total(c.past(64 * mid, a.group)) > rank)
                lo = mid;
            else
                hi = mid;
        }
        const int here = lo < 0 ? c.units : c.past(64 * lo, a.group), beyond = c.past(64 * (lo + 1), a.group);
        rank -= wave_total(beyond);
        int upto = here - beyond;      // of this x: a sequence's are units - here .. units - beyond - 1
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o, 64);
            upto += lane >= o ? v : 0;
        }
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > rank));
        auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
        u.s = s0 + l;
        u.seq = {of(c.seq.start), of(c.seq.n), of(c.seq.len)};
        u.keys = of(c.keys);
        u.columns = of(c.columns);
        u.first = kBlockColumns * (of(c.units) - of(here) + rank - (of(upto) - (of(here) - of(beyond))));
        return true;
    }
    return false;
}

// the key tiles the unit's columns see
template <int kTile>
__device__ __forceinline__ void unit_tiles(const AttendArgs& a, const Unit& u, int& t0, int& t1) {
    const int pos0 = u.seq.len + u.first / a.group;
    const int pos1 = u.seq.len + (min(u.first + kBlockColumns, u.columns) - 1) / a.group;
    t0 = (a.window > 0 ? max(0, pos0 - a.window + 1) : 0) / kTile;
    t1 = max((min(u.keys, pos1 + 1) + kTile - 1) / kTile, t0 + 1);
}

// blocks the card holds at once
template <int CT, int D>
constexpr int kResidentBlocks = 256 * (D == 256 || (D == 128 && CT == SE12_STEP_BF16) ? 1 : 2);

// Which units are shared: the first `units` of the order, in parts of about `tiles`
// tiles. Their parts come first, and then the others, the most keys first.
struct Sharing {
    int units, tiles;
};

template <int CT, int D>
__device__ __forceinline__ Sharing sharing_of(const AttendArgs& a, int lane) {
    constexpr int kTile = Form<CT>::kTile;
    if (a.splits == 1) return {0, INT32_MAX};
    const int tiles = max(shared_tiles<kTile>(a, lane, kResidentBlocks<CT, D>), kLeastTiles);
    // (all of them where their order is not that of their keys)
    if (a.b.seqs > 64 || a.window > 0) return {INT32_MAX / a.splits, tiles};
    return {wave_total(load_counts(a, 0, lane, a.b.width << a.page_log2).past((int)min((int64_t)tiles * kTile, (int64_t)INT32_MAX), a.group)), tiles};
}

// tiles of a block of a unit that has `tiles`
__device__ __forceinline__ int part_tiles(const AttendArgs& a, const Sharing& x, int rank, int tiles) {
    if (rank >= x.units) return tiles;
    const int parts = min((tiles + x.tiles - 1) / x.tiles, a.splits);
    return (tiles + parts - 1) / parts;
}

// A block's work, for all KV heads alike: a part (`split`, of `parts`) of the unit of
// this rank, key tiles t0 .. t1 - 1.
struct UnitWork {
    int s, first, start, n;        // s: -1 for none
    int len, keys, columns, t0;
    int t1, rank, split, parts;
};

template <int CT, int D>
__device__ __forceinline__ void write_unit(const AttendArgs& a, int x) {
    constexpr int kTile = Form<CT>::kTile;
    const int lane = threadIdx.x & 63;
    int rank = x, split = 0;
    const Sharing sharing = sharing_of<CT, D>(a, lane);
    if (rank < sharing.units * a.splits) {
        split = rank % a.splits;
        rank /= a.splits;
    } else {
        rank -= sharing.units * (a.splits - 1);
    }
    UnitWork w{-1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    Unit u;
    if (find_unit(a, rank, u)) {
        int t0, t1;
        unit_tiles<kTile>(a, u, t0, t1);
        const int length = part_tiles(a, sharing, rank, t1 - t0), parts = (t1 - t0 + length - 1) / length;
        if (split < parts)
            w = {u.s, u.first, u.seq.start, u.seq.n, u.seq.len, u.keys, u.columns, t0 + split * length, min(t1, t0 + (split + 1) * length),
                 rank, split, parts};
    }
    if (lane == 0) a.units[x] = w;
}

// of a block, the same in all its lanes
__device__ __forceinline__ UnitWork unit_work(const AttendArgs& a, int x) {
    const int4* p = reinterpret_cast<const int4*>(a.units + x);
    const int4 v[3] = {p[0], p[1], p[2]};
    auto of = [](int i) { return __builtin_amdgcn_readfirstlane(i); };
    return {of(v[0].x), of(v[0].y), of(v[0].z), of(v[0].w), of(v[1].x), of(v[1].y), of(v[1].z), of(v[1].w),
            of(v[2].x), of(v[2].y), of(v[2].z), of(v[2].w)};
}

}  // namespace se12step
