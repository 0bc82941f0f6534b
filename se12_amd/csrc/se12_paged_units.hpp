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

constexpr int kFewColumns = 64;           // of a sequence and KV head that se12_paged_attention.hip takes
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
    c.seq = load_seq(a.b, min(s0 + lane, a.b.seqs - 1));
    c.keys = min(c.seq.len + c.seq.n, capacity);
    c.columns = s0 + lane < a.b.seqs ? c.seq.n * a.group : 0;
    c.units = c.columns > kFewColumns ? (c.columns + kBlockColumns - 1) / kBlockColumns : 0;
    c.columns = c.units > 0 ? c.columns : 0;
    return c;
}

// unit `rank` of the order of 64 sequences
__device__ __forceinline__ Unit unit_of(const AttendArgs& a, const UnitCounts& c, int s0, int rank) {
    const int lane = threadIdx.x & 63, most = wave_most(c.units > 0 ? c.keys : 0);
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
    Unit u;
    u.s = s0 + l;
    u.seq = {of(c.seq.start), of(c.seq.n), of(c.seq.len)};
    u.keys = of(c.keys);
    u.columns = of(c.columns);
    u.first = kBlockColumns * (of(c.units) - of(here) + rank - (of(upto) - (of(here) - of(beyond))));
    return u;
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
constexpr int resident_blocks(bool e4m3, int d) { return 256 * (d == 256 || (d == 128 && !e4m3) ? 1 : 2); }

// Which units are shared: of every 64 sequences those that see more than `tiles` tiles,
// `units` of all at most, each in up to `splits` parts of about `tiles` tiles. Tiles: as
// many as make all units' one round of blocks, those of a sequence's units taken as a run
// from the first to the last, so a KV head's parts are as many as a round's blocks and the
// shared units together, and room for twice a round's is enough (a.parts).
struct Sharing {
    int units, splits, tiles;
};

template <int CT, int D>
__device__ __forceinline__ Sharing sharing_of(const AttendArgs& a, int lane) {
    constexpr int kTile = Form<CT>::kTile, kResident = resident_blocks(CT == SE12_STEP_E4M3, D);
    if (a.parts < 2) return {0, 1, 1};
    const int capacity = a.b.width << a.page_log2;
    int64_t tiles = 0, units = 0;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 64) {
        const UnitCounts c = load_counts(a, s0, lane, capacity);
        const int last = c.keys, first = min(c.seq.len + kBlockColumns / a.group, last);
        const int reach = a.window > 0 ? min(a.window, INT32_MAX - kTile) + kTile : INT32_MAX;
        // (a float holds it closely enough, and is the same for every block)
        tiles += wave_total((int)fminf((float)c.units * (float)(min(first, reach) / 2 + min(last, reach) / 2) / kTile, 1e7f));
        units += wave_total(c.units);
    }
    const int64_t each = max(min(tiles * a.kvh / kResident + 1, (int64_t)1 << 24), (int64_t)kLeastTiles);
    const int splits = (int)max(min(kResident / max(units * a.kvh, (int64_t)1), (int64_t)a.most), (int64_t)2);
    return {a.parts / splits, splits, (int)each};
}

// A block's work, for all KV heads alike: a part of a unit, key tiles t0 .. t1 - 1.
struct UnitWork {
    int s, first, start, len;      // s: -1 for none
    int keys, columns, t0, t1;
    int rank, split, parts;        // which of its `parts`, of which of the shared units
    int splits;                    // places for the parts of a unit
};

// where a part of a KV head's unit is held
__device__ __forceinline__ int64_t part_place(const AttendArgs& a, const UnitWork& u, int kh) {
    return ((int64_t)u.rank * a.kvh + kh) * u.splits + u.split;
}

// What block x does: of every 64 sequences the shared units' parts come first, then the
// others, the most keys first. Behind the blocks' records those of the joins: the shared units.
template <int CT, int D>
__device__ __forceinline__ void write_unit(const AttendArgs& a, int x) {
    constexpr int kTile = Form<CT>::kTile;
    const int lane = threadIdx.x & 63, capacity = a.b.width << a.page_log2;
    const bool join = x >= a.unit_count;
    int index = join ? x - a.unit_count : x, left, before = 0;
    const Sharing sharing = sharing_of<CT, D>(a, lane);
    const int limit = (sharing.tiles * kTile) & ~63;      // (the order is that of 64 keys)
    left = sharing.units;
    UnitWork w{-1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    for (int s0 = 0; s0 < a.b.seqs; s0 += 64) {
        const UnitCounts c = load_counts(a, s0, lane, capacity);
        const int all = wave_total(c.units), shared = left > 0 ? min(wave_total(c.past(limit, a.group)), left) : 0;
        const int first_alone = shared * sharing.splits, count = join ? shared : first_alone + all - shared;
        if (index >= count) {
            index -= count;
            left -= shared;
            before += shared;
            continue;
        }
        const bool alone = !join && index >= first_alone;
        const int rank = alone ? shared + index - first_alone : join ? index : index / sharing.splits;
        const int split = alone || join ? 0 : index - rank * sharing.splits;
        const Unit u = unit_of(a, c, s0, rank);
        int t0, t1;
        unit_tiles<kTile>(a, u, t0, t1);
        const int wanted = alone ? 1 : min((t1 - t0 + sharing.tiles - 1) / sharing.tiles, sharing.splits);
        const int length = (t1 - t0 + wanted - 1) / wanted, parts = (t1 - t0 + length - 1) / length;
        if (split < parts)
            w = {u.s, u.first, u.seq.start, u.seq.len, u.keys, u.columns, t0 + split * length, min(t1, t0 + (split + 1) * length),
                 before + rank, split, parts, sharing.splits};
        break;
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
