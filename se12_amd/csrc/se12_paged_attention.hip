// Attention over a paged key/value cache of BF16 or E4M3 (a scale per page and
// head). Mathematics, per query: s_j = cap(q . k_j kscale_j scaling), o = sum_j
// 2^(s_j - m) vscale_j v_j / sum_j 2^(s_j - m) over the keys it sees (scores in
// base 2), in one pass over the pages: m is the largest score met so far, or up
// to kSlack below it; a tile that passes it by more moves it and what is summed.
//
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16 (A: lane l holds row
// l % 16, inner positions 8 (l / 16) ..; B: the same of column l % 16; D: column
// l % 16, rows 4 (l / 16) ..). Columns are a sequence's (token, query head)
// pairs of one KV head, 16 to a unit. Of a tile of 64 keys, row r of the first
// product's step t is key 16 (r / 4) + 4 t + r % 4, so a lane's scores, as they
// come out, are those of keys 16 (l / 16) .. + 15 of its column: the second
// product's B operand, with V held transposed in its pages as the A operand,
// 16 keys of a column in a lane. So keys, values and probabilities go from
// memory through registers only: no LDS, no exchange between lanes, and the
// scales (one page at least holds 16 keys) are one number per lane and tile.
// Scores, statistics and sums are FP32; a weight, times the values' scale, is rounded to
// BF16, the type of the second product's operands: off by 2^-8 of it at most, as the output
// is by its own rounding, and less in a sum over many keys. (A weight in two BF16 parts
// would double the second product.)
//
// Bound by the bytes of the pages: 32 sequences of up to 4,095 keys, 16 / 8 heads of 256
// in E4M3 (309 MB) take 60 us and 4 to join, 4.9 TB/s; 24 of up to 5,000 in BF16 under a
// window of 4,096 (273 MB) 52 and 4. One sequence of 1,023 keys: 9.4 + 3.8 us, the loads
// that wait for each other (length, table entry, keys) and the second launch.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "se12_paged_attend4.hpp"
#include "se12_paged_units.hpp"

namespace se12step {

constexpr int kColumns = 16;          // columns of a unit
// waves of a launch: one per SIMD of 256 CUs (3 x 65,000 keys, 28 / 4 heads of 128: 31.5
// us, 36 with two, which have two starts and twice the parts to join)
constexpr int kWorkersLog2 = 10, kWorkers = 1 << kWorkersLog2;
constexpr int kAttendThreads = 256;   // four waves, each with tiles of its own

// The work: units of up to 16 columns of one sequence and KV head, each a run of
// key tiles; all units' tiles in one line (sequence, head, column unit, tile),
// cut evenly over the waves, so that sequences of any lengths load them alike.
struct SeqWork {
    Seq seq;
    int keys;      // held and new, as far as the table reaches
    int tile0;     // first tile any query sees
    int tiles;     // tiles of a unit
    int units;     // column units
};

template <int kTile>
__device__ __forceinline__ SeqWork seq_work(const AttendArgs& a, Seq seq) {
    SeqWork w;
    w.seq = seq;
    w.keys = min(seq.len + seq.n, a.b.width << a.page_log2);
    const int low = a.window > 0 ? max(0, seq.len - a.window + 1) : 0;
    w.tile0 = low / kTile;
    const int columns = seq.n * a.group;
    w.units = columns > kFewColumns ? 0 : (columns + kColumns - 1) / kColumns;
    w.tiles = w.units > 0 ? max((w.keys + kTile - 1) / kTile - w.tile0, 1) : 0;
    return w;
}

// 64 sequences' work, one to a lane: the tiles of all heads and units, those of the
// lanes up to it, and of all (the C entry sees to it that 32 bits hold them)
struct Chunk {
    Seq seq;
    int tiles, upto, all;
};

template <int kTile>
__device__ __forceinline__ Chunk load_chunk(const AttendArgs& a, int s0, int lane) {
    Chunk c;
    const int s = s0 + lane;
    c.seq = load_seq(a.b, min(s, a.b.seqs - 1));
    if (s >= a.b.seqs) c.seq.n = 0;
    const SeqWork w = seq_work<kTile>(a, c.seq);
    c.tiles = w.tiles * w.units * a.kvh;
    c.upto = c.tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(c.upto, o, 64);
        c.upto += lane >= o ? u : 0;
    }
    c.all = __builtin_amdgcn_readlane(c.upto, 63);
    return c;
}

// tiles of a worker (workers that are not launched, where there can be no more
// tiles than are, would have none)
__device__ __forceinline__ int64_t tiles_each(int64_t total) { return (total + kWorkers - 1) >> kWorkersLog2; }

// (at / each is below kWorkers; 64-bit division only where it takes one)
__device__ __forceinline__ int worker_of(int64_t at, int64_t each) {
    return ((at | each) >> 32) == 0 ? (int)((uint32_t)at / (uint32_t)each) : (int)(at / each);
}

__device__ __forceinline__ Seq seq_of(const Chunk& c, int l) {
    return {__builtin_amdgcn_readlane(c.seq.start, l), __builtin_amdgcn_readlane(c.seq.n, l), __builtin_amdgcn_readlane(c.seq.len, l)};
}

// (of E2M1: se12_paged_attend4.hpp)
template <int CT, int D>
struct Attend {
    using F = Form<CT>;
    static constexpr int kTile = F::kTile, kPer = F::kPer, kHalves = F::kHalves;
    static constexpr int kSteps = kPer / 4;          // row steps of the first product
    static constexpr int kChunks = D / (4 * kPer);   // 64-byte parts of a key
    static constexpr int kRows = D / 16;             // 16-column parts of the output
    floatx4_t o[kRows];
    float m, l;

    // what the lane holds of its column: runs of four
    template <typename Store>
    __device__ __forceinline__ void each_part(Store store) const {
        const int quarter = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < kRows; ++i) store(16 * i + 4 * quarter, o[i]);
    }

    // one run of tiles of a unit
    __device__ __forceinline__ void run(const AttendArgs& a, int s, const SeqWork& w, int kh, int unit, int tile, int tiles) {
        const int lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
        const int columns = min(kColumns, w.seq.n * a.group - unit * kColumns);
        const bool live = col < columns;
        const int c = unit * kColumns + (live ? col : 0), token = c / a.group;
        const int pos = live ? w.seq.len + token : -1;                       // -1 sees nothing
        const int pos_min = w.seq.len + unit * kColumns / a.group;
        const int pos_max = w.seq.len + (unit * kColumns + columns - 1) / a.group;
        const int reach = a.window > 0 ? a.window : INT32_MAX;
        const int low = max(0, pos_min - reach + 1), high = min(w.keys, pos_max + 1);   // keys some column sees
        const uint16_t* qp = a.q + (w.seq.start + token) * a.q_stride + (int64_t)(kh * a.group + c % a.group) * D + kPer * quarter;
        bf16x8_t qf[kChunks][kHalves];
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
#pragma unroll
            for (int h = 0; h < kHalves; ++h) qf[i][h] = *reinterpret_cast<const bf16x8_t*>(qp + 4 * kPer * i + 8 * h);
#pragma unroll
        for (int i = 0; i < kRows; ++i) o[i] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
        m = -INFINITY;
        l = 0.0f;
        const int t0 = max(w.tile0 + tile, low / kTile), t1 = min(w.tile0 + tile + tiles, (high + kTile - 1) / kTile);
        if (t0 >= t1) return;
        const int P = 1 << a.page_log2;
        // the keys a lane takes: K rows krow + 4 step of a tile, V keys vkey .. + kPer - 1
        const int kgroup = kPer * (col >> 2), krow = kgroup + (col & 3), vkey = kPer * quarter;
        const int64_t page_elems = (int64_t)P * D;
        // a tile's table entries are loaded a tile ahead of their pages, without a
        // branch that would wait for them (a column behind the table's last: that one)
        const int32_t* table = a.b.table + s * a.b.table_stride;
        auto entry = [&](int key) { return table[min(key >> a.page_log2, a.b.width - 1)]; };
        auto held_page = [&](int e) { return (uint32_t)e < (uint32_t)a.pages ? e : 0; };
        uint4 kf[kSteps][kChunks];
        auto load_k = [&](int t, int page) {
            const int64_t at = ((int64_t)held_page(page) * a.kvh + kh) * page_elems + (int64_t)((t * kTile + krow) & (P - 1)) * D + kPer * quarter;
#pragma unroll
            for (int g = 0; g < kSteps; ++g)
#pragma unroll
                for (int i = 0; i < kChunks; ++i) kf[g][i] = load_piece<CT>(a.kc, at + 4 * g * D + 4 * kPer * i);
        };
        int vpage = entry(t0 * kTile + vkey), vpage_next = entry(min(t0 + 1, t1 - 1) * kTile + vkey);
        int kpage_next = entry(min(t0 + 1, t1 - 1) * kTile + kgroup);
        load_k(t0, entry(t0 * kTile + kgroup));
        uint4 vf[kRows];
        float sc[kPer], top = 0.0f, vs = 1.0f;
        bf16x8_t pf[kHalves];
        auto weights = [&]() {
            const float base = (m == -INFINITY ? 0.0f : m) + (CT == SE12_STEP_BF16 ? a.shift : 0.0f);
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                uint32_t u[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float p0 = __builtin_amdgcn_exp2f(sc[8 * h + 2 * k] - base);
                    const float p1 = __builtin_amdgcn_exp2f(sc[8 * h + 2 * k + 1] - base);
                    l += p0 + p1;
                    u[k] = f_to_bf16x2(p0 * vs, p1 * vs);
                }
                pf[h] = __builtin_bit_cast(bf16x8_t, make_uint4(u[0], u[1], u[2], u[3]));
            }
        };
        auto add_values = [&]() {
#pragma unroll
            for (int i = 0; i < kRows; ++i)
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand<CT>(vf[i], h), pf[h], o[i], 0, 0, 0);
        };
        auto column_max = [&](float v) {
            v = fmaxf(v, __shfl_xor(v, 16, 64));
            return fmaxf(v, __shfl_xor(v, 32, 64));
        };
        for (int t = t0;; ++t) {
            bool apart = false;     // a value that is no number may be hidden from some of the columns
            bool higher = false;    // a score passes the maximum by more than kSlack
            for (; t < t1; ++t) {
                const int k0 = t * kTile, key0 = k0 + vkey;
                const int64_t head_page = (int64_t)held_page(vpage) * a.kvh + kh;
                // (what the page of unseen keys holds, its scales too, may be anything)
                const bool held = (uint32_t)vpage < (uint32_t)a.pages && key0 < high && key0 + kPer > low;
                const int next = min(t + 1, t1 - 1), after = min(t + 2, t1 - 1);
                const int kpage_after = entry(after * kTile + kgroup), vpage_after = entry(after * kTile + vkey);
                float ks = 1.0f;
                if constexpr (CT == SE12_STEP_E4M3) {
                    ks = a.k_scale[head_page];
                    vs = a.v_scale[head_page];
                }
                {
                    const int64_t at = head_page * page_elems + (int64_t)col * P + (key0 & (P - 1));
#pragma unroll
                    for (int i = 0; i < kRows; ++i) vf[i] = load_piece<CT>(a.vc, at + 16 * i * P);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int g = 0; g < kSteps; ++g) {
                    floatx4_t d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < kChunks; ++i)
#pragma unroll
                        for (int h = 0; h < kHalves; ++h)
                            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand<CT>(kf[g][i], h), qf[i][h], d, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[4 * g + e] = d[e];
                }
                __builtin_amdgcn_sched_barrier(0);
                load_k(next, kpage_next);
                __builtin_amdgcn_sched_barrier(0);
                const float by = a.c1 * ks;
                if (a.cap > 0.0f) {
#pragma unroll
                    for (int e = 0; e < kPer; ++e)
                        sc[e] = a.cap - 2.0f * a.cap * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(sc[e] * by));
                } else {
#pragma unroll
                    for (int e = 0; e < kPer; ++e) sc[e] *= by;
                }
                const bool inside = k0 + kTile - 1 <= pos_min && k0 + kTile <= w.keys && pos_max - k0 < reach &&
                                    __builtin_amdgcn_ballot_w64(!held) == 0;
                if (!inside) {
                    if constexpr (CT == SE12_STEP_E4M3) vs = held ? vs : 0.0f;   // (of this tile's page)
                    const int from = max(pos - reach + 1, 0) - key0, to = held ? min(pos + 1, w.keys) - key0 : 0;
#pragma unroll
                    for (int e = 0; e < kPer; ++e) sc[e] = (e < from || e >= to) ? -INFINITY : sc[e];
                    const uint4 mask = piece_mask<CT>(low - key0, held ? high - key0 : 0);
                    bool bad = false;
#pragma unroll
                    for (int i = 0; i < kRows; ++i) {
                        vf[i] = masked(vf[i], mask);
                        bad |= has_no_number<CT>(vf[i]);
                    }
                    apart = __builtin_amdgcn_ballot_w64(bad) != 0;
                }
                top = sc[0];
#pragma unroll
                for (int e = 1; e < kPer; ++e) top = fmaxf(top, sc[e]);
                if (t == t0) m = column_max(top);
                higher = __builtin_amdgcn_ballot_w64(top > m + kSlack) != 0;
                vpage = vpage_next;
                vpage_next = vpage_after;
                kpage_next = kpage_after;
                if (higher || apart) break;
                weights();
                add_values();
            }
            if (t >= t1) break;
            // The rare tile, outside the loop, where the sums may stay in accumulation
            // registers: the maximum moves, and what is summed with it; 0 x NaN is
            // NaN, so a value that is no number leaves the product and comes back in
            // the columns that give it a weight.
            const float to = fmaxf(m, column_max(top));
            const float scale = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= scale;
#pragma unroll
            for (int i = 0; i < kRows; ++i) o[i] *= scale;
            weights();
            if (apart) {
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
#pragma unroll
                    for (int kind = 0; kind < (CT == SE12_STEP_E4M3 ? 1 : 3); ++kind) {
                        floatx4_t d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int h = 0; h < kHalves; ++h) {
                            const uint4 v = __builtin_bit_cast(uint4, operand<CT>(vf[i], h));
                            const uint4 is = make_uint4(where_no_number(v.x, kind), where_no_number(v.y, kind),
                                                        where_no_number(v.z, kind), where_no_number(v.w, kind));
                            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, is), pf[h], d, 0, 0, 0);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o[i][e] += d[e] == 0.0f ? 0.0f : kind == 0 ? __builtin_nanf("") : kind == 1 ? INFINITY : -INFINITY;
                    }
                    vf[i] = make_uint4(numbers_only<CT>(vf[i].x), numbers_only<CT>(vf[i].y), numbers_only<CT>(vf[i].z),
                                       numbers_only<CT>(vf[i].w));
                }
            }
            // (a row at a time, for the registers' sake)
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand<CT>(vf[i], h), pf[h], o[i], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
    }
};

// a worker's sums of a run that is not a whole unit: slot 0 where the unit began
// before its run, slot 1 where it goes on after it
__device__ __forceinline__ int64_t part_at(const AttendArgs& a, int worker, int slot) { return ((int64_t)worker * 2 + slot) * a.columns; }

template <int CT, int D>
__global__ __launch_bounds__(kAttendThreads, D == 256 ? 1 : 2) void paged_attention_kernel(AttendArgs a) {
    constexpr int kTile = Form<CT>::kTile;
    const int lane = threadIdx.x & 63;
    const int worker = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * (kAttendThreads / 64) + (threadIdx.x >> 6)));
    // (workers come four to a block; behind them waves for the units of se12_paged_prompt.hip)
    if (worker >= a.workers) {
        if (worker - a.workers < a.unit_count + a.join_count) write_unit<CT, D>(a, worker - a.workers);
        return;
    }
    Chunk chunk = load_chunk<kTile>(a, 0, lane);
    int64_t total = chunk.all;
    for (int s0 = 64; s0 < a.b.seqs; s0 += 64) total += load_chunk<kTile>(a, s0, lane).all;
    const int64_t per = tiles_each(total);
    int64_t at = worker * per;
    const int64_t end = min(at + per, total);
    int64_t before = 0;      // tiles of the sequences before the chunk
    for (int s0 = 0; at < end;) {
        const uint64_t past = __builtin_amdgcn_ballot_w64(before + chunk.upto > at);
        if (!past) {
            before += chunk.all;
            s0 += 64;
            chunk = load_chunk<kTile>(a, s0, lane);
            continue;
        }
        const int of = __builtin_ctzll(past);
        const SeqWork w = seq_work<kTile>(a, seq_of(chunk, of));
        const int in = (int)(at - before) - (__builtin_amdgcn_readlane(chunk.upto, of) - __builtin_amdgcn_readlane(chunk.tiles, of));
        const int line = in / w.tiles, tile = in - line * w.tiles, kh = line / w.units, unit = line - kh * w.units;
        const int tiles = (int)min((int64_t)(w.tiles - tile), end - at);
        Attend<CT, D> x;
        x.run(a, s0 + of, w, kh, unit, tile, tiles);
        const int col = lane & 15, quarter = lane >> 4, c = unit * kColumns + col;
        if (c < w.seq.n * a.group) {
            if (tiles == w.tiles) {
                const float inv = x.l == 0.0f ? 0.0f : 1.0f / x.l;
                uint16_t* out = a.out + ((int64_t)(w.seq.start + c / a.group) * a.heads + kh * a.group + c % a.group) * D;
                x.each_part([&](int at, floatx4_t v) { store4(out + at, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv); });
            } else {
                const int64_t p = part_at(a, worker, tile > 0 ? 0 : 1) + col;
                x.each_part([&](int at, floatx4_t v) { *reinterpret_cast<floatx4_t*>(a.part + p * D + at) = v; });
                if (quarter == 0) {
                    float* ml = a.part + (int64_t)a.workers * 2 * a.columns * D + 2 * p;
                    ml[0] = x.m;
                    ml[1] = x.l;
                }
            }
        }
        at += tiles;
    }
}

// The units that several workers share, from their parts in order: a block (for every
// column, or every fourth) per (sequence, KV head, column unit), or, where those are many
// beside the workers (max_units 0), per worker, which joins the unit that the worker begins
// and others go on with. (1,024 sequences to 1,000 keys, 16 / 8 heads of 256, a block per
// unit: 126 us, and 848 where max_new allows 64 columns; per worker 43 and 60.) D / 4
// lanes take every kParts-th part, the loads of four at once, or of eight where there are
// as many (85 parts at D = 128: 6.8 us by four, 6.1 so; 12 at once are 8.0, for few parts
// 6.8 from 4.6); a part's maximum may lie above those before it, so what is summed moves
// with it.
// Of a grid of blocks [nx][ny] (max_units 0: x a worker) block x, y.
template <int CT, int D>
__device__ __forceinline__ void join_columns(const AttendArgs& a, int max_units, int x, int y, int ny) {
    constexpr int kTile = Form<CT>::kTile;
    constexpr int kLanes = D / 4, kParts = kAttendThreads / kLanes;
    __shared__ float4 sums[kAttendThreads];
    __shared__ float2 mls[kParts];
    const int tid = threadIdx.x, lane = tid & 63, part = tid / kLanes, at = tid % kLanes;
    int unit, kh;
    SeqWork w;
    int64_t first, per;      // the unit's first tile, tiles of a worker
    if (max_units > 0) {
        unit = x % max_units;
        kh = x / max_units % a.kvh;
        const int s = x / max_units / a.kvh;
        const Chunk chunk = load_chunk<kTile>(a, s & ~63, lane);
        w = seq_work<kTile>(a, seq_of(chunk, s & 63));
        if (unit >= w.units || unit * kColumns + y >= w.seq.n * a.group) return;
        int64_t base = __builtin_amdgcn_readlane(chunk.upto, s & 63) - __builtin_amdgcn_readlane(chunk.tiles, s & 63), total = chunk.all;
        for (int s0 = 0; s0 < a.b.seqs; s0 += 64) {
            if (s0 == (s & ~63)) continue;
            const int all = load_chunk<kTile>(a, s0, lane).all;
            total += all;
            base += s0 < s ? all : 0;
        }
        per = tiles_each(total);
        first = base + ((int64_t)kh * w.units + unit) * w.tiles;
    } else {
        Chunk chunk = load_chunk<kTile>(a, 0, lane);
        int64_t total = chunk.all, before = 0;
        for (int s0 = 64; s0 < a.b.seqs; s0 += 64) total += load_chunk<kTile>(a, s0, lane).all;
        per = tiles_each(total);
        const int64_t at = ((int64_t)x + 1) * per;      // where the next worker begins
        if (at >= total) return;
        for (int s0 = 64; before + chunk.all <= at; s0 += 64) {
            before += chunk.all;
            chunk = load_chunk<kTile>(a, s0, lane);
        }
        const int of = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + chunk.upto > at));
        w = seq_work<kTile>(a, seq_of(chunk, of));
        const int in = (int)(at - before) - (__builtin_amdgcn_readlane(chunk.upto, of) - __builtin_amdgcn_readlane(chunk.tiles, of));
        const int line = in / w.tiles, tile = in - line * w.tiles;
        kh = line / w.units;
        unit = line - kh * w.units;
        first = at - tile;
        if (tile == 0 || worker_of(first, per) != x) return;
    }
    const int w0 = worker_of(first, per), w1 = worker_of(first + w.tiles - 1, per);
    if (w0 == w1) return;      // one worker had it all
    const float2* mlp = reinterpret_cast<const float2*>(a.part + (int64_t)a.workers * 2 * a.columns * D);
    for (int col = y; col < kColumns; col += ny) {
        const int c = unit * kColumns + col;
        if (c >= w.seq.n * a.group) break;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto add = [&](int k0, auto batch) {
            constexpr int kBatch = batch.value;
            float2 ml[kBatch];
            float4 v[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int k = k0 + i * kParts;
                const int64_t p = part_at(a, min(k, w1), k == w0 ? 1 : 0) + col;
                ml[i] = mlp[p];
                v[i] = *reinterpret_cast<const float4*>(a.part + p * D + 4 * at);
            }
            float to = m;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) to = k0 + i * kParts <= w1 ? fmaxf(to, ml[i].x) : to;
            const float top = to == -INFINITY ? 0.0f : to, keep = __builtin_amdgcn_exp2f(m - top);
            m = to;
            l *= keep;
            o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (k0 + i * kParts > w1) continue;
                const float by = __builtin_amdgcn_exp2f(ml[i].x - top);
                l += by * ml[i].y;
                o.x += by * v[i].x;
                o.y += by * v[i].y;
                o.z += by * v[i].z;
                o.w += by * v[i].w;
            }
        };
        for (int k0 = w0; k0 <= w1;) {
            const bool many = w1 - k0 >= 4 * kParts;
            many ? add(k0 + part, std::integral_constant<int, 8>{}) : add(k0 + part, std::integral_constant<int, 4>{});
            k0 += kParts * (many ? 8 : 4);
        }
        sums[tid] = o;
        if (at == 0) mls[part] = make_float2(m, l);
        __syncthreads();
        if (tid < kLanes) {
            float to = mls[0].x;
#pragma unroll
            for (int k = 1; k < kParts; ++k) to = fmaxf(to, mls[k].x);
            to = to == -INFINITY ? 0.0f : to;
            o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            l = 0.0f;
#pragma unroll
            for (int k = 0; k < kParts; ++k) {
                const float4 v = sums[k * kLanes + tid];
                const float by = __builtin_amdgcn_exp2f(mls[k].x - to);
                l += by * mls[k].y;
                o.x += by * v.x;
                o.y += by * v.y;
                o.z += by * v.z;
                o.w += by * v.w;
            }
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            store4(a.out + ((int64_t)(w.seq.start + c / a.group) * a.heads + kh * a.group + c % a.group) * D + 4 * tid, o.x * inv, o.y * inv,
                   o.z * inv, o.w * inv);
        }
        __syncthreads();      // sums and mls are free again
    }
}

template <int CT, int D>
__global__ __launch_bounds__(kAttendThreads) void paged_join_kernel(AttendArgs a, int max_units) {
    join_columns<CT, D>(a, max_units, (int)blockIdx.x, (int)blockIdx.y, (int)gridDim.y);
}

// Both joins of a call that may have prompts, behind their kernel: the prompts' units, then the
// others' columns (a launch each: 302 tokens of 4 sequences 41 us for 39).
template <int CT, int D>
__global__ __launch_bounds__(kAttendThreads) void paged_joins_kernel(AttendArgs a, float* prompt_part, int prompt_blocks, int max_units, int nx, int ny) {
    const int block = (int)blockIdx.x - prompt_blocks;
    if (block < 0) {
        a.part = prompt_part;
        join_unit<D>(a, (int)blockIdx.x);
    } else {
        join_columns<CT, D>(a, max_units, block % nx, block / nx, ny);
    }
}

}  // namespace se12step

using namespace se12step;

namespace {

int column_count(const Batch& b, int group) {
    return (int)std::min<int64_t>(kColumns, (int64_t)b.max_new * group);
}

int worker_count(const se12_step_pages* p, const Batch& b, int group) {
    // no more than there can be tiles
    const int64_t tiles = ((int64_t)b.width * p->page_size + 31) / 32;
    const int64_t units = (std::min<int64_t>((int64_t)b.max_new * group, kFewColumns) + kColumns - 1) / kColumns;
    int64_t all = tiles;
    for (const int64_t f : {(int64_t)b.seqs, (int64_t)p->kv_heads, units}) all = std::min<int64_t>(all * f, kWorkers);
    return (int)((all + 3) / 4 * 4);
}

int64_t few_bytes(const se12_step_pages* p, const Batch& b, int group) {
    return ((int64_t)worker_count(p, b, group) * 2 * column_count(b, group) * (p->head_dim + 2) * (int64_t)sizeof(float) + 255) / 256 * 256;
}

PromptPlan plan_of(const se12_step_pages* p, const Batch& b, int group) {
    if ((int64_t)b.max_new * group <= kFewColumns) return {};
    return prompt_plan(b, p->kv_heads, group, p->page_size, p->head_dim, p->dtype);
}

// what one launch holds, and what 32 bits hold of it
const char* limits_error(const se12_step_pages* p, const Batch& b, int group) {
    const int most_threads = (p->dtype == SE12_STEP_E2M1 && p->head_dim == 256 ? 2 : 1) * kAttendThreads;      // (of a block of prompts)
    if ((int64_t)b.tokens * group > INT32_MAX || !grid_fits(plan_of(p, b, group).records * p->kv_heads, most_threads))
        return "too many sequences, tokens and heads for one launch";
    if (std::min<int64_t>(b.seqs, 64) * (((int64_t)b.width * p->page_size + 31) / 32) * (kFewColumns / kColumns) * p->kv_heads > INT32_MAX)
        return "too long a table for so many sequences and heads";
    return nullptr;
}

int64_t all_bytes(const se12_step_pages* p, const Batch& b, int group) {
    const PromptPlan x = plan_of(p, b, group);
    return few_bytes(p, b, group) + x.record_bytes + x.part_bytes;
}

// part: of the prompts' units, NULL where no sequence can have any
template <int CT, int D>
void launch_attend(const AttendArgs& a, float* part, hipStream_t st) {
    constexpr int kWaves = kAttendThreads / 64;
    hipLaunchKernelGGL((paged_attention_kernel<CT, D>), dim3((uint32_t)(((int64_t)a.workers + a.unit_count + a.join_count + kWaves - 1) / kWaves)),
                       dim3(kAttendThreads), 0, st, a);
    const int max_units = (int)((std::min<int64_t>((int64_t)a.b.max_new * a.group, kFewColumns) + kColumns - 1) / kColumns);
    const int64_t units = (int64_t)a.b.seqs * a.kvh * max_units;
    // (half as many again where each can be there: 130 sequences of one token, 8 KV heads of
    // 128, the call 29.7 us a block per unit, 30.8 per worker; 200 of 256 196 either way)
    const bool by_unit = units <= (max_units > 1 ? a.workers : a.workers + a.workers / 2);
    const int nx = by_unit ? (int)units : a.workers, ny = max_units > 1 ? 4 : a.columns;
    if (!part) {
        hipLaunchKernelGGL((paged_join_kernel<CT, D>), dim3(nx, ny), dim3(kAttendThreads), 0, st, a, by_unit ? max_units : 0);
        return;
    }
    AttendArgs prompts = a;
    prompts.part = part;
    launch_prompt(prompts, CT, D, st);
    const int blocks = join_blocks<D>(a);
    hipLaunchKernelGGL((paged_joins_kernel<CT, D>), dim3(blocks + nx * ny), dim3(kAttendThreads), 0, st, a, part, blocks, by_unit ? max_units : 0, nx, ny);
}

template <int CT>
void launch_attend_of(const AttendArgs& a, float* part, int d, hipStream_t st) {
    switch (d) {
        case 64: launch_attend<CT, 64>(a, part, st); break;
        case 128: launch_attend<CT, 128>(a, part, st); break;
        default: launch_attend<CT, 256>(a, part, st);
    }
}

}  // namespace

extern "C" {

int64_t se12_step_paged_attention_workspace(const se12_step_pages* pages, const se12_step_batch* batch, int32_t heads) {
    const char* fn = "se12_step_paged_attention_workspace";
    if (const char* e = paged_error(pages, batch, heads)) return step_fail(fn, e);
    if (batch->tokens == 0) return 0;
    const Batch b = device_batch(batch);
    if (const char* e = limits_error(pages, b, heads / pages->kv_heads)) return step_fail(fn, e);
    return all_bytes(pages, b, heads / pages->kv_heads);
}

int se12_step_paged_attention(const se12_step_pages* pages, const se12_step_batch* batch, const uint16_t* q,
                              int64_t q_stride, uint16_t* out, int32_t heads, float scaling, float softcap,
                              int32_t window, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "se12_step_paged_attention";
    if (const char* e = paged_error(pages, batch, heads)) return step_fail(fn, e);
    if (batch->tokens > 0 && (!q || !out)) return step_fail(fn, "NULL argument");
    if (q_stride < (int64_t)heads * pages->head_dim || q_stride % 8) return step_fail(fn, "q rows must be a multiple of 8 elements apart and hold all heads");
    if (!softcap_fits(softcap) || window < 0) return step_fail(fn, "softcap must be 0, or 2^-60 to 1024, and window 0 or more");
    constexpr float kLog2E = 1.4426950408889634f;
    const float c1 = softcap > 0.0f ? 2.0f * scaling / softcap * kLog2E : scaling * kLog2E;
    if (!(c1 - c1 == 0.0f)) return step_fail(fn, "scaling, or scaling / softcap, must be finite");
    if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(out) % 8) return step_fail(fn, "misaligned tensor");
    if (batch->tokens == 0) return SE12_STEP_OK;
    const Batch b = device_batch(batch);
    const int group = heads / pages->kv_heads;
    if (const char* e = limits_error(pages, b, group)) return step_fail(fn, e);
    if (reinterpret_cast<uintptr_t>(workspace) % 256 || !workspace || workspace_bytes < all_bytes(pages, b, group))
        return step_fail(fn, "workspace missing, misaligned or too small");
    // (q is read until the last wave is done with it)
    const int64_t row = (int64_t)heads * pages->head_dim;
    if (overlap(q, 2 * ((b.tokens - 1) * q_stride + row), out, 2 * b.tokens * row))
        return step_fail(fn, "out overlaps q");
    const PromptPlan plan = plan_of(pages, b, group);
    const int64_t held = (int64_t)b.width * pages->page_size, seen = window > 0 ? std::min<int64_t>(held, window) : held;
    const float shift = kSlack + 1.0f + (float)(64 - __builtin_clzll((uint64_t)seen));
    AttendArgs a{q, q_stride, out, pages->k, pages->v, pages->k_scale, pages->v_scale, b, heads, pages->kv_heads, group, pages->pages,
                 log2_of(pages->page_size), window, c1,
                 softcap * kLog2E, shift, static_cast<float*>(workspace), worker_count(pages, b, group), column_count(b, group),
                 reinterpret_cast<UnitWork*>(static_cast<char*>(workspace) + few_bytes(pages, b, group)),
                 (int)plan.slots + plan.parts, plan.parts / 2, plan.parts, plan.most};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    float* part = plan.records > 0 ? reinterpret_cast<float*>(reinterpret_cast<char*>(a.units) + plan.record_bytes) : nullptr;
    switch (pages->dtype) {
        case SE12_STEP_E2M1: launch_attend_of<SE12_STEP_E2M1>(a, part, pages->head_dim, st); break;
        case SE12_STEP_E4M3: launch_attend_of<SE12_STEP_E4M3>(a, part, pages->head_dim, st); break;
        default: launch_attend_of<SE12_STEP_BF16>(a, part, pages->head_dim, st);
    }
    return step_launched();
}

}  // extern "C"
