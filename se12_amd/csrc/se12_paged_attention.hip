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
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "se12_paged_device.hpp"

namespace se12step {

constexpr int kColumns = 16;          // columns of a unit
constexpr int kFewColumns = 64;       // of a sequence and KV head; with more it is se12_paged_prompt.hip's
constexpr int kAttendThreads = 256;   // four waves, each with tiles of its own
constexpr int kWorkers = 256 * 4;     // waves of a launch: one per SIMD

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
__device__ __forceinline__ SeqWork seq_work(const AttendArgs& a, int s) {
    SeqWork w;
    const int capacity = a.b.width << a.page_log2;
    w.seq = load_seq(a.b, s, capacity);
    w.keys = min(w.seq.len + w.seq.n, capacity);
    const int low = a.window > 0 ? max(0, w.seq.len - a.window + 1) : 0;
    w.tile0 = low / kTile;
    const int columns = w.seq.n * a.group;
    w.units = columns > a.few ? 0 : (columns + kColumns - 1) / kColumns;
    w.tiles = w.units > 0 ? max((w.keys + kTile - 1) / kTile - w.tile0, 1) : 0;
    return w;
}

__device__ __forceinline__ int64_t shfl64(int64_t v, int from) {
    const int lo = __shfl((int)v, from, 64), hi = __shfl((int)(v >> 32), from, 64);
    return ((int64_t)hi << 32) | (uint32_t)lo;
}

// inclusive prefix sums of a wave's values
__device__ __forceinline__ int64_t scan64(int64_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = shfl64(v, lane - o);
        v += lane >= o ? u : 0;
    }
    return v;
}

// tiles of sequence s over all heads and units
template <int kTile>
__device__ __forceinline__ int64_t seq_tiles(const AttendArgs& a, int s) {
    if (s >= a.b.seqs) return 0;
    const SeqWork w = seq_work<kTile>(a, s);
    return (int64_t)w.tiles * w.units * a.kvh;
}

template <int kTile>
__device__ __forceinline__ int64_t all_tiles(const AttendArgs& a, int lane) {
    int64_t total = 0;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 64) total += shfl64(scan64(seq_tiles<kTile>(a, s0 + lane), lane), 63);
    return total;
}

// the sequence that holds tile `at` of the line, and the tile its part begins at
template <int kTile>
__device__ __forceinline__ int seq_of_tile(const AttendArgs& a, int64_t at, int lane, int64_t& base) {
    int64_t before = 0;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 64) {
        const int64_t mine = seq_tiles<kTile>(a, s0 + lane), upto = scan64(mine, lane);
        const uint64_t past = __builtin_amdgcn_ballot_w64(before + upto > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            base = before + shfl64(upto - mine, l);
            return s0 + l;
        }
        before += shfl64(upto, 63);
    }
    base = before;
    return a.b.seqs;
}

template <int CT, int D>
struct Attend {
    using F = Form<CT>;
    static constexpr int kTile = F::kTile, kPer = F::kPer, kHalves = F::kHalves;
    static constexpr int kSteps = kPer / 4;          // row steps of the first product
    static constexpr int kChunks = D / (4 * kPer);   // 64-byte parts of a key
    static constexpr int kRows = D / 16;             // 16-column parts of the output
    floatx4_t o[kRows];
    float m, l;

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
        for (int t = t0; t < t1; ++t) {
            const int k0 = t * kTile, key0 = k0 + vkey;
            const int64_t head_page = (int64_t)held_page(vpage) * a.kvh + kh;
            const int next = min(t + 1, t1 - 1), after = min(t + 2, t1 - 1);
            const int kpage_after = entry(after * kTile + kgroup), vpage_after = entry(after * kTile + vkey);
            uint4 vf[kRows];
            {
                const int64_t at = head_page * page_elems + (int64_t)col * P + (key0 & (P - 1));
#pragma unroll
                for (int i = 0; i < kRows; ++i) vf[i] = load_piece<CT>(a.vc, at + 16 * i * P);
            }
            // (what the page of unseen keys holds, its scales too, may be anything)
            const bool held = (uint32_t)vpage < (uint32_t)a.pages && key0 < high && key0 + kPer > low;
            float ks = 1.0f, vs = 1.0f;
            if constexpr (CT == SE12_STEP_E4M3) {
                ks = a.k_scale[head_page];
                vs = held ? a.v_scale[head_page] : 0.0f;
            }
            float sc[kPer];
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
            load_k(next, kpage_next);
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
            bool apart = false;     // a value that is no number may be hidden from some of the columns
            if (!inside) {
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
            float top = sc[0];
#pragma unroll
            for (int e = 1; e < kPer; ++e) top = fmaxf(top, sc[e]);
            if (__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0) {
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float to = fmaxf(m, top);
                const float scale = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
                m = to;
                l *= scale;
#pragma unroll
                for (int i = 0; i < kRows; ++i) o[i] *= scale;
            }
            const float base = m == -INFINITY ? 0.0f : m;
            bf16x8_t pf[kHalves];
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
            if (apart) {
                // 0 x NaN is NaN, so what is no number leaves the product, and comes
                // back in the columns that give it a weight
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
#pragma unroll
            for (int i = 0; i < kRows; ++i)
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand<CT>(vf[i], h), pf[h], o[i], 0, 0, 0);
            vpage = vpage_next;
            vpage_next = vpage_after;
            kpage_next = kpage_after;
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
    const int64_t total = all_tiles<kTile>(a, lane);
    const int64_t per = (total + a.workers - 1) / a.workers;
    int64_t at = worker * per;
    const int64_t end = min(at + per, total);
    if (at >= end) return;
    int64_t base;
    int s = __builtin_amdgcn_readfirstlane(seq_of_tile<kTile>(a, at, lane, base));
    while (at < end && s < a.b.seqs) {
        const SeqWork w = seq_work<kTile>(a, s);
        const int64_t size = (int64_t)w.tiles * w.units * a.kvh;
        if (at >= base + size) {
            base += size;
            ++s;
            continue;
        }
        const int64_t in = at - base;
        const int tile = (int)(in % w.tiles), unit = (int)(in / w.tiles % w.units), kh = (int)(in / w.tiles / w.units);
        const int tiles = (int)min((int64_t)(w.tiles - tile), end - at);
        Attend<CT, D> x;
        x.run(a, s, w, kh, unit, tile, tiles);
        const int col = lane & 15, quarter = lane >> 4, c = unit * kColumns + col;
        if (c < w.seq.n * a.group) {
            if (tiles == w.tiles) {
                const float inv = x.l == 0.0f ? 0.0f : 1.0f / x.l;
                uint16_t* out = a.out + ((int64_t)(w.seq.start + c / a.group) * a.heads + kh * a.group + c % a.group) * D + 4 * quarter;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    store4(out + 16 * i, x.o[i][0] * inv, x.o[i][1] * inv, x.o[i][2] * inv, x.o[i][3] * inv);
            } else {
                const int64_t p = part_at(a, worker, tile > 0 ? 0 : 1) + col;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    *reinterpret_cast<floatx4_t*>(a.part + p * D + 16 * i + 4 * quarter) = x.o[i];
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

// The units that several workers share, from their parts in order: one block per
// (sequence, KV head, column unit) and column, D / 4 lanes a part.
template <int CT, int D>
__global__ __launch_bounds__(kAttendThreads) void paged_join_kernel(AttendArgs a, int max_units) {
    constexpr int kTile = Form<CT>::kTile;
    __shared__ float4 sums[kAttendThreads];
    __shared__ float ls[kAttendThreads];
    const int tid = threadIdx.x, lane = tid & 63;
    const int unit = (int)(blockIdx.x % max_units), kh = (int)(blockIdx.x / max_units % a.kvh), s = (int)(blockIdx.x / max_units / a.kvh);
    const int col = blockIdx.y, c = unit * kColumns + col;
    const SeqWork w = seq_work<kTile>(a, s);
    if (unit >= w.units || c >= w.seq.n * a.group) return;
    int64_t base = 0, total = 0;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 64) {
        const int64_t mine = seq_tiles<kTile>(a, s0 + lane), upto = scan64(mine, lane);
        if (s >= s0 && s < s0 + 64) base = total + shfl64(upto - mine, s - s0);
        total += shfl64(upto, 63);
    }
    const int64_t per = (total + a.workers - 1) / a.workers;
    const int64_t first = base + ((int64_t)kh * w.units + unit) * w.tiles, last = first + w.tiles - 1;
    const int w0 = (int)(first / per), w1 = (int)(last / per);
    if (w0 == w1) return;      // one worker had it all
    constexpr int kLanes = D / 4, kParts = kAttendThreads / kLanes;
    const float* ml = a.part + (int64_t)a.workers * 2 * a.columns * D;
    float m = -INFINITY;
    for (int k = w0; k <= w1; ++k) m = fmaxf(m, ml[2 * (part_at(a, k, k == w0 ? 1 : 0) + col)]);
    const float top = m == -INFINITY ? 0.0f : m;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
    for (int k = w0 + tid / kLanes; k <= w1; k += kParts) {
        const int64_t p = part_at(a, k, k == w0 ? 1 : 0) + col;
        const float by = __builtin_amdgcn_exp2f(ml[2 * p] - top);
        const float4 v = *reinterpret_cast<const float4*>(a.part + p * D + 4 * (tid % kLanes));
        l += by * ml[2 * p + 1];
        o.x += by * v.x;
        o.y += by * v.y;
        o.z += by * v.z;
        o.w += by * v.w;
    }
    sums[tid] = o;
    ls[tid] = l;
    __syncthreads();
    if (tid >= kLanes) return;
    for (int k = 1; k < kParts; ++k) {
        const float4 v = sums[k * kLanes + tid];
        o.x += v.x;
        o.y += v.y;
        o.z += v.z;
        o.w += v.w;
        l += ls[k * kLanes + tid];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    store4(a.out + ((int64_t)(w.seq.start + c / a.group) * a.heads + kh * a.group + c % a.group) * D + 4 * tid, o.x * inv, o.y * inv,
           o.z * inv, o.w * inv);
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

bool any_many(const Batch& b, int group) { return (int64_t)b.max_new * group > kFewColumns; }

int64_t part_bytes(const se12_step_pages* p, const Batch& b, int group) {
    return few_bytes(p, b, group) + (any_many(b, group) ? prompt_part_bytes(b, p->kv_heads, group, p->page_size, p->head_dim) : 0);
}

template <int CT, int D>
void launch_attend(const AttendArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((paged_attention_kernel<CT, D>), dim3(a.workers / (kAttendThreads / 64)), dim3(kAttendThreads), 0, st, a);
    const int max_units = (int)((std::min<int64_t>((int64_t)a.b.max_new * a.group, kFewColumns) + kColumns - 1) / kColumns);
    hipLaunchKernelGGL((paged_join_kernel<CT, D>), dim3((uint32_t)((int64_t)a.b.seqs * a.kvh * max_units), a.columns), dim3(kAttendThreads), 0,
                       st, a, max_units);
}

}  // namespace

extern "C" {

int64_t se12_step_paged_attention_workspace(const se12_step_pages* pages, const se12_step_batch* batch, int32_t heads) {
    if (const char* e = paged_error(pages, batch, heads)) return step_fail("se12_step_paged_attention_workspace", e);
    if (batch->tokens == 0) return 0;
    return part_bytes(pages, device_batch(batch), heads / pages->kv_heads);
}

int se12_step_paged_attention(const se12_step_pages* pages, const se12_step_batch* batch, const uint16_t* q,
                              int64_t q_stride, uint16_t* out, int32_t heads, float scaling, float softcap,
                              int32_t window, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "se12_step_paged_attention";
    if (const char* e = paged_error(pages, batch, heads)) return step_fail(fn, e);
    if (!q || !out) return step_fail(fn, "NULL argument");
    if (q_stride < (int64_t)heads * pages->head_dim || q_stride % 8) return step_fail(fn, "q rows must be a multiple of 8 elements apart and hold all heads");
    if (!(softcap >= 0.0f) || !(softcap < 1e30f) || window < 0) return step_fail(fn, "softcap and window must be 0 or more");
    if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(out) % 8) return step_fail(fn, "misaligned tensor");
    if (batch->tokens == 0) return SE12_STEP_OK;
    const Batch b = device_batch(batch);
    const int group = heads / pages->kv_heads;
    if (reinterpret_cast<uintptr_t>(workspace) % 256 || !workspace || workspace_bytes < part_bytes(pages, b, group))
        return step_fail(fn, "workspace missing, misaligned or too small");
    if ((int64_t)b.seqs * pages->kv_heads * (kFewColumns / kColumns) > INT32_MAX || !prompt_fits(b, pages->kv_heads, group, pages->page_size))
        return step_fail(fn, "too many sequences, tokens and heads for one launch");
    constexpr float kLog2E = 1.4426950408889634f;
    AttendArgs a{q, q_stride, out, pages->k, pages->v, pages->k_scale, pages->v_scale, b, heads, pages->kv_heads, group, pages->pages,
                 log2_of(pages->page_size), window, softcap > 0.0f ? 2.0f * scaling / softcap * kLog2E : scaling * kLog2E,
                 softcap * kLog2E, static_cast<float*>(workspace), worker_count(pages, b, group), column_count(b, group), kFewColumns,
                 prompt_splits(b, pages->kv_heads, group, pages->page_size)};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool e4m3 = pages->dtype == SE12_STEP_E4M3;
    switch (pages->head_dim) {
        case 64:
            e4m3 ? launch_attend<SE12_STEP_E4M3, 64>(a, st) : launch_attend<SE12_STEP_BF16, 64>(a, st);
            break;
        case 128:
            e4m3 ? launch_attend<SE12_STEP_E4M3, 128>(a, st) : launch_attend<SE12_STEP_BF16, 128>(a, st);
            break;
        default:
            e4m3 ? launch_attend<SE12_STEP_E4M3, 256>(a, st) : launch_attend<SE12_STEP_BF16, 256>(a, st);
    }
    if (any_many(b, group)) {
        a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + few_bytes(pages, b, group));
        launch_prompt(a, e4m3, pages->head_dim, st);
    }
    return step_launched();
}

}  // extern "C"
