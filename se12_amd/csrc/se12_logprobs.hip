// Log probabilities of given tokens, entropy and the most likely alternatives of
// rows of logits. Mathematics: z = cap tanh(x / cap) or x; with the maximum m met so
// far, S = sum e^(z - m) and W = sum e^(z - m) (m - z), both of terms of one sign,
// log p_i = z_i - m - log S and the entropy is log S + W / S. (S is 1 at least: no log p
// is above 0, and a likely token's has the roundings of a small number. A reference of up
// to 8 below the maximum, which moves less often, left 1e-6 in all of them and saved nothing.)
//
// One pass over the logits. A wave takes kChunk of them at a time, 16 to a lane,
// the next chunk's loads in flight. Alternatives: a key per logit, its bits in an
// order that compares as the logits do, then the index from the highest, so no two
// are equal and equal logits go by the lower index. A wave keeps candidates in LDS,
// keys above the top-th best so far; when 128 are full each counts the keys above
// it, which is its place, and the best stay. The first chunk's bar is the top-th
// best of the lanes' own best: what passes it lies in `top` lanes. After that a
// chunk costs a comparison of its largest logit with the bar, and about
// top ln(length / chunk) logits of a row pass.
// The waves of a block and the blocks of a row merge the same way, the latter in a
// second launch, where rows are too few to fill the card with a block each.
//
// Bound by its bytes where rows are many and in FP32: 1,024 of 256,000, top 5, 1,049 MB in
// 186 us, under a cap 192 (5.5 TB/s); in BF16 by its bytes without a cap, 117 us (4.5 TB/s),
// and with one by the arithmetic, 145 (an instruction of a quarter of the rate and eleven
// others to a logit). One FP32 row, top 20: 6.6 + 4.6 us, two launches' latency and the
// rankings; 40 rows of 100,277 in BF16, top 5: 8.0 + 4.6.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "se12_step.h"
#include "se12_step_math.hpp"

namespace se12step {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / 64;
constexpr int kLpPer = 16;                     // logits of a lane and chunk
constexpr int kChunk = 64 * kLpPer;
constexpr int kMaxTop = 32;
constexpr int kKeys = 128;                     // of a wave's buffer: 32 best and a ballot's 64 fit
constexpr int kBlocksWanted = 1024;            // four to a CU
constexpr int kJoinKeys = 8;                   // that a thread of the second launch loads at once
constexpr float kLog2E = 1.4426950408889634f;

// of a part of a row: the maximum (of capped logits in units of log 2), S, and W in units of log 2
struct Stats {
    float m, s, w;
};

struct LogprobArgs {
    const void* logits;
    int64_t stride;
    int vocab, top, slices, slice;             // slice: logits of a block, a multiple of kLpWaves * kChunk
    float cap, half, inv_cap2;                 // base 2: the cap; |x| of the polynomial; 2 log2(e) / cap
    float unit, unit2;                         // of z: to units of 1, and of log 2
    float k[5];                                // the polynomial's coefficients
    const int64_t* tokens;
    float* logprobs;
    float* entropy;
    float* top_logprobs;
    int64_t* top_ids;
    Stats* stats;                              // [rows][slices]
    uint64_t* keys;                            // [rows][slices][top]
};

// bits that compare as the numbers do (0 for nothing, 1 for a NaN)
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);   // -0 ties with 0
    return x != x ? 1u : (u >> 31 ? ~u : u | 0x80000000u);
}

__device__ __forceinline__ float number_of(uint32_t order) {
    return order <= 1u ? __builtin_nanf("") : __uint_as_float(order >> 31 ? order & 0x7FFFFFFFu : ~order);
}

__device__ __forceinline__ uint64_t key_of(float x, int i) { return ((uint64_t)order_of(x) << 32) | (uint32_t)~i; }

__device__ __forceinline__ uint64_t read_lane64(uint64_t v, int l) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)v, l);
}

// LDS is written and read by lanes of one wave, in order
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// A wave's best keys. buf: kKeys of LDS; the first n are candidates.
struct Best {
    uint64_t* buf;
    uint64_t bar;      // keys above it count
    int n, top;

    __device__ __forceinline__ void reset(uint64_t* b, int k) {
        buf = b;
        bar = 0;
        n = 0;
        top = k;
    }

    // The best `top` to the front, in order: a key's place is the number of keys above it,
    // read from LDS, up to eight at a time, by all lanes alike. (A key a time, from registers by
    // readlane, the keys of a block's four waves took 14,000 cycles.)
    template <int kAtOnce>
    __device__ __forceinline__ void settle() {
        const int lane = threadIdx.x & 63;
        if (lane < 8) buf[n + lane] = 0;
        wave_fence();
        const uint64_t a = lane < n ? buf[lane] : 0, b = lane + 64 < n ? buf[lane + 64] : 0;
        int above_a = 0, above_b = 0;
        for (int i = 0; i < n; i += kAtOnce) {
            uint64_t k[kAtOnce];
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) k[e] = buf[i + e];
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) above_a += k[e] > a;
            if (n > 64) {
#pragma unroll
                for (int e = 0; e < kAtOnce; ++e) above_b += k[e] > b;
            }
        }
        wave_fence();
        if (lane < n && above_a < top) buf[above_a] = a;
        if (lane + 64 < n && above_b < top) buf[above_b] = b;
        wave_fence();
        n = min(n, top);
        if (n == top) bar = read_lane64(buf[top - 1], 0);
    }

    __device__ __forceinline__ void offer(uint64_t key) {
        uint64_t in = __builtin_amdgcn_ballot_w64(key > bar);
        if (!in) return;
        if (n + __builtin_popcountll(in) > kKeys) {
            settle<2>();
            in = __builtin_amdgcn_ballot_w64(key > bar);
        }
        if (key > bar) buf[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0))] = key;
        n += __builtin_popcountll(in);
    }

    // Logits up to it are below the bar. (Zero is above a bar just below it; as numbers,
    // -0 and 0 are equal.)
    __device__ __forceinline__ float bar_number() const {
        const uint32_t order = (uint32_t)(bar >> 32);
        return order == 0x7FFFFFFFu ? -1.17549435e-38f : number_of(order);
    }

    // A bar that at least `top` of the lanes' best reach, in the upper 16 bits of the
    // logits' order: the largest that so many do, less one in the last place.
    __device__ __forceinline__ void bar_of_lanes(uint32_t order) {
        const uint32_t mine = order >> 16;
        uint32_t at = 0;
#pragma unroll
        for (int bit = 15; bit >= 0; --bit) {
            const uint32_t next = at | (1u << bit);
            at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine >= next)) >= top ? next : at;
        }
        bar = at ? ((uint64_t)at << 48) - 1 : 0;
    }
};

// Capped logits in units of log 2, z = log2(e) cap tanh(u), u = x / cap, off by 3 units of
// 2^-24 of themselves: up to cap / 2 as x p(x^2), p fitted (kTanh), beyond from e^(2 |u|).
// The same x has the same z wherever it is taken (the product is rounded, not made part of
// a difference), so a maximum's own term is 1.
__device__ __forceinline__ float z_near(const LogprobArgs& a, float x) {
#pragma clang fp contract(off)
    const float q = x * x;
    return x * fmaf(q, fmaf(q, fmaf(q, fmaf(q, a.k[4], a.k[3]), a.k[2]), a.k[1]), a.k[0]);
}

__device__ __forceinline__ float z_of(const LogprobArgs& a, float x) {
    if (a.cap == 0.0f) return x;
    const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(fabsf(x) * a.inv_cap2));
    return fabsf(x) < a.half ? z_near(a, x) : copysignf(fmaf(-2.0f * a.cap, r, a.cap), x);
}

// sums on a maximum moved up to `to`
__device__ __forceinline__ Stats moved(const LogprobArgs& a, Stats v, float to) {
    // (of m = -inf there is no sum; a NaN stays one)
    const float d = v.m == -INFINITY ? 0.0f : (to - v.m) * a.unit2, f = __builtin_amdgcn_exp2f(-d);
    return {to, v.s * f, (v.w + v.s * fminf(d, 1e30f)) * f};
}

// the sums of a wave's lanes, on the largest of their references
__device__ __forceinline__ Stats wave_join(const LogprobArgs& a, Stats v) {
    v = moved(a, v, wave_max(v.m));
    return {v.m, wave_sum(v.s), wave_sum(v.w)};
}

// the logit of the row's given token (false where there is none): two loads, one
// after the other, sent before the row's
template <int DT>
__device__ __forceinline__ bool token_logit(const LogprobArgs& a, int row, float& x) {
    const int64_t t = a.tokens[row];
    const bool valid = t >= 0 && t < a.vocab;
    const int64_t at = (int64_t)row * a.stride + (valid ? t : 0);
    x = DT == SE12_STEP_F32 ? static_cast<const float*>(a.logits)[at] : bf16_to_f(static_cast<const uint16_t*>(a.logits)[at]);
    return valid;
}

// the row's results, by one wave, from its sums and its best keys in order
__device__ __forceinline__ void finish_row(const LogprobArgs& a, int row, Stats v, const Best& best, bool valid, float x) {
    const int lane = threadIdx.x & 63;
    const float log_s = logf(v.s);
    auto logprob = [&](float x) { return v.m == -INFINITY && v.s == 0.0f ? -INFINITY : (z_of(a, x) - v.m) * a.unit - log_s; };
    if (lane == 0) {
        // (a token that there is not: -inf, in a row of numbers)
        const float lp = valid ? logprob(x) : v.s != v.s ? v.s : -INFINITY;
        a.logprobs[row] = lp;
        a.entropy[row] = v.m == -INFINITY && v.s == 0.0f ? 0.0f : log_s + v.w * (1.0f / kLog2E) / v.s;
    }
    if (lane < a.top) {
        const uint64_t k = best.buf[lane];
        a.top_ids[(int64_t)row * a.top + lane] = (int64_t)(uint32_t)~(uint32_t)k;
        a.top_logprobs[(int64_t)row * a.top + lane] = logprob(number_of((uint32_t)(k >> 32)));
    }
}

// What the waves of a block hand to the first of them.
struct Waves {
    uint64_t keys[kLpWaves][kKeys + 8];
    uint64_t bar[kLpWaves];
    int n[kLpWaves];
    Stats sums[kLpWaves];
};

// the block's waves to wave 0; true there, with the best keys in order
__device__ __forceinline__ bool join_waves(const LogprobArgs& a, Stats& v, Best& best, Waves& of) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, top = best.top;
    v = wave_join(a, v);
    if (best.n > 64) best.settle<2>();
    if (lane == 0) {
        of.sums[wave] = v;
        of.n[wave] = best.n;
        of.bar[wave] = best.bar;
    }
    __syncthreads();
    if (wave > 0) return false;
    v = lane < kLpWaves ? of.sums[lane] : Stats{-INFINITY, 0.0f, 0.0f};
    v = wave_join(a, v);
    if (top > 0) {
        // as in a chunk: a bar from the lanes' best, and what passes all bars
        uint64_t key[kLpWaves], most = 0, least = 0;
#pragma unroll
        for (int k = 0; k < kLpWaves; ++k) {
            key[k] = lane < of.n[k] ? of.keys[k][lane] : 0;
            most = max(most, key[k]);
            least = max(least, of.bar[k]);
        }
        wave_fence();
        best.n = 0;
        best.bar_of_lanes((uint32_t)(most >> 32));
        best.bar = max(best.bar, (least ? read_lane64(least, 0) : 1) - 1);
#pragma unroll
        for (int k = 0; k < kLpWaves; ++k) best.offer(key[k]);
        best.settle<8>();
    }
    return true;
}

template <int DT>
__global__ __launch_bounds__(kLpThreads, 6) void logprobs_kernel(LogprobArgs a) {
    constexpr int kVec = DT == SE12_STEP_F32 ? 4 : 8, kVecs = kLpPer / kVec, kSize = 16 / kVec;
    __shared__ Waves waves;
    __shared__ float held[kLpWaves][kChunk];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const char* base = static_cast<const char*>(a.logits) + (int64_t)row * a.stride * kSize;
    // whole 16-byte pieces of the row: logit i is value i + skew of them
    const int skew = (int)((reinterpret_cast<uintptr_t>(base) & 15) / kSize);
    const char* pieces = base - skew * kSize;
    const int first = skew, last = skew + a.vocab;      // values of the pieces that are the row's
    const int per_wave = a.slice / kLpWaves;
    const int begin = slice * a.slice + wave * per_wave, end = min(begin + per_wave, last);
    float token_x = 0.0f;
    bool valid = false;
    if (a.slices == 1) valid = token_logit<DT>(a, row, token_x);
    Best best;
    best.reset(waves.keys[wave], a.top);
    float bar = -INFINITY;                              // no logit up to it counts
    Stats v{-INFINITY, 0.0f, 0.0f};
    uint4 next[kVecs];
    auto load = [&](int at) {
        if (at >= first && at + kChunk <= last) {
            const uint4* p = reinterpret_cast<const uint4*>(pieces + (int64_t)at * kSize) + lane;
#pragma unroll
            for (int j = 0; j < kVecs; ++j) next[j] = p[j * 64];
            return;
        }
        // a piece that is not wholly the row's is read value by value
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            const int i = at + (j * 64 + lane) * kVec;
            if (i >= first && i + kVec <= last) {
                next[j] = *reinterpret_cast<const uint4*>(pieces + (int64_t)i * kSize);
            } else {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    if (i + e < first || i + e >= last) continue;
                    if constexpr (DT == SE12_STEP_F32)
                        w[e] = reinterpret_cast<const uint32_t*>(pieces)[i + e];
                    else
                        w[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(pieces)[i + e] << (16 * (e & 1));
                }
                next[j] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    };
    if (begin < end) load(begin);
    for (int at = begin; at < end; at += kChunk) {
        float x[kLpPer];
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            const uint32_t w[4] = {next[j].x, next[j].y, next[j].z, next[j].w};
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                if constexpr (DT == SE12_STEP_F32)
                    x[j * kVec + e] = __uint_as_float(w[e]);
                else
                    x[j * kVec + e] = __uint_as_float(e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
            }
        }
        const bool edge = at < first || at + kChunk > last;
        if (at + kChunk < end) load(at + kChunk);
        auto index = [&](int k) { return at + (k / kVec * 64 + lane) * kVec + k % kVec; };
        auto outside = [&](int k) { return index(k) < first || index(k) >= last; };
        if (edge) {
#pragma unroll
            for (int k = 0; k < kLpPer; ++k) x[k] = outside(k) ? -INFINITY : x[k];
        }
        float most = x[0];
#pragma unroll
        for (int k = 1; k < kLpPer; ++k) most = fmaxf(most, x[k]);
        if (a.top > 0) {
            // (-inf may stand for no logit of the row beside one that is a NaN)
            if (at == begin) {
                best.bar_of_lanes(most > -INFINITY ? order_of(most) : 0);
                bar = best.bar_number();
            }
            // (a bar or a logit that is a NaN goes the long way as well)
            if (at == begin || __builtin_amdgcn_ballot_w64(!(most <= bar)) != 0) {
                // what passes, a lane's logits one after the other, by way of LDS
                float* mine = held[wave] + lane;
                uint32_t hits = 0;
#pragma unroll
                for (int k = 0; k < kLpPer; ++k) {
                    mine[64 * k] = x[k];
                    hits |= (x[k] <= bar ? 0u : 1u) << k;
                }
                while (__builtin_amdgcn_ballot_w64(hits != 0)) {
                    const int k = hits ? __builtin_ctz(hits) : 0;
                    best.offer(hits && !outside(k) ? key_of(mine[64 * k], index(k) - skew) : 0);
                    hits &= hits - 1;
                }
                bar = best.bar_number();
            }
        }
        most = z_of(a, most);
        if (__builtin_amdgcn_ballot_w64(most > v.m) != 0) v = moved(a, v, fmaxf(v.m, wave_max(most)));
        if (v.m == -INFINITY) {
            // nothing but -inf so far, unless there is a NaN
#pragma unroll
            for (int k = 0; k < kLpPer; ++k) v.s = x[k] != x[k] ? x[k] : v.s;
        } else if (a.cap > 0.0f) {
            // (a logit within cap / 2 takes an instruction of a quarter of the rate and eleven
            // others, one beyond three and sixteen: 1,024 BF16 rows of 256,000 145 us; 152 with
            // the second form, in cap - 2 cap r, off by 2^-22 of the cap, for all)
            float far = 0.0f;
#pragma unroll
            for (int k = 0; k < kLpPer; ++k) far = fmaxf(far, fabsf(x[k]));
            auto add = [&](auto near, auto at_edge) {
#pragma unroll
                for (int k = 0; k < kLpPer; ++k) {
                    float d = v.m - (near.value ? z_near(a, x[k]) : z_of(a, x[k]));
                    if (at_edge.value && outside(k)) d = 1e30f;
                    const float e = __builtin_amdgcn_exp2f(-d);
                    v.s += e;
                    v.w = fmaf(e, d, v.w);
                }
            };
            // (a NaN that the maximum leaves out stays one either way)
            if (edge)
                add(std::false_type{}, std::true_type{});
            else if (__builtin_amdgcn_ballot_w64(far >= a.half) != 0)
                add(std::false_type{}, std::false_type{});
            else
                add(std::true_type{}, std::false_type{});
        } else {
#pragma unroll
            for (int k = 0; k < kLpPer; ++k) {
                const float d = (v.m - x[k]) * kLog2E, e = __builtin_amdgcn_exp2f(-d);
                v.s += e;
                v.w = fmaf(e, fminf(d, 1e30f), v.w);
            }
        }
    }
    if (!join_waves(a, v, best, waves)) return;
    if (a.slices == 1) {
        finish_row(a, row, v, best, valid, token_x);
        return;
    }
    if (lane == 0) a.stats[blockIdx.x] = v;
    if (lane < a.top) a.keys[(int64_t)blockIdx.x * a.top + lane] = lane < best.n ? best.buf[lane] : 0;
}

// the slices of a row
template <int DT>
__global__ __launch_bounds__(kLpThreads) void logprobs_join_kernel(LogprobArgs a) {
    __shared__ Waves waves;
    __shared__ uint64_t held[kLpWaves][kJoinKeys * 64];
    const int row = blockIdx.x;
    float token_x;
    const bool valid = token_logit<DT>(a, row, token_x);
    Best best;
    best.reset(waves.keys[threadIdx.x >> 6], a.top);
    Stats v{-INFINITY, 0.0f, 0.0f};
    const int count = a.slices * a.top;
    const uint64_t* keys = a.keys + (int64_t)row * count;
    uint64_t key[kJoinKeys];
#pragma unroll
    for (int k = 0; k < kJoinKeys; ++k) {
        const int i = k * kLpThreads + threadIdx.x;
        key[k] = i < count ? keys[i] : 0;
    }
    // (a block's slices, 1,024 at most, on a reference of their own)
    for (int i = threadIdx.x; i < a.slices; i += kLpThreads) {
        const Stats x = a.stats[(int64_t)row * a.slices + i];
        const float to = fmaxf(v.m, x.m);
        const Stats p = moved(a, v, to), n = moved(a, x, to);
        v = {to, p.s + n.s, p.w + n.w};
    }
    if (a.top > 0) {
        uint32_t mine = 0, hits = 0;
#pragma unroll
        for (int k = 0; k < kJoinKeys; ++k) mine = max(mine, (uint32_t)(key[k] >> 32));
        best.bar_of_lanes(mine);
        uint64_t* mine64 = held[threadIdx.x >> 6] + (threadIdx.x & 63);
#pragma unroll
        for (int k = 0; k < kJoinKeys; ++k) {
            mine64[64 * k] = key[k];
            hits |= (key[k] > best.bar ? 1u : 0u) << k;
        }
        while (__builtin_amdgcn_ballot_w64(hits != 0)) {
            best.offer(hits ? mine64[64 * __builtin_ctz(hits)] : 0);
            hits &= hits - 1;
        }
        for (int k = kJoinKeys * kLpThreads; k < count; k += kLpThreads) {
            const int i = k + threadIdx.x;
            best.offer(i < count ? keys[i] : 0);
        }
    }
    if (join_waves(a, v, best, waves)) finish_row(a, row, v, best, valid, token_x);
}

}  // namespace se12step

using namespace se12step;

namespace {

// (tanh(u) / u - 1) / u^2 in powers of u^2, |u| <= 1/2: least squares with weights moved to
// where tanh(u) is furthest off (2^-26 of it)
constexpr double kTanh[4] = {-0.33333149552345276, 0.1332598775625229, -0.05305296927690506, 0.01725703850388527};

struct LpLayout {
    int slices, slice;
    int64_t stats_bytes, total;
};

// Slices of a row: as many blocks as fill the card, none smaller than a chunk a
// wave. (+ 7: a row that begins inside a 16-byte piece)
LpLayout logprobs_layout(int32_t rows, int32_t vocab, int32_t top) {
    constexpr int64_t unit = (int64_t)kLpWaves * kChunk;
    const int64_t units = ((int64_t)vocab + 7 + unit - 1) / unit;
    const int64_t want = std::min<int64_t>(units, std::max(1, kBlocksWanted / rows));
    const int64_t slice = (units + want - 1) / want * unit;
    LpLayout l;
    l.slice = (int)slice;
    l.slices = (int)(((int64_t)vocab + 7 + slice - 1) / slice);
    l.stats_bytes = ((int64_t)rows * l.slices * (int64_t)sizeof(Stats) + 15) / 16 * 16;
    l.total = l.slices == 1 ? 0 : l.stats_bytes + (int64_t)rows * l.slices * top * (int64_t)sizeof(uint64_t);
    return l;
}

const char* logprobs_shape_error(int32_t rows, int32_t vocab, int32_t top) {
    if (rows < 0 || vocab < 1 || vocab > (1 << 30)) return "bad shape";
    if (top < 0 || top > kMaxTop || top > vocab) return "top must be 0 to 32 and at most vocab";
    return nullptr;
}

}  // namespace

extern "C" {

int64_t se12_step_logprobs_workspace(int32_t rows, int32_t vocab, int32_t top) {
    if (const char* e = logprobs_shape_error(rows, vocab, top)) return step_fail("se12_step_logprobs_workspace", e);
    return rows == 0 ? 0 : logprobs_layout(rows, vocab, top).total;
}

int se12_step_logprobs(const void* logits, int32_t dtype, int64_t stride, int32_t rows, int32_t vocab, float softcap,
                       const int64_t* tokens, int32_t top, float* logprobs, float* entropy, float* top_logprobs,
                       int64_t* top_ids, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "se12_step_logprobs";
    if (const char* e = logprobs_shape_error(rows, vocab, top)) return step_fail(fn, e);
    if (rows == 0) return SE12_STEP_OK;
    if (!logits || !tokens || !logprobs || !entropy || (top > 0 && (!top_logprobs || !top_ids))) return step_fail(fn, "NULL argument");
    if (dtype != SE12_STEP_BF16 && dtype != SE12_STEP_F32) return step_fail(fn, "logits must be BF16 or FP32");
    if (stride < vocab) return step_fail(fn, "rows overlap");
    if (!(softcap == 0.0f || (softcap >= 0x1p-60f && softcap <= 1024.0f))) return step_fail(fn, "softcap must be 0, or 2^-60 to 1024");
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == SE12_STEP_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(tokens) % 8 ||
        reinterpret_cast<uintptr_t>(logprobs) % 4 || reinterpret_cast<uintptr_t>(entropy) % 4 ||
        reinterpret_cast<uintptr_t>(top_logprobs) % 4 || reinterpret_cast<uintptr_t>(top_ids) % 8)
        return step_fail(fn, "misaligned tensor");
    const LpLayout l = logprobs_layout(rows, vocab, top);
    if (!grid_fits((int64_t)rows * l.slices, kLpThreads)) return step_fail(fn, "too many rows");
    if (l.total > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < l.total))
        return step_fail(fn, "workspace missing, misaligned or too small");
    LogprobArgs a{};
    a.logits = logits;
    a.stride = stride;
    a.vocab = vocab;
    a.top = top;
    a.slices = l.slices;
    a.slice = l.slice;
    a.cap = softcap * kLog2E;
    a.unit = softcap > 0.0f ? 1.0f / kLog2E : 1.0f;
    a.unit2 = softcap > 0.0f ? 1.0f : kLog2E;
    if (softcap > 0.0f) {
        a.inv_cap2 = 2.0f * kLog2E / softcap;
        // (of smaller caps FP32 does not hold the coefficients, and no z is above 2^-14)
        a.half = softcap >= 0x1p-14f ? 0.5f * softcap : 0.0f;
        double k = 1.4426950408889634;
        a.k[0] = (float)k;
        for (int i = 0; i < 4 && a.half > 0.0f; ++i) {
            k /= (double)softcap * softcap;
            a.k[i + 1] = (float)(k * kTanh[i]);
        }
    }
    a.tokens = tokens;
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.top_logprobs = top_logprobs;
    a.top_ids = top_ids;
    a.stats = static_cast<Stats*>(workspace);
    a.keys = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + (l.slices > 1 ? l.stats_bytes : 0));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((uint32_t)((int64_t)rows * l.slices));
    if (dtype == SE12_STEP_F32) {
        hipLaunchKernelGGL(logprobs_kernel<SE12_STEP_F32>, grid, dim3(kLpThreads), 0, st, a);
        if (l.slices > 1) hipLaunchKernelGGL(logprobs_join_kernel<SE12_STEP_F32>, dim3(rows), dim3(kLpThreads), 0, st, a);
    } else {
        hipLaunchKernelGGL(logprobs_kernel<SE12_STEP_BF16>, grid, dim3(kLpThreads), 0, st, a);
        if (l.slices > 1) hipLaunchKernelGGL(logprobs_join_kernel<SE12_STEP_BF16>, dim3(rows), dim3(kLpThreads), 0, st, a);
    }
    return step_launched();
}

}  // extern "C"
