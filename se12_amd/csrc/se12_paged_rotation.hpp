// Norm and position rotation of a token's heads, shared by the append to E2M1 pages
// (se12_paged_e2m1.hip) and the rotation by itself (se12_paged_rotate.hip).
// Mathematics: n = x rsqrt(mean(x^2) + eps) (offset + w), then the pair (a, b) of n by
// angle = position * inv_freq: (a cos - b sin, b cos + a sin) times `scale`; pairs (i, i +
// rotary / 2), or (2 i, 2 i + 1) where interleaved.
//
// A row (token and head) is 8 columns to a lane. Sums of squares and angles in 64 bits,
// each rounded to FP32 once (the mean's root, sine and cosine times scale); all else in
// single FP32 operations, no product kept longer than the next rounding. So keys are the
// same bits whatever append wrote them, and those of the formula in FP32: a digit of a
// quantised key does not depend on how the work was cut. (An append sums a position's angle
// from its run's first, the rotation by itself works each out: theirs may differ in FP32's
// last bit, and one BF16 value in 2^16 by a step.)
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "se12_paged_device.hpp"

namespace se12step {

struct Rotation {
    const float* inv_freq;
    const void* q_norm;
    const void* k_norm;
    double scale, eps;
    float offset;
    int half;              // rotary / 2
    bool f32_norm, interleaved;
};

// eight values as they are loaded (rows are 4 values' bytes apart at least, not 16)
template <int DT>
struct Eight {
    uint32_t w[DT == SE12_STEP_F32 ? 8 : 4];
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        if constexpr (DT == SE12_STEP_F32) {
            const uint4* v = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
            const uint4 a = v[0], b = v[1];
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        } else {
            const uint2* v = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
            const uint2 a = v[0], b = v[1];
            w[0] = a.x, w[1] = a.y, w[2] = b.x, w[3] = b.y;
        }
    }
    __device__ __forceinline__ void values(float x[8]) const {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            x[k] = __uint_as_float(DT == SE12_STEP_F32 ? w[k] : k & 1 ? w[k / 2] & 0xFFFF0000u : w[k / 2] << 16);
    }
};

template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float x[8]) {
    Eight<DT> v;
    v.load(p, i);
    v.values(x);
}

struct Angle {
    double c, s;      // its cosine and sine
};

__device__ __forceinline__ Angle angle_of(double angle) {
    // what is beyond a whole number of quarter turns, in two parts of pi / 2, by the series
    // of sine and cosine: 2^-52 of a whole turn, beside the angle's own rounding
    const double whole = angle * 0.63661977236758134 + 0x1.8p52, k = whole - 0x1.8p52;
    const int turn = __double2loint(whole);
    // (beyond 2^52 quarters a double is whole ones: none left over)
    const double over = fma(-k, 6.123233995736766e-17, fma(-k, 1.5707963267948966, angle));
    const double x = fabs(over) <= 2.0 ? over : angle - angle, x2 = x * x;
    double s = -1.0 / 1307674368000, c = 1.0 / 20922789888000;
    s = fma(s, x2, 1.0 / 6227020800);
    c = fma(c, x2, -1.0 / 87178291200);
    s = fma(s, x2, -1.0 / 39916800);
    c = fma(c, x2, 1.0 / 479001600);
    s = fma(s, x2, 1.0 / 362880);
    c = fma(c, x2, -1.0 / 3628800);
    s = fma(s, x2, -1.0 / 5040);
    c = fma(c, x2, 1.0 / 40320);
    s = fma(s, x2, 1.0 / 120);
    c = fma(c, x2, -1.0 / 720);
    s = fma(s, x2, -1.0 / 6);
    c = fma(c, x2, 1.0 / 24);
    s = fma(s * x2, x, x);
    c = fma(c, x2, -0.5);
    c = fma(c, x2, 1.0);
    const double sn = turn & 1 ? c : s, cs = turn & 1 ? s : c;
    return {(turn + 1) & 2 ? -cs : cs, turn & 2 ? -sn : sn};
}

__device__ __forceinline__ Angle operator+(Angle a, Angle b) { return {fma(a.c, b.c, -a.s * b.s), fma(a.s, b.c, a.c * b.s)}; }

__device__ __forceinline__ float2 turn_of(Angle a, double scale) { return make_float2((float)(a.c * scale), (float)(a.s * scale)); }

// cos and sin of pos * freq, times scale
__device__ __forceinline__ float2 turn_at(int pos, float freq, double scale) { return turn_of(angle_of((double)pos * (double)freq), scale); }

// The angles of kEach places of a run of 16 from place `at`, whose angle is x: halves of them
// in turn, so a place's is its run's first, and then the powers of two it is beyond it, the
// high ones first. `beyond`: 1, 2, 4, 8 places.
template <int kEach, typename Put>
__device__ __forceinline__ void places_of(Angle x, int at, const Angle* beyond, Put put) {
    if constexpr (kEach == 1) {
        put(at, x);
    } else {
        constexpr int kHalf = kEach / 2, kPower = kHalf == 1 ? 0 : kHalf == 2 ? 1 : kHalf == 4 ? 2 : 3;
        places_of<kHalf>(x, at, beyond, put);
        places_of<kHalf>(x + beyond[kPower], at + kHalf, beyond, put);
    }
}

// cos and sin of positions first + from .. first + to - 1 of a run of 16 (first a multiple of
// 16), cs[position][half] (16-byte aligned, 16 positions long), by a block's kThreads, all of which
// call it. Every place's angle comes by sums from the run's first and that of one place. (An
// angle of its own for every place was a quarter of the append's vector instructions. A place's is
// the same whatever else of its run is worked out.) kShared: these two are worked out once, by
// different waves, and go by LDS to the others (9,001 tokens of 16 / 8 heads of 256, 4 us less, but
// two barriers, which cost 57 tokens of 40 sequences 0.5 us).
template <int kThreads, bool kShared>
__device__ __forceinline__ void turn_run16(float2* cs, const Rotation& r, int first, int from, int to) {
    static_assert(kThreads >= 256, "");
    const int half = r.half, tid = (int)threadIdx.x;
    if (half == 0) return;
    int parts = 16;                                  // of the run, each a thread's
    while (parts > 1 && parts * half > kThreads) parts >>= 1;
    const int part = tid / half, f = tid - part * half, each = 16 / parts, at = part * each;
    const bool none = part >= parts || at >= to || at + each <= from;
    Angle beyond[4], x;
    if constexpr (kShared) {
        Angle* two = reinterpret_cast<Angle*>(cs);
        if (tid < 2 * half) {
            const double freq = (double)r.inv_freq[tid < half ? tid : tid - half];
            two[tid] = angle_of(tid < half ? freq : (double)first * freq);
        }
        __syncthreads();
        beyond[0] = two[f];
        x = two[half + f];
        __syncthreads();
        if (none) return;
    } else {
        if (none) return;
        const double freq = (double)r.inv_freq[f];
        beyond[0] = angle_of(freq);
        x = angle_of((double)first * freq);
    }
#pragma unroll
    for (int i = 1; i < 4; ++i) beyond[i] = beyond[i - 1] + beyond[i - 1];
    if (at & 8) x = x + beyond[3];
    if (at & 4) x = x + beyond[2];
    if (at & 2) x = x + beyond[1];
    if (at & 1) x = x + beyond[0];
    auto put = [&](int i, Angle y) {
        if (i >= from && i < to) cs[(i - from) * half + f] = turn_of(y, r.scale);
    };
    switch (each) {
        case 1: places_of<1>(x, at, beyond, put); break;
        case 2: places_of<2>(x, at, beyond, put); break;
        case 4: places_of<4>(x, at, beyond, put); break;
        default: places_of<8>(x, at, beyond, put);      // (half is 128 at most, threads 256)
    }
}

// the sum over 16 lanes side by side, in each of them
__device__ __forceinline__ double row16_sum(double v) {
    auto add = [&](auto control) {
        const int lo = __builtin_amdgcn_mov_dpp(__double2loint(v), control.value, 0xF, 0xF, true);
        const int hi = __builtin_amdgcn_mov_dpp(__double2hiint(v), control.value, 0xF, 0xF, true);
        v += __hiloint2double(hi, lo);
    };
    add(std::integral_constant<int, 0xB1>{});       // (as row16_reduce of se12_step_math.hpp)
    add(std::integral_constant<int, 0x4E>{});
    add(std::integral_constant<int, 0x141>{});
    add(std::integral_constant<int, 0x140>{});
    return v;
}

// offset + w of d weights, in FP32
template <int kThreads>
__device__ __forceinline__ void load_weights(float* to, const Rotation& r, const void* w, int d) {
    for (int i = threadIdx.x; i < d; i += kThreads)
        to[i] = r.offset + (r.f32_norm ? static_cast<const float*>(w)[i] : bf16_to_f(static_cast<const uint16_t*>(w)[i]));
}

// x[8] of a row whose kLanes lanes lie side by side, normed; w: the 8 weights of its columns, share: 1 / head_dim
template <int kLanes>
__device__ __forceinline__ void norm_row(float x[8], double eps, const float* w, double share) {
#pragma clang fp contract(off)
    static_assert(kLanes == 8 || kLanes == 16 || kLanes == 32, "");
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fma((double)x[i], (double)x[i], sum);
    if constexpr (kLanes == 8) {
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor(sum, o, 64);
    } else {
        sum = row16_sum(sum);
        if constexpr (kLanes == 32) sum += __shfl_xor(sum, 16, 64);
    }
    // the inverse root to 2^-45: the card's, and one step of Newton's
    const double mean = sum * share + eps, root = __builtin_amdgcn_rsq(mean);
    const float inv = (float)(root > 0.0 && root < INFINITY ? fma(0.5 * root, fma(-mean * root, root, 1.0), root) : root);
    const float4 w0 = *reinterpret_cast<const float4*>(w), w1 = *reinterpret_cast<const float4*>(w + 4);
    const float f[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (x[i] * inv) * f[i];
}

// x[8], columns c0 .. of a row whose lanes lie side by side, turned by the angles cs[half] of
// its token
__device__ __forceinline__ void turn_row(float x[8], const float2* cs, int c0, int half, bool interleaved) {
#pragma clang fp contract(off)
    if (c0 >= 2 * half) return;
    if (interleaved) {
        const float4* t = reinterpret_cast<const float4*>(cs + c0 / 2);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const float4 u = t[p];
            const float a = x[4 * p], b = x[4 * p + 1], c = x[4 * p + 2], d = x[4 * p + 3];
            x[4 * p] = a * u.x - b * u.y;
            x[4 * p + 1] = b * u.x + a * u.y;
            x[4 * p + 2] = c * u.z - d * u.w;
            x[4 * p + 3] = d * u.z + c * u.w;
        }
        return;
    }
    // The columns half a rotation on, or back, are another lane's: its same four, or where half
    // is no multiple of 8 its other four.
    float o[8];
    auto bring = [&](auto swapped) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int at = c0 + 4 * j, from = 4 * ((int)(threadIdx.x & 63) + (at < half ? at + half : at - half) / 8 - c0 / 8);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                o[4 * j + k] = __int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(x[(swapped.value ? 4 - 4 * j : 4 * j) + k])));
        }
    };
    if (half % 8 == 0)
        bring(std::false_type{});
    else
        bring(std::true_type{});
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int at = c0 + 4 * j;
        const bool first = at < half;
        const uint32_t sign = first ? 0x80000000u : 0u;      // (a - b is a + -b)
        const float4* t = reinterpret_cast<const float4*>(cs + (first ? at : at - half));
        const float4 t0 = t[0], t1 = t[1];
        const float cos[4] = {t0.x, t0.z, t1.x, t1.z}, sin[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float b = o[4 * j + k] * __uint_as_float(__float_as_uint(sin[k]) ^ sign);
            x[4 * j + k] = x[4 * j + k] * cos[k] + b;
        }
    }
}

__device__ __forceinline__ uint4 bf16x8(const float x[8]) {
    return make_uint4(f_to_bf16x2(x[0], x[1]), f_to_bf16x2(x[2], x[3]), f_to_bf16x2(x[4], x[5]), f_to_bf16x2(x[6], x[7]));
}

// The calls' blocks: each has 16 positions side by side of one sequence. A sequence of
// n new tokens touches at most n / 16 + 2 such runs, so sequence s may have blocks
// starts[s] / 16 + 2 s onwards; at one token each, block s.
struct Run16 {
    Seq seq;
    int s, first;        // sequence, first position of the run (a multiple of 16)
    int from, to;        // its new tokens: first + from .. first + to - 1
};

__device__ __forceinline__ Run16 run16_of(const Batch& b, int slot) {
    int s = slot, j = 0;
    if (b.max_new > 1) {
        auto block0 = [&](int i) { return (min(max(b.starts[i], 0), b.tokens) >> 4) + 2 * i; };
        int lo = 0, hi = b.seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (block0(mid) <= slot)
                lo = mid;
            else
                hi = mid;
        }
        s = lo;
        j = slot - block0(s);
    }
    Run16 r;
    r.s = s;
    r.seq = load_seq(b, s);
    const int64_t first = ((int64_t)(r.seq.len >> 4) + j) << 4, left = (int64_t)r.seq.len + r.seq.n - first;
    r.first = (int)first;
    r.from = j == 0 ? r.seq.len - r.first : 0;
    r.to = j < 0 ? 0 : (int)max(min(left, (int64_t)16), (int64_t)0);
    return r;
}

// host
inline int64_t run16_blocks(const Batch& b) {
    return b.max_new == 1 ? b.seqs : (int64_t)(b.tokens >> 4) + 2 * (int64_t)b.seqs;
}

inline const char* rotation_error(const se12_step_rotation* r, int head_dim) {
    if (!r) return "NULL argument";
    if (r->rotary < 0 || r->rotary > head_dim || r->rotary % 8) return "rotary must be a multiple of 8 up to head_dim";
    if (r->rotary > 0 && !r->inv_freq) return "NULL argument";
    if (r->norm_dtype != SE12_STEP_BF16 && r->norm_dtype != SE12_STEP_F32) return "norm weights must be BF16 or FP32";
    if (!(fabs(r->scale) < 0x1p127) || !(r->eps >= 0.0) || !(r->eps - r->eps == 0.0) || !(r->offset - r->offset == 0.0f))
        return "scale, eps and offset must be finite (scale below 2^127), eps not below 0";
    if (reinterpret_cast<uintptr_t>(r->inv_freq) % 16 || reinterpret_cast<uintptr_t>(r->q_norm) % 16 ||
        reinterpret_cast<uintptr_t>(r->k_norm) % 16)
        return "misaligned tensor";
    return nullptr;
}

inline Rotation device_rotation(const se12_step_rotation* r) {
    return {r->inv_freq, r->q_norm, r->k_norm, r->scale, r->eps, r->offset, r->rotary / 2, r->norm_dtype == SE12_STEP_F32, r->interleaved != 0};
}

}  // namespace se12step
