// Appending to a paged cache of E2M1 (4 bits, a scale to 32 columns of a token and
// head), and reading a cache of any type back. Mathematics: rows of q and k normed and
// rotated (se12_paged_rotation.hpp); of 32 columns s = the 8-bit scale nearest to
// max |x| / 6, at most 10240, and each value the E2M1 nearest to x / s, ties to even,
// 6 at most. A code has 2 significant bits and a scale 4, so what is held is a number of
// FP16 and of BF16 alike. A scale is that of its token alone: no later token changes it,
// and nothing is rounded twice.
//
// A block has 16 positions of a sequence and one KV head: its keys, its values and the
// query heads that read it, so a value column's 8 bytes (16 tokens) have one writer and
// the angles serve all its rows. Values meet in LDS, where a column's tokens lie apart.
//
// Append: 9,001 tokens of 7 prompts, 16 / 8 heads normed and rotated, BF16 in. Heads of 256: 241 MB in 55
// to 60 us (4.0 to 4.4 TB/s; a copy 5.0, so 48), bound by the issue of vector instructions: 26.3 of 26.3
// million quarter cycles, 1,390 of them to a wave; LDS is busy for 54%. Heads of 128: 33 us (24 by
// bytes), vector instructions 85% of the cycles; of 64: 25 to 26 (12), 88%. One token 4.6 us, 57 of 40
// sequences 6.4: starts, lengths, table entry and rows, one after the other.
// Read: bound by bytes. 47,604 tokens of 8 heads of 256 from pages of 4 bits: 494 MB in 104 us (4.75
// TB/s; a copy 5.0), of E4M3 585 MB in 130 (4.5), of BF16 780 in 165 (4.7). Values turn in LDS, so that
// rows are written whole.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "se12_paged_rotation.hpp"

namespace se12step {

constexpr int kRowThreads = 256;

struct Append4Args {
    const void* q;
    const void* k;
    const void* v;
    int64_t q_stride, k_stride, v_stride;
    uint8_t* kc;
    uint8_t* vc;
    uint8_t* k_scale;
    uint8_t* v_scale;
    uint16_t* q_out;
    Batch b;
    Rotation r;
    int group, kvh, pages, page_log2;      // group: query heads of a KV head, 0 without q
};

// the scale nearest to amax / 6 (ties to an even byte), and its byte; amax by its bits
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
    if (amax >= 0x7F800000u) return 255u;
    const float a = __uint_as_float(amax), sixth = a * (1.0f / 6.0f);
    // below it (cut to 3 bits of fraction) and half a step on, six times: both exact
    uint32_t byte;
    if (sixth >= 0x1p-14f)
        byte = min((__float_as_uint(sixth) >> 20) - (112u << 3), 226u);
    else
        byte = (uint32_t)(sixth * 0x1p17f);
    const int e = max((int)(byte >> 3), 1);
    const float s = e2m1_scale(byte), middle = 6.0f * (s + __uint_as_float((uint32_t)(e - 19 + 127) << 23));
    byte += a > middle || (a == middle && (byte & 1));
    return min(byte, 226u);
}

// 8 values as codes, the first in the lowest bits
__device__ __forceinline__ uint32_t e2m1x8(const float x[8], float s) {
    if (!(s > 0.0f)) return 0u;            // (NaN: the scale says so)
    const float inv = __builtin_amdgcn_rcpf(s);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // the quotient to its last bit, or a tie would go by the inverse's rounding (beyond 6
        // the conversion gives 6)
        const float t = x[i] * inv;
        y[i] = fmaf(fmaf(-t, s, x[i]), inv, t);
    }
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.0f, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.0f, 3);
}

// kFew: a run's new tokens are half of the rows that kRowThreads work on at once, or fewer.
// kHeads: KV heads of a block, each with kRowThreads of its own (two share the angles: 9,001
// tokens of 8 heads 2 us less than one to a block; few tokens have blocks to spare)
template <int DT, int D, bool kFew, int kHeads>
__global__ __launch_bounds__(kHeads * kRowThreads) void paged_append4_kernel(Append4Args a) {
    constexpr int kLanes = D / 8, kRows = kRowThreads / kLanes, kThreads = kHeads * kRowThreads;
    static_assert(16 <= 2 * kRows, "");
    __shared__ __attribute__((aligned(16))) float2 cs[16 * D / 2];
    __shared__ __attribute__((aligned(16))) float weights[2][D]; // of q's norm and k's
    __shared__ uint32_t all_codes[kHeads][16][kLanes];           // of the values
    __shared__ __attribute__((aligned(16))) uint8_t all_scales[kHeads][2][D / 32][16];
    const int sub = kHeads == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kRowThreads), tid = threadIdx.x % kRowThreads;
    auto& codes = all_codes[sub];
    auto& scales = all_scales[sub];
    const int groups = (a.kvh + kHeads - 1) / kHeads, kh = (int)blockIdx.x % groups * kHeads + sub;
    const Run16 u = run16_of(a.b, (int)blockIdx.x / groups);
    const int n = u.to - u.from;
    if (n <= 0) return;
    const int64_t row0 = u.seq.start + u.first + u.from - u.seq.len;      // of the first token
    const int half = a.r.half;
    turn_run16<kThreads, !kFew>(cs, a.r, u.first, u.from, u.to);
    if (a.r.q_norm && a.group > 0) load_weights<kThreads>(weights[0], a.r, a.r.q_norm, D);
    if (a.r.k_norm) load_weights<kThreads>(weights[1], a.r, a.r.k_norm, D);
    const int P = 1 << a.page_log2, page = page_of(a.b, u.s, u.first >> a.page_log2, a.pages);
    const int64_t page_head = (int64_t)max(page, 0) * a.kvh + kh;
    const int slot0 = u.first & (P - 1);

    // Rows: values (0), keys (1), then the query heads, n tokens of each. A block's threads take
    // kRows tokens of one of them at a time, or of few tokens those of several (in places for a
    // power of two): 57 of 40 sequences, 32 / 8 heads of 128, 6.4 us, 10.6 one at a time; 9,001 of
    // 16 / 8 heads of 256 14 us less one at a time than several, where each lane finds its own. The
    // next rows are on their way while some are worked on (16 tokens of a head of 256 in two turns,
    // both asked for at once: 3 us of 9,001 tokens').
    constexpr int kTurns = kFew ? 1 : 16 / kRows;
    const int lane = tid % kLanes, c0 = 8 * lane, place = tid / kLanes, what_end = kh < a.kvh ? 2 + a.group : 0;
    const int places = n > 1 ? 32 - __builtin_clz(n - 1) : 0;
    auto load = [&](int what, int token) {
        const int t = min(token, n - 1);
        Eight<DT> v;
        if (what == 0)
            v.load(a.v, (row0 + t) * a.v_stride + (int64_t)kh * D + c0);
        else if (what == 1)
            v.load(a.k, (row0 + t) * a.k_stride + (int64_t)kh * D + c0);
        else
            v.load(a.q, (row0 + t) * a.q_stride + (int64_t)(kh * a.group + what - 2) * D + c0);
        return v;
    };
    auto work = [&](const Eight<DT>& from, int what, int t) {
        if (what >= what_end || t >= n) return;
        float x[8];
        from.values(x);
        const int64_t row = row0 + t;
        if (what > 0) {
            const void* w = what == 1 ? a.r.k_norm : a.r.q_norm;
            if (w) norm_row<kLanes>(x, a.r.eps, weights[what == 1] + c0, 1.0 / D);
            if (half > 0) turn_row(x, cs + t * half, c0, half, a.r.interleaved);
            if (what > 1) {
                uint16_t* o = a.q_out + (row * a.group * a.kvh + kh * a.group + what - 2) * D + c0;
                const uint4 v = bf16x8(x);
                reinterpret_cast<uint2*>(o)[0] = make_uint2(v.x, v.y);
                reinterpret_cast<uint2*>(o)[1] = make_uint2(v.z, v.w);
                return;
            }
        }
        // (the larger one, and NaN if there is one: by bits a NaN is above all numbers)
        float most = fabsf(x[0]);
#pragma unroll
        for (int k = 1; k < 8; ++k) most = __builtin_elementwise_maximum(most, fabsf(x[k]));
        uint32_t amax = __float_as_uint(most) & 0x7FFFFFFFu;
        amax = max(amax, (uint32_t)__builtin_amdgcn_mov_dpp((int)amax, 0xB1, 0xF, 0xF, true));       // of four lanes
        amax = max(amax, (uint32_t)__builtin_amdgcn_mov_dpp((int)amax, 0x4E, 0xF, 0xF, true));
        const uint32_t byte = scale_byte(amax), w = e2m1x8(x, e2m1_scale(byte));
        const int slot = u.from + t;
        if (lane % 4 == 0) scales[what][lane / 4][slot] = (uint8_t)byte;
        if (what == 0)
            codes[slot][lane] = w;
        else if (page >= 0)
            *reinterpret_cast<uint32_t*>(a.kc + (page_head * P + slot0 + slot) * (D / 2) + c0 / 2) = w;
    };
    Eight<DT> next[kTurns] = {};
    if constexpr (kFew) {
        auto what_of = [&](int k) { return (k * kRows + place) >> places; };
        auto token_of = [&](int k) { return (k * kRows + place) & ((1 << places) - 1); };
        const int count = ((what_end << places) + kRows - 1) / kRows;
        if (what_of(0) < what_end) next[0] = load(what_of(0), token_of(0));
        __syncthreads();
        for (int k = 0; k < count; ++k) {
            const Eight<DT> here = next[0];
            if (k + 1 < count && what_of(k + 1) < what_end) next[0] = load(what_of(k + 1), token_of(k + 1));
            work(here, what_of(k), token_of(k));
        }
    } else {
#pragma unroll
        for (int j = 0; j < kTurns; ++j)
            if (what_end > 0) next[j] = load(0, j * kRows + place);
        __syncthreads();
        for (int what = 0; what < what_end; ++what) {
            Eight<DT> here[kTurns];
#pragma unroll
            for (int j = 0; j < kTurns; ++j) {
                here[j] = next[j];
                if (what + 1 < what_end) next[j] = load(what + 1, j * kRows + place);
            }
#pragma unroll
            for (int j = 0; j < kTurns; ++j) work(here[j], what, j * kRows + place);
        }
    }
    __syncthreads();
    if (page < 0 || kh >= a.kvh) return;
    for (int c = tid; c < D; c += kRowThreads) {
        uint2* p = reinterpret_cast<uint2*>(a.vc + ((page_head << (a.page_log2 - 4)) + slot0 / 16) * (8 * D)) + c;
        uint2 was = make_uint2(0, 0);
        if (n < 16) was = *p;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int t = 0; t < 16; ++t) w[t / 8] |= ((codes[t][c / 8] >> (4 * (c % 8))) & 15u) << (4 * (t % 8));
        if (n < 16) {      // slots that are not new keep what they hold
            const uint64_t fresh = ((1ull << (4 * n)) - 1) << (4 * u.from);
            w[0] = (w[0] & (uint32_t)fresh) | (was.x & ~(uint32_t)fresh);
            w[1] = (w[1] & (uint32_t)(fresh >> 32)) | (was.y & ~(uint32_t)(fresh >> 32));
        }
        *p = make_uint2(w[0], w[1]);
    }
    for (int i = tid; i < 2 * (D / 32); i += kRowThreads) {
        const int what = i / (D / 32), g = i % (D / 32);
        uint8_t* p = (what == 0 ? a.v_scale : a.k_scale) + (page_head * (D / 32) + g) * P + slot0;
        if (n == 16)
            *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(scales[what][g]);
        else
            for (int t = u.from; t < u.to; ++t) p[t] = scales[what][g][t];
    }
}

// ---------------------------------------------------------------------------
// reading back
// ---------------------------------------------------------------------------

struct ReadArgs {
    const uint8_t* kc;
    const uint8_t* vc;
    const void* k_scale;
    const void* v_scale;
    uint16_t* k;
    uint16_t* v;
    Batch b;
    int kvh, pages, page_log2;
};

// four values of 8 bits times s, in BF16
__device__ __forceinline__ uint2 e4m3x4_values(uint32_t w, float s) {
    typedef float f2_t __attribute__((ext_vector_type(2)));
    const f2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return make_uint2(f_to_bf16x2(a.x * s, a.y * s), f_to_bf16x2(b.x * s, b.y * s));
}

// the two codes of byte `which` of w, times a and b, in BF16
template <int kByte>
__device__ __forceinline__ uint32_t e2m1_values(uint32_t w, float a, float b) {
    typedef float f2_t __attribute__((ext_vector_type(2)));
    const f2_t x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, kByte);
    return f_to_bf16x2(x.x * a, x.y * b);
}

template <int CT, int D>
__global__ __launch_bounds__(kRowThreads) void paged_read_kernel(ReadArgs a) {
    constexpr int kLanes = D / 8, kRows = kRowThreads / kLanes;
    __shared__ __attribute__((aligned(16))) uint16_t tile[16 * (D + 8)];      // values, a token to a row
    const int tid = threadIdx.x, kh = (int)blockIdx.x % a.kvh;
    const Run16 u = run16_of(a.b, (int)blockIdx.x / a.kvh);
    if (u.to <= u.from) return;
    const int P = 1 << a.page_log2, page = page_of(a.b, u.s, u.first >> a.page_log2, a.pages);
    const int64_t page_head = (int64_t)max(page, 0) * a.kvh + kh;
    const int slot0 = u.first & (P - 1), lane = tid % kLanes;
    const int64_t out0 = ((u.seq.start + (int64_t)u.first - u.seq.len) * a.kvh + kh) * D + 8 * lane;       // of slot 0
    // values: two columns to a thread, 16 tokens
    for (int c = 2 * tid; c < D; c += 2 * kRowThreads) {
        uint32_t x[16];      // (token's two columns)
        if constexpr (CT == SE12_STEP_E2M1) {
            const uint4 w = *reinterpret_cast<const uint4*>(a.vc + ((page_head << (a.page_log2 - 4)) + slot0 / 16) * (8 * D) + 8 * c);
            const uint4 sb = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.v_scale) + (page_head * (D / 32) + c / 32) * P + slot0);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w}, bs[4] = {sb.x, sb.y, sb.z, sb.w};
            uint32_t y[2][8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t b = bs[k / 2] >> (16 * (k & 1));
                const float s0 = e2m1_scale(b & 255u), s1 = e2m1_scale((b >> 8) & 255u);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t v = ws[2 * j + k / 4];
                    y[j][k] = (k & 3) == 0 ? e2m1_values<0>(v, s0, s1) : (k & 3) == 1 ? e2m1_values<1>(v, s0, s1)
                              : (k & 3) == 2 ? e2m1_values<2>(v, s0, s1) : e2m1_values<3>(v, s0, s1);
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                x[2 * k] = __builtin_amdgcn_perm(y[1][k], y[0][k], 0x05040100u);
                x[2 * k + 1] = __builtin_amdgcn_perm(y[1][k], y[0][k], 0x07060302u);
            }
        } else {
            uint32_t y[2][8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint8_t* p = a.vc + ((page_head * D + c + j) * P + slot0) * (CT == SE12_STEP_BF16 ? 2 : 1);
                if constexpr (CT == SE12_STEP_BF16) {
                    const uint4 v0 = reinterpret_cast<const uint4*>(p)[0], v1 = reinterpret_cast<const uint4*>(p)[1];
                    const uint32_t v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[j][k] = v[k];
                } else {
                    const float s = static_cast<const float*>(a.v_scale)[page_head];
                    const uint4 v0 = *reinterpret_cast<const uint4*>(p);
                    const uint32_t v[4] = {v0.x, v0.y, v0.z, v0.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint2 z = e4m3x4_values(v[k], s);
                        y[j][2 * k] = z.x;
                        y[j][2 * k + 1] = z.y;
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                x[2 * k] = __builtin_amdgcn_perm(y[1][k], y[0][k], 0x05040100u);
                x[2 * k + 1] = __builtin_amdgcn_perm(y[1][k], y[0][k], 0x07060302u);
            }
        }
#pragma unroll
        for (int t = 0; t < 16; ++t) *reinterpret_cast<uint32_t*>(tile + t * (D + 8) + c) = x[t];
    }
    for (int t = u.from + tid / kLanes; t < u.to; t += kRows) {
        uint4 x;
        const int64_t at = (page_head * P + slot0 + t) * D + 8 * lane;
        if constexpr (CT == SE12_STEP_E2M1) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(a.kc + at / 2);
            const float s = e2m1_scale(static_cast<const uint8_t*>(a.k_scale)[(page_head * (D / 32) + lane / 4) * P + slot0 + t]);
            x = make_uint4(e2m1_values<0>(w, s, s), e2m1_values<1>(w, s, s), e2m1_values<2>(w, s, s), e2m1_values<3>(w, s, s));
        } else if constexpr (CT == SE12_STEP_E4M3) {
            const uint2 w = *reinterpret_cast<const uint2*>(a.kc + at);
            const float s = static_cast<const float*>(a.k_scale)[page_head];
            const uint2 x0 = e4m3x4_values(w.x, s), x1 = e4m3x4_values(w.y, s);
            x = make_uint4(x0.x, x0.y, x1.x, x1.y);
        } else {
            x = *reinterpret_cast<const uint4*>(a.kc + 2 * at);
        }
        *reinterpret_cast<uint4*>(a.k + out0 + (int64_t)t * a.kvh * D) = page >= 0 ? x : make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    for (int t = u.from + tid / kLanes; t < u.to; t += kRows) {
        const uint4 x = *reinterpret_cast<const uint4*>(tile + t * (D + 8) + 8 * lane);
        *reinterpret_cast<uint4*>(a.v + out0 + (int64_t)t * a.kvh * D) = page >= 0 ? x : make_uint4(0, 0, 0, 0);
    }
}

}  // namespace se12step

using namespace se12step;

namespace {

// Heads of 64, whose 16 rows are half of those that kRowThreads work on, are few always: 9,001 tokens of
// 16 / 8 heads 27.3 us, 26.4 a head at a time in pairs of heads, 9 / 3 heads 15.1 and 18.9, 306 tokens of
// 32 / 8 heads 7.6 and 8.8. (Larger heads in pairs where there are two: 6 / 3 heads of 256 29.4, 26.0 one to a
// block; 10 / 5 and 14 / 7 alike.)
template <int DT, int D>
void launch_append4_of(const Append4Args& a, uint32_t runs, hipStream_t st) {
    constexpr int kRows = kRowThreads / (D / 8);
    if (2 * (a.b.max_new < 16 ? a.b.max_new : 16) <= kRows) {
        hipLaunchKernelGGL((paged_append4_kernel<DT, D, true, 1>), dim3(runs * a.kvh), dim3(kRowThreads), 0, st, a);
        return;
    }
    if constexpr (kRows < 2 * 16) {
        if (a.kvh == 1)
            hipLaunchKernelGGL((paged_append4_kernel<DT, D, false, 1>), dim3(runs), dim3(kRowThreads), 0, st, a);
        else
            hipLaunchKernelGGL((paged_append4_kernel<DT, D, false, 2>), dim3(runs * ((a.kvh + 1) / 2)), dim3(2 * kRowThreads), 0, st, a);
    }
}

template <int DT>
void launch_append4(const Append4Args& a, int d, uint32_t runs, hipStream_t st) {
    switch (d) {
        case 64: launch_append4_of<DT, 64>(a, runs, st); break;
        case 128: launch_append4_of<DT, 128>(a, runs, st); break;
        default: launch_append4_of<DT, 256>(a, runs, st);
    }
}

template <int CT>
void launch_read(const ReadArgs& a, int d, uint32_t blocks, hipStream_t st) {
    switch (d) {
        case 64: hipLaunchKernelGGL((paged_read_kernel<CT, 64>), dim3(blocks), dim3(kRowThreads), 0, st, a); break;
        case 128: hipLaunchKernelGGL((paged_read_kernel<CT, 128>), dim3(blocks), dim3(kRowThreads), 0, st, a); break;
        default: hipLaunchKernelGGL((paged_read_kernel<CT, 256>), dim3(blocks), dim3(kRowThreads), 0, st, a);
    }
}

}  // namespace

extern "C" {

int se12_step_paged_append_rotated(const se12_step_pages* pages, const se12_step_batch* batch, const void* q, const void* k,
                                   const void* v, int32_t dtype, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                   int32_t heads, const se12_step_rotation* rotation, uint16_t* q_out, void* stream) {
    const char* fn = "se12_step_paged_append_rotated";
    if (!pages) return step_fail(fn, "NULL argument");
    if (const char* e = paged_error(pages, batch, q ? heads : pages->kv_heads)) return step_fail(fn, e);
    if (pages->dtype != SE12_STEP_E2M1) return step_fail(fn, "the cache must be E2M1");
    if (const char* e = rotation_error(rotation, pages->head_dim)) return step_fail(fn, e);
    if (const char* e = append_error(pages, batch, q, k, v, dtype, q_stride, k_stride, v_stride, heads, q_out)) return step_fail(fn, e);
    if (batch->tokens == 0) return SE12_STEP_OK;
    const Append4Args a{q, k, v, q_stride, k_stride, v_stride, static_cast<uint8_t*>(pages->k), static_cast<uint8_t*>(pages->v),
                        reinterpret_cast<uint8_t*>(pages->k_scale), reinterpret_cast<uint8_t*>(pages->v_scale), q_out,
                        device_batch(batch), device_rotation(rotation), q ? heads / pages->kv_heads : 0, pages->kv_heads,
                        pages->pages, log2_of(pages->page_size)};
    const int64_t runs = run16_blocks(a.b);
    if (!grid_fits(runs * (pages->kv_heads + 1), kRowThreads)) return step_fail(fn, "too many tokens and heads for one launch");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == SE12_STEP_F32)
        launch_append4<SE12_STEP_F32>(a, pages->head_dim, (uint32_t)runs, st);
    else
        launch_append4<SE12_STEP_BF16>(a, pages->head_dim, (uint32_t)runs, st);
    return step_launched();
}

int se12_step_paged_read(const se12_step_pages* pages, const se12_step_batch* batch, uint16_t* k, uint16_t* v, void* stream) {
    const char* fn = "se12_step_paged_read";
    if (!pages) return step_fail(fn, "NULL argument");
    if (const char* e = paged_error(pages, batch, pages->kv_heads)) return step_fail(fn, e);
    if (batch->tokens == 0) return SE12_STEP_OK;
    if (!k || !v) return step_fail(fn, "NULL argument");
    if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16) return step_fail(fn, "misaligned tensor");
    const int64_t bytes = 2 * (int64_t)batch->tokens * pages->kv_heads * pages->head_dim;
    if (overlap(k, bytes, v, bytes)) return step_fail(fn, "k overlaps v");
    const ReadArgs a{static_cast<const uint8_t*>(pages->k), static_cast<const uint8_t*>(pages->v), pages->k_scale, pages->v_scale, k, v,
                     device_batch(batch), pages->kv_heads, pages->pages, log2_of(pages->page_size)};
    const int64_t blocks = run16_blocks(a.b) * pages->kv_heads;
    if (!grid_fits(blocks, kRowThreads)) return step_fail(fn, "too many tokens and heads for one launch");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (pages->dtype == SE12_STEP_E2M1)
        launch_read<SE12_STEP_E2M1>(a, pages->head_dim, (uint32_t)blocks, st);
    else if (pages->dtype == SE12_STEP_E4M3)
        launch_read<SE12_STEP_E4M3>(a, pages->head_dim, (uint32_t)blocks, st);
    else
        launch_read<SE12_STEP_BF16>(a, pages->head_dim, (uint32_t)blocks, st);
    return step_launched();
}

}  // extern "C"
