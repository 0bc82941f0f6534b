// Appending to a paged key/value cache, with the position rotation applied on
// the way. Mathematics: y[i] = x[i] cos(a) - x[j] sin(a), y[j] = x[j] cos(a) +
// x[i] sin(a), j = i + rotary / 2, a = position * inv_freq[i]; a page of E4M3
// holds round(y / scale), scale = 2^e, the least with max |y| <= 448 scale. A
// power of two costs an 8-bit float no precision (its relative step is the same
// at every exponent) and lets a page's scale grow with a later token without
// moving what it holds: old / new is a power of two as well.
//
// One launch. A block owns one (sequence, page, head, K or V), so its scale and
// its bytes have one writer and no order to depend on; further blocks rotate q,
// a wave per token. Angles: position * inv_freq in quarter turns, in 64 bits
// (positions beyond 2^17 would lose a radian's third digit in FP32); sine and cosine
// of what is beyond a whole quarter, up to pi / 4, rounded once, by their series, so that
// q and k are as close to the exact rotation as with FP32 sines and cosines of 64-bit
// angles (in 9,001 tokens 24 E4M3 digits and 840 BF16 ones are not the exact one's; 25 and
// 930 that way; 26 and 1,040 with the fraction turned into an angle in FP32). Bound by the
// bytes of q, k and v at prompt sizes: 9,001 BF16 tokens of 16 and 8 heads of 256 (258 MB)
// take 65 us (68 with a library's sine and cosine; 62 with the card's instructions, whose
// 2^-23 change an E4M3 digit ten times as often); at decode sizes by the launch: 48
// tokens, 7 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "se12_paged_device.hpp"

namespace se12step {

constexpr int kAppendMaxThreads = 1024;
constexpr int kAppendUnits = 4;          // units of 8 values a thread of a prompt's block holds
constexpr int kDirectTokens = 16;        // V of fewer tokens is written value by value

struct AppendArgs {
    const void* q;
    const void* k;
    const void* v;
    int64_t q_stride, k_stride, v_stride;
    void* kc;
    void* vc;
    float* k_scale;
    float* v_scale;
    const float* inv_freq;
    uint16_t* q_out;
    Batch b;
    int kv_blocks, heads, kvh, pages;
    int page_log2, d, half;     // half = rotary / 2
};

template <int DT>
__device__ __forceinline__ float4 load4(const void* p, int64_t i) {
    if constexpr (DT == SE12_STEP_F32) {
        return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    } else {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                           __uint_as_float(u.y & 0xFFFF0000u));
    }
}

// A unit is 8 values of a token's head: columns lo .. lo + 3 and hi .. hi + 3,
// the pairs the rotation mixes (i < half) or, behind the rotated part, neighbours.
__device__ __forceinline__ void unit_columns(int unit, int half, int& lo, int& hi) {
    if (4 * unit < half) {
        lo = 4 * unit;
        hi = lo + half;
    } else {
        lo = 8 * unit;     // 2 half + 8 (unit - half / 4)
        hi = lo + 4;
    }
}

struct Turn {
    float c[4], s[4];
};

__device__ __forceinline__ Turn turn_of(const float* inv_freq, int lo, int pos) {
    const float4 f = *reinterpret_cast<const float4*>(inv_freq + lo);
    const float w[4] = {f.x, f.y, f.z, f.w};
    Turn t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // (to a whole number in the last places of a double's 53 bits)
        const double quarters = (double)pos * (double)w[i] * 0.63661977236758134, whole = quarters + 0x1.8p52;
        const int turn = __double2loint(whole);
        const float x = (float)((quarters - (whole - 0x1.8p52)) * 1.57079632679489662), x2 = x * x;
        const float s = fmaf(x * x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
        const float c = 1.0f + fmaf(x, -0.5f * x, x2 * x2 * fmaf(x2, fmaf(x2, fmaf(x2, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24));
        const uint32_t sn = __float_as_uint(turn & 1 ? c : s), cs = __float_as_uint(turn & 1 ? s : c);
        t.s[i] = __uint_as_float(sn ^ ((uint32_t)(turn & 2) << 30));
        t.c[i] = __uint_as_float(cs ^ ((uint32_t)((turn + 1) & 2) << 30));
    }
    return t;
}

__device__ __forceinline__ void rotate(float* x, const Turn& t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = x[i], b = x[4 + i];
        x[i] = a * t.c[i] - b * t.s[i];
        x[4 + i] = b * t.c[i] + a * t.s[i];
    }
}

__device__ __forceinline__ void put4(float* x, const float4 v) {
    x[0] = v.x;
    x[1] = v.y;
    x[2] = v.z;
    x[3] = v.w;
}

__device__ __forceinline__ uint2 bf16x4(const float* x) { return make_uint2(f_to_bf16x2(x[0], x[1]), f_to_bf16x2(x[2], x[3])); }

// four E4M3 values (round to nearest even; NaN and infinities: NaN)
__device__ __forceinline__ uint32_t e4m3x4(const float* x, float by) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * by, x[1] * by, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * by, x[3] * by, r, true);
}

__device__ __forceinline__ uint32_t e4m3x4_times(uint32_t w, float by) {
    float x[4];
    typedef float f2_t __attribute__((ext_vector_type(2)));
    const f2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = a.x;
    x[1] = a.y;
    x[2] = b.x;
    x[3] = b.y;
    return e4m3x4(x, by);
}

// the least 2^e >= 2^-100 with amax <= 448 * 2^e (448 = 1.75 * 2^8)
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = max((int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0), -100);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// the rows of q, a wave per token: the angles serve all heads
template <int DT>
__device__ __forceinline__ void rotate_q(const AppendArgs& a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int token = ((int)blockIdx.x - a.kv_blocks) * ((int)blockDim.x >> 6) + wave;
    if (token >= a.b.tokens) return;
    // the last sequence that starts at or before the token
    int s = 0, e = a.b.seqs;
    while (e - s > 1) {
        const int mid = (s + e) >> 1;
        if (a.b.starts[mid] <= token)
            s = mid;
        else
            e = mid;
    }
    const Seq seq = load_seq(a.b, s);
    const int i = token - seq.start;
    if (i < 0 || i >= seq.n) return;
    const int units = a.d >> 3, unit = lane & (units - 1), step = 64 / units;
    int lo, hi;
    unit_columns(unit, a.half, lo, hi);
    const bool turned = 4 * unit < a.half;
    Turn t;
    if (turned) t = turn_of(a.inv_freq, lo, seq.len + i);
    for (int h = lane / units; h < a.heads; h += step) {
        const int64_t at = (int64_t)token * a.q_stride + (int64_t)h * a.d;
        float x[8];
        put4(x, load4<DT>(a.q, at + lo));
        put4(x + 4, load4<DT>(a.q, at + hi));
        if (turned) rotate(x, t);
        uint16_t* o = a.q_out + ((int64_t)token * a.heads + h) * a.d;
        *reinterpret_cast<uint2*>(o + lo) = bf16x4(x);
        *reinterpret_cast<uint2*>(o + hi) = bf16x4(x + 4);
    }
}

// What the page holds of older tokens, rounded again to a larger scale: slots
// 0 .. older - 1 of every row. A K row is a token, a V row a column.
__device__ __forceinline__ void rescale_held(uint8_t* page, bool is_v, int d, int page_size, int older, float by) {
    uint32_t* w = reinterpret_cast<uint32_t*>(page);
    if (!is_v) {
        for (int i = threadIdx.x; i < older * d / 4; i += blockDim.x) w[i] = e4m3x4_times(w[i], by);
        return;
    }
    const int per_row = (older + 3) / 4;
    for (int i = threadIdx.x; i < per_row * d; i += blockDim.x) {
        const int r = i / per_row, c = i % per_row, keep = older - 4 * c;   // slots of this word that are older
        uint32_t* p = w + r * (page_size / 4) + c;
        const uint32_t was = *p, now = e4m3x4_times(was, by);
        const uint32_t mask = keep >= 4 ? ~0u : (1u << (8 * keep)) - 1u;
        *p = (now & mask) | (was & ~mask);
    }
}

template <int DT, int CT, int NU>
__global__ __launch_bounds__(kAppendMaxThreads) void paged_append_kernel(AppendArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t tile[];
    __shared__ float most[kAppendMaxThreads / 64];
    if ((int)blockIdx.x >= a.kv_blocks) {
        rotate_q<DT>(a);
        return;
    }
    const int tid = threadIdx.x, P = 1 << a.page_log2, d = a.d;
    const int hv = (int)blockIdx.x % (2 * a.kvh), slot = (int)blockIdx.x / (2 * a.kvh);
    const int head = hv >> 1;
    const bool is_v = hv & 1;
    // Block slots: a sequence of n new tokens touches at most n / P + 2 pages, so
    // sequence s may have slots starts[s] / P + 2 s onwards; at one token each, slot s.
    int s = slot, j = 0;
    if (a.b.max_new > 1) {
        int lo = 0, hi = a.b.seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((min(max(a.b.starts[mid], 0), a.b.tokens) >> a.page_log2) + 2 * mid <= slot)
                lo = mid;
            else
                hi = mid;
        }
        s = lo;
        j = slot - (min(max(a.b.starts[s], 0), a.b.tokens) >> a.page_log2) - 2 * s;
    }
    const Seq seq = load_seq(a.b, s);
    const int page = (seq.len >> a.page_log2) + j;
    if (j < 0 || page >= a.b.width) return;
    const int first = page << a.page_log2;
    const int from = j == 0 ? seq.len - first : 0, to = min(P, seq.len + seq.n - first);   // slots of new tokens
    if (to <= from) return;
    const int id = page_of(a.b, s, page, a.pages);
    if (id < 0) return;

    const int units = d >> 3, count = (to - from) * units;   // units of the block
    const int half = is_v ? d / 2 : a.half;
    const int64_t row0 = seq.start + first + from - seq.len;
    const void* in = is_v ? a.v : a.k;
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
    float x[NU][8];
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        const int u = tid + n * (int)blockDim.x;
        if (u >= count) break;
        int lo, hi;
        unit_columns(u & (units - 1), half, lo, hi);
        const int64_t at = (row0 + u / units) * stride + (int64_t)head * d;
        put4(x[n], load4<DT>(in, at + lo));
        put4(x[n] + 4, load4<DT>(in, at + hi));
    }
    float amax = 0.0f;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        const int u = tid + n * (int)blockDim.x;
        if (u >= count) break;
        if (!is_v) {
            int lo, hi;
            unit_columns(u & (units - 1), half, lo, hi);
            if (lo < half) rotate(x[n], turn_of(a.inv_freq, lo, first + from + u / units));
        }
        if constexpr (CT == SE12_STEP_E4M3) {
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fabsf(x[n][i]) < INFINITY ? fmaxf(amax, fabsf(x[n][i])) : amax;
        }
    }
    const int64_t page_head = (int64_t)id * a.kvh + head;
    constexpr int kBytes = CT == SE12_STEP_E4M3 ? 1 : 2;
    uint8_t* held = static_cast<uint8_t*>(is_v ? a.vc : a.kc) + page_head * P * d * kBytes;
    float by = 1.0f;
    if constexpr (CT == SE12_STEP_E4M3) {
        amax = wave_max(amax);
        if (blockDim.x > 64) {
            if ((tid & 63) == 0) most[tid >> 6] = amax;
            __syncthreads();
            amax = most[0];
            for (int w = 1; w < (int)blockDim.x >> 6; ++w) amax = fmaxf(amax, most[w]);
        }
        float* scale = (is_v ? a.v_scale : a.k_scale) + page_head;
        float now = scale_for(amax);
        if (from > 0) {
            const float was = *scale;
            now = fmaxf(now, was);
            if (now != was) {
                rescale_held(held, is_v, d, P, from, was / now);
                __syncthreads();
            }
        }
        // (every thread has read the old scale: the barrier above, or one wave)
        if (tid == 0) *scale = now;
        by = 1.0f / now;
    }
    const bool staged = is_v && to - from >= kDirectTokens;
    const int row_bytes = P * kBytes + 4;    // LDS: columns four apart are a bank apart
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        const int u = tid + n * (int)blockDim.x;
        if (u >= count) break;
        const int at = from + u / units;
        int c[2];
        unit_columns(u & (units - 1), half, c[0], c[1]);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            if constexpr (CT == SE12_STEP_E4M3) {
                const uint32_t w = e4m3x4(x[n] + 4 * g, by);
                if (!is_v) {
                    *reinterpret_cast<uint32_t*>(held + at * d + c[g]) = w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint8_t* p = staged ? tile + (c[g] + i) * row_bytes + at : held + (c[g] + i) * P + at;
                        *p = (uint8_t)(w >> (8 * i));
                    }
                }
            } else {
                const uint2 w = bf16x4(x[n] + 4 * g);
                if (!is_v) {
                    *reinterpret_cast<uint2*>(held + 2 * (at * d + c[g])) = w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint8_t* p = staged ? tile + (c[g] + i) * row_bytes + 2 * at : held + 2 * ((c[g] + i) * P + at);
                        *reinterpret_cast<uint16_t*>(p) = (uint16_t)((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
                    }
                }
            }
        }
    }
    if (!staged) return;
    __syncthreads();
    constexpr int kPer = 16 / kBytes;        // tokens of 16 bytes
    const int pieces = P / kPer;
    for (int i = tid; i < pieces * d; i += blockDim.x) {
        const int r = i / pieces, t0 = i % pieces * kPer;
        const uint32_t* w = reinterpret_cast<const uint32_t*>(tile + r * row_bytes + t0 * kBytes);
        uint8_t* p = held + (r * P + t0) * kBytes;
        if (t0 >= from && t0 + kPer <= to) {
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            for (int t = max(t0, from); t < min(t0 + kPer, to); ++t) {
                if constexpr (CT == SE12_STEP_E4M3)
                    p[t - t0] = tile[r * row_bytes + t];
                else
                    reinterpret_cast<uint16_t*>(p)[t - t0] = *reinterpret_cast<const uint16_t*>(tile + r * row_bytes + 2 * t);
            }
        }
    }
}

}  // namespace se12step

using namespace se12step;

namespace {

template <int DT, int CT>
void launch_append(const AppendArgs& a, dim3 grid, int threads, int units, size_t lds, hipStream_t st) {
    if (units <= threads)
        hipLaunchKernelGGL((paged_append_kernel<DT, CT, 1>), grid, dim3(threads), lds, st, a);
    else
        hipLaunchKernelGGL((paged_append_kernel<DT, CT, kAppendUnits>), grid, dim3(threads), lds, st, a);
}

}  // namespace

extern "C" {

int se12_step_paged_append(const se12_step_pages* pages, const se12_step_batch* batch, const void* q, const void* k,
                           const void* v, int32_t dtype, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                           int32_t heads, const float* inv_freq, int32_t rotary, uint16_t* q_out, void* stream) {
    const char* fn = "se12_step_paged_append";
    if (!pages) return step_fail(fn, "NULL argument");
    if (const char* e = paged_error(pages, batch, q ? heads : pages->kv_heads)) return step_fail(fn, e);
    if (batch->tokens > 0 && rotary > 0 && !inv_freq) return step_fail(fn, "NULL argument");
    if (rotary < 0 || rotary > pages->head_dim || rotary % 8) return step_fail(fn, "rotary must be a multiple of 8 up to head_dim");
    if (reinterpret_cast<uintptr_t>(inv_freq) % 16) return step_fail(fn, "misaligned tensor");
    if (const char* e = append_error(pages, batch, q, k, v, dtype, q_stride, k_stride, v_stride, heads, q_out)) return step_fail(fn, e);
    if (batch->tokens == 0) return SE12_STEP_OK;
    if (pages->dtype == SE12_STEP_E2M1) {
        const se12_step_rotation r{inv_freq, nullptr, nullptr, 1.0, 0.0, 0.0f, SE12_STEP_BF16, rotary, 0};
        return se12_step_paged_append_rotated(pages, batch, q, k, v, dtype, q_stride, k_stride, v_stride, heads, &r, q_out, stream);
    }
    AppendArgs a{q, k, v, q_stride, k_stride, v_stride, pages->k, pages->v, pages->k_scale, pages->v_scale, inv_freq, q_out,
                 device_batch(batch), 0, q ? heads : 0, pages->kv_heads, pages->pages,
                 log2_of(pages->page_size), pages->head_dim, rotary / 2};
    const int per_token = pages->head_dim / 8;
    const int units = (pages->page_size < a.b.max_new ? pages->page_size : a.b.max_new) * per_token;   // of a block, at most
    const int threads = units <= 64 ? 64 : units <= 256 * kAppendUnits ? 256 : units <= 512 * kAppendUnits ? 512 : kAppendMaxThreads;
    const int64_t slots = a.b.max_new == 1 ? a.b.seqs : (int64_t)(a.b.tokens >> a.page_log2) + 2 * (int64_t)a.b.seqs;
    const int64_t kv_blocks = slots * 2 * pages->kv_heads;
    const int64_t q_blocks = q ? ((int64_t)a.b.tokens + threads / 64 - 1) / (threads / 64) : 0;
    if (!grid_fits(kv_blocks + q_blocks, threads)) return step_fail(fn, "too many tokens and heads for one launch");
    a.kv_blocks = (int)kv_blocks;
    const size_t lds = a.b.max_new < kDirectTokens
                           ? 0 : (size_t)pages->head_dim * (pages->page_size * (pages->dtype == SE12_STEP_E4M3 ? 1 : 2) + 4);
    const dim3 grid((uint32_t)(kv_blocks + q_blocks));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool f32 = dtype == SE12_STEP_F32, e4m3 = pages->dtype == SE12_STEP_E4M3;
    if (f32 && e4m3)
        launch_append<SE12_STEP_F32, SE12_STEP_E4M3>(a, grid, threads, units, lds, st);
    else if (f32)
        launch_append<SE12_STEP_F32, SE12_STEP_BF16>(a, grid, threads, units, lds, st);
    else if (e4m3)
        launch_append<SE12_STEP_BF16, SE12_STEP_E4M3>(a, grid, threads, units, lds, st);
    else
        launch_append<SE12_STEP_BF16, SE12_STEP_BF16>(a, grid, threads, units, lds, st);
    return step_launched();
}

}  // extern "C"
