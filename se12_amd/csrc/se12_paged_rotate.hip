// Norm and rotation of a call's q and k by themselves (for caches of BF16 and E4M3, or a
// program's own): se12_paged_rotation.hpp for the mathematics. A block takes a few tokens
// with all their heads, whose angles it works out once. Bound by the bytes of q and k: 7,987
// tokens of 32 / 8 heads of 128, BF16, normed: 164 MB in 35 us (4.7 TB/s; a copy 5.0). 24 tokens 6.1
// us: starts, lengths and rows, one after the other.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "se12_paged_rotation.hpp"

namespace se12step {

constexpr int kRotateThreads = 256;

struct RotateArgs {
    const void* q;
    const void* k;
    int64_t q_stride, k_stride;
    void* q_out;
    void* k_out;
    Batch b;
    Rotation r;
    int heads, kvh, d, tokens;      // tokens of a block
    double share;                   // 1 / d
};

template <int DT, int OT, int kLanes>
__global__ __launch_bounds__(kRotateThreads) void rotate_heads_kernel(RotateArgs a) {
    constexpr int kRows = kRotateThreads / kLanes;
    __shared__ __attribute__((aligned(16))) float weights[2 * kLanes * 8];      // of q's norm and k's
    extern __shared__ __attribute__((aligned(16))) float2 cs[];      // [tokens][half], then positions
    const int tid = threadIdx.x, half = a.r.half, first = (int)blockIdx.x * a.tokens, n = min(a.tokens, a.b.tokens - first);
    int* pos = reinterpret_cast<int*>(cs + a.tokens * half);
    if (tid < n) {
        // the last sequence that starts at or before the token
        int s = 0, e = a.b.seqs;
        while (e - s > 1) {
            const int mid = (s + e) >> 1;
            if (a.b.starts[mid] <= first + tid)
                s = mid;
            else
                e = mid;
        }
        const Seq seq = load_seq(a.b, s);
        const int i = first + tid - seq.start;
        pos[tid] = i >= 0 && i < seq.n ? seq.len + i : -1;
    }
    if (a.r.q_norm) load_weights<kRotateThreads>(weights, a.r, a.r.q_norm, a.d);
    if (a.r.k_norm) load_weights<kRotateThreads>(weights + kLanes * 8, a.r, a.r.k_norm, a.d);
    __syncthreads();
    for (int i = tid; i < n * half; i += kRotateThreads) {
        const int t = i / half, f = i - t * half;
        cs[i] = turn_at(max(pos[t], 0), a.r.inv_freq[f], a.r.scale);
    }
    __syncthreads();
    const int lane = tid % kLanes, c0 = 8 * lane, all = a.heads + a.kvh;
    const bool live = c0 < a.d;
    for (int i = tid / kLanes; i < n * all; i += kRows) {
        const int t = i / all, h = i - t * all;
        const bool is_q = h < a.heads;
        if (pos[t] < 0) continue;
        const int64_t row = first + t;
        const int head = is_q ? h : h - a.heads;
        float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (live) load8<DT>(is_q ? a.q : a.k, row * (is_q ? a.q_stride : a.k_stride) + (int64_t)head * a.d + c0, x);
        const void* w = is_q ? a.r.q_norm : a.r.k_norm;
        if (w) norm_row<kLanes>(x, a.r.eps, weights + (is_q ? 0 : kLanes * 8) + c0, a.share);
        if (half > 0) turn_row(x, cs + t * half, c0, half, a.r.interleaved);
        if (!live) continue;
        const int64_t to = (row * (is_q ? a.heads : a.kvh) + head) * a.d + c0;
        if constexpr (OT == SE12_STEP_F32) {
            float4* o = reinterpret_cast<float4*>(static_cast<float*>(is_q ? a.q_out : a.k_out) + to);
            o[0] = make_float4(x[0], x[1], x[2], x[3]);
            o[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(is_q ? a.q_out : a.k_out) + to) = bf16x8(x);
        }
    }
}

}  // namespace se12step

using namespace se12step;

namespace {

template <int DT, int OT>
void launch_rotate(const RotateArgs& a, uint32_t blocks, hipStream_t st) {
    const size_t lds = (size_t)a.tokens * (a.r.half * sizeof(float2) + sizeof(int));
    if (a.d <= 64)
        hipLaunchKernelGGL((rotate_heads_kernel<DT, OT, 8>), dim3(blocks), dim3(kRotateThreads), lds, st, a);
    else if (a.d <= 128)
        hipLaunchKernelGGL((rotate_heads_kernel<DT, OT, 16>), dim3(blocks), dim3(kRotateThreads), lds, st, a);
    else
        hipLaunchKernelGGL((rotate_heads_kernel<DT, OT, 32>), dim3(blocks), dim3(kRotateThreads), lds, st, a);
}

}  // namespace

extern "C" int se12_step_rotate_heads(const se12_step_batch* batch, const void* q, const void* k, int32_t dtype, int64_t q_stride,
                                      int64_t k_stride, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                      const se12_step_rotation* rotation, void* q_out, void* k_out, int32_t out_dtype, void* stream) {
    const char* fn = "se12_step_rotate_heads";
    if (!batch) return step_fail(fn, "NULL argument");
    if (!batch->lengths || !batch->starts) return step_fail(fn, "NULL batch tensor");
    if (batch->sequences < 1 || batch->sequences > 65536 || batch->tokens < 0 || batch->tokens > (1 << 30) || batch->max_new < 1)
        return step_fail(fn, "bad batch shape");
    if (reinterpret_cast<uintptr_t>(batch->lengths) % 4 || reinterpret_cast<uintptr_t>(batch->starts) % 4)
        return step_fail(fn, "misaligned tensor");
    if (dtype != SE12_STEP_BF16 && dtype != SE12_STEP_F32) return step_fail(fn, "q and k must be BF16 or FP32");
    if (out_dtype != SE12_STEP_BF16 && out_dtype != SE12_STEP_F32) return step_fail(fn, "outputs must be BF16 or FP32");
    if (head_dim < 8 || head_dim > 256 || head_dim % 8) return step_fail(fn, "head_dim must be a multiple of 8 up to 256");
    if (heads < 1 || heads > 65535 || kv_heads < 0 || kv_heads > 65535) return step_fail(fn, "bad head counts");
    if (const char* e = rotation_error(rotation, head_dim)) return step_fail(fn, e);
    const int64_t q_row = (int64_t)heads * head_dim, k_row = (int64_t)kv_heads * head_dim;
    if (q_stride < q_row || q_stride % 4 || (kv_heads > 0 && (k_stride < k_row || k_stride % 4)))
        return step_fail(fn, "rows must be a multiple of 4 elements apart and hold all heads");
    if (batch->tokens == 0) return SE12_STEP_OK;
    if (!q || !q_out || (kv_heads > 0 && (!k || !k_out))) return step_fail(fn, "NULL argument");
    const uintptr_t piece = dtype == SE12_STEP_F32 ? 16 : 8;
    if (reinterpret_cast<uintptr_t>(q) % piece || reinterpret_cast<uintptr_t>(k) % piece || reinterpret_cast<uintptr_t>(q_out) % 16 ||
        reinterpret_cast<uintptr_t>(k_out) % 16)
        return step_fail(fn, "misaligned tensor");
    // (rows are read and written in any order: only a row may be written over, by itself)
    const int64_t more = batch->tokens - 1, in = dtype == SE12_STEP_F32 ? 4 : 2, to = out_dtype == SE12_STEP_F32 ? 4 : 2;
    struct Span {
        const void* p;
        int64_t bytes;
    };
    const Span from[2] = {{q, in * (more * q_stride + q_row)}, {k, kv_heads > 0 ? in * (more * k_stride + k_row) : 0}};
    const Span out[2] = {{q_out, to * (more + 1) * q_row}, {k_out, kv_heads > 0 ? to * (more + 1) * k_row : 0}};
    const bool same[2] = {q == q_out && dtype == out_dtype && (more == 0 || q_stride == q_row),
                          k == k_out && dtype == out_dtype && (more == 0 || k_stride == k_row)};
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2; ++j)
            if (from[i].bytes > 0 && out[j].bytes > 0 && !(i == j && same[i]) && overlap(from[i].p, from[i].bytes, out[j].p, out[j].bytes))
                return step_fail(fn, "an output overlaps other values of q or k");
    if (kv_heads > 0 && overlap(out[0].p, out[0].bytes, out[1].p, out[1].bytes)) return step_fail(fn, "an output overlaps the other");
    const Batch b{nullptr, 0, batch->lengths, batch->starts, 0, batch->sequences, batch->tokens,
                  batch->max_new < batch->tokens ? batch->max_new : batch->tokens};
    // tokens of a block: four share the start, where there are blocks enough all the same (us with one and
    // with four, BF16. 2,048 tokens: 32 / 8 heads of 128 12.5 and 15.9, 16 / 8 of 256 15.0 and 19.3, 8 / 2 of 128 5.7
    // and 6.1, 2 / 1 of 64 4.2 and 3.8. 4,096: 21.1 and 20.7, 25.9 and 26.7, 11.1 and 9.1, 6.7 and 4.0. 8,192: 41 and
    // 38, 52 and 48, 18 and 13, 10.2 and 5.2)
    RotateArgs a{q, k, q_stride, k_stride, q_out, k_out, b, device_rotation(rotation), heads, kv_heads, head_dim, batch->tokens >= 4096 ? 4 : 1, 1.0 / head_dim};
    const int64_t blocks = ((int64_t)b.tokens + a.tokens - 1) / a.tokens;
    if (!grid_fits(blocks, kRotateThreads) || (int64_t)a.tokens * (heads + kv_heads) > INT32_MAX)
        return step_fail(fn, "too many tokens and heads for one launch");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool f32 = dtype == SE12_STEP_F32, f32_out = out_dtype == SE12_STEP_F32;
    if (f32 && f32_out)
        launch_rotate<SE12_STEP_F32, SE12_STEP_F32>(a, (uint32_t)blocks, st);
    else if (f32)
        launch_rotate<SE12_STEP_F32, SE12_STEP_BF16>(a, (uint32_t)blocks, st);
    else if (f32_out)
        launch_rotate<SE12_STEP_BF16, SE12_STEP_F32>(a, (uint32_t)blocks, st);
    else
        launch_rotate<SE12_STEP_BF16, SE12_STEP_BF16>(a, (uint32_t)blocks, st);
    return step_launched();
}
