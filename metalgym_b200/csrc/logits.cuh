// Controls on logits: penalties for actions that occurred before, biases and
// action masks, as the kernels of logits.cu read them.
//
// Row r, action a, raw logit x, n = occurrences of a in the row's history:
//   n > 0:  x = x > 0 ? x / repetition : x * repetition
//           x = (x - frequency * n) - presence
//   x = x + bias;  an action that the mask leaves out gets -inf.
// Every operation is one rounded fp32 operation (no contraction), so that the
// winner of a draw, a whole number, does not depend on the compiler.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/metalgym_b200.h"

namespace mg {

constexpr int kLogitsMaxActions = 1 << 18;   // the seen-bits of a row fit in 32 KB
constexpr int kLogitsMaxHistory = 1 << 14;   // a count fits in 16 bits

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f32(float* p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_f32(__half* p, float x) { *p = __float2half_rn(x); }

// The occurrences of actions [lo, hi) in one row's history, in shared memory:
// a bit per action, the number of set bits before each word, and a 16-bit
// count per set bit. Whole numbers only, so the order of the atomics that
// fill it does not matter. A row's history names few of its actions: the bits
// cost 1/32 word an action, and only actions that occurred look a count up.
struct HistoryTable {
    uint32_t* seen;    // [words]
    uint16_t* before;  // [words]
    uint32_t* counts;  // two 16-bit counts a word

    __host__ __device__ static int words(int span) { return (span + 31) / 32; }
    __host__ __device__ static int count_words(int span, int history) { return ((span < history ? span : history) + 1) / 2; }
    __host__ __device__ static size_t bytes(int span, int history) {
        return (size_t)words(span) * 4 + (size_t)count_words(span, history) * 4 + (size_t)(words(span) + 1) / 2 * 4;
    }
    __device__ void place(void* smem, int span, int history) {
        seen = static_cast<uint32_t*>(smem);
        counts = seen + words(span);
        before = reinterpret_cast<uint16_t*>(counts + count_words(span, history));
    }
    // Number of occurrences of action lo + i.
    __device__ __forceinline__ int count(int i) const {
        const uint32_t w = seen[i >> 5], bit = 1u << (i & 31);
        if (!(w & bit)) return 0;
        const int at = before[i >> 5] + __popc(w & (bit - 1u));
        return (counts[at >> 1] >> ((at & 1) * 16)) & 0xffff;
    }
};

// Fills the table from entries [0, n) of `history` (every thread of the CTA;
// ends with a barrier). `sums` is a shared array of a word per warp.
__device__ inline void history_fill(const HistoryTable& t, const int32_t* history, int n, int lo, int hi, int capacity,
                                    uint32_t* sums) {
    const int span = hi - lo, words = HistoryTable::words(span), cw = HistoryTable::count_words(span, capacity);
    const int tid = threadIdx.x, nt = blockDim.x;
    for (int i = tid; i < words; i += nt) t.seen[i] = 0;
    for (int i = tid; i < cw; i += nt) t.counts[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += nt) {
        const int a = history[i];
        if (a >= lo && a < hi) atomicOr(&t.seen[(a - lo) >> 5], 1u << ((a - lo) & 31));
    }
    __syncthreads();
    // exclusive scan of the words' bit counts: a contiguous run of words a thread
    const int per = (words + nt - 1) / nt, w0 = min(words, tid * per), w1 = min(words, w0 + per);
    uint32_t own = 0;
    for (int w = w0; w < w1; w++) own += __popc(t.seen[w]);
    uint32_t incl = own;
    const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    uint32_t base = incl - own;
    for (int w = 0; w < warp; w++) base += sums[w];
    for (int w = w0; w < w1; w++) {
        t.before[w] = (uint16_t)base;
        base += __popc(t.seen[w]);
    }
    __syncthreads();
    for (int i = tid; i < n; i += nt) {
        const int a = history[i];
        if (a >= lo && a < hi) {
            const int k = a - lo;
            const int at = t.before[k >> 5] + __popc(t.seen[k >> 5] & ((1u << (k & 31)) - 1u));
            atomicAdd(&t.counts[at >> 1], 1u << ((at & 1) * 16));
        }
    }
    __syncthreads();
}

// One row's controls.
struct RowControls {
    const uint32_t* mask;  // null: every action allowed
    const float* bias;     // null: none
    float repetition, frequency, presence;
    bool history;  // the row's table is filled
};

__device__ __forceinline__ int row_history_len(const mg_logit_controls& c, int row) {
    if (!c.history) return 0;
    return c.history_len ? min(max(c.history_len[row], 0), c.history_max) : c.history_max;
}

__device__ __forceinline__ RowControls row_controls(const mg_logit_controls& c, int row) {
    RowControls r;
    r.mask = c.mask ? c.mask + (int64_t)row * c.mask_stride : nullptr;
    r.bias = c.bias ? c.bias + (int64_t)row * c.bias_stride : nullptr;
    r.repetition = c.repetition ? c.repetition[row] : 1.0f;
    r.frequency = c.frequency ? c.frequency[row] : 0.0f;
    r.presence = c.presence ? c.presence[row] : 0.0f;
    r.history = c.history != nullptr;
    return r;
}

__device__ __forceinline__ bool allowed(const RowControls& r, int a) {
    return !r.mask || ((r.mask[a >> 5] >> (a & 31)) & 1u);
}

// The penalties of an action that occurred n > 0 times.
__device__ __forceinline__ float penalise(const RowControls& r, float x, int n) {
    x = x > 0.0f ? __fdiv_rn(x, r.repetition) : __fmul_rn(x, r.repetition);
    return __fsub_rn(__fsub_rn(x, __fmul_rn(r.frequency, (float)n)), r.presence);
}

}  // namespace mg
