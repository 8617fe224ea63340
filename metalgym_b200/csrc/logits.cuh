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
#include <string.h>

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

template <int NT>
__device__ __forceinline__ void team_sync() {
    if (NT == 32)
        __syncwarp();
    else
        __syncthreads();
}

// Fills the table from entries [0, n) of `history` (every thread of the team:
// a warp or a CTA; ends with a barrier). `sums` is a shared array of a word
// per warp. The first entries of a thread stay in registers between the two
// passes over the history.
template <int NT>
__device__ inline void history_fill(const HistoryTable& t, const int32_t* history, int n, int lo, int hi, int capacity,
                                    uint32_t* sums) {
    const int span = hi - lo, words = HistoryTable::words(span), cw = HistoryTable::count_words(span, capacity);
    const int tid = NT == 32 ? threadIdx.x & 31 : threadIdx.x;
    constexpr int nt = NT, KEEP = 4;
    int kept[KEEP];
#pragma unroll
    for (int k = 0; k < KEEP; k++) kept[k] = tid + k * nt < n ? history[tid + k * nt] : -1;
    for (int i = tid; i < words; i += nt) t.seen[i] = 0;
    for (int i = tid; i < cw; i += nt) t.counts[i] = 0;
    team_sync<NT>();
    auto mark = [&](int a) {
        if (a >= lo && a < hi) atomicOr(&t.seen[(a - lo) >> 5], 1u << ((a - lo) & 31));
    };
#pragma unroll
    for (int k = 0; k < KEEP; k++) mark(kept[k]);
    for (int i = tid + KEEP * nt; i < n; i += nt) mark(history[i]);
    team_sync<NT>();
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
    uint32_t base = incl - own;
    if (NT > 32) {
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        for (int w = 0; w < warp; w++) base += sums[w];
    }
    for (int w = w0; w < w1; w++) {
        t.before[w] = (uint16_t)base;
        base += __popc(t.seen[w]);
    }
    team_sync<NT>();
    auto add = [&](int a) {
        if (a < lo || a >= hi) return;
        const int k = a - lo;
        const int at = t.before[k >> 5] + __popc(t.seen[k >> 5] & ((1u << (k & 31)) - 1u));
        atomicAdd(&t.counts[at >> 1], 1u << ((at & 1) * 16));
    };
#pragma unroll
    for (int k = 0; k < KEEP; k++) add(kept[k]);
    for (int i = tid + KEEP * nt; i < n; i += nt) add(history[i]);
    team_sync<NT>();
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

// ------------------------------------------------------------------ groups
// A row is read in groups of 16 bytes, cut at 16-byte boundaries of memory
// whatever the row's start: a group that the row (or the part [lo, hi) of it)
// fills takes one vector load, the first and last ones element loads.

template <class T>
constexpr int kGroup = 16 / (int)sizeof(T);

// The first action of group 0 of [lo, hi) (at or up to kGroup - 1 before lo),
// and the number of groups.
template <class T>
__device__ __forceinline__ int group_start(const T* row, int lo) {
    return lo - (int)((reinterpret_cast<uintptr_t>(row + lo) & 15) / sizeof(T));
}
template <class T>
__device__ __forceinline__ int group_count(int start, int hi) {
    return (hi - start + kGroup<T> - 1) / kGroup<T>;
}

// The group's values as they lie in memory.
template <class T>
struct RawGroup {
    uint4 w;
};

__device__ __forceinline__ float raw_value(const RawGroup<float>& g, int i) {
    return __uint_as_float(i == 0 ? g.w.x : i == 1 ? g.w.y : i == 2 ? g.w.z : g.w.w);
}
__device__ __forceinline__ float raw_value(const RawGroup<__nv_bfloat16>& g, int i) {
    const uint32_t u = (i >> 1) == 0 ? g.w.x : (i >> 1) == 1 ? g.w.y : (i >> 1) == 2 ? g.w.z : g.w.w;
    return __uint_as_float((i & 1) ? (u & 0xffff0000u) : (u << 16));
}
__device__ __forceinline__ float raw_value(const RawGroup<__half>& g, int i) {
    const uint32_t u = (i >> 1) == 0 ? g.w.x : (i >> 1) == 1 ? g.w.y : (i >> 1) == 2 ? g.w.z : g.w.w;
    return __half2float(__ushort_as_half((unsigned short)((i & 1) ? (u >> 16) : (u & 0xffffu))));
}

// Bits of the group's elements that lie in [lo, hi).
template <class T>
__device__ __forceinline__ uint32_t group_valid(int a, int lo, int hi) {
    constexpr int VE = kGroup<T>;
    uint32_t v = (1u << VE) - 1u;
    if (a < lo) v &= ~0u << (lo - a);
    if (a + VE > hi) v = hi <= a ? 0u : v & ((1u << (hi - a)) - 1u);
    return v;
}

template <class T>
__device__ __forceinline__ RawGroup<T> group_load(const T* row, int a, uint32_t valid) {
    constexpr int VE = kGroup<T>;
    RawGroup<T> g;
    if (valid == (1u << VE) - 1u) {
        g.w = *reinterpret_cast<const uint4*>(row + a);
        return g;
    }
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < VE; i++)
        if ((valid >> i) & 1u) {
            if (sizeof(T) == 4)
                w[i] = reinterpret_cast<const uint32_t*>(row)[a + i];
            else
                w[i >> 1] |= (uint32_t)reinterpret_cast<const unsigned short*>(row)[a + i] << ((i & 1) * 16);
        }
    g.w = make_uint4(w[0], w[1], w[2], w[3]);
    return g;
}

// Writes a group's values; `vec`: out + a is 16-byte aligned where the group is full.
template <class T>
__device__ __forceinline__ void group_store(T* out, int a, uint32_t valid, bool vec, const float* v) {
    constexpr int VE = kGroup<T>;
    T o[VE];
#pragma unroll
    for (int i = 0; i < VE; i++) from_f32(&o[i], v[i]);
    if (vec && valid == (1u << VE) - 1u) {
        uint32_t w[4];
        memcpy(w, o, 16);
        *reinterpret_cast<uint4*>(out + a) = make_uint4(w[0], w[1], w[2], w[3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < VE; i++)
        if ((valid >> i) & 1u) out[a + i] = o[i];
}

// Whether full groups of `row` are 16-byte aligned in `out` too.
template <class T>
__device__ __forceinline__ bool same_alignment(const T* row, const T* out) {
    return ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
}

// VE bits of a bit row from bit `at` on (all of them inside it).
template <int VE>
__device__ __forceinline__ uint32_t bit_window(const uint32_t* words, int at) {
    const uint32_t lo = words[at >> 5], hi = words[(at + VE - 1) >> 5];
    return __funnelshift_r(lo, hi, at & 31) & ((1u << VE) - 1u);
}

// What the controls did to a group: the elements that may be taken, those that
// occurred before, and of these those whose raw logit is positive.
struct GroupControls {
    uint32_t ok, seen, positive;
};

// Raw values of group a -> controlled logits (-inf outside `valid` and where
// the mask says so). The table covers actions from lo.
template <class T>
__device__ __forceinline__ GroupControls group_control(const RowControls& r, const HistoryTable& t, const RawGroup<T>& g, int a,
                                                       int lo, uint32_t valid, float* x) {
    constexpr int VE = kGroup<T>;
    constexpr uint32_t ALL = (1u << VE) - 1u;
    GroupControls c{valid, 0u, 0u};
#pragma unroll
    for (int i = 0; i < VE; i++) x[i] = raw_value(g, i);
    if (r.history) {
        if (valid == ALL) {
            c.seen = bit_window<VE>(t.seen, a - lo);
        } else {
#pragma unroll
            for (int i = 0; i < VE; i++)
                if (((valid >> i) & 1u) && ((t.seen[(a - lo + i) >> 5] >> ((a - lo + i) & 31)) & 1u)) c.seen |= 1u << i;
        }
        if (c.seen) {
#pragma unroll
            for (int i = 0; i < VE; i++)
                if ((c.seen >> i) & 1u) {
                    if (x[i] > 0.0f) c.positive |= 1u << i;
                    x[i] = penalise(r, x[i], t.count(a - lo + i));
                }
        }
    }
    if (r.bias) {
        const float* b = r.bias + a;
        if (valid == ALL && (reinterpret_cast<uintptr_t>(b) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < VE; i += 4) {
                const float4 q = *reinterpret_cast<const float4*>(b + i);
                x[i] = __fadd_rn(x[i], q.x);
                x[i + 1] = __fadd_rn(x[i + 1], q.y);
                x[i + 2] = __fadd_rn(x[i + 2], q.z);
                x[i + 3] = __fadd_rn(x[i + 3], q.w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < VE; i++)
                if ((valid >> i) & 1u) x[i] = __fadd_rn(x[i], b[i]);
        }
    }
    if (r.mask) {
        if (valid == ALL) {
            c.ok = bit_window<VE>(r.mask, a);
        } else {
#pragma unroll
            for (int i = 0; i < VE; i++)
                if (((valid >> i) & 1u) && !((r.mask[(a + i) >> 5] >> ((a + i) & 31)) & 1u)) c.ok &= ~(1u << i);
        }
    }
    if (c.ok != ALL) {
#pragma unroll
        for (int i = 0; i < VE; i++)
            if (!((c.ok >> i) & 1u)) x[i] = -INFINITY;
    }
    return c;
}

// Its gradient factor on seen elements.
template <class T>
__device__ __forceinline__ void group_factor(const RowControls& r, const GroupControls& c, float* g) {
    if (c.seen) {
#pragma unroll
        for (int i = 0; i < kGroup<T>; i++)
            if ((c.seen >> i) & 1u)
                g[i] = ((c.positive >> i) & 1u) ? __fdiv_rn(g[i], r.repetition) : __fmul_rn(g[i], r.repetition);
    }
}

}  // namespace mg
