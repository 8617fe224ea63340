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

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f32(float* p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_f32(__half* p, float x) { *p = __float2half_rn(x); }

// The occurrences of actions [lo, hi) in one row's history, in shared memory:
// a bit per action, the number of set bits before each word, and for each set
// bit (in the order of the actions) its action, a 16-bit count and a place
// for a value. A history names few of a row's actions: the passes over a row
// leave them out by their bits, at 1/32 word an action, and the list is done
// one by one, in an order that does not depend on the atomics that fill the
// table (they add whole numbers).
struct HistoryTable {
    uint32_t* seen;    // [words]
    uint32_t* counts;  // two 16-bit counts a word
    uint32_t* list;    // actions
    float* value;
    uint16_t* before;  // [words]
    int words;

    __host__ __device__ static constexpr int words_of(int span) { return (span + 31) / 32; }
    __host__ __device__ static constexpr int entries(int span, int history) { return span < history ? span : history; }
    __host__ __device__ static constexpr size_t bytes(int span, int history) {
        const int w = words_of(span), n = entries(span, history);
        return (size_t)w * 4 + (size_t)((n + 1) / 2) * 4 + (size_t)n * 8 + (size_t)((w + 1) / 2) * 4;
    }
    __device__ void place(void* smem, int span, int history) {
        const int w = words_of(span), n = entries(span, history);
        seen = static_cast<uint32_t*>(smem);
        counts = seen + w;
        list = counts + (n + 1) / 2;
        value = reinterpret_cast<float*>(list + n);
        before = reinterpret_cast<uint16_t*>(value + n);
        words = 0;
    }
    // Actions that occurred (after history_fill).
    __device__ __forceinline__ int total() const { return before[words - 1] + __popc(seen[words - 1]); }
    __device__ __forceinline__ int count_at(int at) const { return (counts[at >> 1] >> ((at & 1) * 16)) & 0xffff; }
    __device__ __forceinline__ bool has(int i) const { return (seen[i >> 5] >> (i & 31)) & 1u; }
    // Number of occurrences of action lo + i.
    __device__ __forceinline__ int count(int i) const {
        const uint32_t w = seen[i >> 5], bit = 1u << (i & 31);
        return (w & bit) ? count_at(before[i >> 5] + __popc(w & (bit - 1u))) : 0;
    }
};

static_assert(MG_LOGITS_MAX_HISTORY < 1 << 16, "counts and ranks are 16 bits");

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
__device__ inline void history_fill(HistoryTable& t, const int32_t* history, int n, int lo, int hi, int capacity,
                                    uint32_t* sums) {
    const int span = hi - lo, words = HistoryTable::words_of(span), cw = (HistoryTable::entries(span, capacity) + 1) / 2;
    t.words = words;
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
        t.list[at] = (uint32_t)a;
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
    int actions;
};

__device__ __forceinline__ int row_history_len(const mg_logit_controls& c, int row) {
    if (!c.history) return 0;
    return c.history_len ? min(max(c.history_len[row], 0), c.history_max) : c.history_max;
}

__device__ __forceinline__ RowControls row_controls(const mg_logit_controls& c, int row, int actions) {
    RowControls r;
    r.mask = c.mask ? c.mask + (int64_t)row * c.mask_stride : nullptr;
    r.bias = c.bias ? c.bias + (int64_t)row * c.bias_stride : nullptr;
    r.repetition = c.repetition ? c.repetition[row] : 1.0f;
    r.frequency = c.frequency ? c.frequency[row] : 0.0f;
    r.presence = c.presence ? c.presence[row] : 0.0f;
    r.history = c.history != nullptr;
    r.actions = actions;
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

// Bias and mask of action a.
__device__ __forceinline__ float bias_mask(const RowControls& r, float x, int a) {
    if (r.bias) x = __fadd_rn(x, r.bias[a]);
    return allowed(r, a) ? x : -INFINITY;
}
// The controlled logit of action a (raw x); the table covers actions from lo.
__device__ __forceinline__ float controlled(const RowControls& r, const HistoryTable& t, float x, int a, int lo) {
    const int n = r.history ? t.count(a - lo) : 0;
    return bias_mask(r, n > 0 ? penalise(r, x, n) : x, a);
}
// The gradient of the raw logit x of an action that occurred.
__device__ __forceinline__ float seen_gradient(const RowControls& r, float g, float x) {
    return x > 0.0f ? __fdiv_rn(g, r.repetition) : __fmul_rn(g, r.repetition);
}

// ------------------------------------------------------------------ groups
// A row (or a part [lo, hi) of it) is read in groups of eight actions, by vector
// loads, from the first 16-byte boundary of memory on; the up to 7 actions
// before it and behind the last whole group, the edges, are done one by one by
// the first warp of the team. (Eight fp32 logits are two loads: four to a
// group would look up mask, table and bias twice as often.)

constexpr int kGroup = 8;

template <class T>
struct RawGroup {
    uint4 w[kGroup * sizeof(T) / 16];
};

struct RowSpan {
    int body, groups;    // first action of group 0, number of groups
    int lo, head, tail;  // actions before the groups, and behind them
    // The action of lane `lane` of the edges, or -1.
    __device__ __forceinline__ int edge(int lane) const {
        if (lane < head) return lo + lane;
        return lane >= 16 && lane - 16 < tail ? body + groups * kGroup + lane - 16 : -1;
    }
    __device__ __forceinline__ bool edges() const { return (head | tail) != 0; }
};

template <class T>
__device__ __forceinline__ RowSpan row_span(const T* row, int lo, int hi) {
    const int past = (int)((reinterpret_cast<uintptr_t>(row + lo) & 15) / sizeof(T));
    RowSpan s;
    s.lo = lo;
    s.head = min(hi - lo, past ? (int)(16 / sizeof(T)) - past : 0);
    s.body = lo + s.head;
    s.groups = (hi - s.body) / kGroup;
    s.tail = hi - s.body - s.groups * kGroup;
    return s;
}

template <class T>
__device__ __forceinline__ RawGroup<T> group_load(const T* p) {
    RawGroup<T> g;
#pragma unroll
    for (int i = 0; i < (int)(kGroup * sizeof(T) / 16); i++) g.w[i] = reinterpret_cast<const uint4*>(p)[i];
    return g;
}
__device__ __forceinline__ void group_floats(const RawGroup<float>& g, float* x) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        x[4 * i] = __uint_as_float(g.w[i].x);
        x[4 * i + 1] = __uint_as_float(g.w[i].y);
        x[4 * i + 2] = __uint_as_float(g.w[i].z);
        x[4 * i + 3] = __uint_as_float(g.w[i].w);
    }
}
__device__ __forceinline__ void group_floats(const RawGroup<__nv_bfloat16>& g, float* x) {
    const uint32_t u[4] = {g.w[0].x, g.w[0].y, g.w[0].z, g.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void group_floats(const RawGroup<__half>& g, float* x) {
    const uint32_t u[4] = {g.w[0].x, g.w[0].y, g.w[0].z, g.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// Writes a full group; `vec`: p is 16-byte aligned.
__device__ __forceinline__ void group_store(float* p, bool vec, const float* v) {
    if (vec) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        return;
    }
#pragma unroll
    for (int i = 0; i < kGroup; i++) p[i] = v[i];
}
__device__ __forceinline__ void group_store16(void* p, bool vec, const uint32_t* u) {
    if (vec) {
        *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < kGroup; i++) static_cast<unsigned short*>(p)[i] = (unsigned short)(u[i >> 1] >> ((i & 1) * 16));
}
__device__ __forceinline__ void group_store(__nv_bfloat16* p, bool vec, const float* v) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    group_store16(p, vec, u);
}
__device__ __forceinline__ void group_store(__half* p, bool vec, const float* v) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    group_store16(p, vec, u);
}

// The bits of a group in a bit row, from bit `at` on (all of them inside the
// row; the bits above them are not cleared).
__device__ __forceinline__ uint32_t bit_window(const uint32_t* words, int at) {
    const int sh = at & 31;
    const uint32_t* w = words + (at >> 5);
    return __funnelshift_r(w[0], sh + kGroup > 32 ? w[1] : 0u, sh);
}

// What a kernel is compiled for: 0 neither bias nor mask, +1 a bias, +2 a mask or
// (where a pass leaves actions out) a history. Tested once per group at run
// time instead, the absent controls cost 2.7 instructions a logit of 12.
constexpr int kWithBias = 1, kWithMask = 2;

__device__ __forceinline__ void add8(float* x, float a, float b, float c, float d, float e, float f, float g, float h) {
    const float y[8] = {a, b, c, d, e, f, g, h};
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __fadd_rn(x[i], y[i]);
}

// Bias and mask of a full group of actions from a on (-inf where the mask says
// so, and where `skip` has a bit).
template <int WITH>
__device__ __forceinline__ void group_bias_mask(const RowControls& r, int a, uint32_t skip, float* x) {
    if (((WITH & kWithBias) != 0) && r.bias) {
        const float* b = r.bias + a;
        if ((reinterpret_cast<uintptr_t>(b) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < kGroup; i += 4) {
                const float4 q = *reinterpret_cast<const float4*>(b + i);
                x[i] = __fadd_rn(x[i], q.x);
                x[i + 1] = __fadd_rn(x[i + 1], q.y);
                x[i + 2] = __fadd_rn(x[i + 2], q.z);
                x[i + 3] = __fadd_rn(x[i + 3], q.w);
            }
        } else {
            // the aligned twelve around the eight, in three loads, where they lie inside the row (one
            // by one, eight lines a load, they take twice the cycles of everything else in L1)
            const int off = (int)((reinterpret_cast<uintptr_t>(b) >> 2) & 3);
            if (a >= off && a - off + 12 <= r.actions) {
                const float4* q = reinterpret_cast<const float4*>(b - off);
                const float4 u = q[0], v = q[1], w = q[2];
                if (off == 1)
                    add8(x, u.y, u.z, u.w, v.x, v.y, v.z, v.w, w.x);
                else if (off == 2)
                    add8(x, u.z, u.w, v.x, v.y, v.z, v.w, w.x, w.y);
                else
                    add8(x, u.w, v.x, v.y, v.z, v.w, w.x, w.y, w.z);
            } else {
#pragma unroll
                for (int i = 0; i < kGroup; i++) x[i] = __fadd_rn(x[i], b[i]);
            }
        }
    }
    if constexpr ((WITH & kWithMask) != 0) {
        const uint32_t out = r.mask ? skip | ~bit_window(r.mask, a) : skip;
#pragma unroll
        for (int i = 0; i < kGroup; i++) x[i] = (out & (1u << i)) ? -INFINITY : x[i];
    }
}

}  // namespace mg
