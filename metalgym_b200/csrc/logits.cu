// Controlled logits: penalties, biases and action masks (logits.cuh) written
// out, differentiated, drawn from, and under the clipped PPO loss.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>
#include <utility>

#include "logits.cuh"
#include "runtime.h"
#include "metalgym/detail/ptx.cuh"
#include "metalgym/pdl.cuh"
#include "metalgym/rng.h"
#include "metalgym/rowmap.h"

namespace mg {
namespace {

// A team reads one row, or one part of it: a warp (eight rows a CTA) where rows
// are short and many, else a CTA of NT threads, with the row's parts in the
// CTAs of a cluster where rows are few or so long that the rows being read
// would not stay in L2 for the loss's second pass.
constexpr int kWarpRows = 8;  // rows of a CTA of warp teams

template <int NT>
constexpr int kCtaThreads = NT == 32 ? 32 * kWarpRows : NT;
template <int NT>
constexpr int kTeamWarps = NT / 32;

struct TeamPart {
    int rows, actions;
    int span;        // actions of a CTA (a multiple of 256, or all of them)
    int parts;       // CTAs of a row
    int tableBytes;  // shared memory of a team's history table
};

// The team's row and its part [lo, hi); false: no row.
template <int NT>
__device__ __forceinline__ bool team_part(const TeamPart& p, int& row, int& lo, int& hi) {
    if (NT == 32) {
        const unsigned r = blockIdx.x * kWarpRows + (threadIdx.x >> 5);  // (past 2^31 in the last CTA of 2^31 - 1 rows)
        row = (int)r;
        lo = 0;
        hi = p.actions;
        return r < (unsigned)p.rows;
    }
    row = blockIdx.x / p.parts;
    lo = min(p.actions, (int)(blockIdx.x % p.parts) * p.span);
    hi = min(p.actions, lo + p.span);
    return true;
}

// Whether 16-byte boundaries of `a` are ones of `b` too.
__device__ __forceinline__ bool same_alignment(const void* a, const void* b) {
    return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

template <int NT>
__device__ __forceinline__ int team_rank() {
    return NT == 32 ? threadIdx.x & 31 : threadIdx.x;
}

template <int NT>
__device__ __forceinline__ HistoryTable team_table(const TeamPart& p, const mg_logit_controls& c, uint32_t* smem) {
    HistoryTable t;
    t.place(smem + (NT == 32 ? (threadIdx.x >> 5) * (p.tableBytes / 4) : 0), p.span, c.history_max);
    return t;
}

// ------------------------------------------------------------------ control and its gradient

// The work is cut into units of kUnit actions of a row, and the units are dealt
// out evenly and in order to as many CTAs as the GPU holds (or warp teams: a
// row each), so that a CTA fills a row's history table once for all the units
// it has of the row.
constexpr int kUnit = 2048;
constexpr int kControlGroups = 4;  // 16-byte loads of a thread in flight
constexpr int kControlCtas = 5;    // CTAs an SM holds

template <class T, int NT, bool BACKWARD, int WITH>
__device__ __forceinline__ void control_part(const T* x, const T* src, T* y, const RowControls& r, HistoryTable& t,
                                             const mg_logit_controls& c, int row, int lo, int hi, uint32_t* sums) {
    constexpr int VE = kGroup, U = kControlGroups * 16 / (VE * (int)sizeof(T));
    const int tid = team_rank<NT>();
    const bool vec = same_alignment(src, y);
    const RowSpan s = row_span(src, lo, hi);
    if (r.history) {
        history_fill<NT>(t, c.history + (int64_t)row * c.history_stride, row_history_len(c, row), lo, hi, c.history_max, sums);
        // the values of the actions that occurred, before anything is written (the call may be in place)
        for (int j = tid, n = t.total(); j < n; j += NT) {
            const int a = t.list[j];
            const float raw = to_f32(x[a]);
            if (BACKWARD)
                t.value[j] = allowed(r, a) ? seen_gradient(r, to_f32(src[a]), raw) : 0.0f;
            else
                t.value[j] = bias_mask(r, penalise(r, raw, t.count_at(j)), a);
        }
        team_sync<NT>();
    }
    for (int g0 = tid; g0 < s.groups; g0 += NT * U) {
        RawGroup<T> raw[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (g0 + u * NT < s.groups) raw[u] = group_load(src + s.body + (g0 + u * NT) * VE);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (g0 + u * NT >= s.groups) break;
            const int a = s.body + (g0 + u * NT) * VE;
            float v[VE];
            group_floats(raw[u], v);
            if constexpr (!BACKWARD) {
                group_bias_mask<WITH>(r, a, 0u, v);
            } else if ((WITH & kWithMask) && r.mask) {
                const uint32_t ok = bit_window(r.mask, a);
#pragma unroll
                for (int i = 0; i < VE; i++) v[i] = (ok & (1u << i)) ? v[i] : 0.0f;
            }
            group_store(y + a, vec, v);
        }
    }
    if (s.edges() && tid < 32) {
        const int a = s.edge(tid);
        if (a >= 0) {
            const float raw = to_f32(src[a]);
            from_f32(&y[a], !BACKWARD ? bias_mask(r, raw, a) : allowed(r, a) ? raw : 0.0f);
        }
    }
    if (r.history) {
        team_sync<NT>();  // the values replace what the pass wrote for these actions
        for (int j = tid, n = t.total(); j < n; j += NT) from_f32(&y[t.list[j]], t.value[j]);
        team_sync<NT>();
    }
}

template <class T, int NT, bool BACKWARD, int WITH>
__global__ void __launch_bounds__(kCtaThreads<NT>, NT == 32 ? 1 : kControlCtas)
    k_logits_control(const T* logits, int64_t ld, const mg_logit_controls c, const T* dOut, int64_t ldg, T* out,
                     int64_t ldo, const TeamPart part) {
    mg_pdl_trigger();
    mg_pdl_wait();
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t sums[kTeamWarps<NT>];
    HistoryTable t = team_table<NT>(part, c, smem);
    auto run = [&](int row, int lo, int hi) {
        const T* x = logits + (int64_t)row * ld;
        control_part<T, NT, BACKWARD, WITH>(x, BACKWARD ? dOut + (int64_t)row * ldg : x, out + (int64_t)row * ldo, row_controls(c, row, part.actions),
                                      t, c, row, lo, hi, sums);
    };
    if (NT == 32) {
        int row, lo, hi;
        if (team_part<NT>(part, row, lo, hi)) run(row, lo, hi);
        return;
    }
    const int perRow = part.parts;  // units of a row
    const int64_t total = (int64_t)part.rows * perRow;
    int64_t u = total * blockIdx.x / gridDim.x;
    const int64_t end = total * (blockIdx.x + 1) / gridDim.x;
    while (u < end) {
        const int row = (int)(u / perRow), first = (int)(u - (int64_t)row * perRow);
        const int last = (int)min((int64_t)perRow, first + (end - u));
        run(row, first * kUnit, min(part.actions, last * kUnit));
        u += last - first;
    }
}

// ------------------------------------------------------------------ softmax statistics and the race

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) {  // within 2 ulp; results below 2^-126 are 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float log2_fast(float x) {  // within 2^-22 (absolute near 1)
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The largest of a warp's values (NaN ignored).
__device__ __forceinline__ float warp_max(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

// l - m for a logit and the running maximum, kept finite, so that e^-inf = 0
// times it is 0 (a NaN stays one). Subtracted before anything is scaled: logits
// up to the type's largest and lowest numbers stay in range.
__device__ __forceinline__ float below(float l, float m) { return max_nan(l - m, -1e30f); }
__device__ __forceinline__ float exp_fast(float d) { return exp2_fast(d * kLog2e); }

// Running softmax statistics: the maximum m, s = sum e^d, t = sum e^d d with d =
// l - m; entropy = log s - t / s. In the passes m is the same in the threads of
// a warp, s and t are a thread's.
struct Softmax {
    float m = -INFINITY, s = 0.0f, t = 0.0f;
    // Raises m (a whole warp) and returns the factor that carried s over.
    __device__ __forceinline__ float raise(float top) {
        const float d = below(m, top), e = exp_fast(d);
        t = e > 0.0f ? e * (t + s * d) : 0.0f;
        if (!(s != s)) s = s * e;
        m = top;
        return e;
    }
};

// Adds N logits (-inf: not allowed) to a warp's statistics; `raised` is told
// when m rises, before each(i, e^(l - max)) gets every logit's weight. False:
// nothing allowed so far, no weights.
template <int N, class Raised, class Each>
__device__ __forceinline__ bool softmax_group(Softmax& v, const float* x, Raised raised, Each each) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; i++) top = fmaxf(top, x[i]);
    top = warp_max(top);
    if (top > v.m) raised(v.raise(top));
    if (v.m == -INFINITY) {  // a NaN still shows
#pragma unroll
        for (int i = 0; i < N; i++)
            if (x[i] != x[i]) v.s = x[i];
        return false;
    }
    float2 s2 = make_float2(0.0f, 0.0f), t2 = s2;
    const float2 k2 = make_float2(kLog2e, kLog2e), m2 = make_float2(-v.m, -v.m);
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) {  // two at a time (f32x2)
        float2 d = f2add_rn(make_float2(x[i], x[i + 1]), m2);
        d.x = max_nan(d.x, -1e30f);
        d.y = max_nan(d.y, -1e30f);
        const float2 k = f2mul_rn(d, k2), w = make_float2(exp2_fast(k.x), exp2_fast(k.y));
        s2 = f2add_rn(s2, w);
        t2 = f2fma_rn(w, d, t2);
        each(i, w.x);
        each(i + 1, w.y);
    }
    if (N & 1) {
        const float d = below(x[N - 1], v.m), w = exp_fast(d);
        s2.x += w;
        t2.x = fmaf(w, d, t2.x);
        each(N - 1, w);
    }
    v.s += s2.x + s2.y;
    v.t += t2.x + t2.y;
    return true;
}

__device__ __forceinline__ uint32_t race_bits(uint32_t word, int a) { return mg_mix32(word + (uint32_t)a * 0x9E3779B9u); }
__device__ __forceinline__ double race_key(uint32_t h, float l) {
    return (double)l - log(-log1p(-((double)h + 0.5) * (1.0 / 4294967296.0)));
}

// Floats as integers of the same order, and back.
__device__ __forceinline__ int float_order(float x) {
    const int i = __float_as_int(x);
    return i >= 0 ? i : i ^ 0x7fffffff;
}
__device__ __forceinline__ float ordered_float(int i) { return __int_as_float(i >= 0 ? i : i ^ 0x7fffffff); }

// A runner of the race: its key in 32 bits, and what gives the key in 64.
struct Runner {
    float key = -INFINITY, logit = -INFINITY;
    uint32_t bits = 0;
    int action = -1;
};

// Whether a's key is above b's (equal keys: the lower action). 32 bits decide
// where they can: both keys are good to well within the margin.
template <bool GREEDY>
__device__ __forceinline__ bool beats(const Runner& a, const Runner& b) {
    if (a.action < 0 || b.action < 0) return a.action >= 0;
    if (GREEDY) return a.logit > b.logit || (a.logit == b.logit && a.action < b.action);
    const float d = a.key - b.key, margin = 1e-4f * (1.0f + fabsf(b.key));
    if (d > margin) return true;
    if (d < -margin) return false;
    const double ka = race_key(a.bits, a.logit), kb = race_key(b.bits, b.logit);
    return ka > kb || (ka == kb && a.action < b.action);
}

__device__ __forceinline__ Runner runner_xor(const Runner& r, int d) {
    Runner o;
    o.key = __shfl_xor_sync(0xffffffffu, r.key, d);
    o.logit = __shfl_xor_sync(0xffffffffu, r.logit, d);
    o.bits = __shfl_xor_sync(0xffffffffu, r.bits, d);
    o.action = __shfl_xor_sync(0xffffffffu, r.action, d);
    return o;
}

// What the warps of a row tell each other.
struct RowPart {
    Softmax v;
    Runner best;
    float chosen;
};

__device__ __forceinline__ float warp_add(float x) {
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}

// The row's statistics (and best runner) in every thread of its CTAs, merged in
// one fixed order: lanes, warps, CTAs. With several parts the caller ends with
// cluster_sync, so that no CTA leaves while another reads its part.
template <int NT, bool RACE, bool GREEDY>
__device__ inline void row_merge(RowPart& mine, RowPart* warps, int parts, int chosenRank) {
    mine.v.s = warp_add(mine.v.s);
    mine.v.t = warp_add(mine.v.t);
    if (RACE) {
#pragma unroll 1
        for (int d = 16; d; d >>= 1) {
            const Runner o = runner_xor(mine.best, d);
            if (beats<GREEDY>(o, mine.best)) mine.best = o;
        }
    }
    if (NT == 32) return;
    // a lane for each warp of the row's CTAs
    constexpr int W = kTeamWarps<NT>;
    static_assert(NT == 32 || W == 8, "eight warps a CTA: up to two slots a lane");
    const int lane = threadIdx.x & 31;
    if (lane == 0) warps[threadIdx.x >> 5] = mine;
    __syncwarp();  // (the cluster's barrier takes whole warps)
    if (parts == 1)
        __syncthreads();
    else
        cluster_sync();
    Softmax v[2];
    Runner best;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int slot = lane + 32 * k;
        if (slot < parts * W) {
            const RowPart* o = parts == 1 ? warps + slot : cluster_peer(warps, slot / W) + slot % W;
            v[k] = o->v;
            if (RACE && beats<GREEDY>(o->best, best)) best = o->best;
        }
    }
    const float m = warp_max(fmaxf(v[0].m, v[1].m));
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const float d = v[k].m > -INFINITY ? below(v[k].m, m) : 0.0f, f = exp_fast(d);
        s += v[k].s * f;
        if (f > 0.0f) t += f * (v[k].t + v[k].s * d);
    }
    mine.v.m = m;
    mine.v.s = warp_add(s);
    mine.v.t = warp_add(t);
    if (RACE) {
#pragma unroll 1
        for (int d = 16; d; d >>= 1) {
            const Runner o = runner_xor(best, d);
            if (beats<GREEDY>(o, best)) best = o;
        }
        mine.best = best;
    } else if (parts > 1) {
        mine.chosen = cluster_peer(warps, chosenRank)->chosen;
    }
}

// Passes the team's part of a row, controlled but without the actions that
// occurred, to take(l, at, count): whole warps, 16 logits a lane while there
// are as many, then a group a lane, then the edges. (The next loads are left to
// the other warps: holding them in registers cost 7 % more than it hid.)
template <class T, int NT, int WITH, class Take>
__device__ __forceinline__ void row_walk(const T* x, const RowControls& r, const HistoryTable& t, const RowSpan& s, int lo,
                                         Take take) {
    constexpr int VE = kGroup, U = 16 / VE;
    const int tid = team_rank<NT>();
    auto control = [&](const RawGroup<T>& raw, int a, float* l) {
        group_floats(raw, l);
        group_bias_mask<WITH>(r, a, r.history ? bit_window(t.seen, a - lo) : 0u, l);
    };
    int g0 = 0;
    for (; g0 + NT * U <= s.groups; g0 += NT * U) {
        const int a = s.body + (g0 + tid) * VE;
        RawGroup<T> raw[U];
#pragma unroll
        for (int u = 0; u < U; u++) raw[u] = group_load(x + a + u * NT * VE);
        float l[16];
#pragma unroll
        for (int u = 0; u < U; u++) control(raw[u], a + u * NT * VE, l + u * VE);
        take(l, [&](int i) { return a + (i / VE) * (NT * VE) + i % VE; }, std::integral_constant<int, 16>());
    }
    for (; g0 < s.groups; g0 += NT) {
        const int g = g0 + tid, a = s.body + g * VE;
        float l[VE];
        if (g < s.groups) {
            control(group_load(x + a), a, l);
        } else {
#pragma unroll
            for (int i = 0; i < VE; i++) l[i] = -INFINITY;
        }
        take(l, [&](int i) { return a + i; }, std::integral_constant<int, VE>());
    }
    if (s.edges() && tid < 32) {
        const int a = s.edge(tid);
        const float l = a < 0 || (r.history && t.has(a - lo)) ? -INFINITY : bias_mask(r, to_f32(x[a]), a);
        take(&l, [&](int) { return a; }, std::integral_constant<int, 1>());
    }
}

// ------------------------------------------------------------------ draw

// One pass. An action can win only where its time E >= v = (h + 1/2) / 2^32 is
// below the best ratio E / e^(l - m) so far times its own e^(l - m). The test
// takes the upper 16 bits of h, which the last step of mg_mix32 leaves alone,
// as 2^23 + k against 2^23 + 2^16 times that bound (1e-4 more than it, so that
// rounding never hides a winner); only the few that pass take logarithms.
template <class T, int NT, bool GREEDY, int WITH>
__global__ void __launch_bounds__(kCtaThreads<NT>, NT == 32 ? 1 : 4)
    k_logits_sample(const T* logits, int64_t ld, const mg_logit_controls c, uint32_t* rng, int32_t* action,
                    float* logProb, float* entropy, float* value, const TeamPart part) {
    mg_pdl_trigger();
    mg_pdl_wait();
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t sums[kTeamWarps<NT>];
    __shared__ __align__(8) unsigned char slots[kTeamWarps<NT> * sizeof(RowPart)];
    RowPart* warps = reinterpret_cast<RowPart*>(slots);
    int row, lo, hi;
    if (!team_part<NT>(part, row, lo, hi)) return;
    const RowControls r = row_controls(c, row, part.actions);
    HistoryTable t = team_table<NT>(part, c, smem);
    if (r.history)
        history_fill<NT>(t, c.history + (int64_t)row * c.history_stride, row_history_len(c, row), lo, hi, c.history_max, sums);
    const T* x = logits + (int64_t)row * ld;
    uint32_t word = GREEDY ? 0u : rng[row];
    if (!GREEDY) rngNext(word);
    RowPart mine;
    float bound = 3e38f;  // the warp's best ratio E / e^(l - m)
    __shared__ int sharedBound;  // the CTA's, as an ordered log(E / e^l)
    if (NT > 32 && !GREEDY) {
        if (threadIdx.x == 0) sharedBound = 0x7f800000;
        __syncthreads();
    }
    const RowSpan s = row_span(x, lo, hi);
    const int tid = team_rank<NT>();

    // Action a of logit l > -inf in the race: the lane's best runner, and its ratio E / e^(l - m).
    auto enter = [&](float l, int a) {
        const uint32_t h = race_bits(word, a);
        // -log(1 - v): its series below 1 / 64 (the next term is 4e-6 of it), else from 1 - v
        const float u = ((float)h + 0.5f) * 2.3283064e-10f;
        const float time = u < 0.015625f ? u * fmaf(u, fmaf(u, 0.33333333f, 0.5f), 1.0f)
                                         : -kLn2 * log2_fast(((float)(~h) + 0.5f) * 2.3283064e-10f);
        Runner o;
        o.key = fmaf(-kLn2, log2_fast(time), l);
        o.logit = l;
        o.bits = h;
        o.action = a;
        if (beats<false>(o, mine.best)) mine.best = o;
        return time / exp_fast(below(l, mine.v.m));
    };
    // The warp's bound from its lanes' ratios, told to the CTA.
    auto tighten = [&](float ratio) {
        const float least = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(ratio)));
        if (!(least < bound)) return false;
        bound = least;
        if (NT > 32 && (threadIdx.x & 31) == 0) atomicMin(&sharedBound, float_order(kLn2 * log2_fast(least) - mine.v.m));
        return true;
    };
    // One action a lane sets a first bound: without one, all 16 logits of every
    // lane would pass it in the first round (12 us of a CTA's time).
    if (!GREEDY && s.groups >= NT) {
        const int a = s.body + tid * kGroup;
        const float l = r.history && t.has(a - lo) ? -INFINITY : bias_mask(r, to_f32(x[a]), a);
        const float top = warp_max(l);
        if (top > -INFINITY) {
            mine.v.m = top;
            tighten(l > -INFINITY ? fminf(enter(l, a), 3e38f) : 3e38f);
        }
        team_sync<NT>();
    }

    // N logits (every lane of the warp calls it; -inf where a lane has none):
    // the i-th is of action at(i)
    auto take = [&](const float* l, auto at, auto count) {
        constexpr int N = decltype(count)::value;
        if (GREEDY) {
            softmax_group<N>(mine.v, l, [](float) {}, [](int, float) {});
#pragma unroll
            for (int i = 0; i < N; i++)
                if (l[i] > mine.best.logit || (l[i] == mine.best.logit && at(i) < mine.best.action)) {
                    mine.best.logit = l[i];
                    mine.best.action = at(i);
                }
            return;
        }
        uint32_t pass = 0;
        float limit = 0.0f;
        auto raised = [&](float f) { bound = f > 0.0f ? fminf(bound / f, 3e38f) : 3e38f; };
        const bool some = softmax_group<N>(mine.v, l, raised, [&](int i, float e) {
            if (i == 0) {
                if (NT > 32) {  // (3e-7 |m|: the roundings of the sums with m, so that the bound is never too low)
                    const float other = ordered_float(*(volatile int*)&sharedBound) + mine.v.m;
                    bound = fminf(bound, exp_fast(fmaf(3e-7f, fabsf(mine.v.m), other)));
                }
                limit = fminf(bound * 65542.6f, 3e38f);  // 2^16 (1 + 1e-4)
            }
            uint32_t h = word + (uint32_t)at(i) * 0x9E3779B9u;
            h ^= h >> 16;
            h *= 0x7feb352du;
            h ^= h >> 15;
            h *= 0x846ca68bu;
            const float f = __uint_as_float(__byte_perm(h, 0x4B000000u, 0x7632));
            // (negated: the weight of a +infinity is NaN, and it passes)
            if (!(f > fmaf(limit, e, 8388608.0f))) pass |= 1u << i;
        });
        // the lanes' candidates, one a lane at a time, each against the bound that the ones before it left
        auto still = [&](uint32_t bits) {  // those of them that pass under the bound as it is now
            uint32_t out = 0;
            const float now = fminf(bound * 65542.6f, 3e38f);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float f = (float)(race_bits(word, at(i)) >> 16), e = exp_fast(below(l[i], mine.v.m));
                if (!(f > now * e)) out |= 1u << i;
            }
            return out & bits;
        };
        while (some && __any_sync(0xffffffffu, pass != 0)) {
            float ratio = 3e38f;
            if (pass) {
                const int i = __ffs(pass) - 1;
                pass &= pass - 1;
                float li = l[0];
#pragma unroll
                for (int k = 1; k < N; k++) li = k == i ? l[k] : li;
                if (li > -INFINITY) ratio = fminf(enter(li, at(i)), 3e38f);
            }
            if (tighten(ratio) && N > 4 && __any_sync(0xffffffffu, (pass & (pass - 1)) != 0)) pass = still(pass);
        }
    };
    row_walk<T, NT, WITH>(x, r, t, s, lo, take);
    if (r.history) {
        for (int j0 = 0, n = t.total(); j0 < n; j0 += NT) {
            const int j = j0 + tid, a = j < n ? (int)t.list[j] : 0;
            const float l = j < n ? bias_mask(r, penalise(r, to_f32(x[a]), t.count_at(j)), a) : -INFINITY;
            take(&l, [&](int) { return a; }, std::integral_constant<int, 1>());
        }
    }
    row_merge<NT, true, GREEDY>(mine, warps, part.parts, 0);
    if (tid == 0 && lo == 0) {
        const float ls = logf(mine.v.s);
        const bool some = mine.best.action >= 0 || mine.v.s != mine.v.s;
        action[row] = mine.best.action;
        logProb[row] = some ? below(mine.best.logit, mine.v.m) - ls : 0.0f;
        if (entropy) entropy[row] = some ? ls - mine.v.t / mine.v.s : 0.0f;
        if (value) value[row] = to_f32(x[part.actions]);
        if (!GREEDY) rng[row] = word;
    }
    __syncwarp();
    if (NT > 32 && part.parts > 1) cluster_sync();
}

// ------------------------------------------------------------------ loss

struct LossArgs {
    const int32_t* action;
    const float *adv, *advStats, *ret, *oldLogProb;
    float* stats;
    float clip, valueCoef, entropyCoef, scale;
    int* status;
};

// The row's statistics in one pass, its gradient in a second one that reads the
// row again, from L2.
template <class T, int NT, int WITH>
__global__ void __launch_bounds__(kCtaThreads<NT>, NT == 32 ? 1 : 5)
    k_logits_loss(const T* logits, int64_t ld, const mg_logit_controls c, T* dLogits, int64_t ldd, const TeamPart part,
                  const LossArgs L) {
    constexpr int VE = kGroup;
    mg_pdl_trigger();
    mg_pdl_wait();
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t sums[kTeamWarps<NT>];
    __shared__ __align__(8) unsigned char slots[kTeamWarps<NT> * sizeof(RowPart)];
    RowPart* warps = reinterpret_cast<RowPart*>(slots);
    int row, lo, hi;
    if (!team_part<NT>(part, row, lo, hi)) return;
    const int actions = part.actions, tid = team_rank<NT>();
    const RowControls r = row_controls(c, row, part.actions);
    HistoryTable t = team_table<NT>(part, c, smem);
    const T* x = logits + (int64_t)row * ld;
    T* d = dLogits + (int64_t)row * ldd;
    const int act = L.action[row];
    // the row's other inputs in flight with its action
    const float old = L.oldLogProb[row], advRaw = L.adv[row], ret = L.ret ? L.ret[row] : 0.0f;
    const float adv0 = L.advStats ? L.advStats[0] : 0.0f, adv1 = L.advStats ? L.advStats[1] : 1.0f;
    const float valueX = L.ret && lo == 0 ? to_f32(x[actions]) : 0.0f;
    const bool inside = act >= 0 && act < actions;
    auto leaveOut = [&] {
        for (int a = lo + tid; a < hi; a += NT) from_f32(&d[a], 0.0f);
        if (lo == 0 && L.ret && tid == 0) from_f32(&d[actions], 0.0f);
        if (lo == 0 && tid < 5) L.stats[(int64_t)row * 5 + tid] = 0.0f;
    };
    if (!inside || !allowed(r, act)) {  // the same for every CTA of the row
        if (tid == 0 && lo == 0 && !inside && act != -1) record_error(L.status, kDevBadAction);
        leaveOut();
        return;
    }
    if (r.history)
        history_fill<NT>(t, c.history + (int64_t)row * c.history_stride, row_history_len(c, row), lo, hi, c.history_max, sums);
    RowPart mine;
    mine.chosen = act >= lo && act < hi ? controlled(r, t, to_f32(x[act]), act, lo) : 0.0f;
    const RowSpan s = row_span(x, lo, hi);
    auto take = [&](const float* l, auto, auto count) {
        softmax_group<decltype(count)::value>(mine.v, l, [](float) {}, [](int, float) {});
    };
    row_walk<T, NT, WITH>(x, r, t, s, lo, take);
    if (r.history) {
        for (int j0 = 0, n = t.total(); j0 < n; j0 += NT) {
            const int j = j0 + tid;
            float l = -INFINITY;
            if (j < n) {
                const int a = t.list[j];
                const float raw = to_f32(x[a]);
                l = bias_mask(r, penalise(r, raw, t.count_at(j)), a);
                t.value[j] = l;
                if (raw > 0.0f) t.list[j] = (uint32_t)a | 0x80000000u;  // the sign, for the gradient
            }
            take(&l, 0, std::integral_constant<int, 1>());
        }
    }
    row_merge<NT, false, false>(mine, warps, part.parts, act / part.span);
    const float m = mine.v.m, ls = logf(mine.v.s), entropy = ls - mine.v.t / mine.v.s;
    const float logp = below(mine.chosen, m) - ls;
    const float ratio = expf(logp - old);
    const float adv = L.advStats ? (advRaw - adv0) * adv1 : advRaw;
    const float one = ratio * adv, two = fminf(fmaxf(ratio, 1.0f - L.clip), 1.0f + L.clip) * adv;
    const float slope = one <= two ? -adv * ratio : 0.0f;
    // every thread has read the action's logit: the gradient may take its place
    __syncwarp();
    if (NT > 32) {
        if (part.parts > 1)
            cluster_sync();
        else
            __syncthreads();
    }
    if (mine.chosen == -INFINITY) {  // an action that the policy never takes
        leaveOut();
        return;
    }
    // dl = scale (slope (1[a = act] - p) + ent p (ln p + H)) = p (s1 log p + (ent H - slope) scale), + s0 at act
    const float s0 = slope * L.scale, s1 = L.entropyCoef * L.scale, sh = fmaf(L.entropyCoef * L.scale, entropy, -s0);
    // (1e8: times the bounded logarithm, 1e30, a larger s1 could overflow, and 0 times that is NaN)
    const bool vec = same_alignment(x, d), all_nan = !(fabsf(sh) < INFINITY && fabsf(s1) < 1e8f);
    auto gradient = [&](float l, int a) {
        const float q = below(l, m) - ls;
        const float g = exp_fast(q) * fmaf(s1, q, sh);
        return a == act ? g + s0 : g;
    };
    constexpr int U = sizeof(T) == 4 ? 1 : 2;  // (two groups of fp32: 176 us at 1000 x 50001, one 153)
    for (int g0 = tid; g0 < s.groups; g0 += NT * U) {
        RawGroup<T> raw[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (g0 + u * NT < s.groups) raw[u] = group_load(x + s.body + (g0 + u * NT) * VE);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (g0 + u * NT >= s.groups) break;
            const int a = s.body + (g0 + u * NT) * VE;
            float l[VE];
            group_floats(raw[u], l);
            group_bias_mask<WITH>(r, a, 0u, l);
            const float2 k2 = make_float2(kLog2e, kLog2e), m2 = make_float2(-m, -m), ls2 = make_float2(-ls, -ls);
            const float2 s12 = make_float2(s1, s1), sh2 = make_float2(sh, sh);
#pragma unroll
            for (int i = 0; i < VE; i += 2) {
                float2 q = f2add_rn(make_float2(l[i], l[i + 1]), m2);
                q.x = max_nan(q.x, -1e30f);
                q.y = max_nan(q.y, -1e30f);
                q = f2add_rn(q, ls2);
                const float2 k = f2mul_rn(q, k2), p = make_float2(exp2_fast(k.x), exp2_fast(k.y));
                const float2 o = f2mul_rn(p, f2fma_rn(s12, q, sh2));
                l[i] = o.x;
                l[i + 1] = o.y;
            }
            if ((unsigned)(act - a) < (unsigned)VE) {
#pragma unroll
                for (int i = 0; i < VE; i++) l[i] = a + i == act ? l[i] + s0 : l[i];
            }
            if ((WITH & kWithMask) && r.mask && all_nan) {  // a NaN somewhere in the row: still 0 where the mask says so
                const uint32_t ok = bit_window(r.mask, a);
#pragma unroll
                for (int i = 0; i < VE; i++) l[i] = (ok & (1u << i)) ? l[i] : 0.0f;
            }
            group_store(d + a, vec, l);
        }
    }
    if (s.edges() && tid < 32) {
        const int a = s.edge(tid);
        if (a >= 0) from_f32(&d[a], allowed(r, a) ? gradient(bias_mask(r, to_f32(x[a]), a), a) : 0.0f);
    }
    if (r.history) {  // the actions that occurred, over what the pass wrote for them
        team_sync<NT>();
        for (int j = tid, n = t.total(); j < n; j += NT) {
            const int a = t.list[j] & 0x7fffffff;
            const float g = gradient(t.value[j], a);
            from_f32(&d[a], allowed(r, a) ? ((t.list[j] >> 31) ? __fdiv_rn(g, r.repetition) : __fmul_rn(g, r.repetition)) : 0.0f);
        }
    }
    if (tid == 0 && lo == 0) {
        float* st = L.stats + (int64_t)row * 5;
        float vLoss = 0.0f;
        if (L.ret) {
            const float err = valueX - ret;
            vLoss = 0.5f * L.valueCoef * err * err;
            from_f32(&d[actions], L.valueCoef * err * L.scale);
        }
        st[0] = -fminf(one, two);
        st[1] = vLoss;
        st[2] = entropy;
        st[3] = old - logp;
        st[4] = fabsf(ratio - 1.0f) > L.clip ? 1.0f : 0.0f;
    }
}

// ------------------------------------------------------------------ host

int type_size(int dtype) { return dtype == MG_DTYPE_F32 ? 4 : 2; }
bool type_ok(int dtype) { return dtype == MG_DTYPE_F32 || dtype == MG_DTYPE_BF16 || dtype == MG_DTYPE_F16; }
bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % (unsigned)bytes) == 0; }

// Without its history a call has no tables either: their size goes by history_max.
void leave_out_history(mg_logit_controls* c) {
    c->history = nullptr;
    c->history_len = nullptr;
    c->history_max = 0;
}

// Checks what every call shares and copies the controls; a history that no
// penalty reads is left out.
int check_common(const char* name, const void* logits, int dtype, int64_t ld, const mg_logit_controls* controls, int rows,
                 int actions, int columns, mg_logit_controls* out) {
    const std::string n(name);
    MG_CHECK_ARG(logits, n + ": null logits");
    MG_CHECK_ARG(type_ok(dtype), n + ": unknown dtype");
    MG_CHECK_ARG(aligned(logits, type_size(dtype)), n + ": logits not aligned to their type");
    MG_CHECK_ARG(rows > 0 && actions > 0, n + ": rows and actions must be positive");
    MG_CHECK_ARG(actions <= MG_LOGITS_MAX_ACTIONS, n + ": at most " + std::to_string(MG_LOGITS_MAX_ACTIONS) + " actions");
    MG_CHECK_ARG(ld >= columns, n + ": ld smaller than the row");
    *out = mg_logit_controls{};
    if (!controls) return MG_OK;
    const mg_logit_controls& c = *controls;
    MG_CHECK_ARG(!c.mask || (aligned(c.mask, 4) && (c.mask_stride == 0 || c.mask_stride >= (actions + 31) / 32)),
                 n + ": mask_stride smaller than a row's words (0: one mask for every row)");
    MG_CHECK_ARG(!c.bias || (aligned(c.bias, 4) && (c.bias_stride == 0 || c.bias_stride >= actions)),
                 n + ": bias_stride smaller than the row (0: one bias for every row)");
    MG_CHECK_ARG(c.history || !(c.repetition || c.frequency || c.presence), n + ": penalties need a history");
    MG_CHECK_ARG(!c.history || (c.history_max > 0 && c.history_max <= MG_LOGITS_MAX_HISTORY),
                 n + ": history_max must be in 1.." + std::to_string(MG_LOGITS_MAX_HISTORY));
    MG_CHECK_ARG(!c.history || c.history_stride >= c.history_max || rows == 1, n + ": history_stride smaller than history_max");
    MG_CHECK_ARG(aligned(c.history, 4) && aligned(c.history_len, 4) && aligned(c.repetition, 4) && aligned(c.frequency, 4) &&
                     aligned(c.presence, 4),
                 n + ": a control's buffer is not aligned to its type");
    *out = c;
    if (!c.history || (!c.repetition && !c.frequency && !c.presence)) leave_out_history(out);
    return MG_OK;
}

// How a call's rows are split over teams.
TeamPart plan(int nt, int rows, int actions, int parts, int historyMax) {
    TeamPart p;
    p.rows = rows;
    p.actions = actions;
    p.parts = parts;
    p.span = nt == 32 || parts == 1 ? actions : ((actions + parts - 1) / parts + 255) / 256 * 256;
    p.tableBytes = historyMax ? (int)HistoryTable::bytes(p.span, historyMax) : 0;
    return p;
}

template <int NT>
size_t table_smem(const TeamPart& p) {
    return (size_t)p.tableBytes * (NT == 32 ? kWarpRows : 1);
}

// the largest table (2^18 actions, 2^14 entries); a CTA's eight of warp teams take less
constexpr int kTableSmemMax = 216 * 1024;
static_assert(HistoryTable::bytes(MG_LOGITS_MAX_ACTIONS, MG_LOGITS_MAX_HISTORY) <= kTableSmemMax, "every table that the calls accept");

// A launch of rows x parts CTAs (or warp teams), the parts of a row in one cluster.
template <int NT, class... KArgs, class... Args>
int launch_rows(void (*kern)(KArgs...), const TeamPart& p, cudaStream_t st, const char* what, Args&&... args) {
    const int64_t ctas = NT == 32 ? ((int64_t)p.rows + kWarpRows - 1) / kWarpRows : (int64_t)p.rows * p.parts;
    if (ctas > INT32_MAX) return fail(MG_ERR_ARGUMENT, std::string(what) + ": too many rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kCtaThreads<NT>);
    cfg.dynamicSmemBytes = table_smem<NT>(p);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.parts;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = NT > 32 && p.parts > 1 ? 2 : 1;
    MG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...));
    return check_launch(what);
}

// Parts of a row for the calls that need the whole row's statistics: the
// fewest nanoseconds by what a CTA alone takes a logit, without and with
// controls, and what a cluster of two, four or eight costs the call and each
// row (its CTAs start together, which the GPU grants one cluster at a time).
// Over 1 to 5000 rows of 6000 to 262144 actions of bf16 and fp32 the choice is
// within 0.4 % (draw) and 1.5 % (loss) of the best of the four on average; us
// with 1, 2, 4, 8 parts, all controls:
//   draw   1 x 32768   20.6  14.5  12.4  13.2     loss   1 x 32768   26.4  17.1  12.2  10.8
//         64 x 131072  63.0  45.6  35.7  44.7           64 x 50001   44.9  30.2  28.2  30.7
//        200 x 20000   22.9  20.2  36.1  98.0          200 x 131072   154  92.9  87.0   103
//        592 x 24000   31.8  43.4  82.4   265         1000 x 50001    145   130   169   331
// A loss of more rows than the GPU holds CTAs takes two parts from 128 KB a row
// on: what it reads and writes would not stay in L2 for the second pass (4096 x
// 32768 fp32 without controls 252 us in one part, 224 in two).
int row_parts(int rows, int actions, int size, bool controls, bool loss) {
    const double fixed[2][4] = {{0, 900, 1500, 3800}, {0, 1000, 1100, 2800}};  // [draw, loss][parts 1, 2, 4, 8]
    const double perRow[2][4] = {{0, 16, 110, 470}, {0, 10, 47, 160}}, perLogit[2][2] = {{0.23, 0.41}, {0.19, 0.55}};
    int best = 0;
    double least = 0.0;
    for (int i = 0; i < 4 && (i == 0 || actions >= 2048 << i); i++) {  // (so long that no part is empty)
        const double ns = fixed[loss][i] + perRow[loss][i] * rows + perLogit[loss][controls] * actions / (1 << i);
        if (i == 0 || ns < least) best = i, least = ns;
    }
    if (loss && rows > 5 * num_sms() && (int64_t)actions * size >= 128 << 10) best = std::max(best, 1);
    return 1 << best;
}

enum RowCall { kCallControl, kCallDraw, kCallLoss };

// Whether a warp takes a row, instead of a CTA. A CTA spends about 3000
// instructions on a row whatever its length (merging warps, barriers), a warp
// waits out its loads one after the other, a row's history among them: warps are
// faster where rows are many for their length and their history's, and where
// rows are short. The choice is within 0.7 % (draw, loss) and 1.3 % (control) of
// the better of the two on average over 4 to 8000 rows of 6 to 12000 actions with
// histories of 0 to 2000; us by warps / by CTAs, mask, bias and a history of 64:
//             180 x 300   600 x 1500   1000 x 2816   1000 x 3500   2048 x 4096   8000 x 6000
//   control   4.5 / 6.4    6.7 / 7.3   10.6 / 12.4   13.3 / 13.0   14.4 / 22.8   64.5 / 88.8
//   draw      9.5 / 8.7   14.9 / 15.9  20.1 / 21.1   24.1 / 21.7   24.6 / 41.3    131 / 194
//   loss      8.2 / 9.1   12.6 / 10.2  18.6 / 16.3   23.4 / 18.3   25.3 / 29.8    157 / 152
// and 1000 x 1024 with a history of 512 14.1 / 12.8, 21.1 / 19.3, 18.0 / 15.1.
// Eight history tables beyond 100 KB leave an SM one CTA (4096 x 2048 with a
// history of 1500, draw 137 / 106).
bool warp_teams(RowCall call, int rows, int actions, int historyMax) {
    if (actions <= 256 && historyMax <= 64) return true;
    if (historyMax && HistoryTable::bytes(actions, historyMax) * kWarpRows > 100 * 1024) return false;
    const int64_t r = rows, a = actions, h = historyMax;
    const int sms = num_sms();
    switch (call) {
        case kCallControl: return r > sms && a <= 8192 && a + 9 * h <= 5 * r;
        case kCallDraw: return r > 4 * sms && a <= 12000 && 4 * a + 9 * h <= 12 * r;
        default: return r > sms && a <= 3600 && 2 * a + 8 * h <= 5 * r;
    }
}

// The compiled controls that a call needs; `history`: the pass leaves out the
// actions that occurred. Warp teams take the kernel with all of them.
int needed_controls(const mg_logit_controls& c, bool history) {
    return (c.bias ? kWithBias : 0) | (c.mask || (history && c.history) ? kWithMask : 0);
}

template <class T, int NT, bool BACKWARD, int WITH>
int launch_control(const void* logits, int64_t ld, const mg_logit_controls& c, const void* dOut, int64_t ldg, void* out,
                   int64_t ldo, int rows, int actions, cudaStream_t st) {
    auto kern = k_logits_control<T, NT, BACKWARD, WITH>;
    static std::atomic<uint64_t> done{0};
    MG_TRY(smem_limit_once(kern, kTableSmemMax, done));
    TeamPart p = plan(NT, rows, actions, 1, c.history_max);
    int64_t ctas = ((int64_t)rows + kWarpRows - 1) / kWarpRows;
    if (NT > 32) {
        p.parts = (actions + kUnit - 1) / kUnit;
        const int64_t units = (int64_t)rows * p.parts;
        ctas = std::min(units, (int64_t)num_sms() * kControlCtas);
        p.span = (int)std::min((int64_t)actions, (units + ctas - 1) / ctas * kUnit);
        p.tableBytes = c.history_max ? (int)HistoryTable::bytes(p.span, c.history_max) : 0;
    }
    MG_CUDA_TRY(MG_LAUNCH(kern, (unsigned)ctas, kCtaThreads<NT>, table_smem<NT>(p), st, static_cast<const T*>(logits), ld, c,
                          static_cast<const T*>(dOut), ldg, static_cast<T*>(out), ldo, p));
    return check_launch("k_logits_control");
}

template <class T, bool BACKWARD>
int control(const void* logits, int64_t ld, const mg_logit_controls& c, const void* dOut, int64_t ldg, void* out, int64_t ldo,
            int rows, int actions, cudaStream_t st) {
    auto f = launch_control<T, 32, BACKWARD, BACKWARD ? kWithMask : kWithBias | kWithMask>;
    if (!warp_teams(kCallControl, rows, actions, c.history_max)) {
        switch (needed_controls(c, false)) {
            case 0: f = launch_control<T, 256, BACKWARD, 0>; break;
            case kWithMask: f = launch_control<T, 256, BACKWARD, kWithMask>; break;
            default:  // (no bias in a gradient)
                if constexpr (!BACKWARD)
                    f = c.mask ? launch_control<T, 256, false, kWithBias | kWithMask> : launch_control<T, 256, false, kWithBias>;
        }
    }
    return f(logits, ld, c, dOut, ldg, out, ldo, rows, actions, st);
}

template <class T, int NT, bool GREEDY, int WITH>
int launch_sample(const void* logits, int64_t ld, const mg_logit_controls& c, uint32_t* rng, int32_t* action, float* logProb,
                  float* entropy, float* value, int rows, int actions, cudaStream_t st) {
    auto kern = k_logits_sample<T, NT, GREEDY, WITH>;
    static std::atomic<uint64_t> done{0};
    MG_TRY(smem_limit_once(kern, kTableSmemMax, done));
    const TeamPart p = plan(NT, rows, actions, NT == 32 ? 1 : row_parts(rows, actions, sizeof(T), WITH != 0, false), c.history_max);
    return launch_rows<NT>(kern, p, st, "k_logits_sample", static_cast<const T*>(logits), ld, c, rng, action, logProb, entropy,
                           value, p);
}

template <class T, bool GREEDY>
int sample_rows(const void* logits, int64_t ld, const mg_logit_controls& c, uint32_t* rng, int32_t* action, float* logProb,
                float* entropy, float* value, int rows, int actions, cudaStream_t st) {
    auto f = launch_sample<T, 32, GREEDY, 3>;
    if (!warp_teams(kCallDraw, rows, actions, c.history_max)) {
        switch (needed_controls(c, true)) {
            case 0: f = launch_sample<T, 256, GREEDY, 0>; break;
            case 1: f = launch_sample<T, 256, GREEDY, 1>; break;
            case 2: f = launch_sample<T, 256, GREEDY, 2>; break;
            default: f = launch_sample<T, 256, GREEDY, 3>;
        }
    }
    return f(logits, ld, c, rng, action, logProb, entropy, value, rows, actions, st);
}

template <class T>
int sample(const void* logits, int64_t ld, const mg_logit_controls& c, uint32_t* rng, int32_t* action, float* logProb,
           float* entropy, float* value, int rows, int actions, cudaStream_t st) {
    return rng ? sample_rows<T, false>(logits, ld, c, rng, action, logProb, entropy, value, rows, actions, st)
               : sample_rows<T, true>(logits, ld, c, rng, action, logProb, entropy, value, rows, actions, st);
}

template <class T, int NT, int WITH>
int launch_loss(const void* logits, int64_t ld, const mg_logit_controls& c, void* d, int64_t ldd, int rows, int actions,
                const LossArgs& L, cudaStream_t st) {
    auto kern = k_logits_loss<T, NT, WITH>;
    static std::atomic<uint64_t> done{0};
    MG_TRY(smem_limit_once(kern, kTableSmemMax, done));
    const TeamPart p = plan(NT, rows, actions, NT == 32 ? 1 : row_parts(rows, actions, sizeof(T), WITH != 0, true), c.history_max);
    return launch_rows<NT>(kern, p, st, "k_logits_loss", static_cast<const T*>(logits), ld, c, static_cast<T*>(d), ldd, p, L);
}

template <class T>
int loss(const void* logits, int64_t ld, const mg_logit_controls& c, void* d, int64_t ldd, int rows, int actions,
         const LossArgs& L, cudaStream_t st) {
    auto f = launch_loss<T, 32, 3>;
    if (!warp_teams(kCallLoss, rows, actions, c.history_max)) {
        switch (needed_controls(c, true)) {
            case 0: f = launch_loss<T, 256, 0>; break;
            case 1: f = launch_loss<T, 256, 1>; break;
            case 2: f = launch_loss<T, 256, 2>; break;
            default: f = launch_loss<T, 256, 3>;
        }
    }
    return f(logits, ld, c, d, ldd, rows, actions, L, st);
}

}  // namespace
}  // namespace mg

using namespace mg;

#define MG_BY_TYPE(dtype, call)                                                \
    ((dtype) == MG_DTYPE_F32 ? call<float> : (dtype) == MG_DTYPE_BF16 ? call<__nv_bfloat16> : call<__half>)

extern "C" {

int mg_logits_control(const void* logits, int dtype, int64_t ld, const mg_logit_controls* controls, void* out, int64_t ldo,
                      int rows, int actions, mg_stream_t stream) {
    mg_logit_controls c;
    MG_TRY(check_common("logits_control", logits, dtype, ld, controls, rows, actions, actions, &c));
    MG_CHECK_ARG(out && aligned(out, type_size(dtype)), "logits_control: null or misaligned out");
    MG_CHECK_ARG(ldo >= actions, "logits_control: ldo smaller than the row");
    MG_CHECK_ARG(out != logits || ldo == ld, "logits_control: in place needs ldo = ld");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == MG_DTYPE_F32)
        return control<float, false>(logits, ld, c, nullptr, 0, out, ldo, rows, actions, st);
    if (dtype == MG_DTYPE_BF16)
        return control<__nv_bfloat16, false>(logits, ld, c, nullptr, 0, out, ldo, rows, actions, st);
    return control<__half, false>(logits, ld, c, nullptr, 0, out, ldo, rows, actions, st);
}

int mg_logits_control_backward(const void* logits, int dtype, int64_t ld, const mg_logit_controls* controls,
                               const void* d_out, int64_t ldg, void* d_logits, int64_t ldd, int rows, int actions,
                               mg_stream_t stream) {
    mg_logit_controls c;
    MG_TRY(check_common("logits_control_backward", logits, dtype, ld, controls, rows, actions, actions, &c));
    const int size = type_size(dtype);
    MG_CHECK_ARG(d_out && d_logits && aligned(d_out, size) && aligned(d_logits, size),
                 "logits_control_backward: null or misaligned gradient");
    MG_CHECK_ARG(ldg >= actions && ldd >= actions, "logits_control_backward: ldg or ldd smaller than the row");
    MG_CHECK_ARG(d_out != d_logits || ldg == ldd, "logits_control_backward: in place needs ldd = ldg");
    MG_CHECK_ARG(d_logits != logits || ldd == ld, "logits_control_backward: in place needs ldd = ld");
    // only the repetition penalty and the mask reach the gradient
    c.bias = nullptr;
    if (!c.repetition) leave_out_history(&c);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == MG_DTYPE_F32)
        return control<float, true>(logits, ld, c, d_out, ldg, d_logits, ldd, rows, actions, st);
    if (dtype == MG_DTYPE_BF16)
        return control<__nv_bfloat16, true>(logits, ld, c, d_out, ldg, d_logits, ldd, rows, actions, st);
    return control<__half, true>(logits, ld, c, d_out, ldg, d_logits, ldd, rows, actions, st);
}

int mg_logits_sample(const void* logits, int dtype, int64_t ld, const mg_logit_controls* controls, uint32_t* rng,
                     int32_t* action, float* log_prob, float* entropy, float* value, int rows, int actions,
                     mg_stream_t stream) {
    mg_logit_controls c;
    MG_TRY(check_common("logits_sample", logits, dtype, ld, controls, rows, actions, actions + (value ? 1 : 0), &c));
    MG_CHECK_ARG(action && log_prob, "logits_sample: null action or log_prob");
    MG_CHECK_ARG(aligned(rng, 4) && aligned(action, 4) && aligned(log_prob, 4) && aligned(entropy, 4) && aligned(value, 4),
                 "logits_sample: a buffer is not aligned to its type");
    return MG_BY_TYPE(dtype, sample)(logits, ld, c, rng, action, log_prob, entropy, value, rows, actions,
                                            reinterpret_cast<cudaStream_t>(stream));
}

int mg_logits_policy_loss(const void* logits, int dtype, int64_t ld, const mg_logit_controls* controls,
                          const int32_t* action, const float* adv, const float* adv_stats, const float* ret,
                          const float* old_log_prob, void* d_logits, int64_t ldd, float* stats, int rows, int actions,
                          float clip, float value_coef, float entropy_coef, float grad_scale, mg_stream_t stream) {
    mg_logit_controls c;
    const int columns = actions + (ret ? 1 : 0);
    MG_TRY(check_common("logits_policy_loss", logits, dtype, ld, controls, rows, actions, columns, &c));
    MG_CHECK_ARG(action && adv && old_log_prob && stats, "logits_policy_loss: null argument");
    MG_CHECK_ARG(aligned(action, 4) && aligned(adv, 4) && aligned(adv_stats, 4) && aligned(ret, 4) && aligned(old_log_prob, 4) &&
                     aligned(stats, 4),
                 "logits_policy_loss: a buffer is not aligned to its type");
    MG_CHECK_ARG(d_logits && aligned(d_logits, type_size(dtype)), "logits_policy_loss: null or misaligned d_logits");
    MG_CHECK_ARG(ldd >= columns, "logits_policy_loss: ldd smaller than the row");
    MG_CHECK_ARG(d_logits != logits || ldd == ld, "logits_policy_loss: in place needs ldd = ld");
    MG_CHECK_ARG(clip >= 0.0f, "logits_policy_loss: negative clip");
    LossArgs L{action, adv, adv_stats, ret, old_log_prob, stats, clip, value_coef, entropy_coef, grad_scale, status_ptr()};
    return MG_BY_TYPE(dtype, loss)(logits, ld, c, d_logits, ldd, rows, actions, L,
                                          reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
