// Controlled logits: penalties, biases and action masks (logits.cuh) written
// out, differentiated, drawn from, and under the clipped PPO loss.
#include <math.h>

#include <atomic>
#include <string>

#include "logits.cuh"
#include "runtime.h"
#include "metalgym/detail/ptx.cuh"
#include "metalgym/pdl.cuh"
#include "metalgym/rng.h"
#include "metalgym/rowmap.h"

namespace mg {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// The controlled logit of action a (raw x); the table covers actions from lo.
__device__ __forceinline__ float controlled(const RowControls& r, const HistoryTable& t, float x, int a, int lo) {
    if (r.history) {
        const int n = t.count(a - lo);
        if (n > 0) x = penalise(r, x, n);
    }
    if (r.bias) x = __fadd_rn(x, r.bias[a]);
    return allowed(r, a) ? x : -INFINITY;
}

// ------------------------------------------------------------------ control and its gradient

// One CTA per chunk of `span` actions of a row: in dimension x, row-major.
template <class T, bool BACKWARD>
__global__ void __launch_bounds__(kThreads)
    k_logits_control(const T* logits, int64_t ld, const mg_logit_controls c, const T* dOut, int64_t ldg, T* out,
                     int64_t ldo, int actions, int span, int chunks) {
    mg_pdl_trigger();
    mg_pdl_wait();
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t sums[kWarps];
    const int row = blockIdx.x / chunks, lo = (blockIdx.x % chunks) * span, hi = min(actions, lo + span);
    const RowControls r = row_controls(c, row);
    HistoryTable t;
    t.place(smem, span, c.history_max);
    if (r.history)
        history_fill(t, c.history + (int64_t)row * c.history_stride, row_history_len(c, row), lo, hi, c.history_max, sums);
    const T* x = logits + (int64_t)row * ld;
    T* y = out + (int64_t)row * ldo;
    for (int a = lo + threadIdx.x; a < hi; a += kThreads) {
        if (!BACKWARD) {
            from_f32(&y[a], controlled(r, t, to_f32(x[a]), a, lo));
        } else {
            float g = to_f32(dOut[(int64_t)row * ldg + a]);
            if (r.history && t.count(a - lo) > 0)
                g = to_f32(x[a]) > 0.0f ? __fdiv_rn(g, r.repetition) : __fmul_rn(g, r.repetition);
            from_f32(&y[a], allowed(r, a) ? g : 0.0f);
        }
    }
}

// ------------------------------------------------------------------ softmax statistics and the race

// Running softmax statistics: the maximum m, s = sum e^(l - m), t = sum
// e^(l - m) (l - m); entropy = log s - t / s.
struct Softmax {
    float m = -INFINITY, s = 0.0f, t = 0.0f;
    __device__ __forceinline__ void add(float l) {
        if (l == -INFINITY) return;
        if (l > m) {
            if (m > -INFINITY) {
                const float d = m - l, e = expf(d);
                t = e * (t + s * d);
                s = s * e;
            }
            m = l;
            s += 1.0f;
        } else {
            const float d = l - m, e = expf(d);  // NaN when l is
            s += e;
            if (!(e == 0.0f)) t += e * d;
        }
    }
    __device__ __forceinline__ void merge(const Softmax& o) {
        if (o.m == -INFINITY && o.s == 0.0f) return;
        if (m == -INFINITY && s == 0.0f) {
            *this = o;
            return;
        }
        const float top = fmaxf(m, o.m);
        const float da = m - top, db = o.m - top, ea = expf(da), eb = expf(db);
        const float ta = ea == 0.0f ? 0.0f : ea * (t + s * da), tb = eb == 0.0f ? 0.0f : eb * (o.t + o.s * db);
        s = s * ea + o.s * eb;
        t = ta + tb;
        m = top;
    }
};

// The best key of a race and its action; equal keys: the lower action.
struct Best {
    double key = -INFINITY;
    int action = -1;
    float logit = -INFINITY;
    __device__ __forceinline__ void offer(double k, int a, float l) {
        if (k > key || (k == key && a < action)) {
            key = k;
            action = a;
            logit = l;
        }
    }
};

__device__ __forceinline__ double race_time(uint32_t word, int a) {
    const uint32_t h = mg_mix32(word + (uint32_t)a * 0x9E3779B9u);
    return -log1p(-((double)h + 0.5) * (1.0 / 4294967296.0));
}

template <class V>
__device__ __forceinline__ V warp_xor(V v, int d) {
    return __shfl_xor_sync(0xffffffffu, v, d);
}
__device__ __forceinline__ Softmax shuffle(const Softmax& a, int d) {
    Softmax o;
    o.m = warp_xor(a.m, d);
    o.s = warp_xor(a.s, d);
    o.t = warp_xor(a.t, d);
    return o;
}

// The CTA's statistics in every thread, merged in one fixed order.
__device__ inline Softmax block_softmax(Softmax v, Softmax* slot) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v.merge(shuffle(v, d));
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    Softmax all = slot[0];
    for (int w = 1; w < kWarps; w++) all.merge(slot[w]);
    return all;
}

// ------------------------------------------------------------------ draw

// One CTA per row.
template <class T>
__global__ void __launch_bounds__(kThreads)
    k_logits_sample(const T* logits, int64_t ld, const mg_logit_controls c, uint32_t* rng, int32_t* action,
                    float* logProb, float* entropy, float* value, int actions) {
    mg_pdl_trigger();
    mg_pdl_wait();
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t sums[kWarps];
    __shared__ Softmax stats[kWarps];
    __shared__ Best best[kWarps];
    const int row = blockIdx.x;
    const RowControls r = row_controls(c, row);
    HistoryTable t;
    t.place(smem, actions, c.history_max);
    if (r.history)
        history_fill(t, c.history + (int64_t)row * c.history_stride, row_history_len(c, row), 0, actions, c.history_max, sums);
    const T* x = logits + (int64_t)row * ld;
    uint32_t word = rng ? rng[row] : 0u;
    if (rng) rngNext(word);
    Softmax v;
    Best b;
    for (int a = threadIdx.x; a < actions; a += kThreads) {
        const float l = controlled(r, t, to_f32(x[a]), a, 0);
        v.add(l);
        if (l > -INFINITY) b.offer(rng ? (double)l - log(race_time(word, a)) : (double)l, a, l);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        const double k = warp_xor(b.key, d);
        const int a = warp_xor(b.action, d);
        const float l = warp_xor(b.logit, d);
        if (a >= 0) b.offer(k, a, l);
    }
    if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = b;
    const Softmax all = block_softmax(v, stats);
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWarps; w++)
            if (best[w].action >= 0) b.offer(best[w].key, best[w].action, best[w].logit);
        const float ls = logf(all.s);
        const bool some = b.action >= 0 || all.s != all.s;
        action[row] = b.action;
        logProb[row] = some ? (b.logit - all.m) - ls : 0.0f;
        if (entropy) entropy[row] = some ? ls - all.t / all.s : 0.0f;
        if (value) value[row] = to_f32(x[actions]);
        if (rng) rng[row] = word;
    }
}

// ------------------------------------------------------------------ loss

struct LossArgs {
    const int32_t* action;
    const float *adv, *advStats, *ret, *oldLogProb;
    float* stats;
    float clip, valueCoef, entropyCoef, scale;
    int* status;
};

// One CTA per row: the row's statistics, then its gradient.
template <class T>
__global__ void __launch_bounds__(kThreads)
    k_logits_loss(const T* logits, int64_t ld, const mg_logit_controls c, T* dLogits, int64_t ldd, int actions,
                  const LossArgs L) {
    mg_pdl_trigger();
    mg_pdl_wait();
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t sums[kWarps];
    __shared__ Softmax slot[kWarps];
    const int row = blockIdx.x;
    const RowControls r = row_controls(c, row);
    HistoryTable t;
    t.place(smem, actions, c.history_max);
    const T* x = logits + (int64_t)row * ld;
    T* d = dLogits + (int64_t)row * ldd;
    const int act = L.action[row];
    const bool inside = act >= 0 && act < actions;
    if (!inside || !allowed(r, act)) {
        if (threadIdx.x == 0 && !inside && act != -1) record_error(L.status, kDevBadAction);
        for (int a = threadIdx.x; a < actions + (L.ret ? 1 : 0); a += kThreads) from_f32(&d[a], 0.0f);
        if (threadIdx.x < 5) L.stats[(int64_t)row * 5 + threadIdx.x] = 0.0f;
        return;
    }
    if (r.history)
        history_fill(t, c.history + (int64_t)row * c.history_stride, row_history_len(c, row), 0, actions, c.history_max, sums);
    const float valueX = L.ret ? to_f32(x[actions]) : 0.0f;
    const float lAct = controlled(r, t, to_f32(x[act]), act, 0);
    Softmax v;
    for (int a = threadIdx.x; a < actions; a += kThreads) v.add(controlled(r, t, to_f32(x[a]), a, 0));
    const Softmax all = block_softmax(v, slot);
    const float ls = logf(all.s), entropy = ls - all.t / all.s;
    const float logp = (lAct - all.m) - ls, old = L.oldLogProb[row];
    const float ratio = expf(logp - old);
    const float adv = L.advStats ? (L.adv[row] - L.advStats[0]) * L.advStats[1] : L.adv[row];
    const float one = ratio * adv, two = fminf(fmaxf(ratio, 1.0f - L.clip), 1.0f + L.clip) * adv;
    const float slope = one <= two ? -adv * ratio : 0.0f;
    // every thread has read the action's logit (the gradient may replace it)
    __syncthreads();
    for (int a = threadIdx.x; a < actions; a += kThreads) {
        const float raw = to_f32(x[a]);
        const float l = controlled(r, t, raw, a, 0);
        const float lp = (l - all.m) - ls, p = expf(lp);
        float g = slope * ((a == act ? 1.0f : 0.0f) - p);
        if (p > 0.0f) g += L.entropyCoef * p * (lp + entropy);
        g *= L.scale;
        if (r.history && t.count(a) > 0) g = raw > 0.0f ? __fdiv_rn(g, r.repetition) : g * r.repetition;
        from_f32(&d[a], allowed(r, a) ? g : 0.0f);
    }
    if (threadIdx.x == 0) {
        float* st = L.stats + (int64_t)row * 5;
        float vLoss = 0.0f;
        if (L.ret) {
            const float err = valueX - L.ret[row];
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
    if (!c.repetition && !c.frequency && !c.presence) out->history = nullptr;
    if (!out->history) {
        out->history_len = nullptr;
        out->history_max = 0;
    }
    return MG_OK;
}

constexpr int kChunk = 8192;  // actions of a CTA of the control kernels

template <class T, bool BACKWARD>
int launch_control(const void* logits, int64_t ld, const mg_logit_controls& c, const void* dOut, int64_t ldg, void* out,
                   int64_t ldo, int rows, int actions, cudaStream_t st) {
    const int span = actions < kChunk ? actions : kChunk, chunks = (actions + span - 1) / span;
    MG_CHECK_ARG((int64_t)rows * chunks <= INT32_MAX, "logits_control: too many rows");
    auto kern = k_logits_control<T, BACKWARD>;
    static std::atomic<uint64_t> done{0};
    const size_t smem = c.history ? HistoryTable::bytes(span, c.history_max) : 0;
    MG_TRY(smem_limit_once(kern, 100 * 1024, done));
    MG_CUDA_TRY(MG_LAUNCH(kern, (unsigned)(rows * chunks), kThreads, smem, st, static_cast<const T*>(logits), ld, c,
                          static_cast<const T*>(dOut), ldg, static_cast<T*>(out), ldo, actions, span, chunks));
    return check_launch("k_logits_control");
}

template <class T>
int launch_sample(const void* logits, int64_t ld, const mg_logit_controls& c, uint32_t* rng, int32_t* action, float* logProb,
                  float* entropy, float* value, int rows, int actions, cudaStream_t st) {
    auto kern = k_logits_sample<T>;
    static std::atomic<uint64_t> done{0};
    const size_t smem = c.history ? HistoryTable::bytes(actions, c.history_max) : 0;
    MG_TRY(smem_limit_once(kern, 100 * 1024, done));
    MG_CUDA_TRY(MG_LAUNCH(kern, rows, kThreads, smem, st, static_cast<const T*>(logits), ld, c, rng, action, logProb, entropy,
                          value, actions));
    return check_launch("k_logits_sample");
}

template <class T>
int launch_loss(const void* logits, int64_t ld, const mg_logit_controls& c, void* d, int64_t ldd, int rows, int actions,
                const LossArgs& L, cudaStream_t st) {
    auto kern = k_logits_loss<T>;
    static std::atomic<uint64_t> done{0};
    const size_t smem = c.history ? HistoryTable::bytes(actions, c.history_max) : 0;
    MG_TRY(smem_limit_once(kern, 100 * 1024, done));
    MG_CUDA_TRY(MG_LAUNCH(kern, rows, kThreads, smem, st, static_cast<const T*>(logits), ld, c, static_cast<T*>(d), ldd,
                          actions, L));
    return check_launch("k_logits_loss");
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
        return launch_control<float, false>(logits, ld, c, nullptr, 0, out, ldo, rows, actions, st);
    if (dtype == MG_DTYPE_BF16)
        return launch_control<__nv_bfloat16, false>(logits, ld, c, nullptr, 0, out, ldo, rows, actions, st);
    return launch_control<__half, false>(logits, ld, c, nullptr, 0, out, ldo, rows, actions, st);
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
    if (!c.repetition) c.history = nullptr;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == MG_DTYPE_F32)
        return launch_control<float, true>(logits, ld, c, d_out, ldg, d_logits, ldd, rows, actions, st);
    if (dtype == MG_DTYPE_BF16)
        return launch_control<__nv_bfloat16, true>(logits, ld, c, d_out, ldg, d_logits, ldd, rows, actions, st);
    return launch_control<__half, true>(logits, ld, c, d_out, ldg, d_logits, ldd, rows, actions, st);
}

int mg_logits_sample(const void* logits, int dtype, int64_t ld, const mg_logit_controls* controls, uint32_t* rng,
                     int32_t* action, float* log_prob, float* entropy, float* value, int rows, int actions,
                     mg_stream_t stream) {
    mg_logit_controls c;
    MG_TRY(check_common("logits_sample", logits, dtype, ld, controls, rows, actions, actions + (value ? 1 : 0), &c));
    MG_CHECK_ARG(action && log_prob, "logits_sample: null action or log_prob");
    return MG_BY_TYPE(dtype, launch_sample)(logits, ld, c, rng, action, log_prob, entropy, value, rows, actions,
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
    MG_CHECK_ARG(d_logits && aligned(d_logits, type_size(dtype)), "logits_policy_loss: null or misaligned d_logits");
    MG_CHECK_ARG(ldd >= columns, "logits_policy_loss: ldd smaller than the row");
    MG_CHECK_ARG(d_logits != logits || ldd == ld, "logits_policy_loss: in place needs ldd = ld");
    MG_CHECK_ARG(clip >= 0.0f, "logits_policy_loss: negative clip");
    LossArgs L{action, adv, adv_stats, ret, old_log_prob, stats, clip, value_coef, entropy_coef, grad_scale, status_ptr()};
    return MG_BY_TYPE(dtype, launch_loss)(logits, ld, c, d_logits, ldd, rows, actions, L,
                                          reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
