// Orthogonalised updates: Newton-Schulz steps on the tensor cores and the Muon
// optimiser step around them.
//
//   X0 = U / |U|_F;  G = X X^T (rows <= cols) or X^T X;  B = b G + c G^2;
//   X <- a X + B X (or X B),  (a, b, c) = (3.4445, -4.7750, 2.0315).
//
// Number formats: the operands of the products are fp16 (11 significant
// bits), scaled by 2^10 so that entries from 2^-24 of |U| up are normal
// numbers and the largest (|X|, |G| <= 1.5, |B| <= 12) stay below 2^14. X
// itself is carried in fp32 beside its fp16 copy: with a X taken from the
// 16-bit copy, its rounding would be multiplied by a = 3.4 in every step in
// the directions that U hardly has (4 % of the result's norm off after five
// steps at rank 8 of 128, against 0.06 % this way); bf16 operands would be
// 1.4 % off on full-rank matrices, against 0.2 %.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "logits.cuh"
#include "muon.cuh"
#include "runtime.h"
#include "metalgym/pdl.cuh"

namespace mg {
namespace {

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;

// ------------------------------------------------------------------ U and its norm

// What turns the inputs into U: a copy (orthogonalise) or the momentum.
struct MuonInput {
    const void* x;  // orthogonalise: [batch][rows][ld]
    int64_t ld, stride;
    const float* grad;  // muon: dense rows
    float* momentum;
    const float* normPartial;
    int nNorm;
    float maxGradNorm, decay;
    int nesterov;
    float* normSqOut;
};

struct MuonShape {
    int rows, cols, ldx;  // ldx: row stride of X in the workspace
};

constexpr int kPrepThreads = 256;
constexpr int kPrepParts = 64;  // CTAs (and norm partials) per matrix

// U into X32 (not yet divided by its norm) and one 64-bit sum of squares a CTA:
// the squares of any finite fp32 U neither overflow nor vanish in 64 bits.
template <class T, bool MUON>
__global__ void __launch_bounds__(kPrepThreads)
    k_muon_prepare(const MuonInput in, MuonShape s, float* x32, double* partial) {
    mg_pdl_trigger();
    mg_pdl_wait();
    __shared__ float sScale;
    __shared__ double sSum[kPrepThreads / 32];
    const int b = blockIdx.y;
    if (MUON) {
        if (threadIdx.x < 32) {  // the clip factor, as the Adam step forms it
            float sum = 0.0f;
            for (int i = threadIdx.x; i < in.nNorm; i += 32) sum = __fadd_rn(sum, in.normPartial[i]);
            sum = warp_sum(sum);
            if (threadIdx.x == 0) {
                const float norm = __fsqrt_rn(sum);
                sScale = (in.maxGradNorm > 0.0f && norm > in.maxGradNorm)
                             ? __fdiv_rn(in.maxGradNorm, __fadd_rn(norm, 1e-6f))
                             : 1.0f;
                if (blockIdx.x == 0 && b == 0 && in.normSqOut) *in.normSqOut = sum;
            }
        }
        __syncthreads();
    }
    double sum = 0.0;
    for (int r = blockIdx.x; r < s.rows; r += gridDim.x) {
        float* dst = x32 + ((int64_t)b * s.rows + r) * s.ldx;
        for (int c = threadIdx.x; c < s.cols; c += kPrepThreads) {
            float u;
            if (MUON) {
                const int64_t i = (int64_t)b * in.stride + (int64_t)r * s.cols + c;
                const float g = __fmul_rn(in.grad[i], sScale);
                const float m = __fadd_rn(__fmul_rn(in.decay, in.momentum[i]), g);
                in.momentum[i] = m;
                u = in.nesterov ? __fadd_rn(g, __fmul_rn(in.decay, m)) : m;
            } else {
                u = to_f32(static_cast<const T*>(in.x)[(int64_t)b * in.stride + (int64_t)r * in.ld + c]);
            }
            dst[c] = u;
            sum += (double)u * (double)u;
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if ((threadIdx.x & 31) == 0) sSum[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kPrepThreads / 32; w++) sum += sSum[w];
        partial[(int64_t)b * kPrepParts + blockIdx.x] = sum;
    }
}

// X = U / |U| (0 for a zero U), and its fp16 copy.
__global__ void __launch_bounds__(kPrepThreads)
    k_muon_normalise(MuonShape s, float* x32, __half* x16, const double* partial, int parts) {
    mg_pdl_trigger();
    mg_pdl_wait();
    __shared__ double sInv;
    const int b = blockIdx.y;
    if (threadIdx.x == 0) {
        double sum = 0.0;
        for (int i = 0; i < parts; i++) sum += partial[(int64_t)b * kPrepParts + i];
        sInv = sum == 0.0 ? 0.0 : 1.0 / sqrt(sum);
    }
    __syncthreads();
    for (int r = blockIdx.x; r < s.rows; r += gridDim.x) {
        const int64_t at = ((int64_t)b * s.rows + r) * s.ldx;
        for (int c = threadIdx.x; c < s.cols; c += kPrepThreads) {
            const float v = (float)((double)x32[at + c] * sInv);
            x32[at + c] = v;
            x16[at + c] = __float2half_rn(v * kNsScale);
        }
    }
}

template <int KIND, bool A_MN, bool B_MN>
int launch_product(const CUtensorMap& ta, const CUtensorMap& tb, const NsProduct& p, int batch, cudaStream_t st) {
    auto kern = k_ns_product<KIND, A_MN, B_MN>;
    static std::atomic<uint64_t> done{0};
    MG_TRY(smem_limit_once(kern, NsTile::SMEM_BYTES, done));
    const int tm = (p.M + NsTile::BM - 1) / NsTile::BM, tn = (p.N + NsTile::BN - 1) / NsTile::BN;
    MG_CUDA_TRY(MG_LAUNCH(kern, dim3(tn, tm, batch), 128, NsTile::SMEM_BYTES, st, ta, tb, p));
    return check_launch("k_ns_product");
}

struct Workspace {
    double* partial;
    float* x32;
    __half* x16[2];
    __half *g16, *b16;
    size_t bytes;
};

int round8(int n) { return (n + 7) / 8 * 8; }

Workspace layout(int batch, int rows, int cols, void* base) {
    Workspace w;
    size_t at = 0;
    char* p = static_cast<char*>(base);
    auto take = [&](size_t bytes) {
        void* q = p ? p + at : nullptr;
        at += (bytes + 255) / 256 * 256;
        return q;
    };
    const size_t s = std::min(rows, cols), x = (size_t)batch * rows * round8(cols), g = (size_t)batch * s * round8((int)s);
    w.partial = static_cast<double*>(take((size_t)batch * kPrepParts * 8));
    w.x32 = static_cast<float*>(take(x * 4));
    w.x16[0] = static_cast<__half*>(take(x * 2));
    w.x16[1] = static_cast<__half*>(take(x * 2));
    w.g16 = static_cast<__half*>(take(g * 2));
    w.b16 = static_cast<__half*>(take(g * 2));
    w.bytes = at;
    return w;
}

constexpr int kMaxSide = 1 << 16;

int check_shape(const char* name, int batch, int rows, int cols) {
    const std::string n(name);
    MG_CHECK_ARG(batch > 0 && rows > 0 && cols > 0, n + ": batch, rows and cols must be positive");
    MG_CHECK_ARG(batch <= 65535 && rows <= kMaxSide && cols <= kMaxSide,
                 n + ": at most 65535 matrices of at most 65536 rows and columns");
    return MG_OK;
}

int check_workspace(const char* name, int batch, int rows, int cols, int steps, void* workspace, size_t bytes) {
    const std::string n(name);
    MG_CHECK_ARG(steps >= 1 && steps <= 16, n + ": steps must be in 1..16");
    MG_CHECK_ARG(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, n + ": null or misaligned workspace");
    const size_t need = layout(batch, rows, cols, nullptr).bytes;
    MG_CHECK_ARG(bytes >= need, n + ": the workspace has " + std::to_string(bytes) + " bytes, mg_muon_workspace gives " +
                                    std::to_string(need));
    return MG_OK;
}

// The Newton-Schulz steps on what k_muon_prepare left; the last product's
// epilogue writes `fin`.
int newton_schulz(const Workspace& w, int batch, int rows, int cols, int steps, int parts, const NsFinal& fin, cudaStream_t st) {
    const MuonShape shape{rows, cols, round8(cols)};
    MG_CUDA_TRY(MG_LAUNCH(k_muon_normalise, dim3(std::min(rows, 512), batch), kPrepThreads, 0, st, shape, w.x32, w.x16[0],
                          w.partial, parts));
    MG_TRY(check_launch("k_muon_normalise"));
    const bool wide = rows <= cols;  // G = X X^T, else X^T X
    const int s = std::min(rows, cols), l = std::max(rows, cols), lds = round8(s);
    CUtensorMap mx[2], mg16, mb16;
    for (int i = 0; i < 2; i++) MG_TRY(make_tmap_f16_3d(&mx[i], w.x16[i], cols, rows, batch, shape.ldx, NsTile::BM));
    CUtensorMap mxk[2];  // boxes of 64 rows, for X as an operand whose K index is the row
    for (int i = 0; i < 2; i++) MG_TRY(make_tmap_f16_3d(&mxk[i], w.x16[i], cols, rows, batch, shape.ldx, 64));
    MG_TRY(make_tmap_f16_3d(&mg16, w.g16, s, s, batch, lds, NsTile::BM));
    MG_TRY(make_tmap_f16_3d(&mb16, w.b16, s, s, batch, lds, NsTile::BM));
    NsProduct p{};
    p.status = status_ptr();
    for (int i = 0; i < steps; i++) {
        const int cur = i & 1;
        p.M = p.N = s;
        p.K = l;
        p.ldo = lds;
        p.out16 = w.g16;
        p.a = 0.0f;
        MG_TRY(wide ? (launch_product<kNsGram, false, false>(mx[cur], mx[cur], p, batch, st))
                    : (launch_product<kNsGram, true, true>(mxk[cur], mxk[cur], p, batch, st)));
        p.K = s;
        p.out16 = w.b16;
        p.g16 = w.g16;
        p.b = kNsB;
        p.c = kNsC;
        MG_TRY((launch_product<kNsPoly, false, false>(mg16, mg16, p, batch, st)));
        p.M = rows;
        p.N = cols;
        p.K = s;
        p.ldo = shape.ldx;
        p.x32 = w.x32;
        p.out16 = w.x16[cur ^ 1];
        p.a = kNsA;
        p.last = i + 1 == steps;
        if (p.last) p.fin = fin;
        MG_TRY(wide ? (launch_product<kNsApply, false, true>(mb16, mxk[cur], p, batch, st))
                    : (launch_product<kNsApply, false, false>(mx[cur], mb16, p, batch, st)));
    }
    return MG_OK;
}

template <class T, bool MUON>
int prepare(const MuonInput& in, const Workspace& w, int batch, int rows, int cols, int* parts, cudaStream_t st) {
    const MuonShape shape{rows, cols, round8(cols)};
    *parts = std::min(rows, kPrepParts);
    MG_CUDA_TRY(MG_LAUNCH((k_muon_prepare<T, MUON>), dim3(*parts, batch), kPrepThreads, 0, st, in, shape, w.x32, w.partial));
    return check_launch("k_muon_prepare");
}

bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % (unsigned)bytes) == 0; }

}  // namespace
}  // namespace mg

using namespace mg;

extern "C" {

int mg_muon_workspace(int batch, int rows, int cols, size_t* bytes) {
    MG_CHECK_ARG(bytes, "muon_workspace: null output");
    MG_TRY(check_shape("muon_workspace", batch, rows, cols));
    *bytes = layout(batch, rows, cols, nullptr).bytes;
    return MG_OK;
}

int mg_orthogonalize(const void* x, int dtype, int64_t ld, int64_t batch_stride, void* out, int out_dtype, int64_t ldo,
                     int64_t out_stride, int batch, int rows, int cols, int steps, void* workspace,
                     size_t workspace_bytes, mg_stream_t stream) {
    MG_CHECK_ARG(x && out, "orthogonalize: null argument");
    MG_TRY(check_shape("orthogonalize", batch, rows, cols));
    MG_CHECK_ARG(dtype == MG_DTYPE_F32 || dtype == MG_DTYPE_BF16 || dtype == MG_DTYPE_F16, "orthogonalize: unknown dtype");
    MG_CHECK_ARG(out_dtype == MG_DTYPE_BF16 || out_dtype == MG_DTYPE_F16, "orthogonalize: out_dtype must be bf16 or f16");
    MG_CHECK_ARG(aligned_to(x, dtype == MG_DTYPE_F32 ? 4 : 2) && aligned_to(out, 2),
                 "orthogonalize: a matrix is not aligned to its type");
    MG_CHECK_ARG(ld >= cols && ldo >= cols, "orthogonalize: ld or ldo smaller than the row");
    MG_CHECK_ARG(batch == 1 || (batch_stride >= (int64_t)(rows - 1) * ld + cols && out_stride >= (int64_t)(rows - 1) * ldo + cols),
                 "orthogonalize: the matrices of the batch overlap");
    MG_TRY(check_workspace("orthogonalize", batch, rows, cols, steps, workspace, workspace_bytes));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const Workspace w = layout(batch, rows, cols, workspace);
    MuonInput in{};
    in.x = x;
    in.ld = ld;
    in.stride = batch_stride;
    int parts = 0;
    if (dtype == MG_DTYPE_F32)
        MG_TRY((prepare<float, false>(in, w, batch, rows, cols, &parts, st)));
    else if (dtype == MG_DTYPE_BF16)
        MG_TRY((prepare<__nv_bfloat16, false>(in, w, batch, rows, cols, &parts, st)));
    else
        MG_TRY((prepare<__half, false>(in, w, batch, rows, cols, &parts, st)));
    NsFinal fin{};
    fin.out = out;
    fin.outBf16 = out_dtype == MG_DTYPE_BF16;
    fin.ld = ldo;
    fin.stride = out_stride;
    return newton_schulz(w, batch, rows, cols, steps, parts, fin, st);
}

int mg_muon_step(float* master, const float* grad, float* momentum, void* weights, int64_t batch_stride, int batch,
                 int rows, int cols, const float* norm_partial, int n_norm_partials, float max_grad_norm, float lr,
                 float scale, float momentum_decay, int nesterov, float weight_decay, int steps, float* norm_sq_out,
                 void* workspace, size_t workspace_bytes, mg_stream_t stream) {
    MG_CHECK_ARG(master && grad && momentum && weights, "muon_step: null argument");
    MG_TRY(check_shape("muon_step", batch, rows, cols));
    MG_CHECK_ARG(aligned_to(master, 4) && aligned_to(grad, 4) && aligned_to(momentum, 4) && aligned_to(weights, 2),
                 "muon_step: a matrix is not aligned to its type");
    MG_CHECK_ARG(batch == 1 || batch_stride >= (int64_t)rows * cols, "muon_step: the matrices of the batch overlap");
    MG_CHECK_ARG(n_norm_partials >= 0 && (norm_partial || n_norm_partials == 0), "muon_step: null norm_partial");
    MG_CHECK_ARG(n_norm_partials > 0 || (!(max_grad_norm > 0.0f) && !norm_sq_out),
                 "muon_step: clipping and norm_sq_out need norm partials");
    MG_CHECK_ARG(std::isfinite(lr) && std::isfinite(scale) && std::isfinite(weight_decay) && std::isfinite(momentum_decay),
                 "muon_step: lr, scale, weight_decay and momentum_decay must be finite");
    MG_TRY(check_workspace("muon_step", batch, rows, cols, steps, workspace, workspace_bytes));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const Workspace w = layout(batch, rows, cols, workspace);
    MuonInput in{};
    in.grad = grad;
    in.momentum = momentum;
    in.stride = batch_stride;
    in.normPartial = norm_partial;
    in.nNorm = n_norm_partials;
    in.maxGradNorm = max_grad_norm;
    in.decay = momentum_decay;
    in.nesterov = nesterov;
    in.normSqOut = norm_sq_out;
    int parts = 0;
    MG_TRY((prepare<float, true>(in, w, batch, rows, cols, &parts, st)));
    NsFinal fin{};
    fin.master = master;
    fin.weights = static_cast<__nv_bfloat16*>(weights);
    fin.ld = cols;
    fin.stride = batch_stride;
    fin.keep = 1.0f - lr * weight_decay;
    fin.rate = lr * scale;
    return newton_schulz(w, batch, rows, cols, steps, parts, fin, st);
}

}  // extern "C"
