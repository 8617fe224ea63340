// Orthogonalised updates: Newton-Schulz steps on the tensor cores and the Muon
// optimiser step around them.
//
//   X0 = U / |U|_F;  G = X X^T (rows <= cols) or X^T X;  B = b G + c G^2;
//   X <- a X + B X (or X B),  (a, b, c) = (3.4445, -4.7750, 2.0315),
//
// the quintic iteration and optimiser that K. Jordan et al. published ("Muon: An
// optimizer for hidden layers in neural networks", 2024).
//
// Number formats: the operands of the products are sums of two fp16 numbers
// (22 significant bits), scaled by 2^10 so that entries from 2^-24 of |U| up
// are normal numbers and the largest (|X|, |G| <= 1.5, |B| <= 12) stay below
// 2^14. X itself is carried in fp32 beside its two parts, since a X multiplies
// its rounding by a = 3.4 in every step in the directions that U hardly has.
// Measured against the exact iteration, of the result's norm: 2e-6 to 5e-5 (129
// x 1000 .. 4096 x 4096; full rank, rank 1/16 over a floor of 1e-3, rows from 1
// to 1e-4), as fp32 products by a library are (1e-6 to 2e-5); products of one
// fp16 number were 5e-4 to 2e-3 off, in less than half the time at 4096 x 4096
// (1510 us; 3230 this way, 3780 once the power cap holds), 0.85 of it at 333 x
// 1001 (117 / 138).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "logits.cuh"
#include "muon.cuh"
#include "muon_small.cuh"
#include "runtime.h"
#include "metalgym/pdl.cuh"

namespace mg {
namespace {

struct MuonShape {
    int rows, cols, ldx;  // ldx: row stride of X in the workspace
};

constexpr int kPrepThreads = 256;
constexpr int kPrepWarps = kPrepThreads / 32;
constexpr int kPrepMaxParts = 1024;  // CTAs (and norm partials) per matrix at most

// U into X32 (not yet divided by its norm) and one 64-bit sum of squares a CTA,
// in which the squares of any finite fp32 U neither overflow nor vanish. A
// thread takes V columns of a row at a time.
template <class T, bool MUON, int V>
__global__ void __launch_bounds__(kPrepThreads)
    k_muon_prepare(const MuonInput in, MuonShape s, float* x32, double* partial) {
    mg_pdl_trigger();
    mg_pdl_wait();
    __shared__ float sScale;
    __shared__ double sSum[kPrepWarps];
    const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (MUON) {
        if (warp == 0) {
            float normSq;
            const float f = muon_clip(in, &normSq);
            if (lane == 0) {
                sScale = f;
                if (blockIdx.x == 0 && b == 0 && in.normSqOut) *in.normSqOut = normSq;
            }
        }
        __syncthreads();
    }
    // the matrix in pieces of V columns, dealt out evenly and in order
    const int perRow = (s.cols + V - 1) / V;
    const int64_t total = (int64_t)s.rows * perRow;
    const int64_t first = total * blockIdx.x / gridDim.x, end = total * (blockIdx.x + 1) / gridDim.x;
    double sum = 0.0;
    for (int64_t i = first + threadIdx.x; i < end; i += kPrepThreads) {
        const int r = (int)(i / perRow), c = (int)(i - (int64_t)r * perRow) * V;
        float* dst = x32 + ((int64_t)b * s.rows + r) * s.ldx + c;
        float u[V];
        if (MUON) {
            const int64_t at = (int64_t)b * in.stride + (int64_t)r * s.cols + c;
            float g[V], m[V];
            if (V == 4) {
                *reinterpret_cast<float4*>(g) = *reinterpret_cast<const float4*>(in.grad + at);
                *reinterpret_cast<float4*>(m) = *reinterpret_cast<const float4*>(in.momentum + at);
            } else {
                g[0] = in.grad[at];
                m[0] = in.momentum[at];
            }
#pragma unroll
            for (int k = 0; k < V; k++) {
                g[k] = __fmul_rn(g[k], sScale);
                m[k] = __fadd_rn(__fmul_rn(in.decay, m[k]), g[k]);
                u[k] = in.nesterov ? __fadd_rn(g[k], __fmul_rn(in.decay, m[k])) : m[k];
            }
            if (V == 4)
                *reinterpret_cast<float4*>(in.momentum + at) = *reinterpret_cast<const float4*>(m);
            else
                in.momentum[at] = m[0];
        } else {
            const T* src = static_cast<const T*>(in.x) + (int64_t)b * in.stride + (int64_t)r * in.ld + c;
            if (V == 4) {
                T raw[4];
                if (sizeof(T) == 4)
                    *reinterpret_cast<float4*>(raw) = *reinterpret_cast<const float4*>(src);
                else
                    *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(src);
#pragma unroll
                for (int k = 0; k < V; k++) u[k] = to_f32(raw[k]);
            } else {
                u[0] = to_f32(src[0]);
            }
        }
        if (V == 4)
            *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(u);
        else
            dst[0] = u[0];
        sum += square_sum<V>(u);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) sSum[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kPrepWarps; w++) sum += sSum[w];
        partial[(int64_t)b * kPrepMaxParts + blockIdx.x] = sum;
    }
}

// X = U / |U| (0 for a zero U), and its two fp16 parts; four columns a thread (the
// workspace's rows are padded to eight).
__global__ void __launch_bounds__(kPrepThreads)
    k_muon_normalise(MuonShape s, float* x32, __half* x16, const double* partial, int parts) {
    mg_pdl_trigger();
    mg_pdl_wait();
    __shared__ double sSum[kPrepWarps];
    const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += kPrepThreads) sum += partial[(int64_t)b * kPrepMaxParts + i];
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) sSum[warp] = sum;
    __syncthreads();
    sum = sSum[0];
    for (int w = 1; w < kPrepWarps; w++) sum += sSum[w];
    const InverseNorm inv(sum);
    const int64_t total = (int64_t)s.rows * s.ldx / 4;
    float4* x = reinterpret_cast<float4*>(x32 + (int64_t)b * s.rows * s.ldx);
    __half* h = x16 + (int64_t)b * s.rows * s.ldx;
    const int64_t lo = (int64_t)gridDim.y * s.rows * s.ldx;
    for (int64_t i = (int64_t)blockIdx.x * kPrepThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kPrepThreads) {
        float4 v = x[i];  // (the padding's values are never read as operands)
        v = make_float4(inv(v.x), inv(v.y), inv(v.z), inv(v.w));
        x[i] = v;
        store_parts4(h + 4 * i, lo, v.x * kNsScale, v.y * kNsScale, v.z * kNsScale, v.w * kNsScale);
    }
}

template <int KIND, int BN, bool A_MN, bool B_MN>
int launch_tiled(const CUtensorMap& ta, const CUtensorMap& tb, NsProduct p, cudaStream_t st) {
    using S = NsTile<BN>;
    auto kern = k_ns_product<KIND, BN, A_MN, B_MN>;
    static std::atomic<uint64_t> done{0};
    MG_TRY(smem_limit_once(kern, S::SMEM_BYTES, done));
    p.tilesM = (p.M + 127) / 128;
    p.tilesN = (p.N + BN - 1) / BN;
    const int64_t units = (int64_t)ns_tiles<KIND, BN>(p.tilesM, p.tilesN) * p.batch;
    if (units > INT32_MAX) return fail(MG_ERR_ARGUMENT, "newton_schulz: too many tiles");
    const int grid = (int)std::min<int64_t>(units, num_sms());
    MG_CUDA_TRY(MG_LAUNCH(kern, grid, S::THREADS, S::SMEM_BYTES, st, ta, tb, p));
    return check_launch("k_ns_product");
}

template <int KIND, bool A_MN, bool B_MN>
int launch_split(const CUtensorMap& ta, const CUtensorMap& tb, NsProduct p, int splits, cudaStream_t st) {
    using S = NsTile<128>;
    auto kern = k_ns_split<KIND, A_MN, B_MN>;
    static std::atomic<uint64_t> done{0};
    MG_TRY(smem_limit_once(kern, S::SMEM_BYTES, done));
    p.tilesM = (p.M + 127) / 128;
    p.tilesN = (p.N + 127) / 128;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ns_tiles<KIND, 128>(p.tilesM, p.tilesN) * p.batch * splits));
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    MG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, ta, tb, p, splits));
    return check_launch("k_ns_split");
}

// Few tiles split a K of four blocks or more over a cluster, while the clusters
// fit the GPU at once (five steps of 512 x 2048: 295 us unsplit, 209 and 166 with
// clusters of two and four; clusters of four on 144 of 148 SMs run in two waves).
// Otherwise the tile with the fewest cycles: whole rounds over the SMs, of 1180
// and 1745 cycles a K block for 128 x 128 and 128 x 256 (the operand bytes of
// both parts at the 55 a cycle that L2 gives an SM), and an epilogue behind the
// last tile (all products by 128 x 128 / by 128 x 256 / by this rule: 8 x 1024 x
// 1024 676 / 800 / 639 us, 2 x 1500 x 4000 1363 / 1098 / 1101, 4096 x 4096 4286 /
// 3425 / 3434, 1500 x 1500 389 / 538 / 390).
template <int KIND, bool A_MN, bool B_MN>
int launch_product(const CUtensorMap& ta, const CUtensorMap& tb, const NsProduct& p, cudaStream_t st) {
    const int64_t tiles = (int64_t)ns_tiles<KIND, 128>((p.M + 127) / 128, (p.N + 127) / 128) * p.batch;
    const int64_t sms = num_sms(), blocks = (p.K + 63) / 64;
    int splits = 1;
    while (splits < 4 && tiles * splits * 2 <= sms * 7 / 8 && blocks >= 4 && blocks >= 2 * splits) splits *= 2;
    if (splits > 1) return launch_split<KIND, A_MN, B_MN>(ta, tb, p, splits, st);
    const int64_t wide = (int64_t)ns_tiles<KIND, 256>((p.M + 127) / 128, (p.N + 255) / 256) * p.batch;
    auto rounds = [&](int64_t n) { return (n + sms - 1) / sms; };
    const int64_t cost128 = rounds(tiles) * 1180 * blocks + 3000, costWide = rounds(wide) * 1745 * blocks + 5000;
    return costWide < cost128 ? launch_tiled<KIND, 256, A_MN, B_MN>(ta, tb, p, st) : launch_tiled<KIND, 128, A_MN, B_MN>(ta, tb, p, st);
}

struct Workspace {
    double* partial;
    float* x32;
    __half* x16[2];  // hi, then lo parts of the batch; G and B likewise
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
    w.partial = static_cast<double*>(take((size_t)batch * kPrepMaxParts * 8));
    w.x32 = static_cast<float*>(take(x * 4));
    w.x16[0] = static_cast<__half*>(take(x * 4));
    w.x16[1] = static_cast<__half*>(take(x * 4));
    w.g16 = static_cast<__half*>(take(g * 4));
    w.b16 = static_cast<__half*>(take(g * 4));
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
    const int64_t quads = (int64_t)rows * shape.ldx / 4;
    const int ctas = (int)std::min<int64_t>((quads + 4 * kPrepThreads - 1) / (4 * kPrepThreads), std::max(1, num_sms() * 8 / batch));
    MG_CUDA_TRY(MG_LAUNCH(k_muon_normalise, dim3(ctas, batch), kPrepThreads, 0, st, shape, w.x32, w.x16[0], w.partial, parts));
    MG_TRY(check_launch("k_muon_normalise"));
    const bool wide = rows <= cols;  // G = X X^T, else X^T X
    const int s = std::min(rows, cols), l = std::max(rows, cols), lds = round8(s);
    CUtensorMap mx[2], mg16, mb16;
    for (int i = 0; i < 2; i++) MG_TRY(make_tmap_f16_3d(&mx[i], w.x16[i], cols, rows, 2 * batch, shape.ldx, 128));
    CUtensorMap mxk[2];  // boxes of 64 rows, for X as an operand whose K index is the row
    for (int i = 0; i < 2; i++) MG_TRY(make_tmap_f16_3d(&mxk[i], w.x16[i], cols, rows, 2 * batch, shape.ldx, 64));
    MG_TRY(make_tmap_f16_3d(&mg16, w.g16, s, s, 2 * batch, lds, 128));
    MG_TRY(make_tmap_f16_3d(&mb16, w.b16, s, s, 2 * batch, lds, 128));
    NsProduct p{};
    p.batch = batch;
    p.status = status_ptr();
    for (int i = 0; i < steps; i++) {
        const int cur = i & 1;
        p.M = p.N = s;
        p.K = l;
        p.ldo = lds;
        p.out16 = w.g16;
        p.a = 0.0f;
        MG_TRY(wide ? (launch_product<kNsGram, false, false>(mx[cur], mx[cur], p, st))
                    : (launch_product<kNsGram, true, true>(mxk[cur], mxk[cur], p, st)));
        p.K = s;
        p.out16 = w.b16;
        p.g16 = w.g16;
        p.b = kNsB;
        p.c = kNsC;
        MG_TRY((launch_product<kNsPoly, false, false>(mg16, mg16, p, st)));
        p.M = rows;
        p.N = cols;
        p.K = s;
        p.ldo = shape.ldx;
        p.x32 = w.x32;
        p.out16 = w.x16[cur ^ 1];
        p.a = kNsA;
        p.last = i + 1 == steps;
        if (p.last) p.fin = fin;
        MG_TRY(wide ? (launch_product<kNsApply, false, true>(mb16, mxk[cur], p, st))
                    : (launch_product<kNsApply, false, false>(mx[cur], mb16, p, st)));
    }
    return MG_OK;
}

template <class T, bool MUON>
int prepare(const MuonInput& in, const Workspace& w, int batch, int rows, int cols, bool vec, int* parts, cudaStream_t st) {
    const MuonShape shape{rows, cols, round8(cols)};
    const int64_t pieces = (int64_t)rows * ((cols + (vec ? 3 : 0)) / (vec ? 4 : 1));
    const int64_t most = std::min<int64_t>(kPrepMaxParts, std::max(1, num_sms() * 8 / batch));
    *parts = (int)std::min<int64_t>((pieces + 4 * kPrepThreads - 1) / (4 * kPrepThreads), most);
    if (vec)
        MG_CUDA_TRY(MG_LAUNCH((k_muon_prepare<T, MUON, 4>), dim3(*parts, batch), kPrepThreads, 0, st, in, shape, w.x32, w.partial));
    else
        MG_CUDA_TRY(MG_LAUNCH((k_muon_prepare<T, MUON, 1>), dim3(*parts, batch), kPrepThreads, 0, st, in, shape, w.x32, w.partial));
    return check_launch("k_muon_prepare");
}

// One kernel for a smaller side of at most 128 and a few steps (muon_small.cuh).
bool small_enough(int rows, int cols, int steps) {
    return std::min(rows, cols) <= kMuonSmallSide && steps <= kMuonSmallSteps;
}

template <int SP, bool WIDE, class T, bool MUON>
int launch_small(const MuonInput& in, const NsProduct& p, float* x32, int steps, bool vec, cudaStream_t st) {
    auto kern = k_muon_small<SP, WIDE, T, MUON>;
    static std::atomic<uint64_t> done{0};
    MG_TRY(smem_limit_once(kern, MuonSmall::SMEM_BYTES, done));
    // a CTA for each 128 of the long side, up to a cluster, while the matrices leave SMs for them
    const int pieces = (std::max(p.M, p.N) + 127) / 128;
    int parts = 1;
    while (parts < kMuonSmallCluster && parts < pieces && (int64_t)p.batch * parts * 2 <= num_sms()) parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.batch * parts));
    cfg.blockDim = dim3(kMuonSmallThreads);
    cfg.dynamicSmemBytes = MuonSmall::SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 2 : 1;
    MG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, in, p, x32, steps, vec ? 1 : 0, parts));
    return check_launch("k_muon_small");
}

template <class T, bool MUON>
int run_small(const MuonInput& in, const Workspace& w, const NsFinal& fin, int batch, int rows, int cols, int steps, bool vec, cudaStream_t st) {
    NsProduct p{};
    p.M = rows;
    p.N = cols;
    p.batch = batch;
    p.ldo = round8(cols);
    p.last = 1;
    p.fin = fin;
    p.status = status_ptr();
    const bool narrow = std::min(rows, cols) <= 64;
    if (rows <= cols)
        return narrow ? launch_small<64, true, T, MUON>(in, p, w.x32, steps, vec, st) : launch_small<128, true, T, MUON>(in, p, w.x32, steps, vec, st);
    return narrow ? launch_small<64, false, T, MUON>(in, p, w.x32, steps, vec, st) : launch_small<128, false, T, MUON>(in, p, w.x32, steps, vec, st);
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
    NsFinal fin{};
    fin.out = out;
    fin.outBf16 = out_dtype == MG_DTYPE_BF16;
    fin.ld = ldo;
    fin.stride = out_stride;
    fin.vec = ldo % 4 == 0 && out_stride % 4 == 0 && aligned_to(out, 8);
    if (small_enough(rows, cols, steps)) {
        const int per = dtype == MG_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
        const bool vec = ld % per == 0 && batch_stride % per == 0 && aligned_to(x, 16);
        if (dtype == MG_DTYPE_F32) return run_small<float, false>(in, w, fin, batch, rows, cols, steps, vec, st);
        if (dtype == MG_DTYPE_BF16) return run_small<__nv_bfloat16, false>(in, w, fin, batch, rows, cols, steps, vec, st);
        return run_small<__half, false>(in, w, fin, batch, rows, cols, steps, vec, st);
    }
    int parts = 0;
    const bool vec = cols % 4 == 0 && ld % 4 == 0 && batch_stride % 4 == 0 && aligned_to(x, dtype == MG_DTYPE_F32 ? 16 : 8);
    if (dtype == MG_DTYPE_F32)
        MG_TRY((prepare<float, false>(in, w, batch, rows, cols, vec, &parts, st)));
    else if (dtype == MG_DTYPE_BF16)
        MG_TRY((prepare<__nv_bfloat16, false>(in, w, batch, rows, cols, vec, &parts, st)));
    else
        MG_TRY((prepare<__half, false>(in, w, batch, rows, cols, vec, &parts, st)));
    return newton_schulz(w, batch, rows, cols, steps, parts, fin, st);
}

int mg_muon_step(float* master, const float* grad, float* momentum, void* weights, int64_t batch_stride, int batch,
                 int rows, int cols, const float* norm_partial, int n_norm_partials, float max_grad_norm, float lr,
                 float scale, float momentum_decay, int nesterov, float weight_decay, int steps, float* norm_sq_out,
                 void* workspace, size_t workspace_bytes, mg_stream_t stream) {
    MG_CHECK_ARG(master && grad && momentum && weights, "muon_step: null argument");
    MG_TRY(check_shape("muon_step", batch, rows, cols));
    MG_CHECK_ARG(aligned_to(master, 4) && aligned_to(grad, 4) && aligned_to(momentum, 4) && aligned_to(weights, 2) &&
                     aligned_to(norm_partial, 4) && aligned_to(norm_sq_out, 4),
                 "muon_step: a buffer is not aligned to its type");
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
    const bool vec = cols % 4 == 0 && batch_stride % 4 == 0 && aligned_to(grad, 16) && aligned_to(momentum, 16);
    NsFinal fin{};
    fin.master = master;
    fin.weights = static_cast<__nv_bfloat16*>(weights);
    fin.ld = cols;
    fin.stride = batch_stride;
    fin.vec = cols % 4 == 0 && batch_stride % 4 == 0 && aligned_to(master, 16) && aligned_to(weights, 8);
    fin.keep = 1.0f - lr * weight_decay;
    fin.rate = lr * scale;
    if (small_enough(rows, cols, steps)) return run_small<float, true>(in, w, fin, batch, rows, cols, steps, vec, st);
    int parts = 0;
    MG_TRY((prepare<float, true>(in, w, batch, rows, cols, vec, &parts, st)));
    return newton_schulz(w, batch, rows, cols, steps, parts, fin, st);
}

}  // extern "C"
