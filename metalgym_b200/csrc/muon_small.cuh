// The whole of an orthogonalisation or Muon step whose smaller side s is at
// most 128, in one kernel: a cluster of up to eight CTAs per matrix.
//
// The Newton-Schulz steps only multiply X by polynomials of G = X X^T, which
// commute: with Q = a I + b G + c G^2 the next X is Q X and the next G is Q G Q.
// So the long side is passed twice in a run of up to three steps, for G and for
// P X with P the product of the Qs, and the steps in between take s x s matrices
// alone, held in shared memory by every CTA of the cluster (the same operations
// on the same bits in each). 17 launches that each wait for the one before took
// 117 us at 2 x 128 x 512 with operands of one part.
//
// Precision: every operand is the sum of two fp16 numbers (22 bits), every
// product three tcgen05 products. P grows to a^k in directions that U hardly
// has, and what G is off there by a^2 in every step, since no X checks it: after
// three steps X is written out (or kept in tensor memory by a CTA of one piece)
// and G taken from it anew. Off the exact iteration, of the result's norm, at 128
// x 512 in five and six steps: 1.2e-4 and 1.9e-4 at rank 1, 3e-5 and 1e-4 at rank
// 8 (fp32 products by a library 1.0e-4 and 2.2e-4, 2e-5 and 1e-4); all steps in
// one run 2.6e-3 and 2.1e-2, 3.2e-4 and 3.5e-3 (a step of 2 x 128 x 512 in 47 us
// of GPU time instead of 57, 128 x 4096 in 69 instead of 106). P is scaled by 2^5,
// the others by 2^10.
#pragma once

#include "logits.cuh"
#include "muon.cuh"
#include "metalgym/detail/tile.cuh"

namespace mg {

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

constexpr int kMuonSmallSide = 128, kMuonSmallRun = 3, kMuonSmallSteps = 2 * kMuonSmallRun, kMuonSmallThreads = 512;
constexpr int kMuonSmallCluster = 8;
constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;

struct MuonSmall {
    static constexpr int MAT = 65536;  // a matrix's or a tile's two fp16 parts
    static constexpr int BAR_OFF = 3 * MAT;
    // All that a CTA can have, more than the 198 KB in use: a CTA waits for its
    // tensor memory without a limit, and its cluster for it. Beside another kernel's
    // clusters that hold tensor memory the two could wait for each other.
    static constexpr int SMEM_BYTES = 227 * 1024;
    static_assert(BAR_OFF + 256 + 1024 /*align*/ <= SMEM_BYTES, "the matrices, barriers and sums");
};

// The sum of N squares. 64-bit conversions run at 16 a cycle and SM, so that
// they, not the loads, would set the pace of a pass (3 of 8 us per 128 x 128
// piece): squares are summed in fp32 wherever that neither overflows nor loses
// small ones, and a CTA's sums in 64 bits.
template <int N>
__device__ __forceinline__ double square_sum(const float* u) {
    float f = 0.0f;
#pragma unroll
    for (int k = 0; k < N; k++) f = fmaf(u[k], u[k], f);
    if (f > 1e-25f && f < 1e30f) return (double)f;
    double d = 0.0;
#pragma unroll
    for (int k = 0; k < N; k++) d += (double)u[k] * (double)u[k];
    return d;
}

// x -> x / norm by fp32 products that stay in range for every norm: 1 / norm =
// p q m with p and q powers of two (0 for a zero norm).
struct InverseNorm {
    float p, q, m;
    __device__ __forceinline__ explicit InverseNorm(double squares) {
        int e = 0;
        m = squares == 0.0 ? 0.0f : (float)frexp(1.0 / sqrt(squares), &e);  // NaN and infinity stay NaN and 0
        const int first = max(-126, min(126, e));
        p = ldexpf(1.0f, first);
        q = ldexpf(1.0f, max(-126, min(126, e - first)));
    }
    __device__ __forceinline__ float operator()(float x) const { return ((x * p) * q) * m; }
};

// The clip factor of mg_adam_step from the norm partials (one warp; lane 0's
// value counts). The squared norm goes to *normSq.
__device__ __forceinline__ float muon_clip(const MuonInput& in, float* normSq) {
    float sum = 0.0f;
    for (int i = threadIdx.x & 31; i < in.nNorm; i += 32) sum = __fadd_rn(sum, in.normPartial[i]);
    sum = warp_sum(sum);
    *normSq = sum;
    const float norm = __fsqrt_rn(sum);
    return (in.maxGradNorm > 0.0f && norm > in.maxGradNorm) ? __fdiv_rn(in.maxGradNorm, __fadd_rn(norm, 1e-6f)) : 1.0f;
}

// Eight consecutive columns of U at (r, c) of matrix b; those from `cols` on are
// 0. `update`: the first pass, which also writes the momentum.
template <class T, bool MUON>
__device__ __forceinline__ void muon_load8(const MuonInput& in, int b, int r, int c, int cols, bool vec, bool update, float scale,
                                           float* u) {
    const int n = min(8, cols - c);
    if (MUON) {
        const int64_t at = (int64_t)b * in.stride + (int64_t)r * cols + c;
        float g[8], m[8];
        if (vec && n == 8) {
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                *reinterpret_cast<float4*>(g + i) = *reinterpret_cast<const float4*>(in.grad + at + i);
                *reinterpret_cast<float4*>(m + i) = *reinterpret_cast<const float4*>(in.momentum + at + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                g[i] = i < n ? in.grad[at + i] : 0.0f;
                m[i] = i < n ? in.momentum[at + i] : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            g[i] = __fmul_rn(g[i], scale);
            if (update) m[i] = __fadd_rn(__fmul_rn(in.decay, m[i]), g[i]);
            u[i] = in.nesterov ? __fadd_rn(g[i], __fmul_rn(in.decay, m[i])) : m[i];
        }
        if (update) {
            if (vec && n == 8) {
#pragma unroll
                for (int i = 0; i < 8; i += 4)
                    *reinterpret_cast<float4*>(in.momentum + at + i) = *reinterpret_cast<const float4*>(m + i);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < n) in.momentum[at + i] = m[i];
            }
        }
    } else {
        const T* x = static_cast<const T*>(in.x) + (int64_t)b * in.stride + (int64_t)r * in.ld + c;
        if (vec && n == 8) {
            T raw[8];
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) * 8 / 16; i++)
                reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(x)[i];
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = to_f32(raw[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = i < n ? to_f32(x[i]) : 0.0f;
        }
    }
}

// Eight values (already scaled) as two fp16 parts into the 16-byte cell at `off`
// of a matrix's first part and the same cell of its second part.
__device__ __forceinline__ void split_store8(uint8_t* mat, uint32_t off, const float* y) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 h = __floats2half2_rn(y[2 * i], y[2 * i + 1]);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(y[2 * i] - f.x, y[2 * i + 1] - f.y);
        hi[i] = *reinterpret_cast<const uint32_t*>(&h);
        lo[i] = *reinterpret_cast<const uint32_t*>(&l);
    }
    *reinterpret_cast<uint4*>(mat + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(mat + 32768 + off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}
__device__ __forceinline__ void split_load8(const uint8_t* mat, uint32_t off, float* y) {
    const uint4 h = *reinterpret_cast<const uint4*>(mat + off), l = *reinterpret_cast<const uint4*>(mat + 32768 + off);
    const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hw[i])), b = __half22float2(*reinterpret_cast<const __half2*>(&lw[i]));
        y[2 * i] = a.x + b.x;
        y[2 * i + 1] = a.y + b.y;
    }
}

// D (+)= A B over K = 16 KS, each operand in two parts: the two mixed products,
// then that of the first parts (one thread). The accumulator is cut off, not
// rounded, at each instruction: with the small products first there are 8 cuts
// of the full sum, not 24 (emulated: a third of the error at rank 1). Tiles are 128 x 128, two blocks of
// 64 columns, 16 KB each, 128-byte swizzled; an operand whose K index is the
// tile's row is MN-major.
template <bool A_MN, bool B_MN, int N, int KS>
__device__ __forceinline__ void split_mma(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
    constexpr uint32_t idesc = idesc_f16_f32(N, A_MN, B_MN);
#pragma unroll
    for (int part = 0; part < 3; part++) {
        const uint32_t ap = a + (part == 0 ? 32768u : 0u), bp = b + (part == 1 ? 32768u : 0u);
#pragma unroll
        for (int k = 0; k < KS; k++) {
            // K-major: 16 columns on, in the second block from 64 on; MN-major: 16 rows on
            const uint64_t ad = A_MN ? smem_desc_sw128(ap + k * 2048, 16384, 1024)
                                     : smem_desc_sw128(ap + (k >> 2) * 16384 + (k & 3) * 32, 16, 1024);
            const uint64_t bd = B_MN ? smem_desc_sw128(bp + k * 2048, 16384, 1024)
                                     : smem_desc_sw128(bp + (k >> 2) * 16384 + (k & 3) * 32, 16, 1024);
            tc_mma_bf16(d, ad, bd, idesc, accumulate || part > 0 || k > 0 ? 1u : 0u);
        }
    }
}

// 32 lanes x N consecutive fp32 columns of tensor memory, N = 16 or 32.
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t taddr, float* v) {
    if constexpr (N == 32) {
        tmem_ld32(taddr, v);
    } else {
        static_assert(N == 16, "16 or 32 columns");
        uint32_t r[16];
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
              "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr));
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
    }
}

// A 32 x 32 piece of X at (row0, col0) of matrix b into x [batch][M][ldo], from
// an accumulator scaled by 2^20 (lane r holds row r in v).
__device__ __forceinline__ void ns_keep(const NsProduct& p, float* x, int b, int row0, int col0, uint8_t* slab, const float* v) {
    const int lane = threadIdx.x & 31, k = lane & 7, col = col0 + 4 * k;
    constexpr float kScale = kNsUnscale * kNsUnscale;
    __syncwarp();  // the slab's last readers are done
#pragma unroll
    for (int i = 0; i < 8; i++)
        *reinterpret_cast<float4*>(slab + ns_slab_offset(lane, i)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    __syncwarp();
    if (col >= p.N) return;  // (the four columns lie inside ldo)
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = 4 * i + (lane >> 3), row = row0 + r;
        const float4 y = *reinterpret_cast<const float4*>(slab + ns_slab_offset(r, k));
        if (row < p.M)
            *reinterpret_cast<float4*>(x + ((int64_t)b * p.M + row) * p.ldo + col) =
                make_float4(y.x * kScale, y.y * kScale, y.z * kScale, y.w * kScale);
    }
}

// SP: the smaller side padded, 64 or 128. WIDE: rows <= cols. x32: X between two
// runs of steps, [batch][rows][ldo].
template <int SP, bool WIDE, class T, bool MUON>
__global__ void __launch_bounds__(kMuonSmallThreads, 1)
    k_muon_small(const MuonInput in, const NsProduct p, float* x32, int steps, int vec, int parts) {
    using S = MuonSmall;
    constexpr int KS = SP / 16, COLS = SP / 4;  // COLS: columns of an s x s matrix that a thread holds
    constexpr int WARPS = kMuonSmallThreads / 32;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *mG = smem, *mQ = smem + S::MAT, *mP = smem + 2 * S::MAT;
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + S::BAR_OFF);  // [2]
    double* sNorm = reinterpret_cast<double*>(bar + 2);
    double* sSum = sNorm + 1;  // [WARPS]
    float* sScale = reinterpret_cast<float*>(sSum + WARPS);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sScale + 1);
    mg_pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = blockIdx.x / parts, rank = blockIdx.x % parts;
    const int rows = p.M, cols = p.N, s = WIDE ? rows : cols, l = WIDE ? cols : rows;
    if (tid == 0) {
        mbar_init(&bar[0], 1);
        mbar_init(&bar[1], 1);
        fence_barrier_init();
    }
    if (warp == 2) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    uint32_t phase[2] = {0, 0};
    auto wait = [&](int i) {
        mbar_wait(&bar[i], phase[i], p.status, kDevTimeoutDone);
        phase[i] ^= 1u;
        __syncwarp();  // loads from tensor memory take whole warps
        tc_fence_after();
    };
    // what the threads wrote to shared memory and read from tensor memory, before the next products
    auto handOver = [&] {
        tc_fence_before();
        fence_async_smem();
        __syncthreads();
        tc_fence_after();
    };
    mg_pdl_wait();
    if (MUON) {
        if (warp == 0) {
            float normSq;
            const float f = muon_clip(in, &normSq);
            if (lane == 0) {
                *sScale = f;
                if (blockIdx.x == 0 && in.normSqOut) *in.normSqOut = normSq;
            }
        }
        __syncthreads();
    }
    const float scale = MUON ? *sScale : 1.0f;
    // this CTA's pieces of 128 along the long side
    const int pieces = (l + 127) / 128, first = (int)((int64_t)pieces * rank / parts), end = (int)((int64_t)pieces * (rank + 1) / parts);
    // eight columns of U: cell g (16 to a tile row) of piece i, zeros outside the matrix
    MuonInput kept{};  // X after a run
    kept.x = x32;
    kept.ld = p.ldo;
    kept.stride = (int64_t)rows * p.ldo;
    bool again = false;
    auto cell = [&](int i, int g, bool update, float* u) {
        const int r = (g >> 4) + (WIDE ? 0 : 128 * i), c = 8 * (g & 15) + (WIDE ? 128 * i : 0);
        if (r < rows && c < cols) {
            if (again)
                muon_load8<float, false>(kept, b, r, c, cols, true, false, 1.0f, u);
            else
                muon_load8<T, MUON>(in, b, r, c, cols, vec != 0, update, scale, u);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) u[k] = 0.0f;
        }
    };
    // cells that a tile has: SP rows of 16 (wide), or 128 rows of SP / 8
    constexpr int CELLS = SP * 16;
    auto cellIndex = [&](int j) { return WIDE || SP == 128 ? j : (j / (SP / 8)) * 16 + j % (SP / 8); };

    constexpr int PER = CELLS / kMuonSmallThreads;  // cells of a thread

    // |U|^2 (and the momentum); the first piece stays in registers for its tile
    double sum = 0.0;
    float held[PER][8];
#pragma unroll 1
    for (int i = end - 1; i >= first; i--)
#pragma unroll
        for (int j = 0; j < PER; j++) {
            cell(i, cellIndex(tid + j * kMuonSmallThreads), true, held[j]);
            sum += square_sum<8>(held[j]);
        }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) sSum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < WARPS; w++) sum += sSum[w];
        *sNorm = sum;
    }
    __syncwarp();
    if (parts > 1) {
        cluster_sync();
        sum = 0.0;
        for (int k = 0; k < parts; k++) sum += *cluster_peer(sNorm, k);
    } else {
        __syncthreads();
        sum = *sNorm;
    }
    InverseNorm inv(sum);
    // the piece of X in `held` into a tile; piece `next` is loaded behind it
    auto load = [&](int i) {
#pragma unroll
        for (int j = 0; j < PER; j++) cell(i, cellIndex(tid + j * kMuonSmallThreads), false, held[j]);
    };
    auto tile = [&](uint8_t* mat, int next) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int g = cellIndex(tid + j * kMuonSmallThreads);
            float u[8];
#pragma unroll
            for (int k = 0; k < 8; k++) u[k] = inv(held[j][k]) * kNsScale;
            split_store8(mat, sw128_offset(g >> 4, g & 15), u);
            if (next < end) cell(next, g, false, held[j]);
        }
        handOver();
    };

    const int q = warp & 3, row = 32 * q + lane, c0 = (warp >> 2) * COLS;
    const uint32_t acc = tmem + ((uint32_t)(32 * q) << 16);
    const bool holds = 32 * q < SP;  // warps 2 and 3 of four have no rows of a 64-row matrix
    const uint32_t aG = smem_u32(mG), aQ = smem_u32(mQ), aP = smem_u32(mP);
    constexpr float kAcc = kNsUnscale * kNsUnscale;  // of a product of two matrices scaled by 2^10
    constexpr int N = WIDE ? 128 : SP;                // columns of a piece of P X
    const int cX = 32 * (warp >> 2);
    const bool holdsX = cX < N && (!WIDE || holds);
    // X of the run before into a tile, out of columns 256 .. of tensor memory, where a CTA of one piece keeps it
    auto retile = [&](uint8_t* mat) {
        if (holdsX) {
            float v[32];
            tmem_ld32(acc + (uint32_t)(256 + cX), v);
#pragma unroll
            for (int k = 0; k < 32; k++) v[k] *= 0.03125f;  // (scaled by 2^15 there)
#pragma unroll
            for (int k = 0; k < 4; k++) split_store8(mat, sw128_offset(row, cX / 8 + k), v + 8 * k);
        }
        handOver();
    };
#pragma unroll 1
    for (;;) {
        const int run = min(steps, kMuonSmallRun);
        // G's part from this CTA's pieces, the tiles alternating between two places
        const bool resident = again && end - first == 1;
        for (int i = first; i < end; i++) {
            const int k = (i - first) & 1;
            uint8_t* mat = k ? mP : mQ;
            if (i - first >= 2) wait(k);
            if (resident)
                retile(mat);
            else
                tile(mat, i + 1);
            if (tid == 0) {
                split_mma<!WIDE, !WIDE, SP, 8>(tmem, smem_u32(mat), smem_u32(mat), i > first);
                tc_commit(&bar[k]);
            }
        }
        if (end - first >= 2) wait((end - first) & 1);
        if (end > first) wait((end - first - 1) & 1);
        if (holds) {
            float v[COLS];
            if (end > first) {
                tmem_load<COLS>(acc + (uint32_t)c0, v);
            } else {
#pragma unroll
                for (int k = 0; k < COLS; k++) v[k] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < COLS / 4; k++)
                *reinterpret_cast<float4*>(mG + tile_offset(row, c0 / 4 + k)) =
                    make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        }
        if (parts > 1) {
            // CTA k sums rows k SP / parts .. of all parts, in their order, and hands
            // them back to all: nobody else reads or writes those rows meanwhile
            __syncwarp();
            cluster_sync();
            const int mine = SP / parts;
            for (int j = tid; j < mine * SP / 4; j += kMuonSmallThreads) {
                const uint32_t off = tile_offset(rank * mine + j / (SP / 4), j % (SP / 4));
                float4 v[kMuonSmallCluster], t;
#pragma unroll
                for (int k = 0; k < kMuonSmallCluster; k++)
                    if (k < parts) v[k] = *reinterpret_cast<const float4*>(cluster_peer(mG, k) + off);
                t = v[0];
#pragma unroll
                for (int k = 1; k < kMuonSmallCluster; k++)
                    if (k < parts) {
                        t.x += v[k].x;
                        t.y += v[k].y;
                        t.z += v[k].z;
                        t.w += v[k].w;
                    }
#pragma unroll
                for (int k = 0; k < kMuonSmallCluster; k++)
                    if (k < parts) *reinterpret_cast<float4*>(const_cast<uint8_t*>(cluster_peer(mG, k)) + off) = t;
            }
            __syncwarp();
            cluster_sync();
        } else {
            __syncthreads();
        }
        // G in two parts, over the fp32 tile (each thread takes its values out first)
        {
            float g[COLS];
            if (holds) {
#pragma unroll
                for (int k = 0; k < COLS / 4; k++)
                    *reinterpret_cast<float4*>(g + 4 * k) = *reinterpret_cast<const float4*>(mG + tile_offset(row, c0 / 4 + k));
            }
            __syncthreads();
            if (holds) {
#pragma unroll
                for (int k = 0; k < COLS; k++) g[k] *= kAcc * kNsScale;
#pragma unroll
                for (int k = 0; k < COLS / 8; k++) split_store8(mG, sw128_offset(row, c0 / 8 + k), g + 8 * k);
            }
        }
        handOver();

        // the steps
        // an accumulator, scaled by 2^10 more than the matrix, into the matrix
        auto take = [&](uint32_t column, uint8_t* mat) {
            if (!holds) return;
            float v[COLS];
            tmem_load<COLS>(acc + column + (uint32_t)c0, v);
#pragma unroll
            for (int k = 0; k < COLS; k++) v[k] *= kNsUnscale;
#pragma unroll
            for (int k = 0; k < COLS / 8; k++) split_store8(mat, sw128_offset(row, c0 / 8 + k), v + 8 * k);
        };
        auto multiply = [&](uint32_t column, uint32_t x, uint32_t y, int bit) {
            if (tid == 0) {
                split_mma<false, false, SP, KS>(tmem + column, x, y, false);
                tc_commit(&bar[bit]);
            }
        };
        // P's products run behind those that the next G waits for, and are taken up
        // while the next product runs.
        for (int step = 0; step < run; step++) {
            const bool more = step + 1 < run;
            multiply(0, aG, aG, 0);
            wait(0);
            if (holds) {  // Q = a I + b G + c G^2
                float v[COLS];
                tmem_load<COLS>(acc + (uint32_t)c0, v);
#pragma unroll
                for (int k = 0; k < COLS / 8; k++) {
                    float g[8];
                    split_load8(mG, sw128_offset(row, c0 / 8 + k), g);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        float y = fmaf(kNsC * kNsUnscale, v[8 * k + i], kNsB * g[i]);  // times 2^10
                        if (c0 + 8 * k + i == row && row < s) y += kNsA * kNsScale;
                        g[i] = y;
                    }
                    split_store8(mQ, sw128_offset(row, c0 / 8 + k), g);
                    if (step == 0) {  // P = Q, scaled by 2^5 throughout
#pragma unroll
                        for (int i = 0; i < 8; i++) g[i] *= 0.03125f;
                        split_store8(mP, sw128_offset(row, c0 / 8 + k), g);
                    }
                }
            }
            handOver();
            if (more) multiply(0, aQ, aG, 0);
            if (step > 0) multiply(128, aQ, aP, 1);
            if (more) {
                wait(0);
                take(0, mG);  // Q G, in G's place
                handOver();
                multiply(0, aQ, aG, 0);
            }
            if (step > 0) {
                wait(1);
                take(128, mP);
            }
            if (more) {
                wait(0);
                take(0, mG);  // Q G Q
            }
            handOver();
        }

        // P X, piece by piece: the next piece's product beside this one's epilogue. The
        // tiles take G's place, the epilogue's slabs Q's.
        uint8_t* slab = mQ + warp * 4096;
        const bool keep = steps > run && end - first == 1;
        auto issue = [&](int i) {
            const int k = (i - first) & 1;
            if (resident)
                retile(mG);
            else
                tile(mG, i + 1);
            if (tid == 0) {
                const uint32_t d = tmem + (keep ? 256 : 128 * k);
                if (WIDE)
                    split_mma<false, true, N, KS>(d, aP, aG, false);
                else
                    split_mma<false, false, N, KS>(d, aG, aP, false);
                tc_commit(&bar[k]);
            }
        };
        if (first < end) {
            if (!resident) load(first);
            issue(first);
        }
        for (int i = first; i < end; i++) {
            const int k = (i - first) & 1;
            wait(k);
            if (keep) break;
            if (i + 1 < end) issue(i + 1);
            const int row0 = 32 * q + (WIDE ? 0 : 128 * i), col0 = cX + (WIDE ? 128 * i : 0);
            if (holdsX && row0 < rows && col0 < cols) {
                float v[32];
                __syncwarp();  // the first warp's lane 0 issued the next product
                tmem_ld32(acc + (uint32_t)(128 * k + cX), v);
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] *= 32.0f;  // to the scale of ns_piece, 2^20
                if (steps > run)
                    ns_keep(p, x32, b, row0, col0, slab, v);
                else
                    ns_piece<kNsApply>(p, b, row0, col0, slab, v, NsFetched<kNsApply>{});
            }
        }
        steps -= run;
        if (steps == 0) break;
        // the next run: X from what this CTA wrote or kept, its slabs' place free
        again = true;
        inv.p = inv.q = inv.m = 1.0f;
        __syncthreads();
        if (end - first > 1) load(first);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace mg
