// The tcgen05 products of a Newton-Schulz step (muon.cu): fp16 operands, fp32
// accumulation in tensor memory, one CTA per 128 x 128 output tile.
//
//   kNsGram   G = X X^T or X^T X, symmetric: the tiles on and above the
//             diagonal are computed, each written to both places
//   kNsPoly   B = b G + c G G, likewise symmetric
//   kNsApply  X <- a X + B X or a X + X B, or in the last step what the caller
//             wants of it
#pragma once

#include <cuda_fp16.h>

#include "metalgym/detail/ptx.cuh"
#include "metalgym/pdl.cuh"

namespace mg {

constexpr float kNsScale = 1024.0f;  // what the fp16 copies are multiplied by
constexpr float kNsUnscale = 1.0f / 1024.0f;

enum NsKind { kNsGram = 0, kNsPoly = 1, kNsApply = 2 };

// What the last step writes: the matrix itself (out), or the optimiser's update.
struct NsFinal {
    void* out;  // bf16 or fp16
    int outBf16;
    float* master;
    __nv_bfloat16* weights;
    int64_t ld, stride;
    float keep, rate;  // master = master * keep - rate * X
};

struct NsProduct {
    int M, N, K;
    int ldo;              // row stride of out16, g16 and x32
    __half* out16;        // [batch][M][ldo], scaled
    const __half* g16;    // kNsPoly
    float* x32;           // kNsApply
    float a, b, c;
    int last;
    NsFinal fin;
    int* status;
};

struct NsTile {
    static constexpr int BM = 128, BN = 128, BK = 64, STAGES = 4;
    static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*align*/ + 256 /*barriers*/;
};

// Instruction descriptor, kind::f16: fp16 A and B, fp32 accumulator, M = 128.
__host__ __device__ constexpr uint32_t idesc_f16_f32(uint32_t n, bool aMnMajor, bool bMnMajor) {
    return (1u << 4) | ((aMnMajor ? 1u : 0u) << 15) | ((bMnMajor ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// 32 columns of one output row.
template <int KIND>
__device__ __forceinline__ void ns_epilogue(const NsProduct& p, int b, int row, int col, bool mirror, const float* v) {
    const int n = min(32, p.N - col);
    const int64_t base = (int64_t)b * p.M * p.ldo;
    if (KIND == kNsApply) {
        float* x = p.x32 + base + (int64_t)row * p.ldo + col;
        __half* h = p.out16 + base + (int64_t)row * p.ldo + col;
        const int64_t at = (int64_t)b * p.fin.stride + (int64_t)row * p.fin.ld + col;
#pragma unroll
        for (int i = 0; i < 32; i++) {
            if (i >= n) break;
            const float y = fmaf(p.a, x[i], v[i] * (kNsUnscale * kNsUnscale));
            if (!p.last) {
                x[i] = y;
                h[i] = __float2half_rn(y * kNsScale);
            } else if (p.fin.master) {
                const float w = __fsub_rn(__fmul_rn(p.fin.master[at + i], p.fin.keep), __fmul_rn(p.fin.rate, y));
                p.fin.master[at + i] = w;
                p.fin.weights[at + i] = __float2bfloat16_rn(w);
            } else if (p.fin.outBf16) {
                static_cast<__nv_bfloat16*>(p.fin.out)[at + i] = __float2bfloat16_rn(y);
            } else {
                static_cast<__half*>(p.fin.out)[at + i] = __float2half_rn(y);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 32; i++) {
        if (i >= n) break;
        float y = v[i] * kNsUnscale;  // scaled by 2^10, as the operands are
        if (KIND == kNsPoly) y = fmaf(p.c, y, p.b * __half2float(p.g16[base + (int64_t)row * p.ldo + col + i]));
        const __half h = __float2half_rn(y);
        p.out16[base + (int64_t)row * p.ldo + col + i] = h;
        if (mirror) p.out16[base + (int64_t)(col + i) * p.ldo + row] = h;
    }
}

template <int KIND, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(128, 1)
    k_ns_product(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const NsProduct p) {
    using S = NsTile;
    mg_pdl_trigger();
    if (KIND != kNsApply && blockIdx.x < blockIdx.y) return;  // the mirror of a tile above the diagonal
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::STAGES * S::STAGE_BYTES);
    uint64_t* empty = full + S::STAGES;
    uint64_t* done = empty + S::STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int m0 = blockIdx.y * S::BM, n0 = blockIdx.x * S::BN, b = blockIdx.z;
    const int nk = (p.K + S::BK - 1) / S::BK;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        fence_barrier_init();
        prefetch_tensormap(&tmA);
        prefetch_tensormap(&tmB);
    }
    if (warp == 2) {
        tmem_alloc(tmem_slot, S::BN);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    mg_pdl_wait();

    if (warp == 0 && lane == 0) {
        int issued = 0;
        for (int kb = 0; kb < nk; kb++) {
            const int s = kb % S::STAGES;
            if (!mbar_wait(&empty[s], ((kb / S::STAGES) & 1) ^ 1, p.status, kDevTimeoutEmpty)) break;
            issued = kb + 1;
            uint8_t* sA = smem + s * S::STAGE_BYTES;
            uint8_t* sB = sA + S::A_BYTES;
            const int k0 = kb * S::BK;
            mbar_arrive_expect_tx(&full[s], S::STAGE_BYTES);
            if (A_MN) {
#pragma unroll
                for (int j = 0; j < S::BM / 64; j++) tma_load_3d(sA + j * 8192, &tmA, m0 + 64 * j, k0, b, &full[s]);
            } else {
                tma_load_3d(sA, &tmA, k0, m0, b, &full[s]);
            }
            if (B_MN) {
#pragma unroll
                for (int j = 0; j < S::BN / 64; j++) tma_load_3d(sB + j * 8192, &tmB, n0 + 64 * j, k0, b, &full[s]);
            } else {
                tma_load_3d(sB, &tmB, k0, n0, b, &full[s]);
            }
        }
        // every issued copy has landed before this CTA can exit
        for (int kb = issued - S::STAGES < 0 ? 0 : issued - S::STAGES; kb < issued; kb++)
            mbar_wait(&full[kb % S::STAGES], (kb / S::STAGES) & 1, p.status, kDevTimeoutFull);
    } else if (warp == 1 && lane == 0) {
        constexpr uint32_t idesc = idesc_f16_f32(S::BN, A_MN, B_MN);
        for (int kb = 0; kb < nk; kb++) {
            const int s = kb % S::STAGES;
            if (!mbar_wait(&full[s], (kb / S::STAGES) & 1, p.status, kDevTimeoutFull)) break;
            tc_fence_after();
            const uint32_t aBase = smem_u32(smem + s * S::STAGE_BYTES), bBase = aBase + S::A_BYTES;
#pragma unroll
            for (int kk = 0; kk < 4; kk++) {
                const uint64_t ad = A_MN ? smem_desc_sw128(aBase + kk * 2048, 8192, 1024)
                                         : smem_desc_sw128(aBase + kk * 32, 16, 1024);
                const uint64_t bd = B_MN ? smem_desc_sw128(bBase + kk * 2048, 8192, 1024)
                                         : smem_desc_sw128(bBase + kk * 32, 16, 1024);
                tc_mma_bf16(tmem, ad, bd, idesc, (kb > 0 || kk > 0) ? 1u : 0u);  // kind::f16: the types are idesc's
            }
            tc_commit(&empty[s]);
        }
        tc_commit(done);  // covers every MMA issued, also after a timeout
    }
    __syncwarp();
    const bool ready = mbar_wait_warp(done, 0, p.status, kDevTimeoutDone);
    tc_fence_after();
    const int row = m0 + warp * 32 + lane;
    if (ready) {
#pragma unroll 1
        for (int c = 0; c < S::BN / 32; c++) {
            float v[32];
            tmem_ld32(tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)(c * 32), v);
            const int col = n0 + c * 32;
            if (row < p.M && col < p.N) ns_epilogue<KIND>(p, b, row, col, blockIdx.x > blockIdx.y, v);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, S::BN);
    }
}

}  // namespace mg
