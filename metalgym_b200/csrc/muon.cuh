// The tcgen05 products of a Newton-Schulz step (muon.cu): operands of two fp16
// parts, fp32 accumulation in tensor memory, persistent CTAs that walk 128 x BN
// output tiles with the accumulator double-buffered in tensor memory, so that
// the epilogue of one tile runs beside the products of the next.
//
// An operand V is hi + lo, hi = fp16(V) and lo = fp16(V - hi): 22 bits. A
// product is lo hi + hi lo + hi hi, three products of fp16 matrices that share
// their loads: a K block of the lo parts of both operands and one of their hi
// parts follow one another through the ring of stages. Two 16-bit matrices are
// also what X, G and B are to memory: the lo parts of a batch lie behind its
// hi parts, so that part and matrix together are a tensor map's third
// coordinate.
//
//   kNsGram   G = X X^T or X^T X, symmetric: only tiles that reach the diagonal
//             or lie above it are computed, and written to both places
//   kNsPoly   B = b G + c G G, likewise symmetric
//   kNsApply  X <- a X + B X or a X + X B, or in the last step what the caller
//             wants of it
//
// Warp roles: 0 TMA producer, 1 MMA issuer, the others epilogue (warp w:
// accumulator lanes 32 (w % 4) .., a part of the columns): 16 at 128-wide tiles,
// where small matrices wait for it, 8 at 256-wide ones, where it runs beside
// the next tile and shared memory is better spent on a fourth stage.
// The epilogue takes 32 x 32 pieces from tensor memory through a swizzled
// 4 KB slab of shared memory: a thread of tcgen05.ld has a row, and rows are
// far apart in memory; out of the slab, eight lanes hold 32 consecutive columns
// of a row, so that X (fp32 and fp16) and G move in whole 128- and 64-byte
// lines. With a row a thread, the same epilogue took 30 us a launch at 128 x 512.
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
    int vec;           // every group of four columns of a row is 16-byte (fp32) and 8-byte (16-bit) aligned
    float keep, rate;  // master = master * keep - rate * X
};

struct NsProduct {
    int M, N, K, batch;
    int tilesM, tilesN;
    int ldo;            // row stride of out16, g16 and x32 (a multiple of 8)
    __half* out16;      // [hi, lo][batch][M][ldo], scaled
    const __half* g16;  // kNsPoly, likewise
    float* x32;         // kNsApply
    float a, b, c;
    int last;
    NsFinal fin;
    int* status;
};

// A tile of 128 x BN. A stage is 64 columns of K of one part of both operands.
template <int BN>
struct NsTile {
    static constexpr int BK = 64, STAGES = BN == 256 ? 4 : 5;
    static constexpr int A_BYTES = 128 * BK * 2, B_BYTES = BN * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int EW = BN == 256 ? 8 : 16, THREADS = 64 + 32 * EW, SLAB = 4096;
    static constexpr int PIECES = BN / (8 * EW);  // 32-column pieces of an epilogue warp
    static constexpr int SLAB_OFF = STAGES * STAGE_BYTES, BAR_OFF = SLAB_OFF + EW * SLAB;
    static constexpr int TMEM_COLS = 2 * BN;
    static constexpr int SMEM_BYTES = BAR_OFF + 256 + 1024 /*align*/;
    static_assert(SMEM_BYTES > 225 * 1024, "no other CTA that holds tensor memory beside it (as in MuonSmall)");
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

// Tiles of one matrix, and the u-th of them; of a symmetric product only those
// that do not lie wholly below the diagonal.
template <int KIND, int BN>
__host__ __device__ __forceinline__ int ns_tiles(int tilesM, int tilesN) {
    if (KIND == kNsApply) return tilesM * tilesN;
    int n = 0;
    for (int i = 0; i < tilesM; i++) n += tilesN - i * 128 / BN;
    return n;
}
template <int KIND, int BN>
__device__ __forceinline__ void ns_tile_at(int u, int tilesN, int& i, int& j) {
    if (KIND == kNsApply) {
        i = u / tilesN;
        j = u % tilesN;
        return;
    }
    i = 0;
    while (u >= tilesN - i * 128 / BN) {
        u -= tilesN - i * 128 / BN;
        i++;
    }
    j = i * 128 / BN + u;
}

__device__ __forceinline__ uint32_t ns_slab_offset(int r, int k) { return (uint32_t)(r * 128 + ((k ^ (r & 7)) << 4)); }

__device__ __forceinline__ uint2 pack_half4(float a, float b, float c, float d) {
    const __half2 x = __floats2half2_rn(a, b), y = __floats2half2_rn(c, d);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// Four values (already scaled) as two parts, `lo` elements apart.
__device__ __forceinline__ void store_parts4(__half* hi, int64_t lo, float a, float b, float c, float d) {
    const uint2 h = pack_half4(a, b, c, d);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h.x)), y = __half22float2(*reinterpret_cast<const __half2*>(&h.y));
    *reinterpret_cast<uint2*>(hi) = h;
    *reinterpret_cast<uint2*>(hi + lo) = pack_half4(a - x.x, b - x.y, c - y.x, d - y.y);
}
// Likewise eight, from 16-byte boundaries on.
__device__ __forceinline__ void store_parts8(__half* hi, int64_t lo, const float* v) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 a = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        const float2 f = __half22float2(a);
        const __half2 b = __floats2half2_rn(v[2 * i] - f.x, v[2 * i + 1] - f.y);
        h[i] = *reinterpret_cast<const uint32_t*>(&a);
        l[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(hi) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(hi + lo) = make_uint4(l[0], l[1], l[2], l[3]);
}
// The sum of four values' parts.
__device__ __forceinline__ float4 parts_sum4(const uint2& h, const uint2& l) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&h.y));
    const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&l.x)), d = __half22float2(*reinterpret_cast<const __half2*>(&l.y));
    return make_float4(a.x + c.x, a.y + c.y, b.x + d.x, b.y + d.y);
}
// B = b G + c G G, scaled by 2^10 as G is; y: the product's accumulator, times 2^-10.
__device__ __forceinline__ float4 ns_poly4(const NsProduct& p, const float4& y, const float4& g) {
    return make_float4(fmaf(p.c, y.x, p.b * g.x), fmaf(p.c, y.y, p.b * g.y), fmaf(p.c, y.z, p.b * g.z), fmaf(p.c, y.w, p.b * g.w));
}
// Elements from the hi to the lo parts of the product's output (and of G).
__device__ __forceinline__ int64_t ns_lo(const NsProduct& p) { return (int64_t)p.batch * p.M * p.ldo; }

// Four columns (from col on) of a row of X; v: the accumulator, x and master:
// what was read there (x 0 where X is not kept).
__device__ __forceinline__ void ns_apply4(const NsProduct& p, int64_t at, int64_t finAt, int col, const float4& v, const float4& x,
                                          const float4& master, bool finVec) {
    float y[4] = {v.x, v.y, v.z, v.w};
    const float xv[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = fmaf(p.a, xv[i], y[i] * (kNsUnscale * kNsUnscale));
    if (!p.last) {
        *reinterpret_cast<float4*>(p.x32 + at) = make_float4(y[0], y[1], y[2], y[3]);
        store_parts4(p.out16 + at, ns_lo(p), y[0] * kNsScale, y[1] * kNsScale, y[2] * kNsScale, y[3] * kNsScale);
        return;
    }
    const int n = min(4, p.N - col);
    const bool vec = finVec && n == 4;
    if (p.fin.master) {
        float* m = p.fin.master + finAt;
        if (vec) {
            const float mv[4] = {master.x, master.y, master.z, master.w};
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = __fsub_rn(__fmul_rn(mv[i], p.fin.keep), __fmul_rn(p.fin.rate, y[i]));
            *reinterpret_cast<float4*>(m) = make_float4(y[0], y[1], y[2], y[3]);
            const __nv_bfloat162 a = __floats2bfloat162_rn(y[0], y[1]), b = __floats2bfloat162_rn(y[2], y[3]);
            *reinterpret_cast<uint2*>(p.fin.weights + finAt) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < n) {
                    const float w = __fsub_rn(__fmul_rn(m[i], p.fin.keep), __fmul_rn(p.fin.rate, y[i]));
                    m[i] = w;
                    p.fin.weights[finAt + i] = __float2bfloat16_rn(w);
                }
        }
    } else if (p.fin.outBf16) {
        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.fin.out) + finAt;
        if (vec) {
            const __nv_bfloat162 a = __floats2bfloat162_rn(y[0], y[1]), b = __floats2bfloat162_rn(y[2], y[3]);
            *reinterpret_cast<uint2*>(o) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < n) o[i] = __float2bfloat16_rn(y[i]);
        }
    } else {
        __half* o = static_cast<__half*>(p.fin.out) + finAt;
        if (vec) {
            *reinterpret_cast<uint2*>(o) = pack_half4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < n) o[i] = __float2half_rn(y[i]);
        }
    }
}

// What the epilogue of a 32 x 32 piece reads: four columns of eight rows a lane
// (eight lanes to a row). It does not depend on the product, so the loads go
// out before the accumulator is waited for.
template <int KIND>
struct NsFetched {
    float4 x[KIND == kNsApply ? 8 : 1];
    uint2 g[KIND == kNsPoly ? 8 : 1], gLo[KIND == kNsPoly ? 8 : 1];
};
template <int KIND>
__device__ __forceinline__ void ns_fetch(const NsProduct& p, int b, int row0, int col0, NsFetched<KIND>& f) {
    const int lane = threadIdx.x & 31, col = col0 + 4 * (lane & 7);
    const int64_t at = ((int64_t)b * p.M + row0 + (lane >> 3)) * p.ldo + col;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (KIND == kNsApply) f.x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (KIND == kNsPoly) f.g[i] = f.gLo[i] = make_uint2(0u, 0u);
        if (col < p.N && row0 + 4 * i + (lane >> 3) < p.M) {
            if (KIND == kNsApply) f.x[i] = ld_f4_now(p.x32 + at + (int64_t)(4 * i) * p.ldo);
            if (KIND == kNsPoly) {
                f.g[i] = *reinterpret_cast<const uint2*>(p.g16 + at + (int64_t)(4 * i) * p.ldo);
                f.gLo[i] = *reinterpret_cast<const uint2*>(p.g16 + ns_lo(p) + at + (int64_t)(4 * i) * p.ldo);
            }
        }
    }
}

// A 32 x 32 piece at (row0, col0) of matrix b's output: lane r holds row r in v.
// Of a symmetric product, pieces below the diagonal are left to their mirror
// pieces above it, which write both: every entry is written once.
template <int KIND>
__device__ __forceinline__ void ns_piece(const NsProduct& p, int b, int row0, int col0, uint8_t* slab, const float* v,
                                         const NsFetched<KIND>& f) {
    const int lane = threadIdx.x & 31;
    __syncwarp();  // the slab's last readers are done
#pragma unroll
    for (int k = 0; k < 8; k++)
        *reinterpret_cast<float4*>(slab + ns_slab_offset(lane, k)) = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    __syncwarp();
    const int64_t base = (int64_t)b * p.M * p.ldo;
    const int k = lane & 7, col = col0 + 4 * k;
    const bool finVec = KIND == kNsApply && p.last && p.fin.vec;
    const bool mirror = KIND != kNsApply && col0 != row0;
    if (col < p.N) {  // then the four columns lie inside ldo
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float4 m[4];
            if (KIND == kNsApply) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int row = row0 + (4 * h + i) * 4 + (lane >> 3);
                    m[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (finVec && p.fin.master && col + 4 <= p.N && row < p.M)
                        m[i] = ld_f4_now(p.fin.master + (int64_t)b * p.fin.stride + (int64_t)row * p.fin.ld + col);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = (4 * h + i) * 4 + (lane >> 3), row = row0 + r;
                float4* cell = reinterpret_cast<float4*>(slab + ns_slab_offset(r, k));
                float4 y = *cell;
                if constexpr (KIND == kNsApply) {
                    if (row < p.M)
                        ns_apply4(p, base + (int64_t)row * p.ldo + col, (int64_t)b * p.fin.stride + (int64_t)row * p.fin.ld + col, col, y,
                                  p.x32 ? f.x[4 * h + i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f), m[i], finVec);
                } else {
                    y.x *= kNsUnscale;  // scaled by 2^10, as the operands are
                    y.y *= kNsUnscale;
                    y.z *= kNsUnscale;
                    y.w *= kNsUnscale;
                    if constexpr (KIND == kNsPoly) y = ns_poly4(p, y, parts_sum4(f.g[4 * h + i], f.gLo[4 * h + i]));
                    if (row < p.M) store_parts4(p.out16 + base + (int64_t)row * p.ldo + col, ns_lo(p), y.x, y.y, y.z, y.w);
                    if (mirror) *cell = y;
                }
            }
        }
    }
    if (!mirror) return;
    __syncwarp();
    // the mirrored piece, row col0 + lane: column row0 + r is this piece's (r, lane)
    const int mrow = col0 + lane;
    if (mrow < p.M) {
        const int64_t at = base + (int64_t)mrow * p.ldo + row0;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (row0 + 8 * q >= p.ldo) break;
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
                y[i] = *reinterpret_cast<const float*>(slab + ns_slab_offset(8 * q + i, lane >> 2) + (lane & 3) * 4);
            store_parts8(p.out16 + at + 8 * q, ns_lo(p), y);
        }
    }
}

// The three products of a K block by one thread: the mixed ones, whose lo stage
// is then free, and that of the hi parts. (The accumulator is cut off, not
// rounded, at every instruction.)
template <int BN, bool A_MN, bool B_MN>
__device__ __forceinline__ void ns_mma_block(uint32_t acc, uint32_t lo, uint32_t hi, uint64_t* emptyLo, uint64_t* emptyHi, bool accumulate) {
    constexpr uint32_t idesc = idesc_f16_f32(BN, A_MN, B_MN);
#pragma unroll
    for (int part = 0; part < 3; part++) {
        const uint32_t a = part == 0 ? lo : hi, b = (part == 1 ? lo : hi) + NsTile<BN>::A_BYTES;
#pragma unroll
        for (int kk = 0; kk < 4; kk++) {
            const uint64_t ad = A_MN ? smem_desc_sw128(a + kk * 2048, 8192, 1024) : smem_desc_sw128(a + kk * 32, 16, 1024);
            const uint64_t bd = B_MN ? smem_desc_sw128(b + kk * 2048, 8192, 1024) : smem_desc_sw128(b + kk * 32, 16, 1024);
            // kind::f16: the types are idesc's
            tc_mma_bf16(acc, ad, bd, idesc, accumulate || part > 0 || kk > 0 ? 1u : 0u);
        }
        if (part == 1) tc_commit(emptyLo);
    }
    tc_commit(emptyHi);
}
// One part (matrix z of the tensor maps) of a K block of both operands into a stage.
template <int BN, bool A_MN, bool B_MN>
__device__ __forceinline__ void ns_load_stage(uint8_t* sA, const CUtensorMap* tmA, const CUtensorMap* tmB, int m0, int n0, int k0, int z,
                                              uint64_t* full) {
    uint8_t* sB = sA + NsTile<BN>::A_BYTES;
    mbar_arrive_expect_tx(full, NsTile<BN>::STAGE_BYTES);
    if (A_MN) {
        tma_load_3d(sA, tmA, m0, k0, z, full);
        tma_load_3d(sA + 8192, tmA, m0 + 64, k0, z, full);
    } else {  // a box of 128 rows
        tma_load_3d(sA, tmA, k0, m0, z, full);
    }
    if (B_MN) {
#pragma unroll
        for (int j = 0; j < BN / 64; j++) tma_load_3d(sB + j * 8192, tmB, n0 + 64 * j, k0, z, full);
    } else {
#pragma unroll
        for (int j = 0; j < BN / 128; j++) tma_load_3d(sB + j * 16384, tmB, k0, n0 + 128 * j, z, full);
    }
}

template <int KIND, int BN, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(NsTile<BN>::THREADS, 1)
    k_ns_product(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const NsProduct p) {
    using S = NsTile<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::BAR_OFF);
    uint64_t* empty = full + S::STAGES;
    uint64_t* tfull = empty + S::STAGES;  // [2]
    uint64_t* tempty = tfull + 2;         // [2]
    uint64_t* done = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    mg_pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int perMatrix = ns_tiles<KIND, BN>(p.tilesM, p.tilesN), units = perMatrix * p.batch;
    const int nk = (p.K + S::BK - 1) / S::BK;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], S::EW);
        }
        mbar_init(done, 1);
        fence_barrier_init();
        prefetch_tensormap(&tmA);
        prefetch_tensormap(&tmB);
    }
    if (warp == 2) {
        tmem_alloc(tmem_slot, S::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    mg_pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
                const int b = u / perMatrix;
                int ti, tj;
                ns_tile_at<KIND, BN>(u - b * perMatrix, p.tilesN, ti, tj);
                for (int h = 0; h < 2 * nk; h++, it++) {  // the lo, then the hi part of each K block
                    const int s = it % S::STAGES;
                    if (!mbar_wait(&empty[s], ((it / S::STAGES) & 1) ^ 1, p.status, kDevTimeoutEmpty)) {
                        ok = false;
                        break;
                    }
                    ns_load_stage<BN, A_MN, B_MN>(smem + s * S::STAGE_BYTES, &tmA, &tmB, ti * 128, tj * BN, (h >> 1) * S::BK,
                                                  (h & 1) ? b : b + p.batch, &full[s]);
                }
            }
            // every issued copy has landed before this CTA can exit
            for (int k = it - S::STAGES < 0 ? 0 : it - S::STAGES; k < it; k++)
                mbar_wait(&full[k % S::STAGES], (k / S::STAGES) & 1, p.status, kDevTimeoutFull);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int it = 0, t = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < units && ok; u += gridDim.x, t++) {
                const int a = t & 1;
                if (!mbar_wait(&tempty[a], ((t >> 1) & 1) ^ 1, p.status, kDevTimeoutEmpty)) break;
                tc_fence_after();
                for (int kb = 0; kb < nk; kb++, it += 2) {
                    const int lo = it % S::STAGES, hi = (it + 1) % S::STAGES;
                    if (!mbar_wait(&full[lo], (it / S::STAGES) & 1, p.status, kDevTimeoutFull) ||
                        !mbar_wait(&full[hi], ((it + 1) / S::STAGES) & 1, p.status, kDevTimeoutFull)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    ns_mma_block<BN, A_MN, B_MN>(tmem + (uint32_t)(a * BN), smem_u32(smem + lo * S::STAGE_BYTES),
                                                 smem_u32(smem + hi * S::STAGE_BYTES), &empty[lo], &empty[hi], kb > 0);
                }
                if (ok) tc_commit(&tfull[a]);
            }
            tc_commit(done);  // covers every MMA issued, also after a timeout
        }
    } else {
        bool gaveUp = false;  // a wait gave up
        const int q = warp & 3, e = warp - 2, part = (e / 4) * (BN * 4 / S::EW);
        uint8_t* slab = smem + S::SLAB_OFF + e * S::SLAB;
        int t = 0;
        for (int u = blockIdx.x; u < units; u += gridDim.x, t++) {
            const int b = u / perMatrix, a = t & 1;
            int ti, tj;
            ns_tile_at<KIND, BN>(u - b * perMatrix, p.tilesN, ti, tj);
            const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(a * BN + part);
#pragma unroll 1
            for (int c = 0; c < S::PIECES; c++) {
                const int at = 32 * c, row0 = ti * 128 + 32 * q, col0 = tj * BN + part + at;
                const bool wanted = row0 < p.M && col0 < p.N && (KIND == kNsApply || col0 >= row0);
                NsFetched<KIND> f;
                if (wanted) ns_fetch<KIND>(p, b, row0, col0, f);
                __syncwarp();  // lanes at a matrix's edge took other branches; loads from tensor memory take whole warps
                if (c == 0) {
                    if (!mbar_wait_warp(&tfull[a], (t >> 1) & 1, p.status, kDevTimeoutDone)) gaveUp = true;
                    if (gaveUp) break;
                    tc_fence_after();
                }
                float v[32];
                tmem_ld32(acc + (uint32_t)at, v);
                if (c == S::PIECES - 1) {  // the accumulator is free for the next tile that uses it
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&tempty[a]);
                }
                if (wanted) ns_piece<KIND>(p, b, row0, col0, slab, v, f);
            }
            if (gaveUp) break;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        mbar_wait_warp(done, 0, p.status, kDevTimeoutDone);
        tc_fence_after();
        tmem_dealloc(tmem, S::TMEM_COLS);
    }
}

// Products of few tiles with K split over the CTAs of a cluster, one 128 x 128
// tile per cluster: a tile's operands come at about 55 bytes a cycle and SM
// from L2, 1180 cycles for a K block whose products take 768, so that few tiles
// with a long K leave most of that rate unused. Every CTA leaves its part of
// the sum in the slabs; CTA r then adds the parts of rows 32 r / splits .. of
// each piece, in their order, and writes them. (512 x 2048: 295 -> 166 us.)
template <int KIND, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(NsTile<128>::THREADS, 1)
    k_ns_split(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const NsProduct p, int splits) {
    using S = NsTile<128>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::BAR_OFF);
    uint64_t* empty = full + S::STAGES;
    uint64_t* done = empty + S::STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    mg_pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % splits, unit = blockIdx.x / splits;
    const int perMatrix = ns_tiles<KIND, 128>(p.tilesM, p.tilesN), b = unit / perMatrix;
    int ti, tj;
    ns_tile_at<KIND, 128>(unit - b * perMatrix, p.tilesN, ti, tj);
    const int m0 = ti * 128, n0 = tj * 128;
    const int blocks = (p.K + S::BK - 1) / S::BK;
    const int kFirst = (int)((int64_t)blocks * rank / splits), kEnd = (int)((int64_t)blocks * (rank + 1) / splits);
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
        tmem_alloc(tmem_slot, 128);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    mg_pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            for (; it < 2 * (kEnd - kFirst); it++) {  // the lo, then the hi part of each K block
                const int s = it % S::STAGES;
                if (!mbar_wait(&empty[s], ((it / S::STAGES) & 1) ^ 1, p.status, kDevTimeoutEmpty)) break;
                ns_load_stage<128, A_MN, B_MN>(smem + s * S::STAGE_BYTES, &tmA, &tmB, m0, n0, (kFirst + (it >> 1)) * S::BK,
                                               (it & 1) ? b : b + p.batch, &full[s]);
            }
            // every issued copy has landed before this CTA can exit
            for (int k = it - S::STAGES < 0 ? 0 : it - S::STAGES; k < it; k++)
                mbar_wait(&full[k % S::STAGES], (k / S::STAGES) & 1, p.status, kDevTimeoutFull);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            for (int it = 0; it < 2 * (kEnd - kFirst); it += 2) {
                const int lo = it % S::STAGES, hi = (it + 1) % S::STAGES;
                if (!mbar_wait(&full[lo], (it / S::STAGES) & 1, p.status, kDevTimeoutFull) ||
                    !mbar_wait(&full[hi], ((it + 1) / S::STAGES) & 1, p.status, kDevTimeoutFull))
                    break;
                tc_fence_after();
                ns_mma_block<128, A_MN, B_MN>(tmem, smem_u32(smem + lo * S::STAGE_BYTES), smem_u32(smem + hi * S::STAGE_BYTES), &empty[lo],
                                              &empty[hi], it > 0);
            }
            tc_commit(done);  // covers every MMA issued, also after a timeout
        }
    }
    const int e = warp - 2, q = warp & 3, row0 = m0 + 32 * q, col0 = n0 + 32 * (e / 4);
    const bool wanted = e >= 0 && row0 < p.M && col0 < p.N && (KIND == kNsApply || col0 >= row0);
    const bool mirror = KIND != kNsApply && wanted && col0 != row0, finVec = KIND == kNsApply && p.last && p.fin.vec;
    uint8_t* slab = smem + S::SLAB_OFF + (e < 0 ? 0 : e) * S::SLAB;
    if (wanted) {
        mbar_wait_warp(done, 0, p.status, kDevTimeoutDone);
        tc_fence_after();
        float v[32];
        tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(32 * (e / 4)), v);
#pragma unroll
        for (int k = 0; k < 8; k++)
            *reinterpret_cast<float4*>(slab + ns_slab_offset(lane, k)) = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    }
    __syncwarp();
    cluster_sync();
    const int share = 32 / splits, first = rank * share;  // rows of a piece that this CTA writes
    const int64_t base = (int64_t)b * p.M * p.ldo;
    if (wanted) {
        const int k = lane & 7, col = col0 + 4 * k;
        for (int r = first + (lane >> 3); r < first + share; r += 4) {
            const int row = row0 + r;
            const bool in = row < p.M && col < p.N;
            uint2 gw = make_uint2(0u, 0u), gLo = gw;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), m = x;
            const int64_t finAt = (int64_t)b * p.fin.stride + (int64_t)row * p.fin.ld + col;
            if (KIND == kNsPoly && in) {
                gw = *reinterpret_cast<const uint2*>(p.g16 + base + (int64_t)row * p.ldo + col);
                gLo = *reinterpret_cast<const uint2*>(p.g16 + ns_lo(p) + base + (int64_t)row * p.ldo + col);
            }
            if (KIND == kNsApply && in) {
                x = ld_f4_now(p.x32 + base + (int64_t)row * p.ldo + col);
                if (finVec && p.fin.master && col + 4 <= p.N) m = ld_f4_now(p.fin.master + finAt);
            }
            const uint32_t off = ns_slab_offset(r, k);
            float4 y = *reinterpret_cast<const float4*>(cluster_peer(slab, 0) + off);
            for (int z = 1; z < splits; z++) {
                const float4 o = *reinterpret_cast<const float4*>(cluster_peer(slab, z) + off);
                y.x += o.x;
                y.y += o.y;
                y.z += o.z;
                y.w += o.w;
            }
            if (KIND == kNsApply) {
                if (in) ns_apply4(p, base + (int64_t)row * p.ldo + col, finAt, col, y, x, m, finVec);
                continue;
            }
            y.x *= kNsUnscale;
            y.y *= kNsUnscale;
            y.z *= kNsUnscale;
            y.w *= kNsUnscale;
            if (KIND == kNsPoly) y = ns_poly4(p, y, parts_sum4(gw, gLo));
            if (in) store_parts4(p.out16 + base + (int64_t)row * p.ldo + col, ns_lo(p), y.x, y.y, y.z, y.w);
            // (rows `first` .. of this CTA's slab are read by nobody else)
            if (mirror) *reinterpret_cast<float4*>(slab + off) = y;
        }
        __syncwarp();
        const int mrow = col0 + lane;  // the mirrored piece, as in ns_piece
        if (mirror && mrow < p.M) {
            for (int r = first; r < first + share && row0 + r < p.ldo; r += 8) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; i++)
                    y[i] = *reinterpret_cast<const float*>(slab + ns_slab_offset(r + i, lane >> 2) + (lane & 3) * 4);
                store_parts8(p.out16 + base + (int64_t)mrow * p.ldo + row0 + r, ns_lo(p), y);
            }
        }
    }
    __syncwarp();    // (the cluster's barrier takes whole warps)
    cluster_sync();  // no CTA leaves while another reads its slabs
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        mbar_wait_warp(done, 0, p.status, kDevTimeoutDone);
        tc_fence_after();
        tmem_dealloc(tmem, 128);
    }
}

}  // namespace mg
