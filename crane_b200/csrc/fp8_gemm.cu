// Codes x codes^T with a scale for each block of 128:  out[m, n] = add[m, n] + sum_b xs[m, b] ws[n / 128, b] sum_{k in b} x[m, k] w[n, k]
//
// The products of a block of 128 columns go through tcgen05.mma (kind::f8f6f4, four of K = 32) into accumulator columns of their own; epilogue warps read those,
// multiply by the block's scale and add them up in f32 registers, while the MMAs fill the next ones.
//
// f8_rows_kernel: 128 weight rows are the MMA's M, up to 2 CW activation rows its N.  All 128 weight rows of a tile share a scale, an activation row's scale is a
// column's: xs * ws of a warp's columns lies in a patch of shared memory that its lanes fill a block ahead.  Fewer tiles than CTAs fit the chip: a cluster
// shares a tile along K and adds its partial tiles through distributed shared memory, every CTA finishing its share of the columns.
#include "fp8.cuh"
#include "tc.cuh"

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace cb {
namespace cg = cooperative_groups;

int f8_err_word(cudaStream_t st, int** out) {
    // a stream's first word may pin memory, which a capture in its strict modes forbids the thread
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    if (const cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode)) return (int)e;
    const int r = tc_err_word(st, out);
    cudaThreadExchangeStreamCaptureMode(&mode);
    return r;
}

struct F8Epi { void* out; const void* add; long long ldo, ldadd; int type; };
__device__ __forceinline__ void f8_put(const F8Epi& e, long long m, int n, float v) {
    if (e.type == F8_F32) {
        if (e.add) v += static_cast<const float*>(e.add)[m * e.ldadd + n];
        static_cast<float*>(e.out)[m * e.ldo + n] = v;
    } else if (e.type == F8_BF16) {
        if (e.add) v += __bfloat162float(static_cast<const bf16*>(e.add)[m * e.ldadd + n]);
        static_cast<bf16*>(e.out)[m * e.ldo + n] = __float2bfloat16_rn(v);
    } else {
        if (e.add) v += __half2float(static_cast<const __half*>(e.add)[m * e.ldadd + n]);
        static_cast<__half*>(e.out)[m * e.ldo + n] = __float2half_rn(v);
    }
}

constexpr int F8_W_BYTES = 128 * 128;
constexpr int F8_EPI = 8;                          // epilogue warps: two have the columns of a quarter of the lanes
struct F8RowsArgs {
    F8Epi ep;
    const float *xs, *ws;
    long long lds, ldws;
    int M, N, KB, nstg, nbuf, cl;
    bool w_static;
    int* err;
};
// CW: activation rows an epilogue warp has; tiles of 2 CW.  Two CTAs an SM while CW <= 32 (113 KB and 256 TMEM columns each).
template <int CW> struct F8RowsCfg {
    static constexpr int NT = 2 * CW, STAGE = F8_W_BYTES + NT * 128;
    static constexpr int BUDGET = (CW <= 32 ? 108 : 200) * 1024, PATCH = F8_EPI * 2 * CW * 4;
    static constexpr int STAGES = (BUDGET - PATCH) / STAGE < 8 ? (BUDGET - PATCH) / STAGE : 8;
    static constexpr int COLS = CW <= 32 ? 256 : 512, BUFS = COLS / NT < 8 ? COLS / NT : 8;
    static constexpr int MAIN = STAGES * STAGE > NT * 512 ? STAGES * STAGE : NT * 512;     // (a partial tile takes the stages' place)
    static constexpr int SMEM = MAIN + PATCH + 1024;
};

//   warp 0: TMA producer    warp 1: TMEM allocator and MMA issuer    warps 2 - 9: epilogue (TMEM lanes 32 (warp % 4) .., CW columns)
template <int CW>
__global__ void __launch_bounds__(64 + 32 * F8_EPI, CW <= 32 ? 2 : 1)
f8_rows_gemm_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const F8RowsArgs a) {
    using Cfg = F8RowsCfg<CW>;
    constexpr int NT = Cfg::NT, STAGE = Cfg::STAGE, STAGES = Cfg::STAGES, BUFS = Cfg::BUFS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[STAGES], empty[STAGES], d_full[BUFS], d_empty[BUFS];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const TcWait wait{&gave_up, a.err};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % a.cl, n0 = blockIdx.x / a.cl * 128, m0 = blockIdx.y * NT;
    const int kb0 = (int)((long long)rank * a.KB / a.cl), kb1 = (int)((long long)(rank + 1) * a.KB / a.cl);

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < BUFS; ++i) { mbar_init(&d_full[i], 1); mbar_init(&d_empty[i], F8_EPI); }
        fence_barrier_init();
    }
    if (warp == 1) { tmem_alloc(&tmem_slot, Cfg::COLS); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch_dependents();

    float acc[CW];
    const int q = warp & 3, part = (warp - 2) >> 2;
    if (warp == 0) {
        if (lane == 0) {
            tma_prefetch_desc(&tmW); tma_prefetch_desc(&tmX);
            const int npre = a.w_static ? min(kb1 - kb0, STAGES) : 0;
            for (int i = 0; i < npre; ++i) {
                mbar_arrive_expect_tx(&full[i], STAGE);
                tma_load_2d(sm + i * STAGE, &tmW, &full[i], (kb0 + i) * 128, n0);
            }
            pdl_wait();
            int s = 0; uint32_t ph = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (kb - kb0 >= npre) {
                    wait(&empty[s], ph ^ 1);
                    mbar_arrive_expect_tx(&full[s], STAGE);
                    tma_load_2d(sm + s * STAGE, &tmW, &full[s], kb * 128, n0);
                }
                tma_load_2d(sm + s * STAGE + F8_W_BYTES, &tmX, &full[s], kb * 128, m0);
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
            wait.drain();
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = make_idesc_e4m3(128, NT);
        int s = 0, b = 0; uint32_t ph = 0, bph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            wait(&d_empty[b], bph ^ 1);
            wait(&full[s], ph);
            tc_fence_after();
            const uint32_t at = smem_u32(sm + s * STAGE);
            const uint64_t wd = make_smem_desc_sw128(at), xd = make_smem_desc_sw128(at + F8_W_BYTES);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_e4m3(tmem + (uint32_t)(b * NT), wd + (uint64_t)(2 * k), xd + (uint64_t)(2 * k), idesc, (uint32_t)(k != 0));
                umma_commit(&empty[s]);
                umma_commit(&d_full[b]);
            }
            __syncwarp();
            if (++s == STAGES) { s = 0; ph ^= 1; }
            if (++b == BUFS) { b = 0; bph ^= 1; }
        }
    } else {
        pdl_wait();
        float* patch = reinterpret_cast<float*>(sm + Cfg::MAIN) + (warp - 2) * 2 * CW;
        const float* xs = a.xs + m0 + part * CW;
        const float* ws = a.ws + (long long)(n0 / 128) * a.ldws;
        constexpr int PER = (CW + 31) / 32;
        float nx[PER];
        auto fetch = [&](int kb) {                  // scales of this lane's columns
            const float w = __ldg(ws + kb);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int c = lane + 32 * i;
                nx[i] = (CW >= 32 || c < CW) && m0 + part * CW + c < a.M ? w * __ldg(xs + kb * a.lds + c) : 0.f;
            }
        };
        fetch(kb0);
#pragma unroll
        for (int j = 0; j < CW; ++j) acc[j] = 0.f;
        int b = 0; uint32_t bph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            float* mine = patch + ((kb - kb0) & 1) * CW;
#pragma unroll
            for (int i = 0; i < PER; ++i) if (CW >= 32 || lane < CW) mine[lane + 32 * i] = nx[i];
            if (kb + 1 < kb1) fetch(kb + 1);
            __syncwarp();
            wait(&d_full[b], bph);
            tc_fence_after();
            const uint32_t d = tmem + (uint32_t)(b * NT + part * CW) + ((uint32_t)(q * 32) << 16);
            constexpr int STEP = CW < 16 ? 8 : 16;
#pragma unroll
            for (int c = 0; c < CW; c += STEP) {
                uint32_t r[STEP];
                if constexpr (STEP == 8) tmem_ld8_async(d + c, r); else tmem_ld16_async(d + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < STEP; j += 4) {
                    const float4 sc = *reinterpret_cast<const float4*>(mine + c + j);
                    acc[c + j] = fmaf(__uint_as_float(r[j]), sc.x, acc[c + j]);
                    acc[c + j + 1] = fmaf(__uint_as_float(r[j + 1]), sc.y, acc[c + j + 1]);
                    acc[c + j + 2] = fmaf(__uint_as_float(r[j + 2]), sc.z, acc[c + j + 2]);
                    acc[c + j + 3] = fmaf(__uint_as_float(r[j + 3]), sc.w, acc[c + j + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&d_empty[b]);
            if (++b == BUFS) { b = 0; bph ^= 1; }
        }
        const int n = n0 + q * 32 + lane;
        if (a.cl == 1) {
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                const int m = m0 + part * CW + j;
                if (m < a.M && n < a.N) f8_put(a.ep, m, n, acc[j]);
            }
        } else {
            // every stage has landed and been read: this CTA's MMAs are complete
            named_bar_sync(1, 32 * F8_EPI);
#pragma unroll
            for (int j = 0; j < CW; ++j) reinterpret_cast<float*>(sm)[(part * CW + j) * 128 + q * 32 + lane] = acc[j];
        }
    }
    if (a.cl > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        __syncwarp();
        cluster.sync();
        if (warp >= 2) {
            const int row = q * 32 + lane, n = n0 + row;
            for (int c = rank + part * a.cl; c < NT && m0 + c < a.M; c += 2 * a.cl) {
                float v = 0.f;
                for (int r = 0; r < a.cl; ++r) v += cluster.map_shared_rank(reinterpret_cast<float*>(sm), r)[c * 128 + row];
                if (n < a.N) f8_put(a.ep, m0 + c, n, v);
            }
        }
        __syncwarp();
        cluster.sync();                              // nobody leaves while its shared memory is still being read
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, Cfg::COLS); }
}

template <int CW>
static int f8_rows_gemm_t(cudaStream_t st, const F8Linear& p, int M, int N, int K, bool pdl) {
    using Cfg = F8RowsCfg<CW>;
    F8RowsArgs a = {};
    a.ep = F8Epi{p.out, p.add, p.ldo, p.ldadd, p.type};
    a.xs = p.x.scales; a.lds = p.x.lds; a.ws = p.ws; a.ldws = p.ldws;
    a.M = M; a.N = N; a.KB = f8_blocks(K); a.w_static = p.w_static;
    if (const int e = f8_err_word(st, &a.err)) return e;
    CUtensorMap tmW, tmX;
    if (!tc_tmap_encode(&tmW, p.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)N, (uint64_t)K, (uint64_t)p.ldw, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tc_tmap_encode(&tmX, p.x.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)M, (uint64_t)K, (uint64_t)p.x.ld, Cfg::NT, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return -1001;
    const int tn = (N + 127) / 128, tm = (M + Cfg::NT - 1) / Cfg::NT;
    if (tm > 65535) return -1000;
    const long long tiles = (long long)tn * tm, slots = (long long)tc_device_sms() * (CW <= 32 ? 2 : 1);
    a.cl = (int)std::max<long long>(1, std::min<long long>(std::min(8, a.KB), slots / tiles));
    static SmemOptIn seen;
    if (const int e = ensure_dyn_smem(f8_rows_gemm_kernel<CW>, (size_t)Cfg::SMEM, seen)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tn * a.cl, tm); cfg.blockDim = dim3(64 + 32 * F8_EPI); cfg.dynamicSmemBytes = Cfg::SMEM; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (a.cl > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = a.cl; attr[na].val.clusterDim.y = 1; attr[na].val.clusterDim.z = 1;
        ++na;
    }
    if (pdl) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        ++na;
    }
    cfg.attrs = attr; cfg.numAttrs = na;
    return (int)cudaLaunchKernelEx(&cfg, f8_rows_gemm_kernel<CW>, tmW, tmX, a);
}

int f8_linear_launch(cudaStream_t st, const F8Linear& p, int M, int N, int K, bool pdl) {
    if (M == 0 || N == 0) return 0;
    if (M <= 16) return f8_rows_gemm_t<8>(st, p, M, N, K, pdl);
    if (M <= 32) return f8_rows_gemm_t<16>(st, p, M, N, K, pdl);
    if (M <= 64) return f8_rows_gemm_t<32>(st, p, M, N, K, pdl);
    return f8_rows_gemm_t<64>(st, p, M, N, K, pdl);
}

}  // namespace cb
