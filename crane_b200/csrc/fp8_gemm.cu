// Codes x codes^T with a scale for each block of 128:  out[m, n] = add[m, n] + sum_b xs[m, b] ws[n / 128, b] sum_{k in b} x[m, k] w[n, k]
//
// The products of a block of 128 columns go through tcgen05.mma (kind::f8f6f4, four of K = 32) into accumulator columns of their own; epilogue warps read those,
// multiply by the block's scale and add them up in f32 registers, while the MMAs fill the next ones.
//
// f8_rows_gemm_kernel, up to some hundred rows: 128 weight rows are the MMA's M, up to 128 activation rows its N.  All weight rows of a tile share a scale, an activation
// row's scale is a column's: xs * ws of a warp's columns lies in a patch of shared memory that its lanes fill a stage ahead.  Fewer tiles than SMs: a cluster shares a tile
// along K and adds its partial tiles through distributed shared memory.
// f8_pair_kernel, more rows: tiles of 256 x 256 over pairs of CTAs, a kernel for each way the results leave.
#include "fp8.cuh"
#include "fp8_tiles.h"
#include "tc.cuh"

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

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

// A load that stays where it is written, ahead of waits that it overlaps (the compiler may move __ldg down to its use), of what the kernel ahead has written
__device__ __forceinline__ float f8_fetch(const float* p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}

// An accumulator has been read: behind tcgen05.wait::ld its values are in registers, so all that the arrival orders is the next MMAs' writes behind these reads, which have happened.  Nothing
// that this thread wrote is handed over with it, so it may be a relaxed one; as a release at cluster scope it waited, once a block of K, for everything the thread had in flight.
__device__ __forceinline__ void f8_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }

struct F8Epi { void* out; const void* add; long long ldo, ldadd; int type; };
template <typename T> __device__ __forceinline__ T f8_round(float v);
template <> __device__ __forceinline__ float f8_round<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 f8_round<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half f8_round<__half>(float v) { return __float2half_rn(v); }
__device__ __forceinline__ float f8_wide(float v) { return v; }
__device__ __forceinline__ float f8_wide(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float f8_wide(__half v) { return __half2float(v); }

// columns n .. n + 3 of row m; `vec`: they lie on the boundary that a vector store wants
template <typename T>
__device__ __forceinline__ void f8_put4_t(const F8Epi& e, bool vec, int N, long long m, int n, const float* s) {
    T* o = static_cast<T*>(e.out) + m * e.ldo + n;
    const T* a = e.add ? static_cast<const T*>(e.add) + m * e.ldadd + n : nullptr;
    if (vec && n + 4 <= N) {
        using V = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
        alignas(16) T h[4];
        if (a) *reinterpret_cast<V*>(h) = *reinterpret_cast<const V*>(a);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = f8_round<T>(a ? f8_wide(h[i]) + s[i] : s[i]);
        *reinterpret_cast<V*>(o) = *reinterpret_cast<const V*>(h);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (n + i < N) o[i] = f8_round<T>(a ? f8_wide(a[i]) + s[i] : s[i]);
    }
}
__device__ __forceinline__ void f8_put4(const F8Epi& e, bool vec, int N, long long m, int n, const float* s) {
    if (e.type == F8_F32) f8_put4_t<float>(e, vec, N, m, n, s);
    else if (e.type == F8_BF16) f8_put4_t<bf16>(e, vec, N, m, n, s);
    else f8_put4_t<__half>(e, vec, N, m, n, s);
}

constexpr int F8_W_BYTES = 128 * 128;
constexpr int F8_EPI = 8;                          // epilogue warps: two have the columns of a quarter of the lanes
constexpr int F8_CH = 2;                           // blocks of K a stage: the issuing warp pays as much for a stage's waits and commits as for its MMAs
struct F8RowsArgs {
    F8Epi ep;
    const float *xs, *ws;
    long long lds, ldws;
    int M, N, KB, cl, tiles_n;
    bool vec, w_static;
    int* err;
};
// Tiles of NT = 2 CW activation rows; an epilogue warp has CW of them.  Two CTAs an SM while CW <= 24 (113 KB and 256 TMEM columns each, so that what fits an SM by
// its shared memory fits it by its TMEM).
template <int CW, int OCC> struct F8RowsCfg {
    static constexpr int NT = 2 * CW, PART = F8_W_BYTES + NT * 128, STAGE = F8_CH * PART;           // PART: a block of K
    static constexpr int TILE = NT * 512;                                                           // a tile of f32 sums
    static constexpr bool PUSH = CW == 8;
    static constexpr int ROOM = PUSH ? 21 * 512 : 0;                                                // sums that other CTAs send: ceil(NT / cl) x cl rows
    static constexpr int PATCH = F8_EPI * 2 * F8_CH * CW * 4;
    static constexpr int BUDGET = (OCC == 2 ? 110 : 216) * 1024, STAGES = (BUDGET - PATCH - ROOM) / STAGE;
    static constexpr int MAIN = STAGES * STAGE > TILE ? STAGES * STAGE : TILE, SMEM = MAIN + PATCH + ROOM + 1024;      // (the tile takes the stages' place)
    static constexpr int COLS = OCC == 2 ? 256 : 512, STEP = CW <= 8 ? 16 : CW <= 16 ? 32 : CW <= 32 ? 64 : 128;
    static constexpr int BUFS = COLS / (F8_CH * STEP) < 8 ? COLS / (F8_CH * STEP) : 8;
    static_assert(STAGES >= 2 && BUFS >= 2 && SMEM <= (OCC == 2 ? 112 : 226) * 1024, "fits");
};

// U rows of a tile, `step` rows apart, whose partial sums lie R times, at p[r] + row * 128 floats: added in the order of r and stored, four columns a lane.
template <int R, int U, typename P>
__device__ __forceinline__ void f8_join(const F8Epi& e, bool vec, int N, int rows, int first, int step, int m0, int n, P&& at) {
    for (int c = first; c < rows; c += U * step) {
        float4 v[R][U];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int u = 0; u < U; ++u) v[r][u] = c + u * step < rows ? at(r, c + u * step) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (c + u * step >= rows) break;
            float s[4] = {v[0][u].x, v[0][u].y, v[0][u].z, v[0][u].w};
#pragma unroll
            for (int r = 1; r < R; ++r) { s[0] += v[r][u].x; s[1] += v[r][u].y; s[2] += v[r][u].z; s[3] += v[r][u].w; }
            f8_put4(e, vec, N, m0 + c + u * step, n, s);
        }
    }
}

//   warp 0: TMA producer    warp 1: TMEM allocator and MMA issuer    warps 2 - 9: epilogue (TMEM lanes 32 (warp % 4) .., CW columns)
template <int CW, int OCC>
__global__ void __launch_bounds__(64 + 32 * F8_EPI, OCC)
f8_rows_gemm_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const F8RowsArgs a) {
    using Cfg = F8RowsCfg<CW, OCC>;
    constexpr int NT = Cfg::NT, PART = Cfg::PART, STAGE = Cfg::STAGE, STAGES = Cfg::STAGES, BUFS = Cfg::BUFS, STEP = Cfg::STEP;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[STAGES], empty[STAGES], d_full[BUFS], d_empty[BUFS];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const TcWait wait{&gave_up, a.err};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % a.cl, tile = blockIdx.x / a.cl, n0 = tile % a.tiles_n * 128, m0 = tile / a.tiles_n * NT;
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
    __syncwarp();
    if (Cfg::PUSH && a.cl > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");     // (this CTA is there: others may write to its memory)
    pdl_launch_dependents();

    const int q = warp & 3, part = (warp - 2) >> 2, rows = min(NT, a.M - m0);
    if (warp == 0) {
        if (lane == 0) {
            tma_prefetch_desc(&tmW); tma_prefetch_desc(&tmX);
            auto weights = [&](int kb, int st) {
                const int n = min(F8_CH, kb1 - kb);
                mbar_arrive_expect_tx(&full[st], n * PART);
                for (int c = 0; c < n; ++c) tma_load_2d(sm + st * STAGE + c * PART, &tmW, &full[st], (kb + c) * 128, n0);
            };
            const int npre = a.w_static ? STAGES : 0;
            for (int i = 0; i < npre && kb0 + i * F8_CH < kb1; ++i) weights(kb0 + i * F8_CH, i);
            pdl_wait();
            int s = 0; uint32_t ph = 0;
            for (int kb = kb0, i = 0; kb < kb1; kb += F8_CH, ++i) {
                if (i >= npre) { wait(&empty[s], ph ^ 1); weights(kb, s); }
                for (int c = 0; c < min(F8_CH, kb1 - kb); ++c) tma_load_2d(sm + s * STAGE + c * PART + F8_W_BYTES, &tmX, &full[s], (kb + c) * 128, m0);
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
            wait.drain();
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = make_idesc_e4m3(128, NT);
        int s = 0, b = 0; uint32_t ph = 0, bph = 0;
        for (int kb = kb0; kb < kb1; kb += F8_CH) {
            wait(&d_empty[b], bph ^ 1);
            wait(&full[s], ph);
            tc_fence_after();
            const uint32_t at = smem_u32(sm + s * STAGE), d = tmem + (uint32_t)(b * F8_CH * STEP);
            const bool two = kb + 1 < kb1;
            if (elect_one()) {
                static_assert(F8_CH == 2, "the last stage may have one");
                const uint64_t wd = make_smem_desc_sw128(at), xd = make_smem_desc_sw128(at + F8_W_BYTES);
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_e4m3(d, wd + (uint64_t)(2 * k), xd + (uint64_t)(2 * k), idesc, (uint32_t)(k != 0));
                if (two) {
                    const uint64_t wd1 = make_smem_desc_sw128(at + PART), xd1 = make_smem_desc_sw128(at + PART + F8_W_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_e4m3(d + STEP, wd1 + (uint64_t)(2 * k), xd1 + (uint64_t)(2 * k), idesc, (uint32_t)(k != 0));
                }
                umma_commit(&empty[s]);
                umma_commit(&d_full[b]);
            }
            __syncwarp();
            if (++s == STAGES) { s = 0; ph ^= 1; }
            if (++b == BUFS) { b = 0; bph ^= 1; }
        }
        // TMEM is given back as soon as it has been read: a CTA that waits for its cluster holds none that another cluster's CTA may be waiting for
        named_bar_sync(2, 32 + 32 * F8_EPI);
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::COLS);
    } else {
        pdl_wait();
        float* patch = reinterpret_cast<float*>(sm + Cfg::MAIN + Cfg::ROOM) + (warp - 2) * 2 * F8_CH * CW;
        const float* ws = a.ws + (long long)(n0 / 128) * a.ldws;
        constexpr int PER = (CW + 31) / 32;
        const float* xs[PER];                       // scales of the columns that this lane fetches for its warp (behind the last: any)
#pragma unroll
        for (int i = 0; i < PER; ++i) xs[i] = a.xs + min(m0 + part * CW + min(lane + 32 * i, CW - 1), a.M - 1);
        float nx[2][F8_CH][PER], nw[2][F8_CH];      // of the next stage and the one behind it: a stage of few rows takes less time than a load
        auto fetch = [&](int u, int kb) {
#pragma unroll
            for (int c = 0; c < F8_CH; ++c) {
                const int k = min(kb + c, kb1 - 1);
                nw[u][c] = f8_fetch(ws + k);
#pragma unroll
                for (int i = 0; i < PER; ++i) nx[u][c][i] = f8_fetch(xs[i] + k * a.lds);
            }
        };
        fetch(0, kb0); fetch(1, kb0 + F8_CH);
        uint64_t acc[CW / 2];                       // pairs of columns
#pragma unroll
        for (int j = 0; j < CW / 2; ++j) acc[j] = 0;
        int b = 0; uint32_t bph = 0;
        for (int k0 = kb0; k0 < kb1; k0 += 2 * F8_CH)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int kb = k0 + u * F8_CH;
            if (kb >= kb1) break;
            float* mine = patch + u * F8_CH * CW;
#pragma unroll
            for (int c = 0; c < F8_CH; ++c)
#pragma unroll
                for (int i = 0; i < PER; ++i) if (CW % 32 == 0 || lane + 32 * i < CW) mine[c * CW + lane + 32 * i] = nx[u][c][i] * nw[u][c];
            if (kb + 2 * F8_CH < kb1) fetch(u, kb + 2 * F8_CH);
            __syncwarp();
            wait(&d_full[b], bph);
            tc_fence_after();
#pragma unroll
            for (int h = 0; h < F8_CH; ++h) {
                if (h > 0 && kb + h >= kb1) break;
                const uint32_t d = tmem + (uint32_t)((b * F8_CH + h) * STEP + part * CW) + ((uint32_t)(q * 32) << 16);
                const float* scales = mine + h * CW;
                constexpr int GRP = CW % 32 == 0 ? 32 : CW % 24 == 0 ? 24 : CW;           // columns read at a time
#pragma unroll
                for (int c = 0; c < CW; c += GRP) {
                    uint32_t r[GRP];
#pragma unroll
                    for (int i = 0; i + 16 <= GRP; i += 16) tmem_ld16_async(d + c + i, r + i);
                    if constexpr (GRP % 16 == 8) tmem_ld8_async(d + c + GRP - 8, r + GRP - 8);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < GRP; j += 4) {
                        const ulonglong2 sc = *reinterpret_cast<const ulonglong2*>(scales + c + j);
                        acc[(c + j) / 2] = f2_fma(f2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), sc.x, acc[(c + j) / 2]);
                        acc[(c + j) / 2 + 1] = f2_fma(f2(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])), sc.y, acc[(c + j) / 2 + 1]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) f8_arrive(smem_u32(&d_empty[b]));
            if (++b == BUFS) { b = 0; bph ^= 1; }
        }
        tc_fence_before();
        asm volatile("bar.arrive 2, %0;" ::"n"(32 + 32 * F8_EPI) : "memory");
        // the sums, a row of 128 a column of the tile: to the CTA that finishes the row, or in place of this CTA's stages (its MMAs are complete, all of them)
        const int row0 = part * CW;
        if (Cfg::PUSH && a.cl > 1) {
            asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
            const uint32_t room = smem_u32(sm + Cfg::MAIN) + (uint32_t)(rank * 128 + q * 32 + lane) * 4;
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                float lo, hi;
                f2_split(acc[j / 2], lo, hi);
                const int c = row0 + j;
                if (c < rows) {
                    uint32_t to;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(room + (uint32_t)(c / a.cl * a.cl * 512)), "r"(c % a.cl));
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(j & 1 ? hi : lo) : "memory");
                }
            }
        } else {
            float* tile = reinterpret_cast<float*>(sm) + q * 32 + lane;
#pragma unroll
            for (int j = 0; j < CW; j += 2) {
                float lo, hi;
                f2_split(acc[j / 2], lo, hi);
                tile[(row0 + j) * 128] = lo;
                tile[(row0 + j + 1) * 128] = hi;
            }
            if (a.cl == 1) {
                named_bar_sync(1, 32 * F8_EPI);
                f8_join<1, 4>(a.ep, a.vec, a.N, rows, warp - 2, F8_EPI, m0, n0 + 4 * lane, [&](int, int c) { return reinterpret_cast<const float4*>(sm)[c * 32 + lane]; });
            }
        }
    }
    __syncwarp();
    if (a.cl > 1) {
        if (Cfg::PUSH) {
            if (warp < 2) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
            cluster_sync_all();                      // the other CTAs' sums are here; nobody touches this CTA's memory any more
            if (warp >= 2) {
                const int i = warp - 2;              // row i of this CTA's is the tile's row rank + i cl
                const float4* p = reinterpret_cast<const float4*>(sm + Cfg::MAIN) + (size_t)i * a.cl * 32 + lane;
                if (rank + i * a.cl < rows) {
                    float4 v[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) v[r] = r < a.cl ? p[r * 32] : make_float4(0.f, 0.f, 0.f, 0.f);
                    float s[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
                    for (int r = 1; r < 8; ++r) { s[0] += v[r].x; s[1] += v[r].y; s[2] += v[r].z; s[3] += v[r].w; }
                    f8_put4(a.ep, a.vec, a.N, m0 + rank + i * a.cl, n0 + 4 * lane, s);
                }
            }
        } else {
            cluster_sync_all();
            if (warp >= 2) {
                cg::cluster_group cluster = cg::this_cluster();
                const int first = rank * F8_EPI + warp - 2, step = a.cl * F8_EPI;
                float4* mine = reinterpret_cast<float4*>(sm) + lane;
                auto at = [&](int r, int c) { return r < a.cl ? cluster.map_shared_rank(mine, r)[c * 32] : make_float4(0.f, 0.f, 0.f, 0.f); };
                if (a.cl <= 2) f8_join<2, 4>(a.ep, a.vec, a.N, rows, first, step, m0, n0 + 4 * lane, at);
                else if (a.cl <= 4) f8_join<4, 2>(a.ep, a.vec, a.N, rows, first, step, m0, n0 + 4 * lane, at);
                else f8_join<8, 1>(a.ep, a.vec, a.N, rows, first, step, m0, n0 + 4 * lane, at);
            }
            __syncwarp();
            cluster_sync_all();                      // nobody leaves while its shared memory is still being read
        }
    }
}

static bool f8_vec_out(const F8Linear& p) {
    const long long e = f8_bytes(p.type);
    return reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.ldo * e % 16 == 0 && (!p.add || (reinterpret_cast<uintptr_t>(p.add) % 16 == 0 && p.ldadd * e % 16 == 0));
}

template <int CW, int OCC>
static int f8_rows_smem() {
    static SmemOptIn seen;
    return ensure_dyn_smem(f8_rows_gemm_kernel<CW, OCC>, (size_t)F8RowsCfg<CW, OCC>::SMEM, seen);
}

// CTAs that share a tile: as many as fit the chip with every tile at work at once (clusters live inside a GPC, so not all SMs take part: of sixteen SMs' worth of
// clusters of eight, two CTAs an SM, 33 fit), more than two blocks of K each.  us for 2 / 4 / 6 / 8 CTAs a tile: 1 row, 4096 x 2048 5.6 / 4.8 / 4.7 / 5.0, 2048 x 6144 10.0 / 6.9 / 6.0 / 5.8,
// 4096 x 12288 18.8 / 12.7 / 11.5 / 10.5; 6144 x 4096 (48 tiles; 45 clusters of six fit) 9.1 / 7.2 / 11.1 / 10.1; 12288 x 2048 (96 tiles; 93 of three) 1: 8.4, 2: 7.2, 3: 11.1.
template <int CW, int OCC>
static int f8_rows_cluster(long long tiles, int KB) {
    static std::atomic<int> known[CB_MAX_DEV][9];
    int dev = 0, best = 1;
    if (f8_rows_smem<CW, OCC>() || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= CB_MAX_DEV) return 1;
    for (int cl = 2; cl <= 8 && 2 * cl < KB; ++cl) {
        int n = known[dev][cl].load(std::memory_order_relaxed);
        if (!n) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(cl); cfg.blockDim = dim3(64 + 32 * F8_EPI); cfg.dynamicSmemBytes = F8RowsCfg<CW, OCC>::SMEM;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = cl; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr; cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&n, f8_rows_gemm_kernel<CW, OCC>, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
            known[dev][cl].store(++n, std::memory_order_relaxed);
        }
        if (tiles <= n - 1) best = cl;
    }
    return best;
}

template <int CW, int OCC>
static int f8_rows_gemm_t(cudaStream_t st, const F8Linear& p, int M, int N, int K, bool pdl) {
    using Cfg = F8RowsCfg<CW, OCC>;
    F8RowsArgs a = {};
    a.ep = F8Epi{p.out, p.add, p.ldo, p.ldadd, p.type};
    a.xs = p.x.scales; a.lds = p.x.lds; a.ws = p.ws; a.ldws = p.ldws;
    a.M = M; a.N = N; a.KB = f8_blocks(K); a.w_static = p.w_static; a.vec = f8_vec_out(p);
    a.err = p.err;
    if (!a.err) if (const int e = f8_err_word(st, &a.err)) return e;
    CUtensorMap tmW, tmX;
    if (!tc_tmap_encode(&tmW, p.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)N, (uint64_t)K, (uint64_t)p.ldw, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tc_tmap_encode(&tmX, p.x.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)M, (uint64_t)K, (uint64_t)p.x.ld, Cfg::NT, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return -1001;
    const long long tiles = (long long)((N + 127) / 128) * ((M + Cfg::NT - 1) / Cfg::NT);
    if (tiles > 0x0fffffffLL) return -1000;
    a.tiles_n = (N + 127) / 128;
    if (const int e = f8_rows_smem<CW, OCC>()) return e;
    a.cl = f8_rows_cluster<CW, OCC>(tiles, a.KB);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * a.cl)); cfg.blockDim = dim3(64 + 32 * F8_EPI); cfg.dynamicSmemBytes = Cfg::SMEM; cfg.stream = st;
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
    return (int)cudaLaunchKernelEx(&cfg, f8_rows_gemm_kernel<CW, OCC>, tmW, tmX, a);
}

// =====================================================================================
// Many activation rows: tiles of 256 rows x 256 weight rows over a pair of CTAs (cta_group::2).  A CTA has 128 of the activation rows and brings half of the weight rows;
// an epilogue thread has one activation row and half of the columns, so that its scale is one product a block of K.
// A persistent pair an SM pair takes tiles in turn; MMAs run up to two blocks of K ahead of the epilogue, into the next tile too.  Tiles left over for the last turn, or
// for the only one, are cut into 2 or 4 strips of columns when that many pairs are free.
// What bounds it (8192 x 24576 x 4096: 705 - 730 us in some calls, 2 340 TFLOP/s; 843 in seconds of them, 1 960, at the 1.2 - 1.28 GHz that the power limit leaves; the MMAs and stores alone
// 2 700 at 1.3 GHz): the two accumulators.  A block's MMAs take 512 cycles, its epilogue 440 (TMEM reads and 256 FMA issues a scheduler, next to MMAs that read and write the same TMEM), the
// hand-overs between them (commit, wait, arrival at the even CTA) some 600 more, so that a block passes every 800.  Measured and left: two MMAs of 128 columns, for four accumulators
// (1 850 TFLOP/s; by themselves MMAs of 256, 128 and 64 columns take 128, 64 and 43 cycles), sixteen epilogue warps, 32 columns a read, two producers, two issuing warps (no gain).
// =====================================================================================
struct F8PairArgs {
    F8Epi ep;
    const float *xs, *ws;
    long long lds, ldws;
    int M, N, KB, tiles_m, tiles_n, pairs;
    int whole, items, cut;             // tiles 0 .. whole - 1 as they are, then strips of 256 / cut columns: `items` together
    bool tma, w_static;
    int* err;
};
struct F8PairCfg {
    static constexpr int A_BYTES = 128 * 128, STAGE = A_BYTES + 128 * 128, PATCH = F8_EPI * 8192;
    static constexpr int STAGES = (226 * 1024 - PATCH - 1024) / STAGE;
    static constexpr int SMEM = STAGES * STAGE + PATCH + 1024;
};
// 32 rows x up to C columns of a warp (those below N), a row a lane, through a patch of 32 x 32 f32 (16-byte pieces swizzled by the row), so that stores (and the addend's loads) cover
// pieces of rows.  The addition is f32.  Addends are read ahead of all stores: result and addend may be the same memory, so the compiler keeps a load behind every store that is written
// before it (8192 x 24576 x 64 f32 669 us so, 345 ahead).
template <typename T, int C, bool ADD>
__device__ __forceinline__ void f8_store_rows(const F8Epi& e, int M, int N, int m0, int n0, const float* v, uint8_t* patch, int lane) {
    using V = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
    const int r0 = lane >> 3, p0 = lane & 7;
#pragma unroll
    for (int c = 0; c < C; c += 32) {
        if (n0 + c >= N) break;
#pragma unroll
        for (int p = 0; p < 8; ++p) *reinterpret_cast<float4*>(patch + sw128_off(lane, p)) = make_float4(v[c + 4 * p], v[c + 4 * p + 1], v[c + 4 * p + 2], v[c + 4 * p + 3]);
        __syncwarp();
        const int n = n0 + c + p0 * 4;
        const T* add = ADD ? static_cast<const T*>(e.add) + n : nullptr;
        V g[8];
        if (ADD && n + 4 <= N) {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (m0 + 4 * i + r0 < M) g[i] = *reinterpret_cast<const V*>(add + (long long)(m0 + 4 * i + r0) * e.ldadd);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + r0, m = m0 + r;
            const float4 u = *reinterpret_cast<const float4*>(patch + sw128_off(r, p0));
            if (m >= M || n >= N) continue;
            T* o = static_cast<T*>(e.out) + (long long)m * e.ldo + n;
            const float w[4] = {u.x, u.y, u.z, u.w};
            if (n + 4 <= N) {
                alignas(16) T h[4];
                if (ADD) *reinterpret_cast<V*>(h) = g[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = f8_round<T>(ADD ? f8_wide(h[j]) + w[j] : w[j]);
                *reinterpret_cast<V*>(o) = *reinterpret_cast<const V*>(h);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) if (n + j < N) o[j] = f8_round<T>(ADD ? f8_wide(add[(long long)m * e.ldadd + j]) + w[j] : w[j]);
            }
        }
        __syncwarp();
    }
}

// The same for rows that lie on no 16-byte boundaries: a value a lane, a row at a time.  Addends are read eight rows at a time, ahead of those rows' stores: result and addend may be the
// same memory, so the compiler keeps a load behind every store that is written before it.
template <typename P, typename T, int C>
__device__ __forceinline__ void f8_store_odd(const F8Epi& e, int M, int N, int m0, int n0, const float* v, uint8_t* patch, int lane) {
    constexpr int PER = 16 / (int)sizeof(P), W = 8 * PER;
    const T* add = sizeof(P) == 4 ? static_cast<const T*>(e.add) : nullptr;
    const int rows = min(32, M - m0);
#pragma unroll
    for (int c = 0; c < C; c += W) {
        if (n0 + c >= N) break;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            alignas(16) P h[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) h[i] = f8_round<P>(c + p * PER + i < C ? v[c + p * PER + i < C ? c + p * PER + i : 0] : 0.f);
            *reinterpret_cast<uint4*>(patch + sw128_off(lane, p)) = *reinterpret_cast<const uint4*>(h);
        }
        __syncwarp();
        for (int q = lane; q < W && n0 + c + q < N; q += 32) {
            const int at = q * (int)sizeof(P), n = n0 + c + q;
            T* o = static_cast<T*>(e.out) + (long long)m0 * e.ldo + n;
            const T* a = add ? add + (long long)m0 * e.ldadd + n : nullptr;
#pragma unroll 1
            for (int r = 0; r < rows; r += 8) {
                T x[8];
                if (add) {
#pragma unroll
                    for (int i = 0; i < 8; ++i, a += e.ldadd) if (r + i < rows) x[i] = *a;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i, o += e.ldo) {
                    const float h = f8_wide(*reinterpret_cast<const P*>(patch + sw128_off(r + i, at >> 4) + (at & 15)));
                    if (r + i < rows) *o = f8_round<T>(add ? f8_wide(x[i]) + h : h);
                }
            }
        }
        __syncwarp();
    }
}

// The same rows by TMA, two pieces of 128 bytes a row under way: the tiles of all SMs end together, and what they store then (64 KB each) takes the chip longer than the two blocks
// of K that the MMAs run ahead.
template <typename T, int C>
__device__ __forceinline__ void f8_store_tma(const CUtensorMap* map, int M, int N, int m0, int n0, const float* v, uint8_t* patch, uint32_t& phases, int lane) {
    constexpr int PER = 16 / (int)sizeof(T), W = 8 * PER;
#pragma unroll
    for (int c = 0; c < C; c += W) {
        if (n0 + c >= N || m0 >= M) break;
        uint8_t* to = patch + f8_half(phases) * 4096;
        if (lane == 0) tma_store_wait_read<1>();
        __syncwarp();
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            alignas(16) T h[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) h[i] = f8_round<T>(v[c + p * PER + i]);
            *reinterpret_cast<uint4*>(to + sw128_off(lane, p)) = *reinterpret_cast<const uint4*>(h);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) { tma_store_2d(map, to, n0 + c, m0); tma_store_commit(); }
        f8_half_stored(phases);
    }
}

// One tile, or strip, of an epilogue warp: C columns of each lane's row
// How results leave has a kernel each: with other ways beside its own, the loop over K comes out slower (8192 x 24576 x 4096 bf16 745 us with all three in one, so 711)
enum { F8_PLAIN, F8_ADD, F8_ODD };                    // rows on 16-byte boundaries without an addend, with one, rows on others
struct F8Ring { uint64_t *full, *empty; int b; uint32_t phases; };
template <int C, typename T, int WAY>
__device__ __forceinline__ void f8_pair_tile(const F8PairArgs& a, const CUtensorMap* tmO, const float* xs, const float* ws, uint32_t lanes, F8Ring& ring, const TcWait& wait, int m0, int n0, int N,
                                             uint8_t* patch, int lane) {
    constexpr int BUFS = 256 / C;
    if (WAY != F8_PLAIN && a.ep.add && m0 + lane < a.M) {      // the addend's lines come to L2 while the MMAs run (8192 x 24576 x 64 f32 421 us without, 345 so)
        const char* row = reinterpret_cast<const char*>(static_cast<const T*>(a.ep.add) + (long long)(m0 + lane) * a.ep.ldadd + n0);
        for (int c = 0; c < (N - n0) * (int)sizeof(T); c += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + c));
    }
    float v[C];
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = 0.f;
    // scales are on their way AHEAD blocks of K before their use: a narrow strip's block takes less time than a load
    constexpr int AHEAD = C == 128 ? 1 : 2;
    float nx[AHEAD], nw[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        nx[u] = f8_fetch(xs); nw[u] = f8_fetch(ws);
        if (u + 1 < a.KB) { xs += a.lds; ++ws; }
    }
    for (int k0 = 0; k0 < a.KB; k0 += AHEAD)
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        const int kb = k0 + u;
        if (kb >= a.KB) break;
        const float sc = nx[u] * nw[u];
        wait(&ring.full[ring.b], (ring.phases >> ring.b) & 1);
        tc_fence_after();
        const uint32_t d = lanes + (uint32_t)(ring.b * 2 * C);
        uint32_t r[2][16];
        tmem_ld16_async(d, r[0]);
        if (kb + AHEAD < a.KB) { nx[u] = f8_fetch(xs); nw[u] = f8_fetch(ws); xs += a.lds; ++ws; }
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < C; c += 16) {
            const int k = (c >> 4) & 1;
            if (c + 16 < C) tmem_ld16_async(d + c + 16, r[k ^ 1]);
#pragma unroll
            for (int j = 0; j < 16; j += 2)
                f2_split(f2_fma(f2(__uint_as_float(r[k][j]), __uint_as_float(r[k][j + 1])), f2(sc, sc), f2(v[c + j], v[c + j + 1])), v[c + j], v[c + j + 1]);
            if (c + 16 < C) tmem_ld_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) f8_arrive(peer_smem(&ring.empty[ring.b], 0));
        ring.phases ^= 1u << ring.b;
        if (++ring.b == BUFS) ring.b = 0;
    }
    if constexpr (WAY == F8_PLAIN && C * sizeof(T) >= 128) {
        if (a.tma) { f8_store_tma<T, C>(tmO, a.M, N, m0, n0, v, patch, ring.phases, lane); return; }
    }
    if (lane == 0) tma_store_wait_read<0>();          // (the whole tiles' stores have left the patch)
    __syncwarp();
    if constexpr (WAY != F8_ODD) f8_store_rows<T, C, WAY == F8_ADD>(a.ep, a.M, N, m0, n0, v, patch, lane);
    else if (a.ep.add) f8_store_odd<float, T, C>(a.ep, a.M, N, m0, n0, v, patch, lane);
    else f8_store_odd<T, T, C>(a.ep, a.M, N, m0, n0, v, patch, lane);
}

// Registers: 384 threads x 168 at the launch = 128 x 72 (warps 0 - 3) + 256 x 216 (the epilogue: 128 sums and 32 of the next products a thread)
constexpr int F8_PAIR_THREADS = 128 + 32 * F8_EPI, F8_REGS_LOW = 72, F8_REGS_EPI = 216;
static_assert(128 * F8_REGS_LOW + 32 * F8_EPI * F8_REGS_EPI <= F8_PAIR_THREADS * 168, "the shares come out of the launch's registers");
//   warp 0: TMA producer    warp 1: TMEM allocator and (even CTA) MMA issuer    warps 4 - 11: epilogue (32 rows from 32 (warp % 4), half of the columns)
template <typename T, int WAY>
__global__ void __launch_bounds__(F8_PAIR_THREADS, 1) __cluster_dims__(2, 1, 1)
f8_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmW32,
               const __grid_constant__ CUtensorMap tmO, const F8PairArgs a) {
    using Cfg = F8PairCfg;
    constexpr int STAGE = Cfg::STAGE, STAGES = Cfg::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[STAGES];                 // of the even CTA: both CTAs' operands of a stage
    __shared__ uint64_t empty[STAGES], d_full[8];     // of each CTA
    __shared__ uint64_t d_empty[8];                   // of the even CTA: accumulator drained by the epilogue warps of both
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, KB = a.KB;
    const TcWait wait{&gave_up, a.err, peer_smem(&gave_up, rank ^ 1)};

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 8; ++i) { mbar_init(&d_full[i], 1); mbar_init(&d_empty[i], 2 * F8_EPI); }
        fence_barrier_init();
    }
    __syncwarp();
    if (warp == 1) { tmem_alloc_pair(&tmem_slot, 512); tmem_relinquish_pair(); }
    tc_fence_before();
    __syncthreads();
    __syncwarp();
    cluster_sync_all();                               // the pair's barriers are initialised before either CTA signals the other's
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch_dependents();

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F8_REGS_LOW));
        if (warp == 0 && lane == 0) {
            tma_prefetch_desc(&tmX); tma_prefetch_desc(&tmW); tma_prefetch_desc(&tmW32);
            auto weights = [&](int st, int kb, const F8Item& it) {
                const uint32_t bar = peer_smem(&full[st], 0);
                uint8_t* to = sm + st * STAGE + Cfg::A_BYTES;
                const int rows = it.width / 2, n = it.n0 + rank * rows;
                if (rank == 0) mbar_arrive_expect_tx(&full[st], 2 * (Cfg::A_BYTES + rows * 128));
                if (rows == 128) tma_load_2d_pair(to, &tmW, bar, kb * 128, n);
                else {
                    tma_load_2d_pair(to, &tmW32, bar, kb * 128, n);
                    if (rows == 64) tma_load_2d_pair(to + 32 * 128, &tmW32, bar, kb * 128, n + 32);
                }
            };
            int npre = 0, s = 0; uint32_t ph = 0;
            if (a.w_static) {                         // the weights' first stages go out before the dependency wait
                npre = min(KB, STAGES);
                const F8Item it = f8_item(a, pair);
                for (int i = 0; i < npre; ++i) weights(i, i, it);
            }
            pdl_wait();
            for (int i = pair; i < a.items; i += a.pairs) {
                const F8Item it = f8_item(a, i);
                const int m0 = it.mt * 256 + rank * 128;
                for (int kb = 0; kb < KB; ++kb) {
                    if (npre > 0) --npre;
                    else { wait(&empty[s], ph ^ 1); weights(s, kb, it); }
                    tma_load_2d_pair(sm + s * STAGE, &tmX, peer_smem(&full[s], 0), kb * 128, m0);
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
            }
        } else if (warp == 1 && rank == 0) {
            int s = 0, b = 0, width = 256; uint32_t ph = 0, phases = 0;       // phases: a bit an accumulator
            for (int i = pair; i < a.items; i += a.pairs) {
                const F8Item it = f8_item(a, i);
                if (it.width != width) {              // from whole tiles to strips: their accumulators lie elsewhere, so all have to be free
                    for (int o = 0; o < 512 / width; ++o) wait(&d_empty[o], ((phases >> o) & 1) ^ 1);
                    width = it.width; b = 0;
                }
                const uint32_t idesc = make_idesc_e4m3(256, width);
                for (int kb = 0; kb < KB; ++kb) {
                    wait(&full[s], ph);
                    wait(&d_empty[b], ((phases >> b) & 1) ^ 1);
                    tc_fence_after();
                    const uint32_t at = smem_u32(sm + s * STAGE);
                    const uint64_t xd = make_smem_desc_sw128(at), wd = make_smem_desc_sw128(at + Cfg::A_BYTES);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) umma_e4m3_pair(tmem + (uint32_t)(b * width), xd + (uint64_t)(2 * k), wd + (uint64_t)(2 * k), idesc, (uint32_t)(k != 0));
                        umma_commit_pair(&empty[s]);
                        umma_commit_pair(&d_full[b]);
                    }
                    __syncwarp();
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                    phases ^= 1u << b;
                    if (++b * width == 512) b = 0;
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F8_REGS_EPI));
        pdl_wait();
        const int q = warp & 3, part = (warp - 4) >> 2;
        uint8_t* patch = sm + STAGES * STAGE + (warp - 4) * 8192;
        int width = 256;
        F8Ring ring = {d_full, d_empty, 0, 0};
        for (int i = pair; i < a.items; i += a.pairs) {
            const F8Item it = f8_item(a, i);
            if (it.width != width) { width = it.width; ring.b = 0; }
            const int m0 = it.mt * 256 + rank * 128 + q * 32, cw = width / 2, n0 = it.n0 + part * cw;
            const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(part * cw);
            const float* xs = a.xs + min(m0 + lane, a.M - 1);
            const float* ws = a.ws + (long long)min(n0 / 128, (a.N - 1) / 128) * a.ldws;
            const int N = min(a.N, n0 + cw);
            if (width == 256) f8_pair_tile<128, T, WAY>(a, &tmO, xs, ws, lanes, ring, wait, m0, n0, N, patch, lane);
            else if (width == 128) f8_pair_tile<64, T, WAY>(a, &tmO, xs, ws, lanes, ring, wait, m0, n0, N, patch, lane);
            else f8_pair_tile<32, T, WAY>(a, &tmO, xs, ws, lanes, ring, wait, m0, n0, N, patch, lane);
        }
        if (lane == 0) tma_store_wait_read<0>();      // (the writes themselves are complete when the grid is)
    }
    tc_fence_before();
    __syncthreads();
    __syncwarp();
    cluster_sync_all();                               // neither CTA leaves while the other's MMAs read its operands or its warps signal here
    wait.drain();
    if (warp == 1) { tc_fence_after(); tmem_dealloc_pair(tmem, 512); }
}

template <typename T, int WAY>
static int f8_pair_t(cudaStream_t st, const F8Linear& p, int M, int N, int K, bool pdl) {
    using Cfg = F8PairCfg;
    F8PairArgs a = {};
    a.ep = F8Epi{p.out, p.add, p.ldo, p.ldadd, p.type};
    a.xs = p.x.scales; a.lds = p.x.lds; a.ws = p.ws; a.ldws = p.ldws;
    a.M = M; a.N = N; a.KB = f8_blocks(K); a.w_static = p.w_static;
    a.tiles_m = (M + 255) / 256; a.tiles_n = (N + 255) / 256;
    const int pairs = tc_device_sms() / 2;
    const F8Turns turns = f8_turns(M, N, pairs);
    a.whole = turns.whole; a.items = turns.items; a.cut = turns.cut;
    a.pairs = std::min(a.items, pairs);
    a.err = p.err;
    if (!a.err) if (const int err = f8_err_word(st, &a.err)) return err;
    CUtensorMap tmX, tmW, tmW32, tmO;
    if (!tc_tmap_encode(&tmX, p.x.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)M, (uint64_t)K, (uint64_t)p.x.ld, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tc_tmap_encode(&tmW, p.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)N, (uint64_t)K, (uint64_t)p.ldw, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tc_tmap_encode(&tmW32, p.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)N, (uint64_t)K, (uint64_t)p.ldw, 32, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return -1001;
    a.tma = WAY == F8_PLAIN && (long long)N * (long long)sizeof(T) % 16 == 0;      // (a row that ends inside 16 bytes would be written to their end)
    tmO = tmX;
    if (a.tma && !tc_tmap_encode(&tmO, p.out, std::is_same<T, float>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : std::is_same<T, bf16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                 (uint64_t)M, (uint64_t)N, (uint64_t)p.ldo, 32, 128 / sizeof(T), CU_TENSOR_MAP_SWIZZLE_128B)) return -1001;
    static SmemOptIn seen;
    if (const int err = ensure_dyn_smem(f8_pair_kernel<T, WAY>, (size_t)Cfg::SMEM, seen)) return err;
    return launch_k(f8_pair_kernel<T, WAY>, dim3(2 * a.pairs), dim3(F8_PAIR_THREADS), Cfg::SMEM, st, pdl, tmX, tmW, tmW32, tmO, a);
}
template <typename T>
static int f8_pair_p(cudaStream_t st, const F8Linear& p, int M, int N, int K, bool pdl) {
    if (!f8_vec_out(p)) return f8_pair_t<T, F8_ODD>(st, p, M, N, K, pdl);
    return p.add ? f8_pair_t<T, F8_ADD>(st, p, M, N, K, pdl) : f8_pair_t<T, F8_PLAIN>(st, p, M, N, K, pdl);
}
static int f8_pair_launch(cudaStream_t st, const F8Linear& p, int M, int N, int K, bool pdl) {
    switch (p.type) {
        case F8_F32:  return f8_pair_p<float>(st, p, M, N, K, pdl);
        case F8_BF16: return f8_pair_p<bf16>(st, p, M, N, K, pdl);
        case F8_F16:  return f8_pair_p<__half>(st, p, M, N, K, pdl);
        default: return -1000;
    }
}

// More than 64 rows: us by fits to what the kernels take (M x N x K, <CW 32> / <48> / <64> / pairs):
//   77 x 4096 x 2048 7.1 / 7.8 / 8.3 / 11.5   77 x 12288 x 2048 15.9 / 11.0 / 12.9 / 13.3   128 x 4096 x 12288 18.2 / 22.6 / 19.0 / 48   128 x 24576 x 4096 42 / 48 / 41 / 39
//   256 x 4096 x 4096 13.0 / 16.3 / 13.8 / 19.1   256 x 12288 x 2048 25.7 / 21.3 / 25.7 / 14.1   512 x 2048 x 6144 17.2 / 21.8 / 17.5 / 26.8   512 x 4096 x 2048 16.9 / 20.3 / 13.3 / 13.0
//   700 x 2048 x 6144 - / 22.0 / 28.2 / 29.3   1024 x 4096 x 4096 - / - / 40.7 / 22.2
//   4096 x 12288 x 128 168 / 134 / 124 / 21.9   4096 x 12288 x 512 200 / 168 / 157 / 40   1500 x 13624 x 116 73 / 59 / 55 / 13.8   82 x 22704 x 1058 22.7 / 18.4 / 21.0 / 15.3
//   2935 x 560 x 1340 14.5 / 17.4 / 11.7 / 10.7   5512 x 480 x 8249 64 / 55 / 72 / 39   291 x 8344 x 801 19.1 / 16.5 / 17.8 / 9.5   66 x 3616 x 378 5.0 / 5.6 / 6.3 / 6.4
// Each turn of CTAs takes t0 us, its launch and its stores, and c us a block of K.  Pairs stay: a turn is their blocks of K, 0.45 us each whatever the width of a strip (strips
// shorten the last turn by little: 1111 x 4096 x 2048 20.5 / 18.7, 256 x 24576 x 4096 38.4 / 37.1, none 400 x 4096 x 4096 19.7 / 20.4), and the part of the stores that the next tile's MMAs do not cover.  Over 48 sizes drawn between 65 x 64 x 64 and 8192 x 24576 x 12288 the choice takes
// 0.1 % longer than the best of the four.
template <int CW>
static double f8_rows_us(int M, int N, int KB, double t0, double c) {
    const long long tiles = (long long)((N + 127) / 128) * ((M + 2 * CW - 1) / (2 * CW));
    const int cl = f8_rows_cluster<CW, 1>(tiles, KB), sms = tc_device_sms();
    const long long turns = cl > 1 ? 1 : (tiles + sms - 1) / sms;
    return (double)turns * (t0 + c * ((KB + cl - 1) / cl)) + (cl > 1 ? 0.3 * cl : 0.);
}

int f8_linear_launch(cudaStream_t st, const F8Linear& p, int M, int N, int K, bool pdl) {
    if (M == 0 || N == 0) return 0;
    if ((long long)((M + 255) / 256) * ((N + 255) / 256) > 0x1fffffffLL) return -1000;
    if (M <= 64) {
        // Two CTAs an SM where there are more tiles than SMs; else one with room for three times the stages.  us, one / two: 1 row 12288 x 2048 7.0 / 8.4, 4096 x 12288 11.1 / 12.8,
        // 24576 x 4096 (192 tiles) 23.3 / 18.6; 16 rows 12288 x 2048 7.6 / 9.1, 24576 x 4096 24.8 / 19.2; 48 rows 8.9 / 11.5, 26.8 / 21.0
        const bool two = (N + 127) / 128 > tc_device_sms();
        if (M <= 16) return two ? f8_rows_gemm_t<8, 2>(st, p, M, N, K, pdl) : f8_rows_gemm_t<8, 1>(st, p, M, N, K, pdl);
        if (M <= 32) return two ? f8_rows_gemm_t<16, 2>(st, p, M, N, K, pdl) : f8_rows_gemm_t<16, 1>(st, p, M, N, K, pdl);
        if (M <= 48) return two ? f8_rows_gemm_t<24, 2>(st, p, M, N, K, pdl) : f8_rows_gemm_t<24, 1>(st, p, M, N, K, pdl);
        return f8_rows_gemm_t<32, 1>(st, p, M, N, K, pdl);
    }
    const int KB = f8_blocks(K), pairs = tc_device_sms() / 2, turns = (f8_turns(M, N, pairs).items + pairs - 1) / pairs;
    const double us32 = f8_rows_us<32>(M, N, KB, 4.2, 0.295), us48 = f8_rows_us<48>(M, N, KB, 5.2, 0.38), us64 = f8_rows_us<64>(M, N, KB, 5.9, 0.49);
    const double us_pair = 4.6 + 0.45 * turns * KB + 1.5 * (turns - 1), us_rows = std::min(us32, std::min(us48, us64));
    if (us_pair < us_rows) return f8_pair_launch(st, p, M, N, K, pdl);
    if (us_rows == us32) return f8_rows_gemm_t<32, 1>(st, p, M, N, K, pdl);
    if (us_rows == us48) return f8_rows_gemm_t<48, 1>(st, p, M, N, K, pdl);
    return f8_rows_gemm_t<64, 1>(st, p, M, N, K, pdl);
}

}  // namespace cb
