// Low-rank adapters of prompts (lora.cuh): many rows of 16 bits, ranks from 17 to 64.  A cluster of CTAs has 128 neighbouring rows, one adapter after the other, as in lora.cu: its CTAs each
// take a share of k for T = X A^T, add their shares up in distributed shared memory, and each take a share of the n columns of out = add + s T B^T.  T and its split into two parts: lora.cu.
//
// Both products are tcgen05's, 128 rows by the rank and by 64 columns, operands in 128-byte rows that come in by 16-byte copies (rows of other adapters as zeros), sums in TMEM.  Bound by the
// bytes of add and out: a step's 64 rows of B and 64 columns of add have a ring of three, its results leave through the room that add came in, a warp's own rows.  Two CTAs an SM: one waits
// for its products while the other stores.  As many CTAs share a tile, 8 at most, as lie on the SMs at once: fixed work (sums through the cluster, T's parts) grows with them.
// 8192 rows x 4096 -> 24 576, rank 64, bf16: 208 us (883 MB: 137); by 8 CTAs 260, by 2 381; the next step's products ahead of a step's stores, with one step less under way, 237;
// X A^T by mma.sync from global memory, by 8, 337; lora.cu 401.
#include <cuda_fp16.h>

#include <algorithm>

#include "lora.cuh"
#include "tc.cuh"

namespace cb {
namespace {

constexpr int THREADS = 256, ROWS = 128, NC = 64, ST = 3;
constexpr int PART = ROWS * 128, PITCH = NC * 2 + 16, B_BYTES = NC * 128, STAGE = B_BYTES + ROWS * PITCH, CHUNK = PART + 64 * 128, SMEM = 2 * PART + ST * STAGE + 1024;

template <typename X> constexpr bool HALF = false;
template <> constexpr bool HALF<__half> = true;
template <typename X> __device__ __forceinline__ float2 two(uint32_t w) {
    if constexpr (HALF<X>) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(bf16lo(w), bf16hi(w));
}
template <typename X> __device__ __forceinline__ uint32_t pack(float a, float b) {
    if constexpr (HALF<X>) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    else return pack_bf16(a, b);
}
// what `hi` leaves of v; nothing of an infinity (inf - inf would make a NaN of it)
__device__ __forceinline__ float rest(float v, float hi) { return fabsf(hi) < INFINITY ? v - hi : 0.f; }
__device__ __forceinline__ uint4 piece(const void* p, bool in) { return in ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0); }
__device__ __forceinline__ void to_l2(const void* p, int bytes) { asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory"); }

template <typename X, int RP>
__global__ void __launch_bounds__(THREADS, 2)
lora_tile_kernel(Lora l, int slots) {
    constexpr int LDT = RP + 4;                                      // RP: the rank, rounded up
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + (-smem_u32(raw) & 1023);
    unsigned char* ring = sm + 2 * PART;
    float* share = reinterpret_cast<float*>(ring + ST * STAGE - ROWS * LDT * 4);      // this CTA's shares of T, read by the cluster (not in the first stage)
    static_assert(ST * STAGE - ROWS * LDT * 4 >= STAGE, "the first stage is asked for ahead of them");
    static_assert(CHUNK <= 2 * PART && STAGE + 2 * CHUNK <= ST * STAGE && STAGE % 1024 == 0, "rooms of X and A");
    __shared__ int which_s[ROWS], gave_up;
    __shared__ float down_s[ROWS];                                   // powers of two that take the rows of T back out of f16's range
    __shared__ unsigned lead_s[4];                                   // rows that are the first of their adapter
    __shared__ uint32_t tmem_s;
    __shared__ uint64_t bar;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    if (tid == 0) { gave_up = 0; mbar_init(&bar, 1); fence_barrier_init(); }
    pdl_wait();
    if (warp == 0) { tmem_alloc(&tmem_s, 64); tmem_relinquish(); }
    uint32_t cl;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(cl));
    const int cr = (int)cluster_rank(), nc = (int)cl, tile = blockIdx.x / nc / slots, slot = blockIdx.x / nc % slots;
    const TcWait wait{&gave_up, l.err};
    if (tid < ROWS) {
        const int r = tile * ROWS + tid, v = r < l.m ? __ldg(l.which + r) : -2;
        which_s[tid] = r >= l.m ? -2 : (unsigned)v < (unsigned)l.adapters ? v : -1;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Behind the allocation: a kernel that allocates and then waits for this one must not come ahead of it.  Nor do two kernels wait for one another's columns while their CTAs wait for
    // one another: those that take more than TMEM has beside two of these CTAs leave no room for them in shared memory.
    pdl_launch_dependents();
    const uint32_t tmem = tmem_s;
    if (tid < ROWS) {
        const int v = which_s[tid];
        bool lead = v != -2;
        if (lead && tid && which_s[tid - 1] == v) lead = false;
        for (int i = 0; lead && i + 1 < tid; ++i) lead = which_s[i] != v;
        const unsigned m = __ballot_sync(0xffffffffu, lead);
        if (lane == 0) lead_s[warp] = m;
    }
    __syncthreads();
    const X* x = reinterpret_cast<const X*>(l.x) + (long long)tile * ROWS * l.ldx;
    const X* add = reinterpret_cast<const X*>(l.add) + (l.add ? (long long)tile * ROWS * l.ldadd : 0);
    X* out = reinterpret_cast<X*>(l.out) + (long long)tile * ROWS * l.ldo;
    const int nb = (l.n + NC - 1) / NC, c0 = (int)((long long)nb * cr / nc) * NC, c1 = min((int)((long long)nb * (cr + 1) / nc) * NC, l.n), steps = c1 > c0 ? (c1 - c0 + NC - 1) / NC : 0;
    const int kc = (l.k + 63) / 64, k0 = (int)((long long)kc * cr / nc), chunks = (int)((long long)kc * (cr + 1) / nc) - k0, ksteps = (l.rank + 15) / 16;
    uint32_t phase = 0;
    int turn = 0;
    for (int word = 0; word < 4; ++word)
    for (unsigned leads = lead_s[word]; leads; leads &= leads - 1) {
        // ---- the next adapter among the rows ----
        if (turn++ % slots != slot) continue;                        // another cluster's
        const int w = which_s[word * 32 + __ffs(leads) - 1];
        if (w < 0) {                                                 // none: add goes through
            if (l.add != l.out)
                for (int i = tid; i < ROWS * ((c1 - c0) / 8); i += THREADS) {
                    const int r = i / ((c1 - c0) / 8), c = c0 + i % ((c1 - c0) / 8) * 8;
                    if (which_s[r] == w) *reinterpret_cast<uint4*>(out + r * l.ldo + c) = piece(add + r * l.ldadd + c, l.add);
                }
            continue;
        }
        const X* A = reinterpret_cast<const X*>(l.a) + (size_t)w * l.rank * l.k;
        const X* B = reinterpret_cast<const X*>(l.b) + ((size_t)w * l.n + c0) * l.rank;
        // ---- a step's rows of B and columns of add: a thread has the same 16-byte piece of every 32nd row ----
        const int fp = tid & 7, fr = tid >> 3;
        uint32_t x_in = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) x_in |= (uint32_t)(which_s[fr + 32 * i] == w) << i;
        const uint32_t add_in = l.add ? x_in : 0;
        const uint32_t base = smem_u32(ring);
        auto copy = [](uint32_t dst, const void* src, bool in) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory"); };
        auto fetch = [&](int step) {
            const uint32_t st = base + step % ST * STAGE;
            const int off = step * NC;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = fr + 32 * i;
                const bool in = fp * 8 < l.rank && c0 + off + r < c1;
                if (fp < 2 * ksteps) copy(st + sw128_off(r, fp), in ? B + (size_t)(off + r) * l.rank + fp * 8 : B, in);
            }
            if (add_in) {
                const bool here = c0 + off + fp * 8 < c1;
                const X* src = add + (long long)fr * l.ldadd + c0 + off + fp * 8;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (here && (add_in >> i & 1)) copy(st + B_BYTES + (fr + 32 * i) * PITCH + fp * 16, src + (long long)(32 * i) * l.ldadd, true);
            }
        };
        auto commit = []() { asm volatile("cp.async.commit_group;" ::: "memory"); };
        // ... and of X and A: 64 of k, in the rooms of T's parts and of the second and third stage
        auto room = [&](int c) { return c % 3 ? ring + STAGE + (c % 3 - 1) * CHUNK : sm; };
        auto fetch_x = [&](int c) {
            const uint32_t st = smem_u32(room(c));
            const int at = (k0 + c) * 64 + fp * 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = at < l.k && (x_in >> i & 1);
                copy(st + sw128_off(fr + 32 * i, fp), in ? x + (long long)(fr + 32 * i) * l.ldx + at : x, in);
            }
#pragma unroll
            for (int i = 0; i < (RP + 31) / 32; ++i) {
                const int r = fr + 32 * i;
                const bool in = at < l.k && r < l.rank;
                if (r < RP) copy(st + PART + sw128_off(r, fp), in ? A + (size_t)r * l.k + at : A, in);
            }
        };
        const int row = (warp & 3) * 32 + lane, half = warp >> 2;     // TMEM's lanes of a warp are its rows, half of the columns
        const uint32_t mine_d = tmem + ((uint32_t)(warp & 3) << 21);
        // ---- this CTA's share of T ----
        if (chunks > 0) fetch_x(0);
        commit();
        if (chunks > 1) fetch_x(1);
        commit();
        if (l.add && tid < ROWS && which_s[tid] == w && c1 > c0) to_l2(add + tid * l.ldadd + c0, (min(c1, c0 + 8 * NC) - c0) * 2);
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            if (c) { wait(&bar, phase); phase ^= 1; }                // (its room is the next one's but one)
            fence_proxy_async();
            __syncthreads();
            if (warp == 0) {
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t xd = make_smem_desc_sw128(smem_u32(room(c))), ad = make_smem_desc_sw128(smem_u32(room(c) + PART));
                    constexpr uint32_t id = HALF<X> ? make_idesc_f16(ROWS, RP) : make_idesc_bf16(ROWS, RP);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) umma_bf16(tmem, xd + 2 * ks, ad + 2 * ks, id, c > 0 || ks > 0);
                    umma_commit(&bar);
                }
                __syncwarp();
            }
            if (c + 2 < chunks) fetch_x(c + 2);
            else if (c + 2 == chunks && steps) fetch(0);
            commit();
        }
        if (chunks < 2 && steps) fetch(0);
        commit();
        if (chunks) { wait(&bar, phase); phase ^= 1; tc_fence_after(); }
        {
            uint32_t d[RP / 2];
            if constexpr (RP == 64) tmem_ld32(mine_d + half * 32, d);
            else tmem_ld16_async(mine_d + half * 16, d);
            tmem_ld_wait();
            tc_fence_before();
#pragma unroll
            for (int i = 0; i < RP / 2; i += 4)
                *reinterpret_cast<uint4*>(share + row * LDT + half * (RP / 2) + i) = chunks ? make_uint4(d[i], d[i + 1], d[i + 2], d[i + 3]) : make_uint4(0, 0, 0, 0);
        }
        // ---- the cluster's sum: the order is the same every time ----
        if (nc > 1) cluster_sync_all(); else __syncthreads();
        const float s = l.scales ? __ldg(l.scales + w) : 1.f;
#pragma unroll 1
        for (int i = tid; i < ROWS * RP / 4; i += THREADS) {         // (whole rounds of the block)
            const int r = i / (RP / 4), q = i % (RP / 4);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f), y[8];
            const float* p = share + r * LDT + q * 4;
#pragma unroll
            for (int c = 0; c < 8; ++c)                              // (all on their way before the first is added)
                if (c < nc) asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(y[c].x), "=f"(y[c].y), "=f"(y[c].z), "=f"(y[c].w) : "r"(peer_smem(p, c)));
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (c < nc) { v.x += y[c].x; v.y += y[c].y; v.z += y[c].z; v.w += y[c].w; }
            v.x *= s; v.y *= s; v.z *= s; v.w *= s;
            if constexpr (HALF<X>) {
                float top = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
#pragma unroll
                for (int o = RP / 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const uint32_t e = __float_as_uint(fminf(fmaxf(top, 0x1p-100f), 0x1p120f)) >> 23;
                const float up = top < INFINITY ? __uint_as_float((268 - e) << 23) : 1.f;      // the largest of the row to [2^14, 2^15)
                v.x *= up; v.y *= up; v.z *= up; v.w *= up;
                if (q == 0) down_s[r] = top < INFINITY ? __uint_as_float((e - 14) << 23) : 1.f;
            }
            const uint32_t h0 = pack<X>(v.x, v.y), h1 = pack<X>(v.z, v.w);
            const float2 a = two<X>(h0), b = two<X>(h1);
            const uint32_t at = sw128_off(r, q >> 1) + (q & 1) * 8;
            *reinterpret_cast<uint2*>(sm + at) = make_uint2(h0, h1);
            *reinterpret_cast<uint2*>(sm + PART + at) = make_uint2(pack<X>(rest(v.x, a.x), rest(v.y, a.y)), pack<X>(rest(v.z, b.x), rest(v.w, b.y)));
        }
        fence_proxy_async();
        if (nc > 1) cluster_sync_all(); else __syncthreads();        // every CTA has read the shares: their room is free, and their owner may leave
        // ---- out = add + T B^T, a step of 64 columns after the other ----
        if (steps > 1) fetch(1);
        commit();
        const float down = HALF<X> ? down_s[row] : 1.f;
        uint32_t out_in = 0;                                         // out of shared memory: 8 rows at a time, four lanes each
#pragma unroll
        for (int i = 0; i < 4; ++i) out_in |= (uint32_t)(which_s[(warp & 3) * 32 + i * 8 + g] == w) << i;
        X* dst = out + (long long)((warp & 3) * 32 + g) * l.ldo + c0 + half * 32 + t * 8;
        const uint64_t hi_d = make_smem_desc_sw128(smem_u32(sm)), lo_d = make_smem_desc_sw128(smem_u32(sm + PART));
        constexpr uint32_t id = HALF<X> ? make_idesc_f16(ROWS, NC) : make_idesc_bf16(ROWS, NC);
#pragma unroll 1
        for (int step = 0; step < steps; ++step) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            fence_proxy_async();
            tc_fence_before();
            __syncthreads();                                         // the step is there, the one before it gone
            unsigned char* st = ring + step % ST * STAGE;
            if (warp == 0) {
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t bd = make_smem_desc_sw128(smem_u32(st));
                    for (int ks = 0; ks < ksteps; ++ks) {
                        umma_bf16(tmem, lo_d + 2 * ks, bd + 2 * ks, id, ks > 0);
                        umma_bf16(tmem, hi_d + 2 * ks, bd + 2 * ks, id, 1);
                    }
                    umma_commit(&bar);
                }
                __syncwarp();
            }
            if (step + 2 < steps) fetch(step + 2);
            commit();
            uint4* mine = reinterpret_cast<uint4*>(st + B_BYTES + row * PITCH + half * 64);
            uint4 av[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) av[i] = l.add ? mine[i] : make_uint4(0, 0, 0, 0);
            wait(&bar, phase);
            phase ^= 1;
            tc_fence_after();
            uint32_t d[32];
            tmem_ld32(mine_d + half * 32, d);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t a[4] = {av[i].x, av[i].y, av[i].z, av[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = two<X>(a[j]);
                    a[j] = pack<X>(fmaf(__uint_as_float(d[8 * i + 2 * j]), down, f.x), fmaf(__uint_as_float(d[8 * i + 2 * j + 1]), down, f.y));
                }
                mine[i] = make_uint4(a[0], a[1], a[2], a[3]);
            }
            __syncwarp();
            if (c0 + step * NC + half * 32 + t * 8 < c1)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (out_in >> i & 1)
                        *reinterpret_cast<uint4*>(dst + (long long)(i * 8) * l.ldo + step * NC) =
                            *reinterpret_cast<const uint4*>(st + B_BYTES + ((warp & 3) * 32 + i * 8 + g) * PITCH + half * 64 + t * 16);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        tc_fence_before();
        __syncthreads();                                             // (T's parts and the stages may be written again)
    }
    if (warp == 0) { wait.drain(); tc_fence_after(); tmem_dealloc(tmem, 64); }
}

template <typename X, int RP>
int launch(cudaStream_t st, const Lora& l, bool pdl) {
    static SmemOptIn seen;
    auto kernel = lora_tile_kernel<X, RP>;
    if (const int e = ensure_dyn_smem(kernel, (size_t)SMEM, seen)) return e;
    const int tiles = (l.m + ROWS - 1) / ROWS;
    int cluster = 8;                                                 // (a power of two: what the sums' loads are counted by)
    while (cluster > 1 && tiles * cluster > 2 * tc_device_sms()) cluster /= 2;
    const int slots = std::min(l.adapters + 1, std::max(2, tc_device_sms() / 2 / tiles));      // a tile's adapters are dealt out in turn to so many clusters
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)tiles * cluster * slots); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, kernel, l, slots);
}
template <typename X> int launch_rank(cudaStream_t st, const Lora& l, bool pdl) {
    return l.rank <= 32 ? launch<X, 32>(st, l, pdl) : launch<X, 64>(st, l, pdl);
}

}  // namespace

int lora_tiles_launch(cudaStream_t st, const Lora& l, bool pdl) { return l.type == LORA_BF16 ? launch_rank<bf16>(st, l, pdl) : launch_rank<__half>(st, l, pdl); }

}  // namespace cb
