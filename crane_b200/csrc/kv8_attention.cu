// Attention over an 8-bit paged cache (kv8.cuh): out = sum over visible i of softmax_i(scale q . k_i) v_i, a query at position p sees the positions up to p.
//
// e4m3 codes are exact in f16, so products run on f16 tensor cores with f32 sums.  Queries are scaled to the range of f16 by a power of two of their own (f32 ones
// are two f16 parts, 22 bits).  The scales stay out of the operands: a page's key scale multiplies its scores, its value scale joins the exponent,
//     p'_i = 2^(s_i + log2 vs_i - m),  m = running max of s_i + log2 vs_i,   out = sum p'_i v-code_i / sum p'_i / vs_i,
// so that the largest weight, scaled values counted in, always sits at the same place of f16's range.  m is a whole number: log2 vs - m is exact, and the exponent is rounded
// once, where it is small for the weights that count.
#include <cuda_fp16.h>

#include <climits>

#include "kv8.cuh"
#include "tc.cuh"

namespace cb {
namespace {

constexpr int TILE = 64;                       // positions a step
constexpr float P_SHIFT = 14.f;                // weights run up to 2^14: f16 holds those down to 2^-28 of the largest with 11 bits

struct Args {
    const void* q; long long ldq, ldqh;
    void* out; long long ldo, ldoh;
    float scale2, scale2_rest;                 // scale * log2 e, and what f32 leaves of it
    Kv8Deal d;
    float* work;                               // [2 * CTAs][rows of a group of rows][D + 2]
    int* err;
};

template <int M> using Units = Kv8Units<M, TILE>;

// ---- fragments -------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void lds16(uint32_t a, uint32_t* r) { asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a)); }
__device__ __forceinline__ void lds8(uint32_t a, uint32_t* r) { asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a)); }
__device__ __forceinline__ uint32_t half2_of(uint32_t codes, int which) {        // codes 2 * which and the next -> f16x2, exact
    uint32_t r;
    const uint16_t c = (uint16_t)(which ? codes >> 16 : codes);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
    return r;
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t pack_f16(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ float2 unpack_f16(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<bf16>(bf16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// Shared memory of a step: keys, values [64 positions][D] in boxes of at most 128 columns, swizzled by TMA; scales of its pages
template <int D> struct Step {
    static constexpr int BOX = D < 128 ? D : 128, PLANES = D / BOX, PLANE = TILE * BOX, BYTES = 2 * PLANES * PLANE;
};
template <int BOX> __device__ __forceinline__ uint32_t piece(int r, int c) { return BOX == 128 ? sw128_off(r, c) : sw64_off(r, c); }

// A warp has 16 query rows and takes 16 positions at a time.  Which position and column a place of a fragment stands for is free as long as both operands agree; this
// order lets a lane read its codes 16 bytes at a time without bank conflicts and leave 16 neighbouring columns of the result:
//   place n of 8 positions: position pos8(n);  contraction of D: lane t of a quad has the 16-byte pieces t and t + 4 of a row of 128 (t of a row of 64)
//   columns: place n of the 8 of an MMA: piece col8(n) of a row (or 8 bytes of one of 64), the MMA's number the column in it
template <int D> __device__ __forceinline__ int pos8(int n) { return D == 64 ? n : (n & 1) * 4 + (n >> 1); }
__device__ __forceinline__ int col8(int n) { return (n & 1) * 4 + (n >> 1); }

template <int D, typename T, int TG, int MG>
struct Small {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int WARPS = TG * MG, THREADS = WARPS * 32 + 32, M = 16 * MG, SL = TILE / 16 / TG;      // SL: 16-position slices of a tile that a warp has
    static constexpr int NT = D / 8;                                        // MMAs across the columns
    static constexpr int KS = D / 16;                                       // ... along them
    static constexpr bool QREG = !(F32 && D >= 128) && D < 256;             // query fragments stay in registers
    static constexpr int QBYTES = QREG ? 0 : MG * KS * 512 * (F32 ? 2 : 1);
    static constexpr int JOIN = (TG > 1 ? TG / 2 : 1) * MG * 32 * (NT * 4 + 4) * 4;      // sums on their way between warps
    static constexpr int CTAS = D == 256 && (F32 || MG > 1) ? 1 : MG > 1 ? 1 : 2;        // resident on an SM
    static constexpr int ROOM = (227 * 1024) / CTAS - 1024 - 1024 - 2048 - JOIN - QBYTES;
    static constexpr int STAGES = ROOM / Step<D>::BYTES > 8 ? 8 : ROOM / Step<D>::BYTES;
    static constexpr int SMEM = STAGES * Step<D>::BYTES + JOIN + QBYTES + 1024 + 512;
    static_assert(STAGES >= 2, "two steps at least");
};

template <int D, typename T, int TG, int MG>
__global__ void __launch_bounds__(Small<D, T, TG, MG>::THREADS, Small<D, T, TG, MG>::CTAS)
small_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Args a) {
    using S = Small<D, T, TG, MG>;
    using St = Step<D>;
    constexpr int M = S::M, NT = S::NT, KS = S::KS, STAGES = S::STAGES;
    constexpr bool F32 = S::F32;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
    float* join = reinterpret_cast<float*>(sm + STAGES * St::BYTES);
    uint32_t* qs = reinterpret_cast<uint32_t*>(sm + STAGES * St::BYTES + S::JOIN);
    __shared__ uint64_t full[STAGES], empty[STAGES];
    __shared__ float4 meta[STAGES][4];                       // of each 16 positions: ks, log2 vs, 1 / vs, and whether there is a page
    __shared__ long long sums[KV8_SHARES + 1];
    __shared__ int gave_up;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        gave_up = 0;
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], S::WARPS); }
        fence_barrier_init();
        tma_prefetch_desc(&map_k); tma_prefetch_desc(&map_v);
    }
    const TcWait wait{&gave_up, a.err};
    pdl_wait();
    const long long total = kv8_count<Units<M>>(a.d, sums);
    const long long begin = kv8_range(total, gridDim.x, blockIdx.x), end = kv8_range(total, gridDim.x, blockIdx.x + 1);
    pdl_launch_dependents();
    if (begin >= end) return;
    Units<M> u = kv8_find<Units<M>>(a.d, sums, begin);

    if (warp == S::WARPS) {
        // ---- copies: a box per page (64 positions of it at most) and plane ----
        const int P = a.d.p.page, rows = min(P, TILE), boxes = TILE / rows;
        int stage = 0;
        uint32_t parity = 1;
        for (long long step = begin; step < end;) {
            const int t0 = (int)(step - u.first), t1 = (int)min((long long)u.tiles, end - u.first), n = (t1 - t0) * boxes;
            for (int base = 0; base < n; base += 32) {
                // a lane looks up one box: its row in the pool and its scales
                int row = -1;
                float4 sc = make_float4(0.f, 0.f, 0.f, 0.f);
                if (base + lane < n) {
                    const int pos = t0 * TILE + (base + lane) * rows, page = pos < u.q.len ? kv8_page(a.d.s, a.d.p, u.b, pos / P) : -1;
                    if (page >= 0) {
                        row = (page * a.d.p.kv_heads + u.head) * P + pos % P;
                        const float2 kv = *reinterpret_cast<const float2*>(a.d.p.scales + ((size_t)page * a.d.p.kv_heads + u.head) * 2);
                        const float vs = fmaxf(kv.y, 0x1p-120f);
                        sc = make_float4(kv.x, log2f(vs), __frcp_rn(vs), 1.f);
                    }
                }
                for (int i = base; i < min(n, base + 32); i += boxes) {
                    wait(&empty[stage], parity);
                    unsigned char* st = sm + stage * St::BYTES;
                    const int from = (i - base + (lane & 3) * 16 / rows) & 31;
                    float4 m;
                    m.x = __shfl_sync(0xffffffffu, sc.x, from); m.y = __shfl_sync(0xffffffffu, sc.y, from);
                    m.z = __shfl_sync(0xffffffffu, sc.z, from); m.w = __shfl_sync(0xffffffffu, sc.w, from);
                    if (lane < 4) meta[stage][lane] = m;
                    __syncwarp();
                    if (lane == 0) mbar_arrive_expect_tx(&full[stage], St::BYTES);
                    __syncwarp();
                    for (int j = 0; j < boxes; ++j) {
                        int r = __shfl_sync(0xffffffffu, row, i - base + j);
                        if (r < 0) r = a.d.p.pages * a.d.p.kv_heads * P;       // behind the pool: zeros come
                        if (lane < 2 * St::PLANES) {
                            const int pl = lane >> 1;
                            tma_load_2d(st + (lane & 1) * St::PLANES * St::PLANE + pl * St::PLANE + j * rows * St::BOX, lane & 1 ? &map_v : &map_k, &full[stage], pl * St::BOX, r);
                        }
                    }
                    if (++stage == STAGES) { stage = 0; parity ^= 1; }
                }
            }
            step = u.first + t1;
            if (step < end && !u.next(a.d)) break;
        }
        __syncwarp();
        // (the last copies have landed when the consumers' last waits return)
        if (lane == 0) wait.drain();
        return;
    }

    // ---- products ----
    const int g = lane >> 2, t = lane & 3, mg = warp % MG, tg = warp / MG;
    int stage = 0;
    uint32_t parity = 0;
    for (long long step = begin; step < end;) {
        const int t0 = (int)(step - u.first), t1 = (int)min((long long)u.tiles, end - u.first);
        // ---- the unit's queries: fragments, and the factor that a row's scores take ----
        uint32_t qf[S::QREG ? KS : 1][4], ql[S::QREG && F32 ? KS : 1][4];
        float factor[2], fine[2];                            // ... and what f32 leaves of it
        int pmax[2], wmin = INT_MAX;                         // last visible position of rows g and g + 8; the warp's rows all see the positions up to wmin
        {
            float v[2][D / 4];                               // this lane's columns of both rows
            int row[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                row[r] = u.grp * M + mg * 16 + g + r * 8;
                const int tok = row[r] / a.d.group, h = u.head * a.d.group + row[r] % a.d.group;
                const bool in = tok < u.q.n;
                pmax[r] = in ? u.q.first + tok : -1;
                if (in) wmin = min(wmin, pmax[r]);
                const T* src = reinterpret_cast<const T*>(a.q) + (long long)(u.q.s0 + (in ? tok : 0)) * a.ldq + (long long)h * a.ldqh;
                float top = 0.f;
#pragma unroll
                for (int p = 0; p < D / 64; ++p) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float y = in ? to_f<T>(src[p * 64 + t * 16 + j]) : 0.f;
                        v[r][p * 16 + j] = y;
                        top = y != y ? INFINITY : fmaxf(top, fabsf(y));
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // 2^e that takes the row's largest magnitude to [2^14, 2^15); rows of less than 2^-100 count as zeros, rows with an infinity or a NaN give NaN
                const uint32_t ex = __float_as_uint(fmaxf(top, 0x1p-100f)) >> 23;
                const float up = __uint_as_float((uint32_t)(268 - ex) << 23);
                factor[r] = top < INFINITY ? a.scale2 * __uint_as_float((ex - 14) << 23) : NAN;
                fine[r] = a.scale2_rest * __uint_as_float((ex - 14) << 23);
#pragma unroll
                for (int j = 0; j < D / 4; ++j) v[r][j] = top < INFINITY ? v[r][j] * up : 0.f;
            }
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                uint32_t f[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = v[i & 1][4 * s + (i >> 1) * 2], y = v[i & 1][4 * s + (i >> 1) * 2 + 1];
                    f[i] = pack_f16(x, y);
                    if (F32) { const float2 h = unpack_f16(f[i]); lo[i] = pack_f16(x - h.x, y - h.y); }
                }
                if constexpr (S::QREG) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) { qf[s][i] = f[i]; if (F32) ql[F32 ? s : 0][i] = lo[i]; }
                } else {
                    if (tg == 0) {
                        uint4* d = reinterpret_cast<uint4*>(qs) + (mg * KS + s) * 32 + lane;
                        d[0] = make_uint4(f[0], f[1], f[2], f[3]);
                        if (F32) d[MG * KS * 32] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            }
            if constexpr (!S::QREG) named_bar_sync(1, S::WARPS * 32);
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) wmin = min(wmin, __shfl_xor_sync(0xffffffffu, wmin, o));
        float o_acc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) { o_acc[j][0] = o_acc[j][1] = o_acc[j][2] = o_acc[j][3] = 0.f; }
        float m_row[2] = {-INFINITY, -INFINITY}, l_row[2] = {0.f, 0.f};

        for (int tile = t0; tile < t1; ++tile) {
            wait(&full[stage], parity);
            const uint32_t kb = smem_u32(sm + stage * St::BYTES), vb = kb + St::PLANES * St::PLANE;
#pragma unroll
            for (int sl = 0; sl < S::SL; ++sl) {
                const int s16 = tg * S::SL + sl, r0 = s16 * 16, pos0 = tile * TILE + r0;
                const float4 sc = meta[stage][s16];
                const bool edge = pos0 + 15 > wmin;          // not all of the warp's rows see all of it
                if (__all_sync(0xffffffffu, sc.w == 0.f || (pos0 > pmax[0] && pos0 > pmax[1]))) continue;
                // ---- scores ----
                float s_acc[2][4];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    s_acc[nt][0] = s_acc[nt][1] = s_acc[nt][2] = s_acc[nt][3] = 0.f;
                    float odd_acc[4] = {0.f, 0.f, 0.f, 0.f}, lo_acc[4] = {0.f, 0.f, 0.f, 0.f};      // f32: short chains, the tensor core cuts its sums off where f32 rounds
                    const int r = r0 + nt * 8 + pos8<D>(g);
#pragma unroll
                    for (int p = 0; p < D / 64; ++p) {       // pieces t, t + 4 of each plane
                        uint32_t w[4];
                        lds16(kb + (p / 2) * St::PLANE + piece<St::BOX>(r, (p & 1) * 4 + t), w);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t b0 = half2_of(w[i], 0), b1 = half2_of(w[i], 1);
                            if constexpr (S::QREG) {
                                if (F32) mma_f16(lo_acc, ql[F32 ? p * 4 + i : 0], b0, b1);
                                mma_f16(F32 && (i & 1) ? odd_acc : s_acc[nt], qf[p * 4 + i], b0, b1);
                            } else {
                                const uint4* qd = reinterpret_cast<const uint4*>(qs) + (mg * KS + p * 4 + i) * 32 + lane;
                                if (F32) { const uint4 f = qd[MG * KS * 32]; const uint32_t x[4] = {f.x, f.y, f.z, f.w}; mma_f16(lo_acc, x, b0, b1); }
                                const uint4 f = qd[0]; const uint32_t x[4] = {f.x, f.y, f.z, f.w};
                                mma_f16(F32 && (i & 1) ? odd_acc : s_acc[nt], x, b0, b1);
                            }
                        }
                    }
                    if (F32)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s_acc[nt][e] += odd_acc[e] + lo_acc[e];
                }
                // ---- weights ----
                const float f[2] = {factor[0] * sc.x, factor[1] * sc.x};
                float mx[2] = {-INFINITY, -INFINITY};
                uint32_t hidden = 0;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int pos = pos0 + nt * 8 + pos8<D>(2 * t + (e & 1));
                        if (edge && pos > pmax[e >> 1]) hidden |= 1u << (nt * 4 + e);
                        else mx[e >> 1] = fmaxf(mx[e >> 1], fmaf(s_acc[nt][e], f[e >> 1], sc.y));
                    }
                float corr[2], mref[2];
                bool far = false;                            // scores whose last bit is worth more than a weight: their exponents are differences of rounded numbers
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                    const float mn = fmaxf(m_row[r], ceilf(mx[r]));
                    mref[r] = mn == -INFINITY ? 0.f : sc.y - (mn - P_SHIFT);
                    corr[r] = m_row[r] == mn ? 1.f : ex2(m_row[r] - mn);
                    m_row[r] = mn;
                    far |= fabsf(mn) > 0x1p20f && fabsf(mn) < INFINITY;
                }
                if (__any_sync(0xffffffffu, far)) {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s_acc[nt][e] = fmaf(s_acc[nt][e], f[e >> 1], sc.y) - m_row[e >> 1];
                    far = true;
                }
                if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
                    l_row[0] *= corr[0]; l_row[1] *= corr[1];
#pragma unroll
                    for (int j = 0; j < NT; ++j) { o_acc[j][0] *= corr[0]; o_acc[j][1] *= corr[0]; o_acc[j][2] *= corr[1]; o_acc[j][3] *= corr[1]; }
                }
                float ps[2] = {0.f, 0.f};
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float p = far ? ex2(s_acc[nt][e] + P_SHIFT) : F32 ? ex2(fmaf(s_acc[nt][e], f[e >> 1], fmaf(s_acc[nt][e], fine[e >> 1] * sc.x, mref[e >> 1]))) : ex2(fmaf(s_acc[nt][e], f[e >> 1], mref[e >> 1]));
                        if (hidden >> (nt * 4 + e) & 1) p = 0.f;
                        s_acc[nt][e] = p;
                        ps[e >> 1] += p;
                    }
                l_row[0] = fmaf(ps[0], sc.z, l_row[0]);
                l_row[1] = fmaf(ps[1], sc.z, l_row[1]);
                uint32_t pa[4], pl[4], vis[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {                // rows g, g + 8 of positions 0 - 7, then of 8 - 15
                    const float x = s_acc[i >> 1][(i & 1) * 2], y = s_acc[i >> 1][(i & 1) * 2 + 1];
                    pa[i] = pack_f16(x, y);
                    if (F32) { const float2 h = unpack_f16(pa[i]); pl[i] = pack_f16(x - h.x, y - h.y); }
                    const int p0 = pos0 + (i >> 1) * 8;
                    vis[i] = (p0 + pos8<D>(2 * t) <= pmax[i & 1] ? 0x3c00u : 0u) | (p0 + pos8<D>(2 * t + 1) <= pmax[i & 1] ? 0x3c000000u : 0u);
                }
                // ---- values: two positions' codes side by side ----
                const int ra = r0 + pos8<D>(2 * t), rb = r0 + pos8<D>(2 * t + 1);
#pragma unroll
                for (int pl8 = 0; pl8 < St::PLANES; ++pl8) {
                    constexpr int W = St::BOX == 128 ? 4 : 2;            // words of four columns that a lane has of a row
                    uint32_t x[4][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = (i & 1 ? rb : ra) + (i >> 1) * 8;
                        if constexpr (St::BOX == 128) lds16(vb + pl8 * St::PLANE + piece<128>(r, col8(g)), x[i]);
                        else lds8(vb + piece<64>(r, g >> 1) + (g & 1) * 8, x[i]);
                    }
                    bool odd = false;                        // a NaN among values that not all rows see: 0 * NaN must not reach the others
                    if (edge) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int w = 0; w < W; ++w) {
                                odd |= (((x[i][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
                            }
                        odd = __any_sync(0xffffffffu, odd);
                    }
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        uint32_t lo[2], hi[2];               // columns 4 w, 4 w + 1 and 4 w + 2, 4 w + 3, of positions 0 - 7 and 8 - 15
#pragma unroll
                        for (int i = 0; i < 2; ++i) { lo[i] = __byte_perm(x[2 * i][w], x[2 * i + 1][w], 0x5140); hi[i] = __byte_perm(x[2 * i][w], x[2 * i + 1][w], 0x7362); }
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t b0 = half2_of(c < 2 ? lo[0] : hi[0], c & 1), b1 = half2_of(c < 2 ? lo[1] : hi[1], c & 1);
                            float* acc = o_acc[pl8 * W * 4 + w * 4 + c];
                            if (odd) {
                                const __half2 n0 = __hisnan2(*reinterpret_cast<__half2*>(&b0)), n1 = __hisnan2(*reinterpret_cast<__half2*>(&b1));
                                const uint32_t m0 = *reinterpret_cast<const uint32_t*>(&n0), m1 = *reinterpret_cast<const uint32_t*>(&n1);
                                float seen[4] = {0.f, 0.f, 0.f, 0.f};
                                mma_f16(seen, vis, m0, m1);
#pragma unroll
                                for (int e = 0; e < 4; ++e) if (seen[e] > 0.f) acc[e] = NAN;
                                if (m0 & 0xffffu) b0 &= 0xffff0000u;
                                if (m0 >> 16) b0 &= 0xffffu;
                                if (m1 & 0xffffu) b1 &= 0xffff0000u;
                                if (m1 >> 16) b1 &= 0xffffu;
                            }
                            if constexpr (F32) {             // (and long sums are f32 additions)
                                float part[4] = {0.f, 0.f, 0.f, 0.f};
                                mma_f16(part, pl, b0, b1);
                                mma_f16(part, pa, b0, b1);
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[e] += part[e];
                            } else {
                                mma_f16(acc, pa, b0, b1);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[stage]);
            if (++stage == STAGES) { stage = 0; parity ^= 1; }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l_row[r] += __shfl_xor_sync(0xffffffffu, l_row[r], 1);
            l_row[r] += __shfl_xor_sync(0xffffffffu, l_row[r], 2);
        }
        // ---- the warps that share rows add up, half of them into the other half each time ----
#pragma unroll
        for (int h = TG / 2; h >= 1; h /= 2) {
            named_bar_sync(1, S::WARPS * 32);
            float* d = join + ((size_t)((tg % h) * MG + mg) * (NT * 4 + 4)) * 32 + lane;
            if (tg >= h && tg < 2 * h) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[(j * 4 + e) * 32] = o_acc[j][e];
                d[(NT * 4) * 32] = m_row[0]; d[(NT * 4 + 1) * 32] = m_row[1]; d[(NT * 4 + 2) * 32] = l_row[0]; d[(NT * 4 + 3) * 32] = l_row[1];
            }
            named_bar_sync(1, S::WARPS * 32);
            if (tg < h) {
                float c0[2], c1[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float mo = d[(NT * 4 + r) * 32], mn = fmaxf(m_row[r], mo);
                    c0[r] = m_row[r] == -INFINITY ? 0.f : exp2f(m_row[r] - mn);
                    c1[r] = mo == -INFINITY ? 0.f : exp2f(mo - mn);
                    m_row[r] = mn;
                    l_row[r] = l_row[r] * c0[r] + d[(NT * 4 + 2 + r) * 32] * c1[r];
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o_acc[j][e] = o_acc[j][e] * c0[e >> 1] + d[(j * 4 + e) * 32] * c1[e >> 1];
            }
        }
        if (tg == 0) {
            const bool whole = t0 == 0 && t1 == u.tiles;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = mg * 16 + g + r * 8, tok = (u.grp * M + row) / a.d.group, h = u.head * a.d.group + (u.grp * M + row) % a.d.group;
                if (whole) {
                    if (tok >= u.q.n) continue;
                    T* dst = reinterpret_cast<T*>(a.out) + (long long)(u.q.s0 + tok) * a.ldo + (long long)h * a.ldoh;
                    const float inv = l_row[r] == 0.f ? 0.f : 1.f / l_row[r];
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int col = D == 64 ? (2 * t + e) * 8 + j : (j / 16) * 128 + col8(2 * t + e) * 16 + j % 16;
                            dst[col] = from_f<T>(o_acc[j][2 * r + e] * inv);
                        }
                } else {
                    const int slot = kv8_slot(blockIdx.x, begin, step);
                    float* dst = a.work + ((size_t)slot * M + row) * (D + 2);
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int col = D == 64 ? (2 * t + e) * 8 + j : (j / 16) * 128 + col8(2 * t + e) * 16 + j % 16;
                            dst[col] = o_acc[j][2 * r + e];
                        }
                    if (t == 0) { dst[D] = m_row[r]; dst[D + 1] = l_row[r]; }
                }
            }
        }
        step = u.first + t1;
        if (step < end && !u.next(a.d)) break;
    }
    if (tid == 0) wait.drain();
}

// Adds up the parts of the units that lie with several CTAs.  Block x: unit boundaries between CTAs x and x + 1, if the unit does not reach back to CTA x - 1's steps.
template <int D, typename T, int M, int TILE>
__global__ void __launch_bounds__(128)
join_kernel(Args a, int ctas) {
    using Units = Kv8Units<M, TILE>;
    __shared__ long long sums[KV8_SHARES + 1];
    pdl_wait();
    pdl_launch_dependents();
    const long long total = kv8_count<Units>(a.d, sums);
    const int c = blockIdx.x;
    const long long begin = kv8_range(total, ctas, c), end = kv8_range(total, ctas, c + 1);
    if (begin >= end || end >= total) return;
    const Units u = kv8_find<Units>(a.d, sums, end - 1);          // the last unit of CTA c
    if (u.first + u.tiles <= end || u.first < begin) return;         // ... ends there, or begins ahead of it
    const int last = kv8_owner(total, ctas, u.first + u.tiles - 1);
    const int rows = (int)min((long long)M, (long long)u.q.n * a.d.group - (long long)u.grp * M);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int row = blockIdx.y * 4 + warp; row < rows; row += 4 * gridDim.y) {
        float o[D / 32], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) o[j] = 0.f;
        for (int k = c; k <= last; ++k) {
            const int slot = k == c ? kv8_slot(c, begin, u.first) : kv8_slot(k, 0, 0);
            const float* src = a.work + ((size_t)slot * M + row) * (D + 2);
            const float mo = src[D], lo = src[D + 1], mn = fmaxf(m, mo);
            const float c0 = m == -INFINITY ? 0.f : exp2f(m - mn), c1 = mo == -INFINITY ? 0.f : exp2f(mo - mn);
            m = mn;
            l = l * c0 + lo * c1;
#pragma unroll
            for (int j = 0; j < D / 32; ++j) o[j] = o[j] * c0 + src[j * 32 + lane] * c1;
        }
        const int rr = u.grp * M + row, tok = rr / a.d.group, h = u.head * a.d.group + rr % a.d.group;
        T* dst = reinterpret_cast<T*>(a.out) + (long long)(u.q.s0 + tok) * a.ldo + (long long)h * a.ldoh;
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) dst[j * 32 + lane] = from_f<T>(o[j] * inv);
    }
}

// Rows of a kv head from which on a sequence goes through kv8_flash.cu: 16-bit ones of 64 and 128 columns.
constexpr int FLASH_FROM = 65;
bool flash_takes(int type, int dim, int group, int max_rows) { return type != KV8_F32 && dim <= 128 && (long long)group * max_rows >= FLASH_FROM; }
// Rows of a group of queries: 16 where no sequence brings more, else 32 or 64.  (Beside kv8_flash.cu 16: most of what is left are decoded tokens.)
int rows_of(int group, int dim, int max_rows, bool flash) {
    const long long r = (long long)group * max_rows;
    return r <= 16 || flash ? 16 : r <= 32 || dim == 256 ? 32 : 64;
}
template <typename T>
int join_flash(cudaStream_t st, const Args& a) {
    auto k = a.d.p.dim == 64 ? join_kernel<64, T, KV8_FLASH_ROWS, 128> : join_kernel<128, T, KV8_FLASH_ROWS, 128>;
    return launch_k(k, dim3(tc_device_sms() - 1, 16), dim3(128), 0, st, true, a, tc_device_sms());
}

template <int D, typename T, int TG, int MG>
int launch(cudaStream_t st, const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, bool pdl) {
    using S = Small<D, T, TG, MG>;
    static SmemOptIn seen;
    if (const int e = ensure_dyn_smem(small_kernel<D, T, TG, MG>, (size_t)S::SMEM, seen)) return e;
    const int ctas = tc_device_sms() * S::CTAS;
    if (const int e = launch_k(small_kernel<D, T, TG, MG>, dim3(ctas), dim3(S::THREADS), S::SMEM, st, pdl, mk, mv, a)) return e;
    return launch_k(join_kernel<D, T, S::M, TILE>, dim3(ctas - 1, S::M / 16), dim3(128), 0, st, true, a, ctas);
}
template <int D, typename T>
int launch_rows(cudaStream_t st, const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, int rows, bool pdl) {
    if (rows == 16) return launch<D, T, 4, 1>(st, mk, mv, a, pdl);
    if (rows == 32) return launch<D, T, 4, 2>(st, mk, mv, a, pdl);
    if constexpr (D < 256) return launch<D, T, 2, 4>(st, mk, mv, a, pdl);
    return -1000;
}
template <typename T>
int launch_dim(cudaStream_t st, const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, int rows, bool pdl) {
    switch (a.d.p.dim) {
        case 64: return launch_rows<64, T>(st, mk, mv, a, rows, pdl);
        case 128: return launch_rows<128, T>(st, mk, mv, a, rows, pdl);
        case 256: return launch_rows<256, T>(st, mk, mv, a, rows, pdl);
    }
    return -1000;
}

}  // namespace

size_t kv8_attention_bytes(int type, int heads, int kv_heads, int dim, int rows, int seqs, int max_rows) {
    if (!rows || !seqs) return 0;
    const bool flash = flash_takes(type, dim, heads / kv_heads, max_rows);
    const size_t small = (size_t)tc_device_sms() * 2 * 2 * rows_of(heads / kv_heads, dim, max_rows, flash), large = flash ? (size_t)tc_device_sms() * 2 * KV8_FLASH_ROWS : 0;
    return (small > large ? small : large) * (dim + 2) * 4;
}

int kv8_attention_launch(cudaStream_t st, const Kv8Attention& k, const Kv8Pool& pool, const Kv8Seqs& s, bool pdl) {
    if (s.rows == 0 || s.seqs == 0) return 0;
    const int group = k.heads / pool.kv_heads;
    const bool flash = flash_takes(k.q.type, pool.dim, group, k.max_rows);
    const int rows = rows_of(group, pool.dim, k.max_rows, flash), box = pool.dim < 128 ? pool.dim : 128;
    const uint64_t n = (uint64_t)pool.pages * pool.kv_heads * pool.page;
    CUtensorMap mk, mv;
    const CUtensorMapSwizzle sw = box == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    const uint32_t box_rows = pool.page < TILE ? pool.page : TILE;
    if (!tc_tmap(&mk, pool.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, n, pool.dim, pool.dim, box_rows, box, sw) ||
        !tc_tmap(&mv, pool.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, n, pool.dim, pool.dim, box_rows, box, sw)) return (int)cudaErrorInvalidValue;
    const double scale2 = (double)k.scale * 1.4426950408889634074;
    const Args a = {k.q.p, k.q.ld, k.q.ldh, k.out, k.ldo, k.ldoh, (float)scale2, (float)(scale2 - (double)(float)scale2), Kv8Deal{s, pool, group, 0, flash ? FLASH_FROM - 1 : 1LL << 62}, reinterpret_cast<float*>(k.work), k.err};
    if (k.q.type == KV8_F32) return launch_dim<float>(st, mk, mv, a, rows, pdl);
    if (const int e = k.q.type == KV8_BF16 ? launch_dim<bf16>(st, mk, mv, a, rows, pdl) : launch_dim<__half>(st, mk, mv, a, rows, pdl)) return e;
    if (!flash) return 0;
    Args f = a;
    f.d.lo = FLASH_FROM;
    f.d.hi = 1LL << 62;
    if (const int e = kv8_flash_launch(st, k, f.d, true)) return e;
    return k.q.type == KV8_BF16 ? join_flash<bf16>(st, f) : join_flash<__half>(st, f);
}

}  // namespace cb
