// Attention over an 8-bit paged cache (kv8.cuh): out = sum over visible i of softmax_i(scale q . k_i) v_i, a query at position p sees the positions up to p.
//
// e4m3 codes are exact in f16, so products run on f16 tensor cores with f32 sums.  Queries are scaled to the range of f16 by a power of two of their own (f32 ones
// are two f16 parts, 22 bits).  The scales stay out of the operands: a page's key scale multiplies its scores, its value scale joins the exponent,
//     p'_i = 2^(s_i + log2 vs_i - m),  m = running max of s_i + log2 vs_i,   out = sum p'_i v-code_i / sum p'_i / vs_i,
// so that the largest weight, scaled values counted in, always sits at the same place of f16's range.  m is a whole number: log2 vs - m is exact, and the exponent is rounded
// once, where it is small for the weights that count.
//
// Bound by bytes where there are few rows: a lane reads fragments of codes as they lie in shared memory (TMA, swizzled), two conversions for four codes, no transposition: 64 sequences of up
// to 8192 positions, 32 heads over 8, 128 columns: 529 MB in 113 us, 4.7 TB/s (of 6.46 measured); issue slots 36 %, eight warps an SM that wait for one another's latencies.
// By what it gave there: 16 positions a warp at a time 182, 32 of two tiles 145, a warp that brings the queries a unit ahead 129, four steps of a unit's own in the deal 113.
// Many rows (f32, or 256 columns) are bound by mma.sync: 44 % of its cycles, 16 or 32 rows beside conversions that every warp makes for itself.
#include <cuda_fp16.h>

#include <climits>

#include "kv8.cuh"
#include "tc.cuh"

namespace cb {
namespace {

constexpr float P_SHIFT = 14.f;                // weights run up to 2^14: f16 holds those down to 2^-28 of the largest with 11 bits

struct Args {
    const void* q; long long ldq, ldqh;
    void* out; long long ldo, ldoh;
    float scale2, scale2_rest;                 // scale * log2 e, and what f32 leaves of it
    Kv8Deal d;
    Kv8Join* joins;                            // [CTAs]
    float* work;                               // parts [2 * CTAs][rows of a group of rows][D + 2]
    int* err;
    bool vec;                                  // rows and heads of q and out start on 16-byte boundaries
};

// ---- fragments -------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void lds16(uint32_t a, uint32_t* r) { asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a)); }
__device__ __forceinline__ void lds8(uint32_t a, uint32_t* r) { asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a)); }
// four codes -> f16x2 of the first two and of the others, exact
__device__ __forceinline__ void halves_of(uint32_t codes, uint32_t& a, uint32_t& b) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(a), "=r"(b) : "r"(codes));
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

// Sixteen neighbouring columns; vec: on 16-byte boundaries
template <typename T> __device__ __forceinline__ void load16(const T* p, bool vec, float* y) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 16 * (int)sizeof(T) / 16; ++i) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
            const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
            for (int j = 0; j < 16 / (int)sizeof(T); ++j) y[i * (16 / (int)sizeof(T)) + j] = to_f<T>(e[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = to_f<T>(p[j]);
    }
}
template <typename T, int N> __device__ __forceinline__ void store_row(T* p, bool vec, const float* y) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < N * (int)sizeof(T) / 16; ++i) {
            __align__(16) T e[16 / sizeof(T)];
#pragma unroll
            for (int j = 0; j < 16 / (int)sizeof(T); ++j) e[j] = from_f<T>(y[i * (16 / (int)sizeof(T)) + j]);
            reinterpret_cast<uint4*>(p)[i] = *reinterpret_cast<const uint4*>(e);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) p[j] = from_f<T>(y[j]);
    }
}

// Shared memory of a step: keys, values [TILE positions][D] in boxes of at most 128 columns, swizzled by TMA
template <int D> struct Step {
    static constexpr int TILE = D == 256 ? 32 : 64;                         // positions
    static constexpr int BOX = D < 128 ? D : 128, PLANES = D / BOX, PLANE = TILE * BOX, BYTES = 2 * PLANES * PLANE;
};
template <int BOX> __device__ __forceinline__ uint32_t piece(int r, int c) { return BOX == 128 ? sw128_off(r, c) : sw64_off(r, c); }

// A warp has 16 query rows, up to 128 columns of the result, and takes 32 positions at a time: two slices of 16.  Which position and column a place of a fragment stands for is
// free as long as both operands agree; this order lets a lane read its codes 16 bytes at a time without bank conflicts and leave 16 neighbouring columns of the result:
//   place n of 8 positions: position pos8(n);  contraction of D: lane t of a quad has the 16-byte pieces t and t + 4 of a row of 128 (t of a row of 64)
//   columns: place n of the 8 of an MMA: piece col8(n) of a row (or 8 bytes of one of 64), the MMA's number the column in it
template <int D> __device__ __forceinline__ int pos8(int n) { return D == 64 ? n : (n & 1) * 4 + (n >> 1); }
__device__ __forceinline__ int col8(int n) { return (n & 1) * 4 + (n >> 1); }

// Four warps, a fifth that copies and a sixth that brings the queries of the next unit while they work, two such CTAs an SM: the four share rows (MG), columns of the result (CW)
// and positions (TG)
template <int D, typename T, int MG>
struct Small {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int TILE = Step<D>::TILE, DC = D < 128 ? D : 128, CW = D / DC, TG = 4 / (MG * CW), M = 16 * MG, WARPS = 4, THREADS = 192;
    static constexpr int SL = TILE / 16 / TG;                               // slices of a tile that a warp has: one (it takes those of two tiles together) or more
    static constexpr int AT_ONCE = SL == 1 ? 2 : 1;                         // tiles
    static constexpr int NT = DC / 8;                                       // MMAs across the columns
    static constexpr int KS = D / 16;                                       // ... along them
    static constexpr int QBYTES = MG * KS * 512 * (F32 ? 2 : 1), QB = QBYTES > 16 * 1024 ? 1 : 2;          // query fragments, and for how many units
    static constexpr int JOIN = (TG > 1 ? TG / 2 : 0) * MG * CW * 32 * (NT * 4 + 4) * 4;                   // sums on their way between warps
    static constexpr int CTAS = 2;                                          // resident on an SM (three, of 128 registers a thread: 189 us for a round of 64 sequences, two 145)
    static constexpr int ROOM = (227 * 1024) / CTAS - 1024 - 2816 - JOIN - QB * QBYTES - 1024;
    static constexpr int STAGES = ROOM / Step<D>::BYTES > 8 ? 8 : ROOM / Step<D>::BYTES;
    static constexpr int SMEM = STAGES * Step<D>::BYTES + JOIN + QB * QBYTES + 1024;
    static_assert(STAGES >= 3 && MG * CW * TG == 4 && SL * TG * 16 == TILE && (SL == 1 || SL % 2 == 0), "");
};

template <int D, typename T, int MG>
__global__ void __launch_bounds__(Small<D, T, MG>::THREADS, Small<D, T, MG>::CTAS)
small_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Args a) {
    using S = Small<D, T, MG>;
    using St = Step<D>;
    constexpr int M = S::M, NT = S::NT, KS = S::KS, STAGES = S::STAGES, TILE = S::TILE, TG = S::TG, CW = S::CW;
    constexpr bool F32 = S::F32;
    using Units = Kv8Units<M, TILE, 4>;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
    float* join = reinterpret_cast<float*>(sm + STAGES * St::BYTES);
    uint32_t* qs = reinterpret_cast<uint32_t*>(sm + STAGES * St::BYTES + S::JOIN);
    __shared__ uint64_t full[STAGES], empty[STAGES], q_full[2], q_empty[2];
    __shared__ float down_s[2][M];                           // what takes a row's scaled queries back
    __shared__ float4 meta[STAGES][TILE / 16];               // of each 16 positions: ks, log2 vs, 1 / vs, and whether there is a page
    __shared__ long long sums[KV8_SHARES + 1];
    __shared__ int gave_up;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        gave_up = 0;
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], S::WARPS); }
        for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], S::WARPS); }
        fence_barrier_init();
        tma_prefetch_desc(&map_k); tma_prefetch_desc(&map_v);
    }
    const TcWait wait{&gave_up, a.err};
    pdl_wait();
    const long long total = kv8_count<Units>(a.d, sums);
    const long long begin = kv8_range(total, gridDim.x, blockIdx.x), end = kv8_range(total, gridDim.x, blockIdx.x + 1);
    pdl_launch_dependents();
    if (tid == 0) a.joins[blockIdx.x].rows = 0;
    if (begin >= end) return;
    Units u = kv8_find<Units>(a.d, sums, begin);
    const int group = a.d.group;

    if (warp == S::WARPS) {
        // ---- copies: a box per page (TILE positions of it at most) and plane ----
        const int P = a.d.p.page, rows = min(P, TILE), boxes = TILE / rows;
        int stage = 0;
        uint32_t parity = 1;
        for (long long step = begin; step < end;) {
            const int t0 = u.tile_at(step), t1 = u.tile_at(u.stop(end)), n = (t1 - t0) * boxes;
            for (int base = 0; base < n; base += 32) {
                // a lane looks up one box: its row in the pool and its scales
                int row = a.d.p.pages * a.d.p.kv_heads * P;                  // behind the pool: zeros come
                float4 sc = make_float4(0.f, 0.f, 1.f, 0.f);
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
                    if (lane < TILE / 16) meta[stage][lane] = m;
                    __syncwarp();
                    if (lane == 0) mbar_arrive_expect_tx(&full[stage], St::BYTES);
                    __syncwarp();
                    // a lane has one box of keys or of values
                    const int j = lane / (2 * St::PLANES), r = __shfl_sync(0xffffffffu, row, (i - base + j) & 31);
                    if (j < boxes) {
                        const int pl = lane / 2 % St::PLANES;
                        tma_load_2d(st + (lane & 1) * St::PLANES * St::PLANE + pl * St::PLANE + j * rows * St::BOX, lane & 1 ? &map_v : &map_k, &full[stage], pl * St::BOX, r);
                    }
                    if (++stage == STAGES) { stage = 0; parity ^= 1; }
                }
            }
            step = u.stop(end);
            if (step < end && !u.next(a.d)) break;
        }
        __syncwarp();
        if (lane == 0) wait.drain();
        return;
    }

    const int g = lane >> 2, t = lane & 3;
    if (warp == S::WARPS + 1) {
        // ---- queries: fragments ----
        int buf = 0;
        uint32_t parity = 1;
        for (long long step = begin; step < end;) {
            wait(&q_empty[buf], parity);
            uint32_t* q = qs + buf * (S::QBYTES / 4);
#pragma unroll 1
            for (int i = 0; i < 2 * MG; ++i) {               // rows g and g + 8 of each 16
                const int r = i & 1, mg = i >> 1, row = u.grp * M + mg * 16 + g + r * 8, tok = row / group, h = u.head * group + row % group;
                const bool in = tok < u.q.n;
                const T* src = reinterpret_cast<const T*>(a.q) + (long long)(u.q.s0 + (in ? tok : 0)) * a.ldq + (long long)h * a.ldqh;
                float v[D / 4], top = 0.f;                   // this lane's columns of the row
#pragma unroll
                for (int p = 0; p < D / 64; ++p) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[p * 16 + j] = 0.f;
                    if (in) load16<T>(src + p * 64 + t * 16, a.vec, v + p * 16);
                }
#pragma unroll
                for (int j = 0; j < D / 4; ++j) top = v[j] != v[j] ? INFINITY : fmaxf(top, fabsf(v[j]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // 2^e that takes the row's largest magnitude to [2^14, 2^15); rows of less than 2^-100 count as zeros, rows with an infinity or a NaN give NaN
                const uint32_t ex = __float_as_uint(fmaxf(top, 0x1p-100f)) >> 23;
                const float up = __uint_as_float((uint32_t)(268 - ex) << 23);
                if (t == 0) down_s[buf][mg * 16 + g + r * 8] = top < INFINITY ? __uint_as_float((ex - 14) << 23) : NAN;
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {            // registers r and r + 2 of the fragment
                        const float x = top < INFINITY ? v[4 * s + 2 * c] * up : 0.f, y = top < INFINITY ? v[4 * s + 2 * c + 1] * up : 0.f;
                        const uint32_t f = pack_f16(x, y);
                        uint32_t* d = q + ((mg * KS + s) * 32 + lane) * 4 + r + 2 * c;
                        d[0] = f;
                        if (F32) { const float2 hf = unpack_f16(f); d[MG * KS * 128] = pack_f16(x - hf.x, y - hf.y); }
                    }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[buf]);
            if (++buf == S::QB) { buf = 0; parity ^= 1; }
            step = u.stop(end);
            if (step < end && !u.next(a.d)) break;
        }
        return;
    }

    // ---- products ----
    const int mg = warp % MG, cw = warp / MG % CW, tg = warp / (MG * CW);
    int stage = 0, buf = 0;
    uint32_t parity = 0, q_parity = 0;
    for (long long step = begin; step < end;) {
        const int t0 = u.tile_at(step), t1 = u.tile_at(u.stop(end));
        // ---- the unit's rows: what their scores are multiplied by, what they see ----
        float factor[2], fine[F32 ? 2 : 1];                  // ... and what f32 leaves of it
        int pmax[2], wmin = INT_MAX;                         // last visible position of rows g and g + 8; the warp's rows all see the positions up to wmin
        wait(&q_full[buf], q_parity);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = u.grp * M + mg * 16 + g + r * 8, tok = row / group;
            const bool in = tok < u.q.n;
            pmax[r] = in ? u.q.first + tok : -1;
            if (in) wmin = min(wmin, pmax[r]);
            const float down = down_s[buf][mg * 16 + g + r * 8];
            factor[r] = a.scale2 * down;
            if (F32) fine[F32 ? r : 0] = a.scale2_rest * down;
        }
        const uint4* qf = reinterpret_cast<const uint4*>(qs + buf * (S::QBYTES / 4)) + mg * KS * 32 + lane;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) wmin = min(wmin, __shfl_xor_sync(0xffffffffu, wmin, o));
        float o_acc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) { o_acc[j][0] = o_acc[j][1] = o_acc[j][2] = o_acc[j][3] = 0.f; }
        float m_row[2] = {-INFINITY, -INFINITY}, l_row[2] = {0.f, 0.f};
        uint32_t odd = 0;

        for (int tile = t0; tile < t1; tile += S::AT_ONCE) {
            const int stage2 = stage + 1 == STAGES ? 0 : stage + 1;
            const bool two = S::AT_ONCE == 1 || tile + 1 < t1;
            wait(&full[stage], parity);
            if (S::AT_ONCE == 2 && two) wait(&full[stage2], parity ^ (stage2 == 0));
#pragma unroll 1
            for (int sl = 0; sl < S::SL; sl += 2) {
                // ---- slices k = 0, 1: where they lie, what they are worth ----
                uint32_t kb[2];
                int pos0[2];
                float4 sc[2];
                const int s16 = tg * S::SL + sl;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int st = S::AT_ONCE == 2 && k ? stage2 : stage, s = S::AT_ONCE == 2 ? s16 : s16 + k;
                    kb[k] = smem_u32(sm + st * St::BYTES) + s * 16 * St::BOX;
                    pos0[k] = (tile + (S::AT_ONCE == 2 ? k : 0)) * TILE + s * 16;
                    sc[k] = meta[st][s];
                }
                if (!two) { sc[1] = make_float4(0.f, 0.f, 1.f, 0.f); }
                const bool edge = pos0[1] + 15 > wmin || sc[0].w == 0.f || sc[1].w == 0.f;      // not all of the warp's rows see all of it
                if (edge && __all_sync(0xffffffffu, (sc[0].w == 0.f || (pos0[0] > pmax[0] && pos0[0] > pmax[1])) && (sc[1].w == 0.f || (pos0[1] > pmax[0] && pos0[1] > pmax[1])))) continue;
                // ---- scores ----
                float s_acc[2][2][4];
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s_acc[k][nt][e] = 0.f;
#pragma unroll
                for (int p = 0; p < D / 64; ++p) {           // pieces t, t + 4 of each plane
                    uint32_t w[2][2][4];
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt) lds16(kb[k] + (p / 2) * St::PLANE + piece<St::BOX>(nt * 8 + pos8<D>(g), (p & 1) * 4 + t), w[k][nt]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 q4 = qf[(p * 4 + i) * 32];
                        const uint32_t x[4] = {q4.x, q4.y, q4.z, q4.w};
                        uint32_t z[4] = {0, 0, 0, 0};
                        if (F32) { const uint4 l4 = qf[MG * KS * 32 + (p * 4 + i) * 32]; z[0] = l4.x; z[1] = l4.y; z[2] = l4.z; z[3] = l4.w; }
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int nt = 0; nt < 2; ++nt) {
                                uint32_t b0, b1;
                                halves_of(w[k][nt][i], b0, b1);
                                if (F32) mma_f16(s_acc[k][nt], z, b0, b1);
                                mma_f16(s_acc[k][nt], x, b0, b1);
                            }
                    }
                }
                // ---- weights ----
                float f[2][2], mx[2] = {-INFINITY, -INFINITY};
                uint32_t hidden = 0;
#pragma unroll
                for (int k = 0; k < 2; ++k) { f[k][0] = factor[0] * sc[k].x; f[k][1] = factor[1] * sc[k].x; }
                if (edge) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (sc[k].w == 0.f || pos0[k] + nt * 8 + pos8<D>(2 * t + (e & 1)) > pmax[e >> 1]) hidden |= 1u << (k * 8 + nt * 4 + e);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (edge) {
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (!(hidden >> (k * 8 + nt * 4 + e) & 1)) mx[e >> 1] = fmaxf(mx[e >> 1], fmaf(s_acc[k][nt][e], f[k][e >> 1], sc[k].y));
                    } else {
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], fmaf(s_acc[k][nt][e], f[k][e >> 1], sc[k].y));
                    }
                }
                float corr[2];
                bool far = false;                            // scores whose last bit is worth more than a weight: their exponents are differences of rounded numbers
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                    const float mn = fmaxf(m_row[r], ceilf(mx[r]));
                    corr[r] = m_row[r] == mn ? 1.f : ex2(m_row[r] - mn);
                    m_row[r] = mn;
                    far |= fabsf(mn) > 0x1p20f && fabsf(mn) < INFINITY;
                }
                if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
                    l_row[0] *= corr[0]; l_row[1] *= corr[1];
#pragma unroll
                    for (int j = 0; j < NT; ++j) { o_acc[j][0] *= corr[0]; o_acc[j][1] *= corr[0]; o_acc[j][2] *= corr[1]; o_acc[j][3] *= corr[1]; }
                }
                if (__any_sync(0xffffffffu, far)) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s_acc[k][nt][e] = ex2(fmaf(s_acc[k][nt][e], f[k][e >> 1], sc[k].y) - m_row[e >> 1] + P_SHIFT);
                } else {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float b[2] = {m_row[0] == -INFINITY ? 0.f : sc[k].y - (m_row[0] - P_SHIFT), m_row[1] == -INFINITY ? 0.f : sc[k].y - (m_row[1] - P_SHIFT)};
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                s_acc[k][nt][e] = ex2(fmaf(s_acc[k][nt][e], f[k][e >> 1], F32 ? fmaf(s_acc[k][nt][e], fine[F32 ? e >> 1 : 0] * sc[k].x, b[e >> 1]) : b[e >> 1]));
                    }
                }
                if (edge)
#pragma unroll
                    for (int i = 0; i < 16; ++i) if (hidden >> i & 1) s_acc[i >> 3][i >> 2 & 1][i & 3] = 0.f;
                uint32_t pa[2][4], pl[F32 ? 2 : 1][4];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float (&s)[2][4] = s_acc[k];
                    l_row[0] = fmaf((s[0][0] + s[0][1]) + (s[1][0] + s[1][1]), sc[k].z, l_row[0]);
                    l_row[1] = fmaf((s[0][2] + s[0][3]) + (s[1][2] + s[1][3]), sc[k].z, l_row[1]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {            // rows g, g + 8 of positions 0 - 7, then of 8 - 15
                        const float x = s[i >> 1][(i & 1) * 2], y = s[i >> 1][(i & 1) * 2 + 1];
                        pa[k][i] = pack_f16(x, y);
                        if (F32) { const float2 hf = unpack_f16(pa[k][i]); pl[F32 ? k : 0][i] = pack_f16(x - hf.x, y - hf.y); }
                    }
                }
                // ---- values: two positions' codes side by side ----
                constexpr int W = St::BOX == 128 ? 4 : 2;                // words of four columns that a lane has of a row
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t x[4][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = pos8<D>(2 * t + (i & 1)) + (i >> 1) * 8;
                        const uint32_t vb = kb[k] + (St::PLANES + cw) * St::PLANE;
                        if constexpr (St::BOX == 128) lds16(vb + piece<128>(r, col8(g)), x[i]);
                        else lds8(vb + piece<64>(r, g >> 1) + (g & 1) * 8, x[i]);
                    }
                    if (edge) {                              // a NaN among values that some row does not see: 0 * NaN must not reach that one; those that see it look it up
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool page = sc[k].w != 0.f;
                            if (page && pos0[k] + pos8<D>(2 * t + (i & 1)) + (i >> 1) * 8 <= wmin) continue;      // (all see it: it stays)
#pragma unroll
                            for (int w = 0; w < W; ++w) {
                                const uint32_t n = (((x[i][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
                                if (page) odd |= n;
                                x[i][w] &= ~(n * 255u);
                            }
                        }
                    }
#pragma unroll
                    for (int w = 0; w < W; ++w)
#pragma unroll
                        for (int c2 = 0; c2 < 2; ++c2) {     // columns 4 w + 2 c2 and the next
                            uint32_t b[2][2];                // column, positions 0 - 7 and 8 - 15
#pragma unroll
                            for (int i = 0; i < 2; ++i) halves_of(__byte_perm(x[2 * i][w], x[2 * i + 1][w], c2 ? 0x7362 : 0x5140), b[0][i], b[1][i]);
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                float* acc = o_acc[w * 4 + c2 * 2 + c];
                                if constexpr (F32) {         // (long sums are f32 additions: the tensor core cuts its sums off where f32 rounds)
                                    float part[4] = {0.f, 0.f, 0.f, 0.f};
                                    mma_f16(part, pl[F32 ? k : 0], b[c][0], b[c][1]);
                                    mma_f16(part, pa[k], b[c][0], b[c][1]);
#pragma unroll
                                    for (int e = 0; e < 4; ++e) acc[e] += part[e];
                                } else {
                                    mma_f16(acc, pa[k], b[c][0], b[c][1]);
                                }
                            }
                        }
                }
            }
            __syncwarp();
            if (lane == 0) { mbar_arrive(&empty[stage]); if (S::AT_ONCE == 2 && two) mbar_arrive(&empty[stage2]); }
#pragma unroll
            for (int i = 0; i < S::AT_ONCE; ++i) if (i == 0 || two) { if (++stage == STAGES) { stage = 0; parity ^= 1; } }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_empty[buf]);
        if (++buf == S::QB) { buf = 0; q_parity ^= 1; }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l_row[r] += __shfl_xor_sync(0xffffffffu, l_row[r], 1);
            l_row[r] += __shfl_xor_sync(0xffffffffu, l_row[r], 2);
        }
        if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
            for (int pos = max(wmin == INT_MAX ? INT_MAX : wmin + 1, t0 * TILE); pos < min(t1 * TILE, u.q.len); ++pos) {
                const int page = kv8_page(a.d.s, a.d.p, u.b, pos / a.d.p.page);
                if (page < 0) continue;
                const unsigned char* v = a.d.p.v + (((size_t)page * a.d.p.kv_heads + u.head) * a.d.p.page + pos % a.d.p.page) * D + cw * 128;
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        if ((__ldg(v + (D == 64 ? (2 * t + e) * 8 : col8(2 * t + e) * 16) + j) & 0x7f) == 0x7f) {
                            if (pos <= pmax[0]) o_acc[j][e] = NAN;
                            if (pos <= pmax[1]) o_acc[j][2 + e] = NAN;
                        }
            }
        }
        // ---- the warps that share rows and columns add up, half of them into the other half each time ----
#pragma unroll
        for (int h = TG / 2; h >= 1; h /= 2) {
            named_bar_sync(1, S::WARPS * 32);
            float* d = join + (size_t)((tg % h) * (MG * CW) + cw * MG + mg) * 32 * (NT * 4 + 4) + lane;
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
                    c0[r] = m_row[r] == -INFINITY ? 0.f : m_row[r] == mn ? 1.f : ex2(m_row[r] - mn);
                    c1[r] = mo == -INFINITY ? 0.f : mo == mn ? 1.f : ex2(mo - mn);
                    m_row[r] = mn;
                    l_row[r] = l_row[r] * c0[r] + d[(NT * 4 + 2 + r) * 32] * c1[r];
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o_acc[j][e] = o_acc[j][e] * c0[e >> 1] + d[(j * 4 + e) * 32] * c1[e >> 1];
            }
        }
        if (tid == 0 && u.begins(step, end)) a.joins[blockIdx.x] = kv8_join(a.d, u, M, total, gridDim.x, blockIdx.x, begin);
        if (tg == 0) {
            const bool whole = u.whole(step, end);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = mg * 16 + g + r * 8, tok = (u.grp * M + row) / group, h = u.head * group + (u.grp * M + row) % group;
                // 16 neighbouring columns a lane and half (8 of rows of 64)
                const float inv = !whole ? 1.f : l_row[r] == 0.f ? 0.f : 1.f / l_row[r];
                T* dst = reinterpret_cast<T*>(a.out) + (long long)(u.q.s0 + tok) * a.ldo + (long long)h * a.ldoh + cw * 128;
                float* part = a.work + ((size_t)kv8_slot(blockIdx.x, begin, step) * M + row) * (D + 2);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int col = D == 64 ? (2 * t + e) * 8 : col8(2 * t + e) * 16;
                    float y[NT];
#pragma unroll
                    for (int j = 0; j < NT; ++j) y[j] = o_acc[j][2 * r + e] * inv;
                    if (!whole) {
#pragma unroll
                        for (int j = 0; j < NT; j += 2) *reinterpret_cast<float2*>(part + cw * 128 + col + j) = make_float2(y[j], y[j + 1]);
                    } else if (tok < u.q.n) store_row<T, NT>(dst + col, a.vec, y);
                }
                if (!whole && t == 0 && cw == 0) { part[D] = m_row[r]; part[D + 1] = l_row[r]; }
            }
        }
        step = u.stop(end);
        if (step < end && !u.next(a.d)) break;
    }
    if (tid == 0) wait.drain();
}

// Adds up the parts of the units that lie with several CTAs.  Block x: the unit that CTA x began and did not end; its rows by turns, the parts by turns of its warps.
template <int D, typename T, int M>
__global__ void __launch_bounds__(128)
join_kernel(Args a) {
    constexpr int V = D / 32;                                        // columns of a lane
    __shared__ float o_s[4][D], l_s[4];
    pdl_wait();
    pdl_launch_dependents();
    const Kv8Join u = a.joins[blockIdx.x];
    const int c = blockIdx.x, parts = u.last - c + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto store = [&](int row, int j, float y) {
        const int rr = u.grp * M + row, tok = rr / a.d.group, h = u.head * a.d.group + rr % a.d.group;
        reinterpret_cast<T*>(a.out)[(long long)(u.s0 + tok) * a.ldo + (long long)h * a.ldoh + j] = from_f<T>(y);
    };
    constexpr int B = 8;                                             // parts on their way at once
    if (parts <= B) {                                                // a row a warp
        for (int row = blockIdx.y * 4 + warp; row < u.rows; row += 4 * gridDim.y) {
            float m[B], s[B], y[B][V], top = -INFINITY, l = 0.f;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                m[i] = -INFINITY;
                if (i >= parts) continue;
                const float* src = a.work + ((size_t)(i ? kv8_slot(c + i, 0, 0) : u.slot) * M + row) * (D + 2);
                m[i] = src[D];
                s[i] = src[D + 1];
#pragma unroll
                for (int j = 0; j < V; ++j) y[i][j] = src[lane + j * 32];
            }
#pragma unroll
            for (int i = 0; i < B; ++i) top = fmaxf(top, m[i]);
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = 0.f;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                if (i >= parts) continue;
                const float f = m[i] == -INFINITY ? 0.f : m[i] == top ? 1.f : ex2(m[i] - top);
                l = fmaf(s[i], f, l);
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = fmaf(y[i][j], f, o[j]);
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int j = 0; j < V; ++j) store(row, lane + j * 32, o[j] * inv);
        }
        return;
    }
    for (int row = blockIdx.y; row < u.rows; row += gridDim.y) {
        const float* first = a.work + ((size_t)u.slot * M + row) * (D + 2);
        auto part = [&](int k) { return k == 0 ? first : a.work + ((size_t)kv8_slot(c + k, 0, 0) * M + row) * (D + 2); };
        float top = -INFINITY;
        for (int k = lane; k < parts; k += 32) top = fmaxf(top, part(k)[D]);
        top = warp_max(top);
        float o[V], l = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = 0.f;
        for (int k0 = warp; k0 < parts; k0 += 4 * B) {
            float m[B], s[B], y[B][V];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const float* src = part(min(k0 + 4 * i, parts - 1));
                m[i] = src[D];
                s[i] = src[D + 1];
#pragma unroll
                for (int j = 0; j < V; j += 2) { const float2 v = *reinterpret_cast<const float2*>(src + lane * 2 + j * 32); y[i][j] = v.x; y[i][j + 1] = v.y; }
            }
#pragma unroll
            for (int i = 0; i < B; ++i) {
                if (k0 + 4 * i >= parts) continue;
                const float f = m[i] == -INFINITY ? 0.f : m[i] == top ? 1.f : ex2(m[i] - top);
                l = fmaf(s[i], f, l);
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = fmaf(y[i][j], f, o[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < V; j += 2) *reinterpret_cast<float2*>(&o_s[warp][lane * 2 + j * 32]) = make_float2(o[j], o[j + 1]);
        if (lane == 0) l_s[warp] = l;
        __syncthreads();
        l = (l_s[0] + l_s[1]) + (l_s[2] + l_s[3]);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        for (int j = threadIdx.x; j < D; j += 128) store(row, j, ((o_s[0][j] + o_s[1][j]) + (o_s[2][j] + o_s[3][j])) * inv);
        __syncthreads();
    }
}

// Rows of a kv head from which on a sequence goes through kv8_flash.cu: 16-bit ones of 64 and 128 columns.  Us, here / there, 32 heads over 8 of 128, bf16, sequences that bring 96, 128, 256 and
// 512 rows of a kv head.  Eight with nothing ahead of them: 24, 23, 30, 51 / 50, 50, 51, 55; behind 1000 positions: 37, 44, 68, 120 / 58, 61, 62, 81; behind 8000: 139, 177, 333, 645 / 119,
// 119, 121, 192; 16 behind 8000: 255, 332, 640, 1262 / 186, 186, 191, 327; one: 39, 44, 59, 100 / 56, 58, 62, 75.  Its launches cost 20 us where there is little to do, rows here cost 70 where
// there is much from the first group of 32 behind the 64th row on; the lengths, which tell, are on the device only.
constexpr int FLASH_FROM = 65;
bool flash_takes(int type, int dim, int group, int max_rows) { return type != KV8_F32 && dim <= 128 && (long long)group * max_rows >= FLASH_FROM; }
// Rows of a group of queries: 16, or 32 where some sequence may bring many and none goes to kv8_flash.cu.  Us, 16 / 32 / 64 rows: portions of 500 tokens, 16 heads over 8, f32 231 / 177 /
// 190; up to 9 drafts, 32 heads over 8, bf16 45 / 52 / 87; 23 sequences, portions of up to 333 tokens among decoded ones, f32 245 / 234 / 267.
int rows_of(int group, int max_rows, bool flash) { return flash || (long long)group * max_rows <= 64 ? 16 : 32; }
template <typename T>
int join_flash(cudaStream_t st, const Args& a) {
    auto k = a.d.p.dim == 64 ? join_kernel<64, T, KV8_FLASH_ROWS> : join_kernel<128, T, KV8_FLASH_ROWS>;
    return launch_k(k, dim3(tc_device_sms() - 1, 64), dim3(128), 0, st, true, a);
}

template <int D, typename T, int MG>
int launch(cudaStream_t st, const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, bool pdl) {
    using S = Small<D, T, MG>;
    static SmemOptIn seen;
    if (const int e = ensure_dyn_smem(small_kernel<D, T, MG>, (size_t)S::SMEM, seen)) return e;
    const int ctas = tc_device_sms() * S::CTAS;
    if (const int e = launch_k(small_kernel<D, T, MG>, dim3(ctas), dim3(S::THREADS), S::SMEM, st, pdl, mk, mv, a)) return e;
    return launch_k(join_kernel<D, T, S::M>, dim3(ctas - 1, S::M / 4), dim3(128), 0, st, true, a);
}
template <int D, typename T>
int launch_rows(cudaStream_t st, const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, int rows, bool pdl) {
    return rows == 16 ? launch<D, T, 1>(st, mk, mv, a, pdl) : launch<D, T, 2>(st, mk, mv, a, pdl);
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
    const size_t small = (size_t)tc_device_sms() * 2 * 2 * rows_of(heads / kv_heads, max_rows, flash), large = flash ? (size_t)tc_device_sms() * 2 * KV8_FLASH_ROWS : 0;
    return kv8_joins(2 * tc_device_sms()) + (small > large ? small : large) * (dim + 2) * 4;
}

int kv8_attention_launch(cudaStream_t st, const Kv8Attention& k, const Kv8Pool& pool, const Kv8Seqs& s, bool pdl) {
    if (s.rows == 0 || s.seqs == 0) return 0;
    const int group = k.heads / pool.kv_heads;
    const bool flash = flash_takes(k.q.type, pool.dim, group, k.max_rows);
    const int rows = rows_of(group, k.max_rows, flash), box = pool.dim < 128 ? pool.dim : 128;
    const uint64_t n = (uint64_t)pool.pages * pool.kv_heads * pool.page;
    CUtensorMap mk, mv;
    const CUtensorMapSwizzle sw = box == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    const int tile = pool.dim == 256 ? 32 : 64;
    const uint32_t box_rows = pool.page < tile ? pool.page : tile;
    if (!tc_tmap(&mk, pool.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, n, pool.dim, pool.dim, box_rows, box, sw) ||
        !tc_tmap(&mv, pool.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, n, pool.dim, pool.dim, box_rows, box, sw)) return (int)cudaErrorInvalidValue;
    const int per = k.q.type == KV8_F32 ? 4 : 8;
    const bool vec = (reinterpret_cast<uintptr_t>(k.q.p) | reinterpret_cast<uintptr_t>(k.out)) % 16 == 0 && (k.q.ld | k.q.ldh | k.ldo | k.ldoh) % per == 0;
    const double scale2 = (double)k.scale * 1.4426950408889634074;
    const Args a = {k.q.p, k.q.ld, k.q.ldh, k.out, k.ldo, k.ldoh, (float)scale2, (float)(scale2 - (double)(float)scale2), Kv8Deal{s, pool, group, 0, flash ? FLASH_FROM - 1 : 1LL << 62}, reinterpret_cast<Kv8Join*>(k.work), reinterpret_cast<float*>(reinterpret_cast<char*>(k.work) + kv8_joins(2 * tc_device_sms())), k.err, vec};
    const int e = k.q.type == KV8_F32 ? launch_dim<float>(st, mk, mv, a, rows, pdl) : k.q.type == KV8_BF16 ? launch_dim<bf16>(st, mk, mv, a, rows, pdl) : launch_dim<__half>(st, mk, mv, a, rows, pdl);
    if (e) return e;
    if (!flash) return 0;
    Args f = a;
    f.d.lo = FLASH_FROM;
    f.d.hi = 1LL << 62;
    if (const int e = kv8_flash_launch(st, k, f.d, f.joins, f.work, true)) return e;
    return k.q.type == KV8_BF16 ? join_flash<bf16>(st, f) : join_flash<__half>(st, f);
}

}  // namespace cb
