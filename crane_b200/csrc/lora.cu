// Low-rank adapters of many requests (lora.cuh).  One kernel: a cluster of CTAs has a tile of rows that go through the same adapter.  Its CTAs each take a share of the
// k columns of T = X A^T, add their shares up in distributed shared memory, and then each take a share of the n columns of out = add + s T B^T.  T never leaves the SMs;
// there is no workspace and nothing to wait for outside the cluster.
//
// T is f32 and multiplied by the adapter's scale before it is split into two parts of the weights' type (bf16: 16 bits; f16: 22, each row moved into f16's range by a power of
// two of its own), so that the rank's sum loses nothing that a 16-bit result could show.  f32 weights or rows: tf32 parts, hi hi + lo hi + hi lo, 2^-22 of each product.
//
// Bound by bytes in principle: for single rows those of A and B, for prompts those of add and out.  Which k a place of a fragment stands for is free as long as both operands agree, so a
// lane takes 16 neighbouring bytes of a row straight from global memory, and the columns of a result are dealt so that a lane leaves eight neighbours.  Up to 384 rows any 16 that share
// an adapter are a tile; beyond, 64 neighbours, one adapter after the other, the first few of them by clusters of their own, and add and B come in through a ring of stages.
// 8192 rows x 4096 -> 24 576, rank 64, bf16: 401 us (883 MB: 137): fixed work of a CTA (its sums, the cluster's, T's parts) 84, X A^T 50; add, B, products and stores, some 70 each,
// one behind the other (leaving any one out saves its 70): eight warps in step, which is why lora_tiles.cu has these.  Without the ring 570.  One row 5.6, 33 rows of 20 adapters, f32, 25.6 (36 MB: 5.6).
#include <cuda_fp16.h>

#include <algorithm>

#include "lora.cuh"
#include "tc.cuh"

namespace cb {
namespace {

constexpr int THREADS = 256, WARPS = 8;

template <typename T> constexpr int TYPE = 0;
template <> constexpr int TYPE<bf16> = 1;
template <> constexpr int TYPE<__half> = 2;
template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<bf16>(bf16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// N neighbouring elements as they lie, `have` of them there (VEC: all or none, aligned); the rest zeros
template <typename T, int N> struct Piece {
    static constexpr int W = N * (int)sizeof(T) / 4;
    uint32_t w[W];
    __device__ __forceinline__ float at(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else {
            const unsigned short u = (unsigned short)(w[i / 2] >> (16 * (i & 1)));
            if constexpr (TYPE<T> == 1) return __uint_as_float((uint32_t)u << 16);
            else return __half2float(__ushort_as_half(u));
        }
    }
};
// Any boundary: the aligned 16 bytes that hold one of them, moved into place.  RO: nobody writes them while the kernel runs.
template <typename T, int N, bool VEC, bool RO = true>
__device__ __forceinline__ Piece<T, N> load(const T* p, int have) {
    Piece<T, N> r;
    constexpr int W = Piece<T, N>::W;
    auto get = [](const uint4* q) { if constexpr (RO) return __ldg(q); else return *q; };
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = 0;
        if (have >= N) {
            if constexpr (W < 4) {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
                r.w[0] = v.x; r.w[1] = v.y;
            } else {
#pragma unroll
                for (int i = 0; i < W; i += 4) { const uint4 v = get(reinterpret_cast<const uint4*>(p) + i / 4); r.w[i % W] = v.x; r.w[(i + 1) % W] = v.y; r.w[(i + 2) % W] = v.z; r.w[(i + 3) % W] = v.w; }
            }
        }
    } else {
        constexpr int B = (W + 3) / 4 + 1;                           // aligned pieces that may hold something of it
        uint32_t w[4 * B + 1];
        const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15), n = min(have, N) * (int)sizeof(T);
        const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)15);
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const uint4 v = n > 0 && 16 * i < off + n ? get(q + i) : make_uint4(0, 0, 0, 0);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
        w[4 * B] = 0;
#pragma unroll
        for (int s = 2; s >= 1; s >>= 1)
            if (off >> 2 & s)
#pragma unroll
                for (int i = 0; i + s <= 4 * B; ++i) w[i] = w[i + s];
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = sizeof(T) == 4 ? w[i] : __funnelshift_r(w[i], w[i + 1], (off & 2) * 8);
        if (n < N * (int)sizeof(T))
#pragma unroll
            for (int i = 0; i < W; ++i) r.w[i] &= n >= 4 * i + 4 ? 0xffffffffu : n <= 4 * i ? 0u : 0xffffu;
    }
    return r;
}
// Eight neighbours, `have` of them there
template <typename T, bool VEC> __device__ __forceinline__ void store8(T* p, int have, const T* y) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(y);
    constexpr int W = 2 * (int)sizeof(T);
    if constexpr (VEC) {
        if (have >= 8)
#pragma unroll
            for (int q = 0; q < W / 4; ++q) reinterpret_cast<uint4*>(p)[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int q = 0; q < 8; ++q) if (q < have) p[q] = y[q];
    } else if (have >= 8) {                                          // 32 bits at a time, a single one at either end of an odd row
        if (reinterpret_cast<uintptr_t>(p) & 2) {
            p[0] = y[0];
#pragma unroll
            for (int q = 0; q < 3; ++q) *reinterpret_cast<uint32_t*>(p + 1 + 2 * q) = __funnelshift_r(w[q], w[q + 1], 16);
            p[7] = y[7];
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) reinterpret_cast<uint32_t*>(p)[q] = w[q];
        }
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) if (q < have) p[q] = y[q];
    }
}

template <typename W> __device__ __forceinline__ void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (TYPE<W> == 1)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tf32(float v) { uint32_t r; asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v)); return r; }
// what `hi` leaves of v; nothing of an infinity (inf - inf would make a NaN of it)
__device__ __forceinline__ float rest(float v, float hi) { return fabsf(hi) < INFINITY ? v - hi : 0.f; }
__device__ __forceinline__ uint32_t tf32_rest(float v, uint32_t hi) { return tf32(rest(v, __uint_as_float(hi))); }

template <typename X, typename W, int MT, int RT>
struct Shape {
    static constexpr bool T32 = sizeof(X) == 4;                      // tf32 products; else those of the 16-bit type
    static constexpr int ROWS = 16 * MT, RP = 8 * RT, LDT = RP + 4;
    static constexpr int MPW = MT == 1 || RT == 16 ? 1 : 2, MW = MT / MPW, KW = WARPS / MW;      // X A^T: row tiles of a warp, warps along the rows, along k
    static constexpr int EM = MT == 1 ? 1 : 2, EW = MT / EM, CW = WARPS / EW;                    // T B^T: the same, along n
    static constexpr int EB = MT > 1 ? 1 : T32 && RT > 4 ? 1 : 2;    // blocks of 32 columns a warp has under way
    static constexpr int KS = T32 ? RT : RT / 2;                     // MMAs along the rank
    static constexpr int T_BYTES = ROWS * LDT * 4, FRAG = MT * KS * 32 * 16;
    // Many rows: the columns of a step, add and B, come in through a ring of stages
    static constexpr int NC = CW * 32, ADD = ROWS * NC * (int)sizeof(X), STAGE = ADD + NC * RP * (int)sizeof(W);
    static constexpr int T_ROOM = 2 * T_BYTES;                       // shares of T (this CTA's, read by the cluster) and T; the stages come into the same room
    static constexpr int CTAS = MT == 1 || 2 * FRAG + 3 * STAGE <= 112 * 1024 ? 2 : 1;               // resident on an SM
    static constexpr int FITS = ((CTAS == 2 ? 112 : 222) * 1024 - 2 * FRAG) / STAGE, STAGES = MT == 1 || FITS < 2 ? 0 : FITS > 4 ? 4 : FITS;
    static constexpr int ROOM = STAGES * STAGE > T_ROOM ? STAGES * STAGE : T_ROOM, SMEM = 2 * FRAG + ROOM;      // ahead of those the two parts of T
};

// o += T B^T over 16 of the rank: EM row tiles from `er` on, 32 columns
template <typename X, typename W, int EM, int KS>
__device__ __forceinline__ void multiply(float (&o)[EM][4][4], const Piece<W, 4> (&bv)[4], const uint4* hi_s, const uint4* lo_s, int er, int ks, int lane) {
    if constexpr (sizeof(X) != 4) {
#pragma unroll
        for (int half = 0; half < 2; ++half)                 // (all of the lower parts first: no product waits for the one ahead of it)
#pragma unroll
            for (int i = 0; i < EM; ++i) {
                const uint4 v = (half ? hi_s : lo_s)[((er + i) * KS + ks) * 32 + lane];
                const uint32_t f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) mma16<W>(o[i][j], f, bv[j].w[0], bv[j].w[1]);
            }
    } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            uint32_t bh[4][2], bl[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) { const float v = bv[j].at(2 * s + e); bh[j][e] = tf32(v); if (sizeof(W) == 4) bl[j][e] = tf32_rest(v, bh[j][e]); }
#pragma unroll
            for (int i = 0; i < EM; ++i) {
                const uint4 hv = hi_s[((er + i) * KS + ks * 2 + s) * 32 + lane], lv = lo_s[((er + i) * KS + ks * 2 + s) * 32 + lane];
                const uint32_t fh[4] = {hv.x, hv.y, hv.z, hv.w}, fl[4] = {lv.x, lv.y, lv.z, lv.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (sizeof(W) == 4) mma_tf32(o[i][j], fh, bl[j][0], bl[j][1]);
                    mma_tf32(o[i][j], fl, bh[j][0], bh[j][1]);
                    mma_tf32(o[i][j], fh, bh[j][0], bh[j][1]);
                }
            }
        }
    }
}

template <typename X, typename W, int MT, int RT, bool VEC>
__global__ void __launch_bounds__(THREADS, Shape<X, W, MT, RT>::CTAS)
lora_kernel(Lora l, bool gather, int slots) {
    using S = Shape<X, W, MT, RT>;
    constexpr bool T32 = S::T32;
    constexpr int ROWS = S::ROWS, LDT = S::LDT, KS = S::KS, MW = S::MW, KW = S::KW, MPW = S::MPW, EM = S::EM, EW = S::EW, CW = S::CW, EB = S::EB;
    extern __shared__ __align__(16) unsigned char sm[];
    uint4* hi_s = reinterpret_cast<uint4*>(sm);
    uint4* lo_s = hi_s + S::FRAG / 16;
    float* share = reinterpret_cast<float*>(sm + 2 * S::FRAG);
    float* ts = share + S::T_BYTES / 4;
    __shared__ int rows_s[ROWS], which_s[ROWS];
    __shared__ float down_s[ROWS];                                   // powers of two that take the rows of T back out of f16's range
    __shared__ int n_rows_s;
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    uint32_t cl;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(cl));
    const int cr = (int)cluster_rank(), nc = (int)cl, tile = blockIdx.x / nc / slots, slot = blockIdx.x / nc % slots;

    // ---- the tile's rows ----
    if (gather) {
        // tile r: rows r and on that go through row r's adapter, if the number of those ahead of r is a multiple of ROWS
        if (warp == 0) {
            const int w = __ldg(l.which + tile);
            int w0 = (unsigned)w < (unsigned)l.adapters ? w : -1, ahead = 0, have = 0;
            for (int i = 0; i < l.m && have < ROWS; i += 32) {
                int v = -2;
                if (i + lane < l.m) { v = __ldg(l.which + i + lane); if ((unsigned)v >= (unsigned)l.adapters) v = -1; }
                const unsigned same = __ballot_sync(0xffffffffu, v == w0);
                const unsigned from = i + 31 < tile ? 0u : i >= tile ? 0xffffffffu : 0xffffffffu << (tile - i);      // rows >= tile
                ahead += __popc(same & ~from);
                const unsigned mine = same & from;
                const int at = have + __popc(mine & ((1u << lane) - 1));
                if ((mine >> lane & 1) && at < ROWS) { rows_s[at] = i + lane; which_s[at] = w0; }
                have = min(ROWS, have + __popc(mine));
                if (i + 31 >= tile && ahead % ROWS) break;
            }
            if (lane == 0) n_rows_s = ahead % ROWS ? 0 : have;
        }
    } else {
        for (int i = tid; i < ROWS; i += THREADS) {
            const int r = tile * ROWS + i;
            rows_s[i] = r;
            int v = r < l.m ? __ldg(l.which + r) : -1;
            which_s[i] = (unsigned)v < (unsigned)l.adapters ? v : -1;
        }
        if (tid == 0) n_rows_s = min(ROWS, l.m - tile * ROWS);
    }
    __syncthreads();
    const int n_rows = n_rows_s;
    if (n_rows == 0) return;                                         // (the whole cluster's CTAs alike)

    const X* x = reinterpret_cast<const X*>(l.x);
    const X* add = reinterpret_cast<const X*>(l.add);
    X* out = reinterpret_cast<X*>(l.out);
    const int nb = (l.n + 31) / 32, nb0 = (int)((long long)nb * cr / nc), nb1 = (int)((long long)nb * (cr + 1) / nc);
    unsigned long long left = n_rows == 64 ? ~0ull : (1ull << n_rows) - 1;
    for (int turn = 0; left;) {
        // ---- the next adapter among the rows that are left ----
        const int w = which_s[__ffsll(left) - 1];
        unsigned long long mine = __ballot_sync(0xffffffffu, lane < ROWS && which_s[lane % ROWS] == w);
        if constexpr (ROWS > 32) mine |= (unsigned long long)__ballot_sync(0xffffffffu, which_s[(lane + 32) % ROWS] == w) << 32;
        mine &= left;
        left &= ~mine;
        if (turn++ % slots != slot) continue;                        // another cluster's adapter
        const W* B = reinterpret_cast<const W*>(l.b) + (size_t)max(w, 0) * l.n * l.rank;
        // ---- the ring: a thread fetches the same piece of every AR-th row of add and of every BR-th row of B, whatever the step ----
        constexpr bool STAGED = VEC && S::STAGES > 0;
        constexpr int ST = S::STAGES, NC = S::NC, CX = NC * (int)sizeof(X) / 16, CB = S::RP * (int)sizeof(W) / 16, EX = 16 / (int)sizeof(X), EWT = 16 / (int)sizeof(W);
        constexpr int AR = THREADS / CX, AK = ROWS / AR, BR = THREADS / CB, BK = NC / BR;
        // (16-byte pieces of a row change places by row, so that what a warp reads of several rows lies in banks of its own)
        auto add_at = [](int row, int c) { return (row * CX + (c ^ (sizeof(X) == 4 ? row & 1 : (row & 1) << 2))) * 16; };
        auto b_at = [](int row, int c) { return (row * CB + (c ^ ((sizeof(W) == 4 ? (row & 1) << 2 : ((row & 1) | (row >> 2 & 2)) << 1) & (CB - 1)))) * 16; };
        const int c0 = nb0 * 32, c1 = min(nb1 * 32, l.n), steps = (c1 - c0 + NC - 1) / NC;
        const X* a_src = nullptr;                                    // the tile's rows are neighbours: one address
        const W* b_src = nullptr;
        uint32_t a_in = 0;
        bool b_in = false;
        auto setup = [&]() {
#pragma unroll
            for (int k = 0; k < AK; ++k) a_in |= (uint32_t)(add && (mine >> (tid / CX + k * AR) & 1)) << k;
            if (add) a_src = add + (long long)(tile * ROWS + tid / CX) * l.ldadd + c0 + tid % CX * EX;
            b_in = tid % CB * EWT < l.rank;
            b_src = B + (b_in ? (size_t)(c0 + tid / CB) * l.rank + tid % CB * EWT : 0);
        };
        auto copy = [](uint32_t dst, const void* src, bool in) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory"); };
        auto fetch = [&](int step) {
            const uint32_t st = smem_u32(sm) + 2 * S::FRAG + step % (ST > 0 ? ST : 1) * S::STAGE;
            const int off = step * NC;
            if (add) {
                const bool here = c0 + off + tid % CX * EX < c1;
                const uint32_t dst = st + add_at(tid / CX, tid % CX);
#pragma unroll
                for (int k = 0; k < AK; ++k) {
                    const bool in = here && (a_in >> k & 1);
                    copy(dst + k * (THREADS * 16), in ? a_src + (long long)(k * AR) * l.ldadd + off : add, in);
                }
            }
            if (w >= 0) {
                const W* src = b_src + (size_t)off * l.rank;
                const uint32_t dst = st + S::ADD + b_at(tid / CB, tid % CB);
                const int left_n = b_in ? c1 - c0 - off - tid / CB : 0;
#pragma unroll
                for (int k = 0; k < BK; ++k) copy(dst + k * (THREADS * 16), k * BR < left_n ? src + (size_t)(k * BR) * l.rank : B, k * BR < left_n);
            }
        };
        auto first = [&]() { for (int i = 0; i < ST - 1; ++i) { if (i < steps) fetch(i); asm volatile("cp.async.commit_group;" ::: "memory"); } };
        if (w >= 0) {
            // ---- this CTA's share of T ----
            const W* A = reinterpret_cast<const W*>(l.a) + (size_t)w * l.rank * l.k;
            float acc[MPW][RT][4];
#pragma unroll
            for (int i = 0; i < MPW; ++i)
#pragma unroll
                for (int j = 0; j < RT; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
            const int mw = warp % MW, kw = warp / MW;
            const X* xr[MPW][2];
#pragma unroll
            for (int i = 0; i < MPW; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = (mw * MPW + i) * 16 + h * 8 + g;
                    xr[i][h] = r < n_rows && (mine >> r & 1) ? x + (long long)rows_s[r] * l.ldx : nullptr;
                }
            const int kc = (l.k + 31) / 32, k0 = (int)((long long)kc * cr / nc), k1 = (int)((long long)kc * (cr + 1) / nc);
#pragma unroll(RT <= 4 ? 4 : RT == 8 && MT == 1 ? 2 : 1)
            for (int c = k0 + kw; c < k1; c += KW) {
                const int at = c * 32 + 8 * t, have = l.k - at;
                Piece<X, 8> xv[MPW][2];
#pragma unroll
                for (int i = 0; i < MPW; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) xv[i][h] = load<X, 8, VEC>(xr[i][h] + at, xr[i][h] ? have : 0);
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    const int r = j * 8 + g;
                    const Piece<W, 8> av = load<W, 8, VEC>(A + (size_t)r * l.k + at, r < l.rank ? have : 0);
                    if constexpr (!T32) {
#pragma unroll
                        for (int s = 0; s < 2; ++s)
#pragma unroll
                            for (int i = 0; i < MPW; ++i) {
                                const uint32_t f[4] = {xv[i][0].w[2 * s], xv[i][1].w[2 * s], xv[i][0].w[2 * s + 1], xv[i][1].w[2 * s + 1]};
                                mma16<W>(acc[i][j], f, av.w[2 * s], av.w[2 * s + 1]);
                            }
                    } else {
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            uint32_t bh[2], bl[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) { bh[e] = tf32(av.at(2 * s + e)); if (sizeof(W) == 4) bl[e] = tf32_rest(av.at(2 * s + e), bh[e]); }
#pragma unroll
                            for (int i = 0; i < MPW; ++i) {
                                uint32_t fh[4], fl[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) { const float v = xv[i][e & 1].at(2 * s + (e >> 1)); fh[e] = tf32(v); fl[e] = tf32_rest(v, fh[e]); }
                                if (sizeof(W) == 4) mma_tf32(acc[i][j], fh, bl[0], bl[1]);
                                mma_tf32(acc[i][j], fl, bh[0], bh[1]);
                                mma_tf32(acc[i][j], fh, bh[0], bh[1]);
                            }
                        }
                    }
                }
            }
            // ---- the warps' sums one after the other, then the cluster's: the order is the same every time ----
            for (int turn = 0; turn < KW; ++turn) {
                if (kw == turn) {
#pragma unroll
                    for (int i = 0; i < MPW; ++i)
#pragma unroll
                        for (int j = 0; j < RT; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float* p = share + ((mw * MPW + i) * 16 + g + 8 * (e >> 1)) * LDT + j * 8 + 2 * t + (e & 1);
                                *p = turn ? *p + acc[i][j][e] : acc[i][j][e];
                            }
                }
                __syncthreads();
            }
            if (nc > 1) cluster_sync_all();
            const float s = l.scales ? __ldg(l.scales + w) : 1.f;
#pragma unroll 1
            for (int i = tid; i < ROWS * S::RP / 4; i += THREADS) {
                const int at = i / (S::RP / 4) * LDT + i % (S::RP / 4) * 4;
                float4 v = *reinterpret_cast<const float4*>(share + at), y[8];
                if (nc > 1) {                                        // (all on their way before the first is added)
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (c < nc) asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(y[c].x), "=f"(y[c].y), "=f"(y[c].z), "=f"(y[c].w) : "r"(peer_smem(share + at, c)));
                    v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (c < nc) { v.x += y[c].x; v.y += y[c].y; v.z += y[c].z; v.w += y[c].w; }
                }
                *reinterpret_cast<float4*>(ts + at) = make_float4(s * v.x, s * v.y, s * v.z, s * v.w);
            }
            if (nc > 1) cluster_sync_all(); else __syncthreads();    // every CTA has read the shares: their room is free, and their owner may leave
            if constexpr (TYPE<W> == 2 && !T32) {
                for (int r = warp; r < ROWS; r += WARPS) {
                    float top = 0.f;
                    for (int i = lane; i < S::RP; i += 32) top = fmaxf(top, fabsf(ts[r * LDT + i]));
                    top = warp_max(top);
                    const uint32_t e = __float_as_uint(fminf(fmaxf(top, 0x1p-100f), 0x1p120f)) >> 23;
                    const float up = top < INFINITY ? __uint_as_float((268 - e) << 23) : 1.f;      // the largest of the row to [2^14, 2^15)
                    for (int i = lane; i < S::RP; i += 32) ts[r * LDT + i] *= up;
                    if (lane == 0) down_s[r] = top < INFINITY ? __uint_as_float((e - 14) << 23) : 1.f;
                }
                __syncthreads();
            }
            for (int i = tid; i < MT * KS * 32; i += THREADS) {
                const int ln = i & 31, ks = i / 32 % KS, mt = i / 32 / KS, gg = ln >> 2, tt = ln & 3;
                uint32_t h[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float* p = ts + (mt * 16 + gg + 8 * (e & 1)) * LDT;
                    if constexpr (T32) {                             // 16 columns of the rank are two MMAs, lane t has columns 4 t .. 4 t + 3
                        const float v = p[ks / 2 * 16 + 4 * tt + (ks & 1) * 2 + (e >> 1)];
                        h[e] = tf32(v);
                        lo[e] = tf32_rest(v, h[e]);
                    } else {
                        const float a = p[ks * 16 + 4 * tt + (e >> 1) * 2], b = p[ks * 16 + 4 * tt + (e >> 1) * 2 + 1];
                        if constexpr (TYPE<W> == 1) {
                            h[e] = pack_bf16(a, b);
                            lo[e] = pack_bf16(rest(a, bf16lo(h[e])), rest(b, bf16hi(h[e])));
                        } else {
                            const __half2 hh = __floats2half2_rn(a, b);
                            const float2 f = __half22float2(hh);
                            const __half2 ll = __floats2half2_rn(rest(a, f.x), rest(b, f.y));
                            h[e] = *reinterpret_cast<const uint32_t*>(&hh);
                            lo[e] = *reinterpret_cast<const uint32_t*>(&ll);
                        }
                    }
                }
                hi_s[i] = make_uint4(h[0], h[1], h[2], h[3]);
                lo_s[i] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            __syncthreads();
        }
        // ---- out = add + T B^T: EB blocks of 32 columns a warp at a time ----
        const int er = warp % EW * EM;                               // this warp's first row tile
        if constexpr (STAGED) {
            if (w >= 0 || add != out) {
                setup();
                first();
                const bool idle = !(mine >> (er * 16) & ((1ull << (16 * EM)) - 1));      // none of this warp's rows
                const int cw = warp / EW * 32;
                uint32_t row_in = 0;
                X* dst[EM][2];
#pragma unroll
                for (int i = 0; i < EM; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int row = (er + i) * 16 + h * 8 + g;
                        const bool in = mine >> row & 1;
                        row_in |= (uint32_t)in << (2 * i + h);
                        dst[i][h] = out + (in ? (long long)rows_s[row] * l.ldo : 0) + c0 + cw + t * 8;
                    }
#pragma unroll 1
                for (int step = 0; step < steps; ++step) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
                    __syncthreads();                                 // the step is there, the one before it read
                    if (step + ST - 1 < steps) fetch(step + ST - 1);
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    if (idle) continue;
                    const unsigned char* st = sm + 2 * S::FRAG + step % ST * S::STAGE;
                    float o[EM][4][4];
#pragma unroll
                    for (int i = 0; i < EM; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
                    if (w >= 0) {
#pragma unroll
                        for (int ks = 0; ks < RT / 2; ++ks) {
                            if (ks * 16 >= l.rank) break;
                            Piece<W, 4> bv[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int row = cw + (g >> 1) * 8 + j * 2 + (g & 1);
                                if constexpr (sizeof(W) == 4) {
                                    const uint4 v = *reinterpret_cast<const uint4*>(st + S::ADD + b_at(row, ks * 4 + t));
                                    bv[j].w[0] = v.x; bv[j].w[1] = v.y; bv[j].w[Piece<W, 4>::W - 2] = v.z; bv[j].w[Piece<W, 4>::W - 1] = v.w;
                                } else {
                                    const uint2 v = *reinterpret_cast<const uint2*>(st + S::ADD + b_at(row, ks * 2 + (t >> 1)) + (t & 1) * 8);
                                    bv[j].w[0] = v.x; bv[j].w[1] = v.y;
                                }
                            }
                            multiply<X, W, EM, KS>(o, bv, hi_s, lo_s, er, ks, lane);
                        }
                    }
                    if (c0 + step * NC + cw + t * 8 < c1)
#pragma unroll
                        for (int i = 0; i < EM; ++i)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                if (!(row_in >> (2 * i + h) & 1)) continue;
                                Piece<X, 8> av;
#pragma unroll
                                for (int q = 0; q < Piece<X, 8>::W; q += 4) {
                                    const uint4 v = add ? *reinterpret_cast<const uint4*>(st + add_at((er + i) * 16 + h * 8 + g, (cw + t * 8) / EX + q / 4)) : make_uint4(0, 0, 0, 0);
                                    av.w[q] = v.x; av.w[q + 1] = v.y; av.w[q + 2] = v.z; av.w[q + 3] = v.w;
                                }
                                const float down = TYPE<W> == 2 && !T32 && w >= 0 ? down_s[(er + i) * 16 + h * 8 + g] : 1.f;
                                __align__(16) X y[8];
#pragma unroll
                                for (int q = 0; q < 8; ++q) y[q] = from_f<X>(fmaf(o[i][q >> 1][2 * h + (q & 1)], down, av.at(q)));
#pragma unroll
                                for (int q = 0; q < Piece<X, 8>::W / 4; ++q) reinterpret_cast<uint4*>(dst[i][h] + step * NC)[q] = reinterpret_cast<const uint4*>(y)[q];
                            }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
            }
        } else if (w >= 0 || add != out)
            for (int b0 = nb0 + warp / EW; b0 < nb1; b0 += CW * EB) {
                Piece<X, 8> av[EB][EM][2];
                float o[EB][EM][4][4];
#pragma unroll
                for (int b = 0; b < EB; ++b) {
                    const int blk = b0 + b * CW, col = blk * 32 + t * 8, have = blk < nb1 ? l.n - col : 0;
#pragma unroll
                    for (int i = 0; i < EM; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int r = (er + i) * 16 + h * 8 + g;
                            const bool in = add && (mine >> r & 1);
                            av[b][i][h] = load<X, 8, VEC, false>(add + (in ? (long long)rows_s[r] * l.ldadd : 0) + col, in ? have : 0);      // (may be out)
#pragma unroll
                            for (int j = 0; j < 4; ++j) o[b][i][j][2 * h] = o[b][i][j][2 * h + 1] = 0.f;
                        }
                }
                if (w >= 0) {
#pragma unroll 2
                    for (int ks = 0; ks < RT / 2; ++ks) {
                        if (ks * 16 >= l.rank) break;
                        Piece<W, 4> bv[EB][4];
#pragma unroll
                        for (int b = 0; b < EB; ++b)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int blk = b0 + b * CW, r = blk * 32 + (g >> 1) * 8 + j * 2 + (g & 1), c = ks * 16 + 4 * t;
                                bv[b][j] = load<W, 4, VEC>(B + (size_t)r * l.rank + c, blk < nb1 && r < l.n ? l.rank - c : 0);
                            }
#pragma unroll
                        for (int b = 0; b < EB; ++b) multiply<X, W, EM, KS>(o[b], bv[b], hi_s, lo_s, er, ks, lane);
                    }
                }
#pragma unroll
                for (int b = 0; b < EB; ++b) {
                    const int blk = b0 + b * CW, col = blk * 32 + t * 8, have = blk < nb1 ? l.n - col : 0;
#pragma unroll
                    for (int i = 0; i < EM; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int r = (er + i) * 16 + h * 8 + g;
                            if (!(mine >> r & 1) || have <= 0) continue;
                            X* p = out + (long long)rows_s[r] * l.ldo + col;
                            const float down = TYPE<W> == 2 && !T32 && w >= 0 ? down_s[r] : 1.f;
                            __align__(16) X y[8];
#pragma unroll
                            for (int q = 0; q < 8; ++q) y[q] = from_f<X>(fmaf(o[b][i][q >> 1][2 * h + (q & 1)], down, av[b][i][h].at(q)));
                            store8<X, VEC>(p, have, y);
                        }
                }
            }
        __syncthreads();                                             // (T's parts and the stages may be written again)
    }
}

template <typename X, typename W, int MT, int RT, bool VEC>
int launch(cudaStream_t st, const Lora& l, bool gather, int cluster, bool pdl) {
    using S = Shape<X, W, MT, RT>;
    static SmemOptIn seen;
    auto kernel = lora_kernel<X, W, MT, RT, VEC>;
    if (const int e = ensure_dyn_smem(kernel, (size_t)S::SMEM, seen)) return e;
    const int tiles = gather ? l.m : (l.m + S::ROWS - 1) / S::ROWS;
    // A tile of neighbours may hold several adapters: they are dealt out in turn to as many clusters as give every SM a CTA, two at least
    const int slots = gather ? 1 : std::min(l.adapters + 1, std::min(16, std::max(2, tc_device_sms() / tiles)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)tiles * cluster * slots); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = S::SMEM; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, kernel, l, gather, slots);
}
template <typename X, typename W, int MT, bool VEC>
int launch_rank(cudaStream_t st, const Lora& l, bool gather, int cluster, bool pdl) {
    if (l.rank <= 16) return launch<X, W, MT, 2, VEC>(st, l, gather, cluster, pdl);
    if (l.rank <= 32) return launch<X, W, MT, 4, VEC>(st, l, gather, cluster, pdl);
    if (l.rank <= 64) return launch<X, W, MT, 8, VEC>(st, l, gather, cluster, pdl);
    return launch<X, W, MT, 16, VEC>(st, l, gather, cluster, pdl);
}
template <typename X, typename W>
int launch_types(cudaStream_t st, const Lora& l, bool vec, bool pdl) {
    // Rows that share an adapter side by side, or as they lie.  Us, rank 16, bf16, 4096 -> 12 288, rows of 1 / 8 / 60 adapters: 200 rows 19 / 20 / 25 against 23 / 24 / 73, 400 rows
    // 26 / 27 / 37 against 26 / 28 / 52, 800 rows 50 / 53 / 53 against 36 / 36 / 58; rank 64, 2048 -> 2048, of 1 / 6 / 40: 300 rows 20 / 20 / 21 against 19 / 21 / 31, 500 rows 31 / 31 / 32
    // against 22 / 26 / 45.
    const bool gather = l.m <= 384;
    const int tiles = gather ? (l.m + 7) / 8 : (l.m + 63) / 64, sms = tc_device_sms();
    int cluster = 1;
    while (cluster < 8 && (!gather || tiles * cluster * 2 <= 2 * sms)) cluster *= 2;
    if (gather) return vec ? launch_rank<X, W, 1, true>(st, l, true, cluster, pdl) : launch_rank<X, W, 1, false>(st, l, true, cluster, pdl);
    return vec ? launch_rank<X, W, 4, true>(st, l, false, cluster, pdl) : launch_rank<X, W, 4, false>(st, l, false, cluster, pdl);
}

}  // namespace

int lora_linear_launch(cudaStream_t st, const Lora& l, bool pdl) {
    if (l.m == 0 || l.n == 0) return 0;
    if (l.rank < 1 || l.rank > LORA_MAX_RANK) return -1000;
    const int xe = l.type == LORA_F32 ? 4 : 2, we = l.w_type == LORA_F32 ? 4 : 2;
    auto on16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool vec = on16(l.x) && on16(l.a) && on16(l.b) && on16(l.out) && (!l.add || on16(l.add)) && (l.ldx * xe) % 16 == 0 && (l.ldo * xe) % 16 == 0 &&
                     (!l.add || (l.ldadd * xe) % 16 == 0) && l.k % 8 == 0 && l.n % 8 == 0 && (l.rank * we) % 16 == 0 && l.rank % 4 == 0 && ((long long)l.k * we) % 16 == 0;
    if (l.type == LORA_F32) {
        if (l.w_type == LORA_F32) return launch_types<float, float>(st, l, vec, pdl);
        if (l.w_type == LORA_BF16) return launch_types<float, bf16>(st, l, vec, pdl);
        if (l.w_type == LORA_F16) return launch_types<float, __half>(st, l, vec, pdl);
    } else if (l.type == l.w_type) {
        // Us, bf16, here / in tiles of 128 rows, neighbours of 1, 6, 40 and 64 adapters, then 6 and 40 in any order.  2048 -> 2048, rank 64: 2048 rows 36, 43, 63, 76, 156, 712 / 37, 38, 70, 101,
        // 113, 568; 9400 rows 131, 135, 163, 182, 645, 3162 / 54, 56, 69, 70, 205, 1122.  4096 -> 12 288, rank 64: 2048 rows 75, 113, 160, 174, 333, 1497 / 76, 77, 129, 199, 224, 1020; rank 32:
        // 66, 91, 124, 137, 247, 973 / 66, 65, 108, 150, 183, 787; 9400 rows 244, 247, 286, 317, 967, 4301 / 178, 206, 200, 199, 607, 3233.  Neighbours of adapters that have less than half a
        // tile of rows each lose a third at most; how many of the adapters rows go through only the device knows.  1200 rows, 2048 -> 2048, of 1, 6 and 40: 29, 30, 49 / 34, 39, 55.  Rank 16,
        // 4096 -> 12 288, 2500 rows: 61, 63, 70 / 64, 63, 126.
        if (vec && l.m >= 2048 && l.rank > 16 && l.rank <= 64) return lora_tiles_launch(st, l, pdl);
        if (l.type == LORA_BF16) return launch_types<bf16, bf16>(st, l, vec, pdl);
        if (l.type == LORA_F16) return launch_types<__half, __half>(st, l, vec, pdl);
    }
    return -1000;
}

}  // namespace cb
