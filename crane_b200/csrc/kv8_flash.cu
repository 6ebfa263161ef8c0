// Attention over an 8-bit paged cache (kv8.cuh) for sequences that bring many rows: 16-bit queries, tcgen05.  The mathematics is kv8_attention.cu's.
//
// 256 query rows x 128 positions x D = 128 are 2 048 cycles of MMAs and as many of the SM's 16 exponentials a cycle.  A CTA has 256 query rows (two tiles of 128, each with its own
// softmax warps, scores and output in TMEM): while one tile's softmax runs, the other's MMAs do.  Codes come in by TMA as they lie.  Four warps turn values into f16 operands, MN-major,
// once for both tiles (e4m3 is exact in f16).  Keys of bf16 queries with 128 columns are operands as they come: such a query is two e4m3 parts, 2^-17 of its row's largest element,
// and the two products take as long as one of f16.  Otherwise keys become f16 as well, K-major.  Weights stay f16: two e4m3 parts would lose those below 2^-19 of the largest, and a
// first token that takes nearly everything is common.  They replace their scores in TMEM and are the A operand from there.
//
// What a step takes, two portions of 4096 rows behind 8192 positions, 32 heads over 8: 4 200 cycles, of which the MMAs fill 2 400: scores to weights 2 400 (720 to the maximum, 1 650 through
// the exponentials), 330 until the MMA warp hears of it, 1 190 of output and next scores, 310 back; the two tiles' chains run half a turn apart.  1 021 us, 832 TFLOP/s of 1 675 measured.
// By what it gave: one thread a row 1 546 -> two (80 registers) 1 215; with keys turned into f16 four warps could not keep three operand slots filled (1 544 with two threads a row);
// every unit four steps of its own in the deal and parts joined a row a warp 1 021.  One pass over the scores with last step's reference, weights held back until it proves good,
// spills: 1 413.
// Work is dealt out by the 128-position step (kv8_units.h): persistent CTAs, whatever the lengths.
#include <cuda_fp16.h>

#include <climits>
#include <type_traits>

#include "kv8.cuh"
#include "tc.cuh"

namespace cb {
namespace {

constexpr int M = KV8_FLASH_ROWS, BN = 128, THREADS = 768;
constexpr float P_SHIFT = 6.f;                 // weights run up to 2^14: the reference trails a row's maximum by up to 8
using Units = Kv8Units<M, BN, 4>;

struct Args {
    const void* q; long long ldq, ldqh;
    void* out; long long ldo, ldoh;
    float scale2, sign;                        // |scale| log2 e; the scale's sign goes with the queries
    Kv8Deal d;
    Kv8Join* joins;                            // [CTAs]
    float* work;                               // parts [2 * CTAs][M][D + 2]
    int* err;
};
// DIRECT (bf16 queries, 128 columns): keys' codes are operands as they come, queries are two e4m3 parts; otherwise keys become f16 as values do
template <int D, bool DIRECT> struct Cfg {
    static constexpr int Q_TILE = 128 * D * 2, SLOT = BN * D * 2, RAW = BN * D;
    static constexpr int NK = DIRECT ? 3 : 0;                               // keys' codes
    static constexpr int NF = DIRECT ? 2 : D == 128 ? 3 : 5, NR = DIRECT ? 2 : D == 128 ? 3 : 4;      // f16 operands (keys and values of a step by turns, or values), their codes
    static constexpr int SMEM = 2 * Q_TILE + NF * SLOT + (NK + NR) * RAW + 1024;
    static constexpr int C_S = 2 * D;                                       // TMEM columns: two outputs, two tiles of scores
    static_assert(C_S + 2 * BN <= 512 && SMEM <= 218 * 1024, "");
};
constexpr int METAS = 8;      // steps whose scales are kept: the softmax is at most five behind the copies

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t half2_of(uint32_t codes, int which) {
    uint32_t r;
    const uint16_t c = (uint16_t)(which ? codes >> 16 : codes);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
    return r;
}
__device__ __forceinline__ uint32_t codes2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) { uint32_t r; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a)); return r; }
template <typename T> __device__ __forceinline__ void pair(uint32_t w, float& a, float& b);
template <> __device__ __forceinline__ void pair<bf16>(uint32_t w, float& a, float& b) { a = bf16lo(w); b = bf16hi(w); }
template <> __device__ __forceinline__ void pair<__half>(uint32_t w, float& a, float& b) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w)); a = f.x; b = f.y; }
template <typename T> __device__ __forceinline__ uint32_t pack(float a, float b);
template <> __device__ __forceinline__ uint32_t pack<bf16>(float a, float b) { return pack_bf16(a, b); }
template <> __device__ __forceinline__ uint32_t pack<__half>(float a, float b) { return pack_f16(a, b); }
// MN-major operand, SWIZZLE_128B: 64 columns (128 B) x 8 positions per 1 KB atom; `lbo` bytes between 64-column groups, 1 KB between groups of 8 positions
__device__ __forceinline__ uint64_t make_smem_desc_mn128(uint32_t smem_addr, uint32_t lbo) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(lbo >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ bool has_nan(uint32_t codes) { return (((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }
// bytes of a word that are NaN codes -> 0
__device__ __forceinline__ uint32_t without_nan(uint32_t codes) {
    const uint32_t n = (((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
    return codes & ~(n * 255u);
}

template <int D, typename T, bool VEC, bool DIRECT>
__global__ void __launch_bounds__(THREADS, 1)
flash_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Args a) {
    using C = Cfg<D, DIRECT>;
    constexpr int NF = C::NF, NR = C::NR, NK = C::NK, HALVES = DIRECT ? 1 : 2;      // items of a step that are converted
    extern __shared__ uint8_t raw_sm[];
    uint8_t* sm = raw_sm + (1024 - (smem_u32(raw_sm) & 1023)) % 1024;
    uint8_t* ring = sm + 2 * C::Q_TILE;
    uint8_t* codes = ring + NF * C::SLOT;
    uint8_t* keys = codes + NR * C::RAW;
    __shared__ uint64_t raw_full[NR], raw_empty[NR], full[NF], empty[NF], k_full[NK + 1], k_empty[NK + 1], q_full[2], s_full[2], p_full[2], o_done[2];
    __shared__ float4 meta[METAS][BN / 16];                  // of each 16 positions: ks, log2 vs, 1 / vs, and whether there is a page
    __shared__ int all_there[METAS];                         // a step's positions all have pages
    __shared__ float factor_s[M], turn_s[2][2][M];           // what the two threads of a row tell one another: by step, by half
    __shared__ long long sums[KV8_SHARES + 1];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up, nan_part[METAS];                 // (a part has a step at least, so the converters are fewer parts ahead)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        gave_up = 0;
        for (int i = 0; i < METAS; ++i) nan_part[i] = -1;
        for (int i = 0; i < NR; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], 4); }
        for (int i = 0; i < NF; ++i) { mbar_init(&full[i], 4); mbar_init(&empty[i], 1); }
        for (int i = 0; i < NK; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 8); mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 8); mbar_init(&o_done[i], 1); }
        fence_barrier_init();
        tma_prefetch_desc(&map_k); tma_prefetch_desc(&map_v);
    }
    pdl_wait();
    const long long total = kv8_count<Units>(a.d, sums);
    const long long begin = kv8_range(total, gridDim.x, blockIdx.x), end = kv8_range(total, gridDim.x, blockIdx.x + 1);
    if (tid == 256) a.joins[blockIdx.x].rows = 0;
    if (begin >= end) return;
    if (warp == 2) { tmem_alloc(&tmem_slot, 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();                                 // (behind the allocation: a kernel that allocates and then waits for this one must not come ahead of it)
    const uint32_t tmem = tmem_slot;
    const TcWait wait{&gave_up, a.err};
    Units u = kv8_find<Units>(a.d, sums, begin);
    const int P = a.d.p.page, group = a.d.group;

    if (warp == 0) {
        // ---- codes: a box per page (64 positions of it at most) ----
        const int rows = min(P, 64), boxes = BN / rows;
        int st = 0, kst = 0, seq = 0;
        uint32_t ph = 1, k_ph = 1;
        for (long long step = begin; step < end;) {
            const int t0 = u.tile_at(step), t1 = u.tile_at(u.stop(end)), n = (t1 - t0) * boxes;
            for (int base = 0; base < n; base += 32) {
                int row = a.d.p.pages * a.d.p.kv_heads * P;                  // behind the pool: zeros come
                float4 sc = make_float4(0.f, 0.f, 1.f, 0.f);
                if (base + lane < n) {
                    const int pos = t0 * BN + (base + lane) * rows, page = pos < u.q.len ? kv8_page(a.d.s, a.d.p, u.b, pos / P) : -1;
                    if (page >= 0) {
                        row = (page * a.d.p.kv_heads + u.head) * P + pos % P;
                        const float2 kv = *reinterpret_cast<const float2*>(a.d.p.scales + ((size_t)page * a.d.p.kv_heads + u.head) * 2);
                        const float vs = fmaxf(kv.y, 0x1p-120f);
                        sc = make_float4(kv.x, log2f(vs), __frcp_rn(vs), 1.f);
                    }
                }
                for (int i = base; i < min(n, base + 32); i += boxes, ++seq) {
                    for (int half = 0; half < 2; ++half) {
                        const bool direct = DIRECT && half == 0;
                        uint64_t* bar = direct ? &k_full[kst] : &raw_full[st];
                        wait(direct ? &k_empty[kst] : &raw_empty[st], direct ? k_ph : ph);
                        if (half == 0) {
                            const int from = (i - base + (lane & 7) * 16 / rows) & 31;
                            float4 m;
                            m.x = __shfl_sync(0xffffffffu, sc.x, from); m.y = __shfl_sync(0xffffffffu, sc.y, from);
                            m.z = __shfl_sync(0xffffffffu, sc.z, from); m.w = __shfl_sync(0xffffffffu, sc.w, from);
                            if (lane < BN / 16) meta[seq % METAS][lane] = m;
                            const bool all = __all_sync(0xffffffffu, m.w != 0.f);
                            if (lane == 0) all_there[seq % METAS] = all;
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive_expect_tx(bar, C::RAW);
                        __syncwarp();
                        const int r = __shfl_sync(0xffffffffu, row, (i - base + lane) & 31);
                        if (lane < boxes) tma_load_2d((direct ? keys + kst * C::RAW : codes + st * C::RAW) + lane * rows * D, half ? &map_v : &map_k, bar, 0, r);
                        if (direct) { if (++kst == NK) { kst = 0; k_ph ^= 1; } }
                        else if (++st == NR) { st = 0; ph ^= 1; }
                    }
                }
            }
            step = u.stop(end);
            if (step < end && !u.next(a.d)) break;
        }
    } else if (warp == 1) {
        // ---- MMAs ----
        constexpr uint32_t id_s = make_idesc_f16(128, BN), id_o = make_idesc_f16(128, D) | (1u << 16);      // (B of P V: MN-major)
        int st = 0, kst = 0, part = 0;
        uint32_t ph = 0, k_ph = 0, p_ph = 0;
        auto scores = [&](int w) {                           // of tile w, with the keys of slot st (DIRECT: kst)
            if (DIRECT && elect_one()) {
                constexpr uint32_t id_8 = make_idesc_e4m3(128, BN);
                const uint64_t qd = make_smem_desc_sw128(smem_u32(sm + w * C::Q_TILE)), kd = make_smem_desc_sw128(smem_u32(keys + kst * C::RAW));
#pragma unroll
                for (int k = 0; k < 8; ++k)                  // the lower parts first
                    umma_e4m3(tmem + C::C_S + w * BN, qd + (uint64_t)((k < 4 ? 1024 : 0) + 2 * (k & 3)), kd + (uint64_t)(2 * (k & 3)), id_8, (uint32_t)(k != 0));
                umma_commit(&s_full[w]);
            }
            if (!DIRECT && elect_one()) {
                const uint64_t qd = make_smem_desc_sw128(smem_u32(sm + w * C::Q_TILE)), kd = make_smem_desc_sw128(smem_u32(ring + st * C::SLOT));
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    umma_bf16(tmem + C::C_S + w * BN, qd + (uint64_t)((k >> 2) * 1024 + 2 * (k & 3)), kd + (uint64_t)((k >> 2) * 1024 + 2 * (k & 3)), id_s, (uint32_t)(k != 0));
                umma_commit(&s_full[w]);
            }
            __syncwarp();
        };
        auto output = [&](int w, int slot, bool first, bool last) {
            if (elect_one()) {
                const uint64_t vd = make_smem_desc_mn128(smem_u32(ring + slot * C::SLOT), BN * 128);
#pragma unroll
                for (int k = 0; k < BN / 16; ++k)
                    umma_ts(tmem + w * D, tmem + C::C_S + (uint32_t)(w * BN + (k >> 1) * 32 + (k & 1) * 8), vd + (uint64_t)(k * 128), id_o, (uint32_t)!(first && k == 0));
                if (last) umma_commit(&o_done[w]);
            }
            __syncwarp();
        };
        auto release = [&](uint64_t* bar) { if (elect_one()) umma_commit(bar); __syncwarp(); };
        auto step_on = [&]() { if (++st == NF) { st = 0; ph ^= 1; } };
        auto wait_keys = [&]() { if (DIRECT) wait(&k_full[kst], k_ph); else wait(&full[st], ph); };
        auto release_keys = [&]() {
            release(DIRECT ? &k_empty[kst] : &empty[st]);
            if (!DIRECT) step_on();
            else if (++kst == NK) { kst = 0; k_ph ^= 1; }
        };
        for (long long step = begin; step < end;) {
            const int t0 = u.tile_at(step), t1 = u.tile_at(u.stop(end));
            if (t0 < t1) {
            wait_keys();
            for (int w = 0; w < 2; ++w) {
                wait(&q_full[w], part & 1);
                tc_fence_after();
                scores(w);
            }
            release_keys();
            for (int t = t0; t < t1; ++t) {
                const bool last = t + 1 == t1;
                const int v = st;
                wait(&full[v], ph);
                step_on();
                for (int w = 0; w < 2; ++w) {
                    wait(&p_full[w], p_ph);
                    tc_fence_after();
                    output(w, v, t == t0, last);
                    if (w == 1) release(&empty[v]);
                    if (!last) {
                        if (w == 0) wait_keys();
                        tc_fence_after();
                        scores(w);
                    }
                }
                p_ph ^= 1;
                if (!last) release_keys();
            }
            ++part;
            }
            step = u.stop(end);
            if (step < end && !u.next(a.d)) break;
        }
    } else if (warp >= 4 && warp < 8) {
        // ---- codes to operands ----
        const int ct = tid - 128;
        int rs = 0, fs = 0, seq = 0, part = 0;
        uint32_t r_ph = 0, f_ph = 1;
        for (long long step = begin; step < end;) {
            const int t0 = u.tile_at(step), t1 = u.tile_at(u.stop(end));
            const int seen = u.q.first + (int)((long long)u.grp * M / group);      // last position that all rows see
            for (int t = t0; t < t1; ++t, ++seq) {
                const bool edge = t * BN + BN - 1 > seen;
                for (int half = 2 - HALVES; half < 2; ++half) {
                    wait(&raw_full[rs], r_ph);
                    wait(&empty[fs], f_ph);
                    const uint8_t* src = codes + rs * C::RAW;
                    uint8_t* dst = ring + fs * C::SLOT;
                    const bool clean = half && (edge || !all_there[seq % METAS]);      // values that some row does not see: nothing of them may reach it
#pragma unroll 4
                    for (int e = 0; e < D / 16; ++e) {
                        const int at = e * 128 + ct, row = at / (D / 16), j = at % (D / 16);
                        uint4 c = *reinterpret_cast<const uint4*>(src + at * 16);
                        if (clean) {
                            const int pos = t * BN + row;
                            if (pos >= u.q.len || meta[seq % METAS][row / 16].w == 0.f) c = make_uint4(0, 0, 0, 0);
                            else if (pos > seen && (has_nan(c.x) || has_nan(c.y) || has_nan(c.z) || has_nan(c.w))) {
                                c.x = without_nan(c.x); c.y = without_nan(c.y); c.z = without_nan(c.z); c.w = without_nan(c.w);
                                nan_part[part % METAS] = part;                          // (the rows that do see it look for it themselves)
                            }
                        }
                        const uint4 lo = make_uint4(half2_of(c.x, 0), half2_of(c.x, 1), half2_of(c.y, 0), half2_of(c.y, 1));
                        const uint4 hi = make_uint4(half2_of(c.z, 0), half2_of(c.z, 1), half2_of(c.w, 0), half2_of(c.w, 1));
                        uint8_t* p = dst + (j >> 2) * (BN * 128);
                        // (lanes of the second 64 columns store their halves the other way round: no two lanes of a store share banks)
                        const int swap = j >> 2;
                        *reinterpret_cast<uint4*>(p + sw128_off(row, (j & 3) * 2 + swap)) = swap ? hi : lo;
                        *reinterpret_cast<uint4*>(p + sw128_off(row, (j & 3) * 2 + (swap ^ 1))) = swap ? lo : hi;
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) { mbar_arrive(&full[fs]); mbar_arrive(&raw_empty[rs]); }
                    if (++rs == NR) { rs = 0; r_ph ^= 1; }
                    if (++fs == NF) { fs = 0; f_ph ^= 1; }
                }
            }
            part += t0 < t1;
            step = u.stop(end);
            if (step < end && !u.next(a.d)) break;
        }
    } else if (warp >= 8) {
        // ---- softmax and results: two threads a row, half of the columns each ----
        const int w = (warp - 8) >> 3, hf = (warp >> 2) & 1, qd = warp & 3, r = w * 128 + qd * 32 + lane, bar = 1 + w * 4 + qd;
        const uint32_t lanes = (uint32_t)(qd * 32) << 16;
        const uint32_t sa = tmem + lanes + C::C_S + w * BN + hf * 64, oa = tmem + lanes + w * D + hf * (D / 2);
        int seq = 0, part = 0;
        uint32_t s_ph = 0;
        for (long long step = begin; step < end;) {
            const int t0 = u.tile_at(step), t1 = u.tile_at(u.stop(end));
            if (tid == 256 && u.begins(step, end)) a.joins[blockIdx.x] = kv8_join(a.d, u, M, total, gridDim.x, blockIdx.x, begin);
            if (t0 == t1) {                                                  // the unit's own steps alone: an empty part
                float* dst = a.work + ((size_t)kv8_slot(blockIdx.x, begin, step) * M + r) * (D + 2);
                for (int c = hf * (D / 2); c < (hf + 1) * (D / 2); c += 2) *reinterpret_cast<float2*>(dst + c) = make_float2(0.f, 0.f);
                if (hf == 0) { dst[D] = -INFINITY; dst[D + 1] = 0.f; }
                step = u.stop(end);
                if (step < end && !u.next(a.d)) break;
                continue;
            }
            // ---- the queries, sixteen rows a warp, D / 8 lanes a row: each row's largest moved to [2^14, 2^15) by a power of two, f16 (or two e4m3 parts) ----
            constexpr int LR = D / 8, RW = 32 / LR;          // lanes a row, rows at a time
#pragma unroll 2
            for (int i = 0; i < 16 / RW; ++i) {
                const int rr = w * 128 + qd * 32 + hf * 16 + i * RW + lane / LR, c = lane % LR;
                const long long row = (long long)u.grp * M + rr;
                const int tok = (int)(row / group), h = u.head * group + (int)(row % group);
                uint32_t v[4] = {0, 0, 0, 0};
                if (tok < u.q.n) {
                    const T* src = reinterpret_cast<const T*>(a.q) + (long long)(u.q.s0 + tok) * a.ldq + (long long)h * a.ldqh + c * 8;
                    if constexpr (VEC) { const uint4 x = __ldg(reinterpret_cast<const uint4*>(src)); v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; }
                    else {
                        const unsigned short* s = reinterpret_cast<const unsigned short*>(src);
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] = __ldg(s + 2 * k) | (uint32_t)__ldg(s + 2 * k + 1) << 16;
                    }
                }
                float x[8], top = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) pair<T>(v[k], x[2 * k], x[2 * k + 1]);
#pragma unroll
                for (int k = 0; k < 8; ++k) top = x[k] != x[k] ? INFINITY : fmaxf(top, fabsf(x[k]));
#pragma unroll
                for (int o = 1; o < LR; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const uint32_t ex = __float_as_uint(fmaxf(top, 0x1p-100f)) >> 23;
                if constexpr (DIRECT) {                                      // each row's largest moved to [2^7, 2^8): two parts hold 8 bits of what is 2^-9 of it and more
                    const float up = top < INFINITY ? a.sign * __uint_as_float((261 - ex) << 23) : NAN;
                    uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float y0 = x[2 * k] * up, y1 = x[2 * k + 1] * up;
                        const uint32_t c8 = codes2(y0, y1);
                        uint32_t h2;
                        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)c8));
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
                        hi[k >> 1] |= c8 << (16 * (k & 1));
                        lo[k >> 1] |= codes2(y0 - f.x, y1 - f.y) << (16 * (k & 1));
                    }
                    uint8_t* dst = sm + w * C::Q_TILE + sw128_off(rr & 127, c >> 1) + (c & 1) * 8;
                    *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2*>(dst + 16384) = make_uint2(lo[0], lo[1]);
                    if (c == 0) factor_s[rr] = fmaxf(a.scale2 * __uint_as_float((ex - 7) << 23), 0x1p-120f);
                    continue;
                }
                const float up = top < INFINITY ? a.sign * __uint_as_float((268 - ex) << 23) : NAN;      // (a row with an infinity or a NaN gives NaN)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = pack_f16(x[2 * k] * up, x[2 * k + 1] * up);
                const int ri = rr & 127;
                *reinterpret_cast<uint4*>(sm + w * C::Q_TILE + (c >> 3) * 16384 + sw128_off(ri, c & 7)) = make_uint4(v[0], v[1], v[2], v[3]);
                if (c == 0) factor_s[rr] = fmaxf(a.scale2 * __uint_as_float((ex - 14) << 23), 0x1p-120f);
            }
            fence_proxy_async();
            named_bar_sync(bar, 64);                         // (both halves' factors)
            if (lane == 0) mbar_arrive(&q_full[w]);
            const float factor = factor_s[r];
            const long long row = (long long)u.grp * M + r;
            const int tok = (int)(row / group), h = u.head * group + (int)(row % group);
            const bool in = tok < u.q.n;
            const int pmax = in ? u.q.first + tok : INT_MAX;                 // last position that the row sees
            const int wmin = __reduce_min_sync(0xffffffffu, pmax);
            float m = -INFINITY, l = 0.f;                                    // reference of the exponents (a whole number, not always the running maximum), this half's sum
            for (int t = t0; t < t1; ++t, ++seq) {
                const float4* mt = meta[seq % METAS] + hf * 4;
                wait(&s_full[w], s_ph);
                s_ph ^= 1;
                tc_fence_after();
                const int kv0 = t * BN + hf * 64;
                if (kv0 + 63 > wmin || !all_there[seq % METAS]) {            // in place, for the code's size
#pragma unroll 1
                    for (int c = 0; c < 64; c += 16) {
                        uint32_t x[16];
                        tmem_ld16_async(sa + c, x);
                        const bool page = mt[c / 16].w != 0.f;
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) if (!page || kv0 + c + j > pmax) x[j] = 0xff800000u;
                        tmem_st16(sa + c, x);
                    }
                    tmem_st_wait();
                }
                float mx = -INFINITY;
#pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    uint32_t x[32];
                    tmem_ld16_async(sa + c0, x);
                    tmem_ld16_async(sa + c0 + 16, x + 16);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 32; c += 16) {
                        float y[2] = {-INFINITY, -INFINITY};
#pragma unroll
                        for (int j = 0; j < 16; ++j) y[j & 1] = fmaxf(y[j & 1], __uint_as_float(x[c + j]));
                        const float2 sc = *reinterpret_cast<const float2*>(mt + (c0 + c) / 16);
                        mx = fmaxf(mx, fmaf(fmaxf(y[0], y[1]), fmaxf(factor * sc.x, 0x1p-126f), sc.y));
                    }
                }
                turn_s[seq & 1][hf][r] = mx;
                named_bar_sync(bar, 64);
                mx = fmaxf(mx, turn_s[seq & 1][hf ^ 1][r]);
                const bool grow = mx > m + 8.f || (m == -INFINITY && mx > -INFINITY);
                if (__any_sync(0xffffffffu, grow)) {                         // (both warps of a row alike)
                    const float mn = fmaxf(m, ceilf(mx)), f = m == -INFINITY ? 0.f : m == mn ? 1.f : ex2(m - mn);
                    l *= f;
                    m = mn;
                    if (t > t0) {                                            // (the scores are there: the MMAs ahead of theirs, the last step's output among them, are done)
#pragma unroll 1
                        for (int c = 0; c < D / 2; c += 16) {
                            uint32_t o[16];
                            tmem_ld16_async(oa + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                            tmem_st16(oa + c, o);
                        }
                    }
                }
                // scores whose last bit is worth more than a weight: their exponents are differences of rounded numbers
                const bool far = __any_sync(0xffffffffu, fabsf(m) > 0x1p20f && fabsf(m) < INFINITY);
                if (far) {
#pragma unroll 1
                    for (int c = 0; c < 64; c += 16) {
                        uint32_t x[16];
                        tmem_ld16_async(sa + c, x);
                        tmem_ld_wait();
                        const float4 sc = mt[c / 16];
                        const float f = fmaxf(factor * sc.x, 0x1p-126f);
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(fmaf(__uint_as_float(x[j]), f, sc.y) - (m == -INFINITY ? 0.f : m));
                        tmem_st16(sa + c, x);
                    }
                    tmem_st_wait();
                }
                const float ref = (m == -INFINITY ? 0.f : m) - P_SHIFT;
#pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    uint32_t x[32], p[16];
                    tmem_ld16_async(sa + c0, x);
                    tmem_ld16_async(sa + c0 + 16, x + 16);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 32; c += 16) {
                        const float4 sc = mt[(c0 + c) / 16];
                        const float f = far ? 1.f : fmaxf(factor * sc.x, 0x1p-126f), b = far ? P_SHIFT : sc.y - ref;
                        float sum[2] = {0.f, 0.f};
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float p0 = ex2(fmaf(__uint_as_float(x[c + 2 * j]), f, b)), p1 = ex2(fmaf(__uint_as_float(x[c + 2 * j + 1]), f, b));
                            sum[0] += p0; sum[1] += p1;
                            p[c / 2 + j] = pack_f16(p0, p1);
                        }
                        l = fmaf(sum[0] + sum[1], sc.z, l);
                    }
                    tmem_st16(sa + c0, p);                                   // in place of the 32 scores
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[w]);
            }
            turn_s[seq & 1][hf][r] = l;
            wait(&o_done[w], part & 1);
            named_bar_sync(bar, 64);
            l += turn_s[seq & 1][hf ^ 1][r];                                 // (the same bits in both)
            named_bar_sync(bar, 64);
            tc_fence_after();
            // a NaN among values that only some rows see was left out of the products: the rows that see it look it up
            uint32_t odd[D / 64];
#pragma unroll
            for (int i = 0; i < D / 64; ++i) odd[i] = 0;
            if (nan_part[part % METAS] == part && in) {
                const int from = max(u.q.first + (int)((long long)u.grp * M / group) + 1, t0 * BN), to = min(min(pmax, u.q.len - 1), t1 * BN - 1);
                for (int pos = max(from, 0); pos <= to; ++pos) {
                    const int page = kv8_page(a.d.s, a.d.p, u.b, pos / P);
                    if (page < 0) continue;
                    const unsigned char* v = a.d.p.v + (((size_t)page * a.d.p.kv_heads + u.head) * P + pos % P) * D + hf * (D / 2);
#pragma unroll
                    for (int i = 0; i < D / 64; ++i)
                        for (int j = 0; j < 32; ++j) if ((v[i * 32 + j] & 0x7f) == 0x7f) odd[i] |= 1u << j;
                }
            }
            const bool whole = u.whole(step, end);
            const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
            T* dst = reinterpret_cast<T*>(a.out) + (long long)(u.q.s0 + (in ? tok : 0)) * a.ldo + (long long)h * a.ldoh + hf * (D / 2);
            float* part_dst = a.work + ((size_t)kv8_slot(blockIdx.x, begin, step) * M + r) * (D + 2);
#pragma unroll
            for (int c = 0; c < D / 2; c += 16) {
                uint32_t o[16];
                tmem_ld16_async(oa + c, o);
                tmem_ld_wait();
                float y[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    y[j] = __uint_as_float(o[j]) * inv;
                    if (odd[c / 32] >> (c % 32 + j) & 1) y[j] = NAN;
                }
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 16; j += 2) *reinterpret_cast<float2*>(part_dst + hf * (D / 2) + c + j) = make_float2(y[j], y[j + 1]);
                } else if (in) {
                    uint32_t k[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) k[j] = pack<T>(y[2 * j], y[2 * j + 1]);
                    if constexpr (VEC) {
                        *reinterpret_cast<uint4*>(dst + c) = make_uint4(k[0], k[1], k[2], k[3]);
                        *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(k[4], k[5], k[6], k[7]);
                    } else {
                        unsigned short* s = reinterpret_cast<unsigned short*>(dst + c);
#pragma unroll
                        for (int j = 0; j < 8; ++j) { s[2 * j] = (unsigned short)k[j]; s[2 * j + 1] = (unsigned short)(k[j] >> 16); }
                    }
                }
            }
            if (!whole && hf == 0) { part_dst[D] = m; part_dst[D + 1] = l; }
            tc_fence_before();
            ++part;
            step = u.stop(end);
            if (step < end && !u.next(a.d)) break;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) { tc_fence_after(); tmem_dealloc(tmem, 512); }
    if (tid == 0) wait.drain();
}

template <int D, typename T>
int launch(cudaStream_t st, const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, bool vec, bool pdl) {
    constexpr bool DIRECT = D == 128 && std::is_same<T, bf16>::value;
    static SmemOptIn seen[2];
    auto kernel = vec ? flash_kernel<D, T, true, DIRECT> : flash_kernel<D, T, false, DIRECT>;
    if (const int e = ensure_dyn_smem(kernel, (size_t)Cfg<D, DIRECT>::SMEM, seen[vec])) return e;
    return launch_k(kernel, dim3(tc_device_sms()), dim3(THREADS), Cfg<D, DIRECT>::SMEM, st, pdl, mk, mv, a);
}

}  // namespace

// Sequences that bring `lo` rows of a kv head and more; parts of units that lie with several CTAs are left in `parts`
int kv8_flash_launch(cudaStream_t st, const Kv8Attention& k, const Kv8Deal& d, Kv8Join* joins, float* parts, bool pdl) {
    const int D = d.p.dim;
    const uint64_t n = (uint64_t)d.p.pages * d.p.kv_heads * d.p.page;
    CUtensorMap mk, mv;
    const uint32_t rows = d.p.page < 64 ? d.p.page : 64;
    if (!tc_tmap(&mk, d.p.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, n, D, D, rows, D, D == 128 && k.q.type == KV8_BF16 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE) ||
        !tc_tmap(&mv, d.p.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, n, D, D, rows, D, CU_TENSOR_MAP_SWIZZLE_NONE)) return (int)cudaErrorInvalidValue;
    const bool vec = (reinterpret_cast<uintptr_t>(k.q.p) | reinterpret_cast<uintptr_t>(k.out)) % 16 == 0 && (k.q.ld | k.q.ldh | k.ldo | k.ldoh) % 8 == 0;
    const Args a = {k.q.p, k.q.ld, k.q.ldh, k.out, k.ldo, k.ldoh, (float)(fabs((double)k.scale) * 1.4426950408889634074), k.scale < 0.f ? -1.f : 1.f, d,
                    joins, parts, k.err};
    if (k.q.type == KV8_BF16) return D == 64 ? launch<64, bf16>(st, mk, mv, a, vec, pdl) : launch<128, bf16>(st, mk, mv, a, vec, pdl);
    return D == 64 ? launch<64, __half>(st, mk, mv, a, vec, pdl) : launch<128, __half>(st, mk, mv, a, vec, pdl);
}

}  // namespace cb
