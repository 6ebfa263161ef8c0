// Verification of drafted tokens (draft.cuh).  With p the target's and q the draft model's softmax at the sequence's temperature:
//   draft j is accepted while u_j q_j(d_j) < p_j(d_j); at the first that is not, and behind the last, one more token follows:
//   argmax_i w_i / -log(noise_i), the lowest index among equals, w = max(p - q, 0) (p where that is zero everywhere), or p behind the last: a race of exponential clocks,
//   drawn in proportion to w as the sampler's whole-vocabulary draw.  Temperature 0: the draft is accepted if it is the row's first maximum, which follows otherwise.
// A NaN logit counts as -inf; where the largest is +inf all of those share the probability; a row without a logit above -inf accepts nothing and gives token -1.
//
// Counts and tokens are those of 64 bits.  The sums of the first reading are not: they are off by SUMS = 2^-16 of themselves at most (an exponential 2^-22, its exponent three roundings
// of 2^-24, which a sum has log2 of the vocabulary of at the mean, 30 at most; a thread's 16 additions of short sums and, in a row that rises all the way, as many steps of its maximum; 13
// joins), 2^-21 as a rule.  They decide where they can.  What lies within that of a border (u q beside p; a key beside the best one, where a difference of p and q makes the keys) is decided by
// sums that the cluster takes again in 64 bits, 60 us for a row of 151 936 (bf16 100): one draft in 30 000.
//
// Two kernels: the first reads every row once and leaves (maximum, its place, sum) of each stretch of it, the second has a cluster of CTAs for each sequence, which
// joins those, walks the drafts and runs the race over the one row that needs it.  Bound by bytes: the rows of both models, one row of noise a sequence.  64 sequences with up to seven
// drafts over 151 936 logits, f32: 101 us, the first 60 (5 TB/s), the second 41 (eight dependent trips to the L2 ahead of a race over 117 MB).  Keys of all places in 64 bits: 306 for the
// second alone.
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "draft.cuh"
#include "tc.cuh"

namespace cb {
namespace {

constexpr int THREADS = 256, RACERS = 512, CLUSTER = 8;
constexpr double LOG2E = 1.4426950408889634, SUMS = 0x1p-16;

struct Part { float top; int at; double sum; };         // of a stretch: its largest logit; greedy: the first place of it; else the sum of exp((x - top) / T)

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<bf16>(bf16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }      // (NaN: -inf)
__device__ __forceinline__ float below(float x, float top) { return x == top ? 0.f : x - top; }      // infinities by themselves
__device__ __forceinline__ double far_below(float x, float top) { return x == top ? 0.0 : (double)x - (double)top; }
// log2 e / T as f32, kept off zero and infinity so that 0 and -inf stay what they are under it
__device__ __forceinline__ float rate(float temp) { return fminf(fmaxf((float)(LOG2E / (double)temp), 0x1p-126f), 0x1p127f); }

template <typename K>
__device__ __forceinline__ int search(int n, int at, K key) {        // the largest b with key(b) <= at, all lanes of a warp together
    int lo = 0;
    while (n > 1) {
        const int step = (n + 31) / 32, i = (int)(threadIdx.x & 31) * step;
        const unsigned m = __ballot_sync(0xffffffffu, i < n && key(lo + i) <= at);
        const int k = m ? 31 - __clz(m) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}
__device__ __forceinline__ int start_of(const Draft& d, int b) { return min(max(__ldg(d.starts + b), 0), d.total); }

__host__ __device__ __forceinline__ int stretch_of(int vocab, int parts) { return ((vocab + parts - 1) / parts + 7) / 8 * 8; }

// N neighbouring values, 16 bytes (f32: 4, else 8) or one
template <typename T, int N> __device__ __forceinline__ void get(const T* p, float* x) {
    if constexpr (N == 1) x[0] = clean(to_f<T>(*p));
    else {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = clean(to_f<T>(e[j]));
    }
}
// A running maximum and the sum of exp2((x - top) c) below it, B values at a time
struct Sum {
    float top = -INFINITY;
    float all = 0.f;
    template <int B> __device__ __forceinline__ void take(const float* x, float c) {
        float m = x[0];
#pragma unroll
        for (int j = 1; j < B; ++j) m = fmaxf(m, x[j]);
        if (m > top) {
            all *= top == -INFINITY ? 0.f : ex2((top - m) * c);
            top = m;
        }
        float s[2] = {0.f, 0.f};
        if (fabsf(top) < INFINITY) {
#pragma unroll
            for (int j = 0; j < B; ++j) s[j & 1] += ex2((x[j] - top) * c);
        } else if (top > 0.f) {                         // +inf: those share
#pragma unroll
            for (int j = 0; j < B; ++j) s[0] += x[j] == top ? 1.f : 0.f;
        }
        all += s[0] + s[1];
    }
};
struct First {                                          // a running maximum and its first place; values come in ascending order of their places
    float top = -INFINITY;
    int at = INT_MAX;
    __device__ __forceinline__ void take(float x, int i) { if (x > top) { top = x; at = i; } }
};

template <typename T>
__global__ void __launch_bounds__(THREADS)
stretch_kernel(Draft d, int parts) {
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.x, part = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool target = row < d.total + d.seqs;
    const int r = target ? row : row - d.total - d.seqs;
    const int b = search(d.seqs, r, [&](int i) { return start_of(d, i) + (target ? i : 0); });
    const float temp = d.temperatures ? __ldg(d.temperatures + b) : 1.f;
    if (!target && !(temp > 0.f)) return;
    const T* x = reinterpret_cast<const T*>(target ? d.logits : d.q) + (long long)r * (target ? d.ld : d.ldq);
    const int len = stretch_of(d.vocab, parts), lo = (int)min((long long)d.vocab, (long long)part * len), hi = min(d.vocab, lo + len);
    const float c = temp > 0.f ? rate(temp) : 1.f;
    constexpr int N = 16 / (int)sizeof(T), U = 4;
    const int skew = (int)(reinterpret_cast<uintptr_t>(x + lo) % 16) / (int)sizeof(T);
    const int a0 = min(hi, lo + (skew ? N - skew : 0)), a1 = a0 + (hi - a0) / N * N;        // what 16-byte loads reach
    float top;
    double s = 0.0;
    int at = INT_MAX;
    if (temp > 0.f) {
        Sum z;
        float v[U * N];
        if (lo + (int)threadIdx.x < a0) { get<T, 1>(x + lo + threadIdx.x, v); z.take<1>(v, c); }
        int i = a0 + threadIdx.x * N;
        for (; i + (U - 1) * THREADS * N < a1; i += U * THREADS * N) {
#pragma unroll
            for (int k = 0; k < U; ++k) get<T, N>(x + i + k * THREADS * N, v + k * N);
            z.take<U * N>(v, c);
        }
        for (; i < a1; i += THREADS * N) { get<T, N>(x + i, v); z.take<N>(v, c); }
        if (a1 + (int)threadIdx.x < hi) { get<T, 1>(x + a1 + threadIdx.x, v); z.take<1>(v, c); }
        top = z.top;
        s = z.all;
    } else {
        First z;
        float v[N];
        if (lo + (int)threadIdx.x < a0) { get<T, 1>(x + lo + threadIdx.x, v); z.take(v[0], lo + threadIdx.x); }
#pragma unroll 4
        for (int i = a0 + threadIdx.x * N; i < a1; i += THREADS * N) {
            get<T, N>(x + i, v);
#pragma unroll
            for (int j = 0; j < N; ++j) z.take(v[j], i + j);
        }
        if (a1 + (int)threadIdx.x < hi) { get<T, 1>(x + a1 + threadIdx.x, v); z.take(v[0], a1 + threadIdx.x); }
        top = z.top;
        at = z.at;
    }
    // ---- the block's ----
    __shared__ float wt[THREADS / 32];
    __shared__ int wa[THREADS / 32];
    __shared__ double wsum[THREADS / 32];
    auto join = [&](float t2, int a2, double s2) {
        const float m = fmaxf(top, t2);
        if (m != -INFINITY) s = s * (double)ex2(below(top, m) * c) + s2 * (double)ex2(below(t2, m) * c);
        at = top > t2 ? at : t2 > top ? a2 : min(at, a2);
        top = m;
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float t2 = __shfl_xor_sync(0xffffffffu, top, o);
        const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
        const double s2 = __shfl_xor_sync(0xffffffffu, s, o);
        join(t2, a2, s2);
    }
    if (lane == 0) { wt[warp] = top; wa[warp] = at; wsum[warp] = s; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < THREADS / 32; ++w) join(wt[w], wa[w], wsum[w]);
        reinterpret_cast<Part*>(d.work)[(long long)row * parts + part] = Part{top, at, top == -INFINITY ? 0.0 : s};
    }
}

// A warp: a row's maximum, its first place and sum
__device__ __forceinline__ Part whole(const Part* p, int parts, double inv_t) {
    const int lane = threadIdx.x & 31;
    Part r = {-INFINITY, INT_MAX, 0.0};
    for (int i = lane; i < parts; i += 32) { const float top = p[i].top; if (top > r.top) { r.top = top; r.at = p[i].at; } }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float top = __shfl_xor_sync(0xffffffffu, r.top, o);
        const int at = __shfl_xor_sync(0xffffffffu, r.at, o);
        r.at = r.top > top ? r.at : top > r.top ? at : min(r.at, at);
        r.top = fmaxf(r.top, top);
    }
    for (int i = lane; i < parts; i += 32) if (p[i].sum > 0.0) r.sum += p[i].sum * exp(far_below(p[i].top, r.top) * inv_t);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r.sum += __shfl_xor_sync(0xffffffffu, r.sum, o);
    return r;
}
__device__ __forceinline__ double share(float x, const Part& p, double inv_t) { return p.sum > 0.0 && x > -INFINITY ? exp(far_below(x, p.top) * inv_t) / p.sum : 0.0; }

// What the warps of a block and the CTAs of a cluster tell one another
struct Room {
    double key[RACERS / 32], best;
    int at[RACERS / 32], best_at;
    int left[RACERS / 32], all_left;
    float rival[RACERS / 32], best_rival;
};
__device__ __forceinline__ double clock_of(float u) { return -log((double)fminf(fmaxf(u, 0x1p-126f), 0x1.fffffep-1f)); }

// A sequence's drafts
constexpr int KEPT = 32;                                // rows of a sequence whose sums stay at hand
struct Holds { int first, close; Part p[KEPT], q[KEPT]; };      // the first draft that does not hold, the first that is too close to call
template <typename T>
struct Drafts {
    const Draft& d;
    int parts, b, s0, n;
    bool greedy;
    double inv_t;
    __device__ __forceinline__ const T* x(int j) const { return reinterpret_cast<const T*>(d.logits) + (long long)(s0 + b + j) * d.ld; }
    __device__ __forceinline__ const T* y(int j) const { return reinterpret_cast<const T*>(d.q) + (long long)(s0 + j) * d.ldq; }
    __device__ __forceinline__ Part target(int j) const { return whole(reinterpret_cast<const Part*>(d.work) + (long long)(s0 + b + j) * parts, parts, inv_t); }
    __device__ __forceinline__ Part draft(int j) const {
        return d.q && !greedy && j < n ? whole(reinterpret_cast<const Part*>(d.work) + (long long)(d.total + d.seqs + s0 + j) * parts, parts, inv_t) : Part{0.f, 0, 0.0};
    }
    // u q and p of a draft whose token is in the vocabulary
    __device__ __forceinline__ void sides(int j, int tok, const Part& p, const Part& q, double& uq, double& pd) const {
        uq = (double)__ldg(d.uniforms + s0 + j) * (d.q ? share(clean(to_f<T>(y(j)[tok])), q, inv_t) : 1.0);
        pd = share(clean(to_f<T>(x(j)[tok])), p, inv_t);
    }
    // The drafts from `from` on, and the row behind the last, a warp each
    __device__ __forceinline__ void look(int from, Holds* h) const {
        if (threadIdx.x == 0) { h->first = n; h->close = INT_MAX; }
        __syncthreads();
        for (int j = from + (int)(threadIdx.x >> 5); j <= n; j += RACERS / 32) {
            const Part p = target(j), q = draft(j);
            if (threadIdx.x & 31) continue;
            if (j < KEPT) { h->p[j] = p; h->q[j] = q; }
            if (j == n) continue;
            const int tok = __ldg(d.tokens + s0 + j);
            bool ok = (unsigned)tok < (unsigned)d.vocab;
            if (ok && greedy) ok = p.top > -INFINITY && tok == p.at;
            else if (ok) {
                double uq, pd;
                sides(j, tok, p, q, uq, pd);
                ok = uq < pd;
                if (uq > 0.0 && fabs(uq - pd) <= 2.25 * SUMS * pd) { atomicMin(&h->close, j); ok = true; }
            }
            if (!ok) atomicMin(&h->first, j);
        }
        __syncthreads();
    }
};
// A row's sum of exp((x - top) / T) in 64 bits, by the whole cluster, a CTA its places lo to hi: the same places in the same order whatever the row's boundary, the same bits everywhere
template <typename T>
__device__ __forceinline__ double again(const T* row, int lo, int hi, float top, double inv_t, Room* room) {
    const int lane = threadIdx.x & 31;
    double s = 0.0;
#pragma unroll 4
    for (int i = lo + threadIdx.x; i < hi; i += RACERS) {
        const float x = clean(to_f<T>(row[i]));
        if (x > -INFINITY) s += exp(far_below(x, top) * inv_t);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) room->key[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < RACERS / 32; ++w) s += room->key[w];
        room->best = s;
    }
    cluster_sync_all();
    s = 0.0;
    if (lane < CLUSTER) asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(s) : "r"(peer_smem(&room->best, lane)) : "memory");
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    cluster_sync_all();                                 // (read: it may be written again)
    return s;
}

// What f32 sums leave open, by a sequence's cluster: 1 + j, drafts from j on are too close to call; -1 - j, the race behind j of them is.  A function of its own, called where nothing else of
// the caller's lives on, so that its registers are no one else's; a third kernel for it took 2 to 4 us more.
template <typename T>
__device__ __noinline__ void settle(const Draft& d, int parts, int b, int s0, int n, double inv_t, int open, Holds* holds, Room* room) {
    const int rank = (int)cluster_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int len = stretch_of(d.vocab, CLUSTER), lo = (int)min((long long)d.vocab, (long long)rank * len), hi = min(d.vocab, lo + len);
    const Drafts<T> drafts{d, parts, b, s0, n, false, inv_t};
    int j = open > 0 ? open - 1 : -1 - open;
    for (bool close = open > 0; close;) {
        Part p = drafts.target(j), q = drafts.draft(j);
        p.sum = again<T>(drafts.x(j), lo, hi, p.top, inv_t, room);
        if (d.q) q.sum = again<T>(drafts.y(j), lo, hi, q.top, inv_t, room);
        double uq, pd;
        drafts.sides(j, __ldg(d.tokens + s0 + j), p, q, uq, pd);
        if (!(uq < pd)) break;
        drafts.look(j + 1, holds);
        j = min(holds->first, holds->close);
        close = j == holds->close;
        __syncthreads();                                // (read: they may be written again)
    }
    // ---- the race, 64 bits throughout ----
    Part p = drafts.target(j), q = drafts.draft(j);
    if (p.sum <= 0.0) {
        if (rank == 0 && threadIdx.x == 0) { d.accepted[b] = j; d.next[b] = -1; }
        return;
    }
    const int sure = j < n && !d.q ? __ldg(d.tokens + s0 + j) : -1;
    const T* x = drafts.x(j);
    const T* y = q.sum > 0.0 ? drafts.y(j) : nullptr;
    const float* u = d.noise + (long long)b * d.ldn;
    if (y) {
        p.sum = again<T>(x, lo, hi, p.top, inv_t, room);
        q.sum = again<T>(y, lo, hi, q.top, inv_t, room);
    }
    int at = INT_MAX;
    for (int pass = 0; pass < 2 && at == INT_MAX; ++pass) {
        double best = 0.0;
        auto meet = [&](double key, int i) { if (key > best || (key == best && i < at)) { best = key; at = i; } };
        auto reduce = [&]() {
            for (int o = 16; o > 0; o >>= 1) { const double k2 = __shfl_xor_sync(0xffffffffu, best, o); meet(k2, __shfl_xor_sync(0xffffffffu, at, o)); }
        };
        for (int i = lo + threadIdx.x; i < hi; i += RACERS) {
            const double w = (i == sure && pass == 0 ? 0.0 : share(clean(to_f<T>(x[i])), p, inv_t)) - (y && pass == 0 ? share(clean(to_f<T>(y[i])), q, inv_t) : 0.0);
            if (w > 0.0) meet(w / clock_of(__ldg(u + i)), i);
        }
        reduce();
        if (lane == 0) { room->key[warp] = best; room->at[warp] = at; }
        __syncthreads();
        if (warp == 0) {
            best = lane < RACERS / 32 ? room->key[lane] : 0.0;
            at = lane < RACERS / 32 ? room->at[lane] : INT_MAX;
            reduce();
            if (lane == 0) { room->best = best; room->best_at = at; }
        }
        cluster_sync_all();
        best = 0.0;
        at = INT_MAX;
        if (lane < CLUSTER) {
            asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(best) : "r"(peer_smem(&room->best, lane)) : "memory");
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(at) : "r"(peer_smem(&room->best_at, lane)) : "memory");
        }
        reduce();
        cluster_sync_all();                             // (read: it may be written again, or its owner leave)
    }
    if (rank == 0 && threadIdx.x == 0) { d.accepted[b] = j; d.next[b] = at; }      // (a row's largest logit always has a key)
}

// A cluster for each sequence: the drafts, then the race
template <typename T>
__global__ void __launch_bounds__(RACERS)
race_kernel(const __grid_constant__ Draft d, int parts) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ Holds holds_s;
    __shared__ Part rows_s[2];
    __shared__ Room room_s;
    __shared__ float bar_s, bars_s[RACERS / 32];
    const int b = blockIdx.x / CLUSTER, rank = (int)cluster_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s0 = start_of(d, b), n = max(start_of(d, b + 1), s0) - s0;
    const float temp = d.temperatures ? __ldg(d.temperatures + b) : 1.f;
    const bool greedy = !(temp > 0.f);
    const double inv_t = greedy ? 1.0 : fmax(1.0 / (double)temp, 0x1p-126);
    const int len = stretch_of(d.vocab, CLUSTER), lo = (int)min((long long)d.vocab, (long long)rank * len), hi = min(d.vocab, lo + len);
    const Drafts<T> drafts{d, parts, b, s0, n, greedy, inv_t};
    drafts.look(0, &holds_s);
    const int j = min(holds_s.first, holds_s.close);    // (the cluster alike)
    auto race = [&]() -> int {                          // 0, or what settle is to settle
        if (j >= KEPT) {
            if (warp == 0) { const Part p = drafts.target(j); if (lane == 0) rows_s[0] = p; }
            else if (warp == 1) { const Part q = drafts.draft(j); if (lane == 0) rows_s[1] = q; }
            __syncthreads();
        }
        const Part p = j < KEPT ? holds_s.p[j] : rows_s[0], q = j < KEPT ? holds_s.q[j] : rows_s[1];
        if (greedy || p.sum <= 0.0) {                       // (the whole cluster alike)
            if (rank == 0 && threadIdx.x == 0) { d.accepted[b] = j; d.next[b] = p.top > -INFINITY ? p.at : -1; }
            return 0;
        }
        const int sure = j < n && !d.q ? __ldg(d.tokens + s0 + j) : -1;      // a draft that was certain: q is 1 there
        const T* x = drafts.x(j);
        const T* y = q.sum > 0.0 ? drafts.y(j) : nullptr;
        const float* u = d.noise + (long long)b * d.ldn;
        const float c = rate(temp), pz = (float)(1.0 / p.sum), qz = q.sum > 0.0 ? (float)(1.0 / q.sum) : 0.f;
        constexpr int N = 16 / (int)sizeof(T);
        const bool wide = ((reinterpret_cast<uintptr_t>(x + lo) | (y ? reinterpret_cast<uintptr_t>(y + lo) : 0) | reinterpret_cast<uintptr_t>(u + lo)) & 15) == 0;
        for (int pass = 0; pass < 2; ++pass) {                           // the second only where p exceeds q nowhere: the race over p itself
            // f32 brackets every key (its p, q and clock are 6e-5 of themselves off at most, a third of what is allowed for).  Places whose upper end stays below the best lower end
            // of the whole row cannot win; the few others' keys are computed in 64 bits.
            float low = 0.f, high = 0.f, second = 0.f;      // best lower end, two best upper ends among this thread's places
            int high_at = 0;
            // p = 2^(x c + bp) in one step where the rounding of its terms stays below 2^-14; not for infinite or far maxima
            const float tp = p.top * c, tq = q.top * c, bp = __log2f(pz) - tp, bq = y ? __log2f(qz) - tq : 0.f;
            const bool near = fabsf(tp) < 500.f && (!y || fabsf(tq) < 500.f);
            auto bracket = [&](int i, float xv, float yv, float uv, float& lo_key, float& hi_key) {
                float pi = near ? ex2(fmaf(xv, c, bp)) : xv == -INFINITY ? 0.f : ex2(below(xv, p.top) * c) * pz;
                const float qi = !y || pass ? 0.f : near ? ex2(fmaf(yv, c, bq)) : yv == -INFINITY ? 0.f : ex2(below(yv, q.top) * c) * qz;
                if (i == sure && pass == 0) pi = 0.f;
                const float slack = 2e-4f * (pi + qi), z = fminf(fmaxf(uv, 0x1p-126f), 0x1.fffffep-1f), w = 1.f - z;
                const float clock = w < 0.02f ? w * fmaf(w, fmaf(w, 0.33333334f, 0.5f), 1.f) : -0.69314718f * __log2f(z), inv = __fdividef(1.f, clock);
                lo_key = (pi - qi - slack) * inv;
                hi_key = (pi - qi + slack) * inv;
            };
            auto all = [&](auto&& f) {                      // f(i, x, y, u) over this thread's places
                if (wide) {
                    const int end = lo + (hi - lo) / N * N;
#pragma unroll 2
                    for (int i = lo + threadIdx.x * N; i < end; i += RACERS * N) {
                        float xv[N], yv[N], uv[N];
                        get<T, N>(x + i, xv);
                        if (y && pass == 0) get<T, N>(y + i, yv);
                        else {
#pragma unroll
                            for (int k = 0; k < N; ++k) yv[k] = -INFINITY;
                        }
#pragma unroll
                        for (int k = 0; k < N; k += 4) { const float4 v = __ldg(reinterpret_cast<const float4*>(u + i + k)); uv[k] = v.x; uv[k + 1] = v.y; uv[k + 2] = v.z; uv[k + 3] = v.w; }
#pragma unroll
                        for (int k = 0; k < N; ++k) f(i + k, xv[k], yv[k], uv[k]);
                    }
                    const int i = end + threadIdx.x;
                    if (i < hi) f(i, clean(to_f<T>(x[i])), y && pass == 0 ? clean(to_f<T>(y[i])) : -INFINITY, __ldg(u + i));
                } else {
#pragma unroll 4
                    for (int i = lo + threadIdx.x; i < hi; i += RACERS) f(i, clean(to_f<T>(x[i])), y && pass == 0 ? clean(to_f<T>(y[i])) : -INFINITY, __ldg(u + i));
                }
            };
            all([&](int i, float xv, float yv, float uv) {
                float a, z;
                bracket(i, xv, yv, uv, a, z);
                low = fmaxf(low, a);
                if (z > high) { second = high; high = z; high_at = i; }
                else second = fmaxf(second, z);
            });
            float bar = warp_max(low);
            if (lane == 0) bars_s[warp] = bar;
            __syncthreads();
            if (warp == 0) {
                bar = warp_max(lane < RACERS / 32 ? bars_s[lane] : 0.f);
                if (lane == 0) bar_s = bar;
            }
            cluster_sync_all();
            bar = 0.f;                                      // (a lane for each CTA)
            if (lane < CLUSTER) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(bar) : "r"(peer_smem(&bar_s, lane)) : "memory");
            bar = warp_max(bar);
            // Keys in 64 bits, with what the sums leave open of them where p and q make them (a sum alone is a factor of all): the best upper end, its place; the best lower end and this
            // thread's other upper ends in case that several places are left
            const bool both = y && pass == 0;
            double best = 0.0;
            int at = INT_MAX, left = 0;
            float rival = 0.f, sure_low = 0.f;
            auto meet = [&](double key, int i) { if (key > best || (key == best && i < at)) { best = key; at = i; } };
            auto exactly = [&](int i, float xv, float yv, float uv) {
                const double pi = share(xv, p, inv_t), qi = yv == -INFINITY ? 0.0 : share(yv, q, inv_t), w = pi - qi, slack = both ? SUMS * (pi + qi) : 0.0;
                if (!(w + slack > 0.0)) return;
                const double key = (w + slack) / clock_of(uv);
                // 1 - 2 slack / (w + slack), the quotient rounded up
                if (both) {
                    sure_low = fmaxf(sure_low, __double2float_rd(key) * (1.f - 2.001f * __fdividef((float)slack, (float)(w + slack))));
                    if (left) rival = fmaxf(rival, __double2float_ru(fmin(key, best)));
                    left += w > slack ? 1 : 2;          // (one that may be 0 is not alone)
                }
                meet(key, i);
            };
            if (high > 0.f && high >= bar) {
                if (second < bar || second <= 0.f) {
                    exactly(high_at, clean(to_f<T>(x[high_at])), y && pass == 0 ? clean(to_f<T>(y[high_at])) : -INFINITY, __ldg(u + high_at));
                } else {
                    all([&](int i, float xv, float yv, float uv) {
                        float a, z;
                        bracket(i, xv, yv, uv, a, z);
                        if (z > 0.f && z >= bar) exactly(i, xv, yv, uv);
                    });
                }
            }
            auto reduce = [&]() {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const double k2 = __shfl_xor_sync(0xffffffffu, best, o);
                    const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
                    meet(k2, a2);
                }
            };
            const int own_at = at;
            const float own = both ? __double2float_ru(best) : 0.f;
            left = __reduce_add_sync(0xffffffffu, left);
            if (__any_sync(0xffffffffu, best > 0.0)) reduce();
            if (lane == 0) { room_s.key[warp] = best; room_s.at[warp] = at; room_s.left[warp] = left; }
            __syncthreads();
            if (warp == 0) {
                const bool here = lane < RACERS / 32;
                best = here ? room_s.key[lane] : 0.0;
                at = here ? room_s.at[lane] : INT_MAX;
                left = __reduce_add_sync(0xffffffffu, here ? room_s.left[lane] : 0);
                reduce();
                if (lane == 0) { room_s.best = best; room_s.best_at = at; room_s.all_left = left; }
            }
            cluster_sync_all();
            best = 0.0;
            at = INT_MAX;
            left = 0;
            if (lane < CLUSTER) {
                asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(best) : "r"(peer_smem(&room_s.best, lane)) : "memory");
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(at) : "r"(peer_smem(&room_s.best_at, lane)) : "memory");
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(left) : "r"(peer_smem(&room_s.all_left, lane)) : "memory");
            }
            reduce();
            cluster_sync_all();                             // (read: it may be written again, or its owner leave)
            if (__reduce_add_sync(0xffffffffu, left) > 1) { // (the cluster alike; both) could another place have the best key, or none?
                rival = warp_max(own_at == at ? rival : fmaxf(rival, own));
                sure_low = warp_max(sure_low);
                if (lane == 0) { room_s.rival[warp] = rival; bars_s[warp] = sure_low; }
                __syncthreads();
                if (threadIdx.x == 0) {
                    for (int w = 0; w < RACERS / 32; ++w) { rival = fmaxf(rival, room_s.rival[w]); sure_low = fmaxf(sure_low, bars_s[w]); }
                    room_s.best_rival = rival;
                    bar_s = sure_low;
                }
                cluster_sync_all();
                rival = sure_low = 0.f;
                if (lane < CLUSTER) {
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(rival) : "r"(peer_smem(&room_s.best_rival, lane)) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(sure_low) : "r"(peer_smem(&bar_s, lane)) : "memory");
                }
                rival = warp_max(rival);
                sure_low = warp_max(sure_low);
                cluster_sync_all();
                if (rival >= sure_low) return -1 - j;
            }
            if (best > 0.0 || pass == 1) {
                if (rank == 0 && threadIdx.x == 0) { d.accepted[b] = j; d.next[b] = best > 0.0 ? at : -1; }      // (a row's largest logit always has a key)
                return 0;
            }
        }
        return 0;
    };
    const int open = j == holds_s.close ? 1 + j : race();
    if (open) settle<T>(d, parts, b, s0, n, inv_t, open, &holds_s, &room_s);
}

int parts_of(int rows, int vocab) {                     // CTAs that share a row: every SM is to have some, stretches of 2048 logits at least and 65 536 at most (SUMS)
    const int most = std::max(1, vocab / 2048), want = (4 * tc_device_sms() + rows - 1) / rows;
    return std::max((vocab + 65535) / 65536, std::min(most, std::min(64, std::max(8, want))));
}

template <typename T>
int launch(cudaStream_t st, const Draft& d, bool pdl) {
    const int rows = d.total + d.seqs + (d.q ? d.total : 0), parts = parts_of(rows, d.vocab);
    if (const int e = launch_k(stretch_kernel<T>, dim3(rows, parts), dim3(THREADS), 0, st, pdl, d, parts)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)d.seqs * CLUSTER); cfg.blockDim = dim3(RACERS); cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CLUSTER; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, race_kernel<T>, d, parts);
}

}  // namespace

size_t draft_bytes(int seqs, int total, int vocab, bool q) {
    if (!seqs) return 0;
    const int rows = total + seqs + (q ? total : 0);
    return (size_t)rows * parts_of(rows, vocab) * sizeof(Part);
}

int draft_verify_launch(cudaStream_t st, const Draft& d, bool pdl) {
    if (d.seqs == 0) return 0;
    switch (d.type) {
        case DRAFT_F32: return launch<float>(st, d, pdl);
        case DRAFT_BF16: return launch<bf16>(st, d, pdl);
        case DRAFT_F16: return launch<__half>(st, d, pdl);
    }
    return -1000;
}

}  // namespace cb
