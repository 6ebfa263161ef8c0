// Verification of drafted tokens (draft.cuh).  With p the target's and q the draft model's softmax at the sequence's temperature:
//   draft j is accepted while u_j q_j(d_j) < p_j(d_j); at the first that is not, and behind the last, one more token follows:
//   argmax_i w_i / -log(noise_i), the lowest index among equals, w = max(p - q, 0) (p where that is zero everywhere), or p behind the last: a race of exponential clocks,
//   drawn in proportion to w as the sampler's whole-vocabulary draw.  Temperature 0: the draft is accepted if it is the row's first maximum, which follows otherwise.
// A NaN logit counts as -inf; where the largest is +inf all of those share the probability; a row without a logit above -inf accepts nothing and gives token -1.
//
// Two kernels: the first reads every row once and leaves (maximum, its place, sum) of each stretch of it, the second has a cluster of CTAs for each sequence, which
// joins those, walks the drafts and runs the race over the one row that needs it.  Bound by bytes: the rows of both models, one row of noise a sequence.
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "draft.cuh"
#include "tc.cuh"

namespace cb {
namespace {

constexpr int THREADS = 256, CLUSTER = 8;
constexpr double LOG2E = 1.4426950408889634;

struct Part { float top; int at; double sum; };         // of a stretch: its largest logit, the first place of it, the sum of exp((x - top) / T)

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<bf16>(bf16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
__device__ __forceinline__ float clean(float x) { return x == x ? x : -INFINITY; }
__device__ __forceinline__ float below(float x, float top) { return x == top ? 0.f : x - top; }      // infinities by themselves
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

// f(i, x) for i in [lo, hi), 16 bytes at a time where the row's address allows
template <typename T, typename F>
__device__ __forceinline__ void each(const T* row, int lo, int hi, F f) {
    constexpr int N = 16 / (int)sizeof(T);
    const int skew = (int)(reinterpret_cast<uintptr_t>(row + lo) % 16) / (int)sizeof(T);
    const int a = min(hi, lo + (skew ? N - skew : 0)), b = a + (hi - a) / N * N;
    for (int i = lo + threadIdx.x; i < a; i += THREADS) f(i, clean(to_f<T>(row[i])));
#pragma unroll 4
    for (int i = a + threadIdx.x * N; i < b; i += THREADS * N) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + i));
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int j = 0; j < N; ++j) f(i + j, clean(to_f<T>(e[j])));
    }
    for (int i = b + threadIdx.x; i < hi; i += THREADS) f(i, clean(to_f<T>(row[i])));
}

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
    float top = -INFINITY, sum = 0.f;
    int at = INT_MAX;
    each<T>(x, lo, hi, [&](int i, float v) {
        if (v > top) {
            sum = top == -INFINITY ? 0.f : sum * ex2((top - v) * c);
            top = v;
            at = i;
        }
        sum += v == -INFINITY ? 0.f : ex2(below(v, top) * c);
    });
    // ---- the block's ----
    __shared__ float wt[THREADS / 32];
    __shared__ int wa[THREADS / 32];
    __shared__ double wsum[THREADS / 32];
    double s = sum;
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
    auto join = [&](const Part& q) {
        const float m = fmaxf(r.top, q.top);
        r.sum = (r.sum > 0.0 ? r.sum * exp((double)below(r.top, m) * inv_t) : 0.0) + (q.sum > 0.0 ? q.sum * exp((double)below(q.top, m) * inv_t) : 0.0);
        r.at = r.top > q.top ? r.at : q.top > r.top ? q.at : min(r.at, q.at);
        r.top = m;
    };
    for (int i = lane; i < parts; i += 32) join(p[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Part q;
        q.top = __shfl_xor_sync(0xffffffffu, r.top, o);
        q.at = __shfl_xor_sync(0xffffffffu, r.at, o);
        q.sum = __shfl_xor_sync(0xffffffffu, r.sum, o);
        join(q);
    }
    return r;
}
__device__ __forceinline__ double share(float x, const Part& p, double inv_t) { return p.sum > 0.0 && x > -INFINITY ? exp((double)below(x, p.top) * inv_t) / p.sum : 0.0; }

// A cluster for each sequence: the drafts, then the race
template <typename T>
__global__ void __launch_bounds__(THREADS)
race_kernel(Draft d, int parts) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ int first_s;
    __shared__ Part rows_s[2];
    __shared__ double key_s[THREADS / 32];
    __shared__ int at_s[THREADS / 32];
    __shared__ double best_s;
    __shared__ int best_at_s;
    const int b = blockIdx.x / CLUSTER, rank = (int)cluster_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s0 = start_of(d, b), n = max(start_of(d, b + 1), s0) - s0;
    const float temp = d.temperatures ? __ldg(d.temperatures + b) : 1.f;
    const bool greedy = !(temp > 0.f);
    const double inv_t = greedy ? 1.0 : fmax(1.0 / (double)temp, 0x1p-126);
    const Part* parts_p = reinterpret_cast<const Part*>(d.work);
    const T* x0 = reinterpret_cast<const T*>(d.logits) + (long long)(s0 + b) * d.ld;
    const T* y0 = reinterpret_cast<const T*>(d.q) + (d.q ? (long long)s0 * d.ldq : 0);
    if (threadIdx.x == 0) first_s = n;
    __syncthreads();
    for (int j = warp; j < n; j += THREADS / 32) {
        const Part p = whole(parts_p + (long long)(s0 + b + j) * parts, parts, inv_t);
        Part q = {};
        if (d.q && !greedy) q = whole(parts_p + (long long)(d.total + d.seqs + s0 + j) * parts, parts, inv_t);
        if (lane == 0) {
            const int tok = __ldg(d.tokens + s0 + j);
            bool ok = (unsigned)tok < (unsigned)d.vocab;
            if (ok && greedy) ok = p.top > -INFINITY && tok == p.at;
            else if (ok) {
                const double qd = d.q ? share(clean(to_f<T>(y0[j * d.ldq + tok])), q, inv_t) : 1.0;
                ok = (double)__ldg(d.uniforms + s0 + j) * qd < share(clean(to_f<T>(x0[j * d.ld + tok])), p, inv_t);
            }
            if (!ok) atomicMin(&first_s, j);
        }
    }
    __syncthreads();
    const int j = first_s;
    if (warp == 0) {
        const Part p = whole(parts_p + (long long)(s0 + b + j) * parts, parts, inv_t);
        if (lane == 0) rows_s[0] = p;
    } else if (warp == 1 && d.q && !greedy && j < n) {
        const Part q = whole(parts_p + (long long)(d.total + d.seqs + s0 + j) * parts, parts, inv_t);
        if (lane == 0) rows_s[1] = q;
    }
    __syncthreads();
    const Part p = rows_s[0], q = j < n && d.q && !greedy ? rows_s[1] : Part{0.f, 0, 0.0};
    if (greedy || p.sum <= 0.0) {                       // (the whole cluster alike)
        if (rank == 0 && threadIdx.x == 0) { d.accepted[b] = j; d.next[b] = p.top > -INFINITY ? p.at : -1; }
        return;
    }
    const int sure = j < n && !d.q ? __ldg(d.tokens + s0 + j) : -1;      // a draft that was certain: q is 1 there
    const T* x = x0 + j * d.ld;
    const T* y = q.sum > 0.0 ? y0 + j * d.ldq : nullptr;
    const float* u = d.noise + (long long)b * d.ldn;
    const float c = rate(temp), pz = (float)(1.0 / p.sum), qz = q.sum > 0.0 ? (float)(1.0 / q.sum) : 0.f;
    const int len = stretch_of(d.vocab, CLUSTER), lo = (int)min((long long)d.vocab, (long long)rank * len), hi = min(d.vocab, lo + len);
    for (int pass = 0; pass < 2; ++pass) {              // the second only where p exceeds q nowhere: the race over p itself
        // f32 tells which places cannot win (its p and q are 1e-5 of themselves off at most, a tenth of what is allowed for); the others' keys are computed in 64 bits
        double best = 0.0;
        float bar = 0.f;
        int at = INT_MAX;
        each<T>(x, lo, hi, [&](int i, float xv) {
            if (xv == -INFINITY || (pass == 0 && i == sure)) return;
            const float yv = y && pass == 0 ? clean(to_f<T>(y[i])) : -INFINITY;
            const float pi = ex2(below(xv, p.top) * c) * pz, qi = yv == -INFINITY ? 0.f : ex2(below(yv, q.top) * c) * qz;
            const float ui = fminf(fmaxf(__ldg(u + i), 0x1p-126f), 0x1.fffffep-1f), clock = -logf(ui);
            if ((pi - qi) + 1e-4f * (pi + qi) <= bar * clock) return;
            const double w = share(xv, p, inv_t) - (yv == -INFINITY ? 0.0 : share(yv, q, inv_t));
            if (!(w > 0.0)) return;
            const double key = w / -log((double)ui);
            if (key > best || (key == best && i < at)) { best = key; at = i; bar = (float)best * 0.9999f; }
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double k2 = __shfl_xor_sync(0xffffffffu, best, o);
            const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
            if (k2 > best || (k2 == best && a2 < at)) { best = k2; at = a2; }
        }
        if (lane == 0) { key_s[warp] = best; at_s[warp] = at; }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < THREADS / 32; ++w)
                if (key_s[w] > best || (key_s[w] == best && at_s[w] < at)) { best = key_s[w]; at = at_s[w]; }
            best_s = best;
            best_at_s = at;
        }
        cluster_sync_all();
        best = 0.0;
        at = INT_MAX;
        for (int r = 0; r < CLUSTER; ++r) {
            double k2;
            int a2;
            asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(k2) : "r"(peer_smem(&best_s, r)) : "memory");
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(a2) : "r"(peer_smem(&best_at_s, r)) : "memory");
            if (k2 > best || (k2 == best && a2 < at)) { best = k2; at = a2; }
        }
        cluster_sync_all();                             // (read: it may be written again, or its owner leave)
        if (best > 0.0 || pass == 1) {
            if (rank == 0 && threadIdx.x == 0) { d.accepted[b] = j; d.next[b] = best > 0.0 ? at : p.at; }
            return;
        }
    }
}

int parts_of(int rows, int vocab) {                     // CTAs that share a row: every SM is to have some, stretches of 2048 logits at least
    const int most = std::max(1, vocab / 2048), want = (4 * tc_device_sms() + rows - 1) / rows;
    return std::min(most, std::min(64, std::max(8, want)));
}

template <typename T>
int launch(cudaStream_t st, const Draft& d, bool pdl) {
    const int rows = d.total + d.seqs + (d.q ? d.total : 0), parts = parts_of(rows, d.vocab);
    if (const int e = launch_k(stretch_kernel<T>, dim3(rows, parts), dim3(THREADS), 0, st, pdl, d, parts)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)d.seqs * CLUSTER); cfg.blockDim = dim3(THREADS); cfg.stream = st;
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
