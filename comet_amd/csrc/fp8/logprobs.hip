// logprobs.hip — rows of scores as distributions: log-probabilities of given columns, entropy, and the best columns, in one pass over the scores.
//
// With z_j = scale * s_j over a row's columns, M = max z, d_j = z_j - M and S = sum exp(d_j):
//   log sum exp(z) = M + log S      log p_j = d_j - log S      entropy = log S + (1 / S) sum exp(d_j) (-d_j)
// S and W = sum exp(d_j) d_j run along with the maximum: when it moves by D, S becomes S exp(-D) and W becomes (W - D S) exp(-D). Every term of the
// entropy is then non-negative, so nothing cancels. A negative scale (distances) is a flip of every score's sign and a positive scale.
//
// The best k columns ride on the same pass: a workgroup keeps the candidates that exceed its k-th best so far in LDS and sorts them when they get many.
// A key is (score, column) in 64 bits, larger is better, equal scores to the lower column; keys are unique, so the result does not depend on the order in
// which candidates arrive. Bound by reading the scores once.
#include "fp8.hpp"

namespace comet {
namespace {

constexpr int kThreads = 256, kEpt = 32, kChunk = kThreads * kEpt;
// candidate buffer: the k best so far and one chunk's survivors. When more than kSoft would be held, the chunk is cut to the keys not below the k-th
// largest of the 256 threads' largest keys: only the k threads above that bound hold survivors, kEpt each.
constexpr int kSoft = 1024, kCap = kLogProbsMaxK + kEpt * kLogProbsMaxK;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Stats { float m, s, w; int bad; };   // maximum, S, W in units of log2 (w = sum e * t, t = d * log2 e); bad: a NaN was seen

__device__ __forceinline__ float exp2_t(float t) { return __builtin_amdgcn_exp2f(t); }

__device__ __forceinline__ void stats_join(Stats& a, float m, float s, float w, int bad, float f) {
    a.bad |= bad;
    const float hi = fmaxf(a.m, m);
    if (hi == -INFINITY) return;
    float ta = (a.m - hi) * f, tb = (m - hi) * f;
    ta = ta < -1e30f ? -1e30f : ta; tb = tb < -1e30f ? -1e30f : tb;      // -inf * 0 below would be NaN
    const float ea = exp2_t(ta), eb = exp2_t(tb);
    a.w = (a.w + ta * a.s) * ea + (w + tb * s) * eb;
    a.s = a.s * ea + s * eb;
    a.m = hi;
}

// order-preserving bits of a finite or infinite float
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) { return __builtin_bit_cast(float, o ^ ((uint32_t)((int32_t)~o >> 31) | 0x80000000u)); }
__device__ __forceinline__ uint64_t make_key(float x, uint32_t col) { return ((uint64_t)ordered(x) << 32) | (0xFFFFFFFFu - col); }   // 0 is no key: it would need a NaN
__device__ __forceinline__ uint32_t key_col(uint64_t k) { return 0xFFFFFFFFu - (uint32_t)k; }

struct Shared {
    uint64_t buf[kCap];
    uint64_t best[kThreads];
    uint64_t cut;
    int total[kThreads / 64];
    int cnt;
    float sm[kThreads / 64], ss[kThreads / 64], sw[kThreads / 64]; int sb[kThreads / 64];
    Stats row;
};

// buf[0 .. cnt) sorted descending, cut to k; every thread returns the new count
__device__ int compact(Shared& sh, int cnt, int k) {
    int p = 64;
    while (p < cnt) p <<= 1;                 // at most 8192 > kCap: the pad beyond kCap is never stored (see below)
    const int top = p < kCap ? p : kCap;
    for (int i = cnt + threadIdx.x; i < top; i += kThreads) sh.buf[i] = 0;
    __syncthreads();
    for (int size = 2; size <= p; size <<= 1) {
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            for (int t = threadIdx.x; t < p / 2; t += kThreads) {
                const int i = 2 * t - (t & (stride - 1)), j = i + stride;
                // bitonic network with every merge descending: the first step of a merge compares mirrored positions
                const int jj = stride == (size >> 1) ? (i & ~(size - 1)) + size - 1 - (i & (size - 1)) : j;
                const int lo = i < jj ? i : jj, hi = i < jj ? jj : i;
                if (hi < kCap) {             // positions from kCap on hold 0, the smallest key: nothing moves there
                    const uint64_t a = sh.buf[lo], b = sh.buf[hi];
                    if (a < b) { sh.buf[lo] = b; sh.buf[hi] = a; }
                }
            }
            __syncthreads();
        }
    }
    return cnt < k ? cnt : k;
}

// Adds this chunk's candidates: bit i of `mask` says that element i of this thread is one, key(i) is its key. thr_key: the k-th best key so far (0: none).
// Uniform across the workgroup; returns the number held.
template <int EPT, class Key>
__device__ int add_candidates(Shared& sh, int cnt, int k, uint32_t mask, Key key, uint64_t& thr_key) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int c = __popc(mask);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
    if (lane == 0) sh.total[wave] = c;
    __syncthreads();
    c = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) c += sh.total[w];
    if (c == 0) { __syncthreads(); return cnt; }
    uint64_t cut = 0;
    if (cnt + c > kSoft) {
        if (cnt > k) { cnt = compact(sh, cnt, k); thr_key = cnt == k ? sh.buf[k - 1] : thr_key; }
        uint64_t mine = 0;
#pragma unroll
        for (int i = 0; i < EPT; i++) if ((mask >> i) & 1u) { const uint64_t q = key(i); mine = q > mine ? q : mine; }
        sh.best[threadIdx.x] = mine;
        if (threadIdx.x == 0) sh.cut = 0;
        __syncthreads();
        int above = 0;
        for (int t = 0; t < kThreads; t++) above += sh.best[t] > mine ? 1 : 0;
        if (mine != 0 && above == k - 1) sh.cut = mine;       // keys are unique: at most one thread; nobody when fewer than k threads hold any
        __syncthreads();
        cut = sh.cut;
        cut = cut > thr_key ? cut : thr_key;
    }
    if (threadIdx.x == 0) sh.cnt = cnt;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EPT; i++) if ((mask >> i) & 1u) {
        const uint64_t q = key(i);
        if (q >= cut) sh.buf[atomicAdd(&sh.cnt, 1)] = q;
    }
    __syncthreads();
    cnt = sh.cnt;
    if ((thr_key == 0 && cnt >= k) || cnt >= k + kThreads) {
        cnt = compact(sh, cnt, k);
        if (cnt == k) thr_key = sh.buf[k - 1];
    }
    __syncthreads();
    return cnt;
}

__device__ void reduce_stats(Shared& sh, Stats st, float f) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) stats_join(st, __shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.w, o, 64), __shfl_xor(st.bad, o, 64), f);
    if (lane == 0) { sh.sm[wave] = st.m; sh.ss[wave] = st.s; sh.sw[wave] = st.w; sh.sb[wave] = st.bad; }
    __syncthreads();
    if (threadIdx.x == 0) {
        Stats a{sh.sm[0], sh.ss[0], sh.sw[0], sh.sb[0]};
        for (int w = 1; w < kThreads / 64; w++) stats_join(a, sh.sm[w], sh.ss[w], sh.sw[w], sh.sb[w], f);
        sh.row = a;
    }
    __syncthreads();
}

template <class T> __device__ __forceinline__ float flip_score(T v, uint32_t sign) {     // -0 becomes +0: the two are one score
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, (float)v) ^ sign) + 0.0f;
}

// a row's outputs from its statistics and its sorted best keys (sh.row, sh.buf[0 .. cnt))
template <class T>
__device__ void finish_row(Shared& sh, int64_t row, const T* x, int count, int cnt, const int32_t* targets, int n_targets, int k, float scale, uint32_t sign,
                           float* logprobs, float* logsum, float* entropy, int32_t* ids, float* top_logprobs) {
    const Stats st = sh.row;
    const bool empty = !st.bad && st.m == -INFINITY;
    const float nan = __builtin_nanf("");
    const float log_s = st.bad ? nan : logf(st.s);
    if (threadIdx.x == 0) {
        logsum[row] = empty ? -INFINITY : st.m * scale + log_s;
        entropy[row] = empty ? 0.0f : log_s - kLn2 * (st.w / st.s);
    }
    for (int t = threadIdx.x; t < n_targets; t += kThreads) {
        const int32_t col = targets[row * n_targets + t];
        float v = -INFINITY;
        if (!empty && col >= 0 && col < count) v = (flip_score(x[col], sign) - st.m) * scale - log_s;
        logprobs[row * n_targets + t] = v;
    }
    for (int i = threadIdx.x; i < k; i += kThreads) {
        const bool has = i < cnt;
        const uint64_t q = has ? sh.buf[i] : 0;
        ids[row * k + i] = has ? (int32_t)key_col(q) : -1;
        top_logprobs[row * k + i] = has ? (unordered((uint32_t)(q >> 32)) - st.m) * scale - log_s : -INFINITY;
    }
}

// Workgroup (row, split): columns [split * span, ...) of the row's count in chunks of 8192, each thread 32 of them in 16-byte pieces.
template <class T>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const T* __restrict__ scores, int64_t ld, int n, const int32_t* __restrict__ counts, float scale, uint32_t sign,
                                                            const int32_t* __restrict__ targets, int n_targets, int k, int splits, float* __restrict__ logprobs,
                                                            float* __restrict__ logsum, float* __restrict__ entropy, int32_t* __restrict__ ids, float* __restrict__ top_logprobs,
                                                            Stats* __restrict__ part_stats, uint64_t* __restrict__ part_keys) {
    __shared__ Shared sh;
    constexpr int V = 16 / sizeof(T), P = kEpt / V;
    const int64_t row = blockIdx.x / (unsigned)splits;
    const int split = (int)(blockIdx.x % (unsigned)splits);
    int count = n;
    if (counts) { count = counts[row]; count = count < 0 ? 0 : (count > n ? n : count); }
    const int chunks = (count + kChunk - 1) / kChunk, per = (chunks + splits - 1) / splits;
    const int c_end = min(chunks, (split + 1) * per);
    const T* x = scores + row * ld;
    const float f = scale * kLog2e;
    Stats st{-INFINITY, 0.0f, 0.0f, 0};
    int cnt = 0;
    uint64_t thr_key = 0;
    for (int c = split * per; c < c_end; c++) {
        const int base = c * kChunk + threadIdx.x * V;
        float v[kEpt];
        if ((c + 1) * (int64_t)kChunk <= count) {
            T t[P][V];
#pragma unroll
            for (int p = 0; p < P; p++) __builtin_memcpy(t[p], x + base + p * (kThreads * V), 16);
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int i = 0; i < V; i++) v[p * V + i] = flip_score(t[p][i], sign);
        } else {
#pragma unroll
            for (int p = 0; p < P; p++) {
                const int64_t col = (int64_t)base + p * (kThreads * V);
                if (col + V <= count) {
                    T t[V];
                    __builtin_memcpy(t, x + col, 16);
#pragma unroll
                    for (int i = 0; i < V; i++) v[p * V + i] = flip_score(t[i], sign);
                } else {
#pragma unroll
                    for (int i = 0; i < V; i++) v[p * V + i] = col + i < count ? flip_score(x[col + i], sign) : -INFINITY;
                }
            }
        }
        float hi = v[0];
#pragma unroll
        for (int i = 0; i < kEpt; i++) { st.bad |= v[i] != v[i] ? 1 : 0; hi = fmaxf(hi, v[i]); }
        hi = fmaxf(hi, st.m);
        if (hi > st.m && st.m > -INFINITY) {
            float t = (st.m - hi) * f;
            t = t < -1e30f ? -1e30f : t;
            const float e = exp2_t(t);
            st.w = (st.w + t * st.s) * e; st.s *= e;
        }
        st.m = hi;
        if (hi > -INFINITY) {
#pragma unroll
            for (int i = 0; i < kEpt; i++) {
                float t = (v[i] - hi) * f;
                t = t < -1e30f ? -1e30f : t;          // a masked entry, or one so far below that exp is 0 and t * 0 must be 0
                const float e = exp2_t(t);
                st.s += e; st.w = __builtin_fmaf(e, t, st.w);
            }
        }
        if (k > 0) {
            const float thr = thr_key ? unordered((uint32_t)(thr_key >> 32)) : -INFINITY;      // later columns lose a tie: strictly greater
            uint32_t mask = 0;
#pragma unroll
            for (int i = 0; i < kEpt; i++) mask |= v[i] > thr ? 1u << i : 0u;                  // false for NaN and for -inf
            cnt = add_candidates<kEpt>(sh, cnt, k, mask, [&](int i) { return make_key(v[i], (uint32_t)(base + (i / V) * (kThreads * V) + i % V)); }, thr_key);
        }
    }
    if (k > 0) cnt = compact(sh, cnt, k);
    reduce_stats(sh, st, f);
    if (splits == 1) {
        finish_row(sh, row, x, count, cnt, targets, n_targets, k, scale, sign, logprobs, logsum, entropy, ids, top_logprobs);
    } else {
        if (threadIdx.x == 0) part_stats[blockIdx.x] = sh.row;
        for (int i = threadIdx.x; i < k; i += kThreads) part_keys[(int64_t)blockIdx.x * k + i] = i < cnt ? sh.buf[i] : 0;
    }
}

// joins a row's splits
template <class T>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(const T* __restrict__ scores, int64_t ld, int n, const int32_t* __restrict__ counts, float scale, uint32_t sign,
                                                                 const int32_t* __restrict__ targets, int n_targets, int k, int splits, float* __restrict__ logprobs,
                                                                 float* __restrict__ logsum, float* __restrict__ entropy, int32_t* __restrict__ ids, float* __restrict__ top_logprobs,
                                                                 const Stats* __restrict__ part_stats, const uint64_t* __restrict__ part_keys) {
    __shared__ Shared sh;
    constexpr int E = 8;
    const int64_t row = blockIdx.x;
    int count = n;
    if (counts) { count = counts[row]; count = count < 0 ? 0 : (count > n ? n : count); }
    const float f = scale * kLog2e;
    Stats st{-INFINITY, 0.0f, 0.0f, 0};
    for (int i = threadIdx.x; i < splits; i += kThreads) { const Stats p = part_stats[row * splits + i]; stats_join(st, p.m, p.s, p.w, p.bad, f); }
    int cnt = 0;
    uint64_t thr_key = 0;
    const int total = splits * k;
    const uint64_t* keys = part_keys + row * total;
    for (int b = 0; b < total; b += kThreads * E) {
        uint64_t q[E];
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < E; i++) { const int at = b + i * kThreads + (int)threadIdx.x; q[i] = at < total ? keys[at] : 0; mask |= q[i] > thr_key ? 1u << i : 0u; }
        cnt = add_candidates<E>(sh, cnt, k, mask, [&](int i) { return q[i]; }, thr_key);
    }
    if (k > 0) cnt = compact(sh, cnt, k);
    reduce_stats(sh, st, f);
    finish_row(sh, row, scores + row * ld, count, cnt, targets, n_targets, k, scale, sign, logprobs, logsum, entropy, ids, top_logprobs);
}

// Splits of a row: enough workgroups for four per CU, none with less than one chunk.
constexpr int64_t kGroups = 1024;
int split_count(int64_t m, int64_t n) {
    const int64_t chunks = std::max<int64_t>(1, ceil_div(n, kChunk));
    return (int)std::min(chunks, std::max<int64_t>(1, kGroups / m));
}

template <class T> void logprobs_t(hipStream_t s, const LogProbsArgs& a) {
    const uint32_t sign = a.scale < 0 ? 0x80000000u : 0u;
    const float scale = std::fabs(a.scale);
    constexpr int64_t kPiece = (int64_t)1 << 24;
    for (int64_t i = 0; i < a.m; i += kPiece) {
        const int64_t m = std::min(kPiece, a.m - i);
        const int splits = split_count(m, a.n);
        Stats* ps = (Stats*)a.work;
        uint64_t* pk = (uint64_t*)((char*)a.work + round_up((int64_t)sizeof(Stats) * m * splits, 16));
        const T* x = (const T*)a.scores + i * a.ld;
        const int32_t* counts = a.counts ? a.counts + i : nullptr;
        const int32_t* targets = a.n_targets ? a.targets + i * a.n_targets : nullptr;
        float* lp = a.n_targets ? a.logprobs + i * a.n_targets : nullptr;
        int32_t* ids = a.k ? a.ids + i * a.k : nullptr;
        float* tl = a.k ? a.top_logprobs + i * a.k : nullptr;
        hipLaunchKernelGGL((logprobs_kernel<T>), dim3((unsigned)(m * splits)), dim3(kThreads), 0, s, x, a.ld, a.n, counts, scale, sign, targets, a.n_targets, a.k, splits,
                           lp, a.logsum + i, a.entropy + i, ids, tl, ps, pk);
        LAUNCH_CHECK();
        if (splits > 1) {
            hipLaunchKernelGGL((logprobs_join_kernel<T>), dim3((unsigned)m), dim3(kThreads), 0, s, x, a.ld, a.n, counts, scale, sign, targets, a.n_targets, a.k, splits,
                               lp, a.logsum + i, a.entropy + i, ids, tl, ps, pk);
            LAUNCH_CHECK();
        }
    }
}
}  // namespace

// an upper bound for every call of at most m rows, n columns and k best: m * splits never exceeds min(m * chunks, max(m, kGroups))
size_t logprobs_work_bytes(int64_t m, int64_t n, int32_t k) {
    const int64_t chunks = std::max<int64_t>(1, ceil_div(n, kChunk));
    if (m <= 0 || chunks == 1) return 0;
    const int64_t parts = std::min(m * chunks, kGroups);
    return (size_t)(round_up((int64_t)sizeof(Stats) * parts, 16) + parts * 8 * k);
}

void launch_logprobs(hipStream_t s, const LogProbsArgs& a) {
    if (a.m <= 0) return;
    if (a.dtype == COMET_F32) logprobs_t<float>(s, a);
    else if (a.dtype == COMET_F16) logprobs_t<_Float16>(s, a);
    else logprobs_t<__bf16>(s, a);
}

}  // namespace comet
