// logprobs.hip — rows of scores as distributions: log-probabilities of given columns, entropy, and the best columns, in one pass over the scores.
//
// With z_j = scale * s_j over a row's columns, M = max z, d_j = z_j - M and S = sum exp(d_j):
//   log sum exp(z) = M + log S      log p_j = d_j - log S      entropy = log S + (1 / S) sum exp(d_j) (-d_j)
// S and W = sum exp(d_j) d_j run along with the maximum: when it moves by D, S becomes S exp(-D) and W becomes (W - D S) exp(-D). Every term of the
// entropy is then non-negative, so nothing cancels. A negative scale (distances) is a flip of every score's sign and a positive scale.
//
// The best k columns ride on the same pass: a workgroup keeps the candidates that exceed its k-th best so far in LDS and sorts them when they get many.
// A key is (score, column) in 64 bits, larger is better, equal scores to the lower column; keys are unique, so the result does not depend on the order in
// which candidates arrive. Candidates wait as the score's own bits over the column's complement and become keys when they are sorted.
//
// What bounds it. Long rows of float32 without the best columns: reading the scores (256 x 1000000: 175 us, 5.9 TB/s). With the best columns, and in 16-bit types,
// the vector instructions of a score: 256 x 1000000 take 196 us with the best 100 whether they are float32 (5.2 TB/s), bfloat16 or float16 (2.6), 1024 x 200000
// 155 and 157; 19 vector instructions a score, the vector units busy 70 - 75 % of the time (11 without the best columns: 1024 x 200000 bfloat16 in 95 us,
// 4.3 TB/s). 1000 ragged rows of up to 30011 bfloat16 take 16 and, with the best 20, 26 us (a call that reads nothing takes 8): one workgroup a row, so the
// longest rows' eight chunks one after the other set the time, and a chunk with candidates costs its workgroup a barrier and the candidates' stores. Rows shorter
// than a chunk: a workgroup each, its numbers loaded one by one (2048 x 300 float32, best 10: 19 us; 2048 x 4096, a whole chunk: 17). Chunks of 16 numbers a
// thread: 32 took 223 us for the first, 8 177 us for 1024 x 200000 bfloat16.
#include "fp8.hpp"
#include "lanes.hpp"

namespace comet {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64, kEpt = 16, kChunk = kThreads * kEpt;
// Candidate buffer: the k best so far and one chunk's survivors. When more than kSoft would be held, the chunk is cut to the keys not below the k-th
// largest of the 256 threads' largest keys: only the k threads above that bound hold survivors, kEpt each. (Up to k = 32 quads of threads do.)
constexpr int kSoft = 512, kCap = kLogProbsMaxK + kEpt * kLogProbsMaxK;
// Splits of a row: as many as keep the workgroups within four per CU, so one for more than 512 rows (float32, best 10: 512 x 300000 in two splits 119 us, 600 in
// one 137, 1024 in one 214: 5.2, 5.3 and 5.7 TB/s). A row of up to four chunks is not split: a second launch costs more than the chunks one after the other
// (1 x 10000, k = 10: 10.6 us a pass, against 14.5 split in three).
constexpr int64_t kGroups = 1024, kWhole = 4;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Stats { float m, s, w; int bad; };   // maximum, S, W in units of log2 (w = sum e * t, t = d * log2 e); bad: a NaN among masked entries only (any other is in s)

__device__ __forceinline__ float exp2_t(float t) { return __builtin_amdgcn_exp2f(t); }

__device__ __forceinline__ void stats_join(Stats& a, float m, float s, float w, int bad, float f) {
    a.bad |= bad;
    const float hi = fmaxf(a.m, m);
    if (hi == -INFINITY) return;
    const float ta = (a.m - hi) * f, tb = (m - hi) * f, ea = exp2_t(ta), eb = exp2_t(tb);
    a.w = (a.w + fmaxf(ta, -1e30f) * a.s) * ea + (w + fmaxf(tb, -1e30f) * s) * eb;       // -inf * 0 would be NaN; a NaN stays in ea, eb
    a.s = a.s * ea + s * eb;
    a.m = hi;
}

// order-preserving bits of a finite or infinite float
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) { return __builtin_bit_cast(float, o ^ ((uint32_t)((int32_t)~o >> 31) | 0x80000000u)); }
__device__ __forceinline__ uint64_t make_key(float x, uint32_t col) { return ((uint64_t)ordered(x + 0.0f /* -0 and 0 are one score */) << 32) | ~col; }   // 0 is no key: it would need a NaN
__device__ __forceinline__ float key_score(uint64_t k) { return unordered((uint32_t)(k >> 32)); }
__device__ __forceinline__ uint32_t key_col(uint64_t k) { return ~(uint32_t)k; }

struct Shared {
    alignas(16) float score[kCap]; uint32_t col[kCap];      // the candidates
    alignas(16) uint64_t best[kThreads];
    __device__ __forceinline__ uint64_t key(int i) const { return make_key(score[i], col[i]); }
    __device__ __forceinline__ void put(int i, uint64_t k) { score[i] = key_score(k); col[i] = key_col(k); }
    uint64_t cut;
    int total[2][kWaves];
    float sm[kWaves], ss[kWaves], sw[kWaves]; int sb[kWaves];
};

struct TopK { int cnt = 0; uint64_t thr = 0; bool sorted = true; int turn = 0; };    // the same in every thread; thr: at least k of the keys so far are not below it (0: unknown)

template <int X> __device__ __forceinline__ uint64_t xor_lane64(uint64_t v) { return ((uint64_t)xor_lane<X>((uint32_t)(v >> 32)) << 32) | xor_lane<X>((uint32_t)v); }

// Sorts N * 256 keys descending, key i * 256 + thread in key[i] of that thread: a bitonic network whose strides below 64 are lane exchanges and whose strides
// of 64 and 128 go through sh.best (256 keys are 33 lane steps and 3 of LDS; counting each key's rank instead was 64-bit compares of all with all, 8 us a
// time with four workgroups on a CU).
template <int N> __device__ void sort_keys(Shared& sh, uint64_t (&key)[N]) {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));        // the network's lane masks are made here: kept across the chunks they crowd the scalar registers out
    auto keep = [&](uint64_t& mine, uint64_t other, bool lower, bool down) { mine = ((mine > other) == (lower == down)) ? mine : other; };
    auto lanes = [&](auto X, int size) {
        constexpr int x = decltype(X)::value;
#pragma unroll
        for (int i = 0; i < N; i++) keep(key[i], xor_lane64<x>(key[i]), (t & x) == 0, ((i * kThreads + t) & size) == 0);
    };
#pragma unroll
    for (int size = 2; size <= N * kThreads; size <<= 1) {
        if constexpr (N == 2) { if (size == 2 * kThreads) { const uint64_t a = key[0], b = key[1]; key[0] = a > b ? a : b; key[1] = a > b ? b : a; } }
#pragma unroll
        for (int stride = 128; stride >= 64; stride >>= 1) {
            if (stride > size / 2) continue;
#pragma unroll
            for (int i = 0; i < N; i++) {
                __syncthreads();
                sh.best[t] = key[i];
                __syncthreads();
                keep(key[i], sh.best[t ^ stride], (t & stride) == 0, ((i * kThreads + t) & size) == 0);
            }
        }
        if (size >= 64) lanes(std::integral_constant<int, 32>{}, size);
        if (size >= 32) lanes(std::integral_constant<int, 16>{}, size);
        if (size >= 16) lanes(std::integral_constant<int, 8>{}, size);
        if (size >= 8) lanes(std::integral_constant<int, 4>{}, size);
        if (size >= 4) lanes(std::integral_constant<int, 2>{}, size);
        lanes(std::integral_constant<int, 1>{}, size);
    }
}

// the same for 64 keys in one wave
__device__ __forceinline__ uint64_t sort_wave(uint64_t key) {
    int t = threadIdx.x & 63;
    asm volatile("" : "+v"(t));
    auto step = [&](auto X, int size) {
        constexpr int x = decltype(X)::value;
        const uint64_t other = xor_lane64<x>(key);
        key = ((key > other) == (((t & x) == 0) == ((t & size) == 0))) ? key : other;
    };
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1) {
        if (size >= 64) step(std::integral_constant<int, 32>{}, size);
        if (size >= 32) step(std::integral_constant<int, 16>{}, size);
        if (size >= 16) step(std::integral_constant<int, 8>{}, size);
        if (size >= 8) step(std::integral_constant<int, 4>{}, size);
        if (size >= 4) step(std::integral_constant<int, 2>{}, size);
        step(std::integral_constant<int, 1>{}, size);
    }
    return key;
}

// the candidates 0 .. cnt sorted descending and cut to k
__device__ void compact(Shared& sh, TopK& tk, int k) {
    const int cnt = tk.cnt, t = threadIdx.x;
    __syncthreads();
    if (cnt <= 64) {
        if (t < 64) {
            const uint64_t key = sort_wave(t < cnt ? sh.key(t) : 0);
            if (t < cnt) sh.put(t, key);
        }
        __syncthreads();
    } else if (cnt <= kThreads) {
        uint64_t key[1] = {t < cnt ? sh.key(t) : 0};
        sort_keys<1>(sh, key);
        if (t < k && t < cnt) sh.put(t, key[0]);            // every thread has read its key before the sort's first barrier
        __syncthreads();
    } else if (cnt <= 2 * kThreads) {
        uint64_t key[2] = {sh.key(t), t + kThreads < cnt ? sh.key(t + kThreads) : 0};
        sort_keys<2>(sh, key);
        if (t < k) sh.put(t, key[0]);                       // k <= 128 < 256 < cnt
        __syncthreads();
    } else {                                                // rows whose best columns crowd into few threads: the k best of the first 512, then of those and the next
        for (int from = 0, held = 0; from < cnt; from += 2 * kThreads - held, held = k) {
            uint64_t key[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int p = i * kThreads + t, at = p < held ? p : from + p - held;
                key[i] = at < cnt ? sh.key(at) : 0;
            }
            sort_keys<2>(sh, key);
            if (t < k) sh.put(t, key[0]);                   // the round's keys lie behind the first k or are in registers
            __syncthreads();
        }
    }
    tk.cnt = cnt < k ? cnt : k;
    tk.sorted = true;
    if (cnt >= k) tk.thr = sh.key(k - 1);
}

// Where the wave's candidates go: `take[i]` holds the lanes whose element i is one, `any` says that the wave has one. Returns the workgroup's number of candidates, `before` those of the lower waves.
template <int EPT> __device__ __forceinline__ int count_candidates(Shared& sh, TopK& tk, bool any, const uint64_t (&take)[EPT], int& before) {
    const int wave = threadIdx.x >> 6;
    int mine = 0;
    if (any) {
#pragma unroll
        for (int i = 0; i < EPT; i++) mine += __popcll(take[i]);
    }
    int* total = sh.total[tk.turn ^= 1];          // two in turn: the other's readers have passed this barrier before it is written again
    if ((threadIdx.x & 63) == 0) total[wave] = mine;
    __syncthreads();
    int all = 0;
    before = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) { const int x = total[w]; all += x; before += w < wave ? x : 0; }
    return all;
}

// Adds this chunk's candidates: take[i] holds the lanes whose element i is one (uniform across the wave). Of `chunk`: best() is the thread's largest key (0:
// none), keep(cut, take) drops what lies below cut, score(i) and col(i) are an element. Returns whether the workgroup had any.
template <int EPT, class Chunk>
__device__ __forceinline__ bool add_candidates(Shared& sh, TopK& tk, int k, bool any, uint64_t (&take)[EPT], const Chunk& chunk) {
    const int lane = threadIdx.x & 63;
    int before, c = count_candidates(sh, tk, any, take, before);
    if (c == 0) return false;
    if (tk.cnt + c > kSoft) {
        if (tk.cnt > k) compact(sh, tk, k);
        uint64_t best[1] = {chunk.best()};
        if (k <= kThreads / 8) {
            // quads stand for their threads: the k quads above the bound hold 4 * EPT keys each, and 64 keys sort in one wave
            const uint64_t p = xor_lane64<1>(best[0]), a = best[0] > p ? best[0] : p, q = xor_lane64<2>(a), quad = a > q ? a : q;
            if ((threadIdx.x & 3) == 0) sh.best[threadIdx.x >> 2] = quad;
            __syncthreads();
            if (threadIdx.x < 64) {
                const uint64_t key = sort_wave(sh.best[threadIdx.x]);
                if ((int)threadIdx.x == k - 1) sh.cut = key;
            }
            __syncthreads();
        }
        if (k > kThreads / 8 || sh.cut == 0) {                // the few columns of a row's end crowd into fewer than k quads
            sort_keys<1>(sh, best);
            if ((int)threadIdx.x == k - 1) sh.cut = best[0];
            __syncthreads();
        }
        // sh.cut: the k-th largest, or 0 when fewer than k threads hold any
        // at least k keys are not below it: the bound for what follows, too
        tk.thr = sh.cut > tk.thr ? sh.cut : tk.thr;
        if (any) chunk.keep(tk.thr, take);
        c = count_candidates(sh, tk, any, take, before);
    }
    if (any) {
        int at = tk.cnt + before;
#pragma unroll
        for (int i = 0; i < EPT; i++) {
            if (!take[i]) continue;
            if ((take[i] >> lane) & 1) {
                const int to = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(take[i] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)take[i], (uint32_t)at));
                sh.score[to] = chunk.score(i); sh.col[to] = chunk.col(i);
            }
            at += __popcll(take[i]);
        }
    }
    tk.cnt += c;
    tk.sorted = false;
    if (tk.cnt >= k + kThreads) compact(sh, tk, k);
    return true;
}

template <int X = 1, class F> __device__ __forceinline__ float reduce_wave(float v, F join) {      // over the 64 lanes, always in the same order
    v = join(v, __builtin_bit_cast(float, xor_lane<X>(__builtin_bit_cast(uint32_t, v))));
    if constexpr (X < 32) return reduce_wave<2 * X>(v, join);
    else return v;
}

// a row's statistics from its threads', in every thread
__device__ Stats reduce_stats(Shared& sh, Stats st, float f) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float wave_max = reduce_wave(st.m, [](float a, float b) { return fmaxf(a, b); });
    if (lane == 0) sh.sm[wave] = wave_max;
    __syncthreads();
    float m = sh.sm[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) m = fmaxf(m, sh.sm[w]);
    float s = 0.0f, w = 0.0f;
    if (m > -INFINITY) {
        const float t = (st.m - m) * f, e = exp2_t(t);
        w = (st.w + fmaxf(t, -1e30f) * st.s) * e;            // -inf * 0 would be NaN; a NaN stays in e
        s = st.s * e;
    }
    auto add = [](float a, float b) { return a + b; };
    s = reduce_wave(s, add); w = reduce_wave(w, add);
    const uint64_t bad = __ballot(st.bad != 0);
    if (lane == 0) { sh.ss[wave] = s; sh.sw[wave] = w; sh.sb[wave] = bad != 0; }
    __syncthreads();
    Stats r{m, 0.0f, 0.0f, 0};
#pragma unroll
    for (int i = 0; i < kWaves; i++) { r.s += sh.ss[i]; r.w += sh.sw[i]; r.bad |= sh.sb[i]; }
    return r;
}

template <bool NEG, class T> __device__ __forceinline__ float signed_score(T v) { return NEG ? -(float)v : (float)v; }

// the score of the thread's first target: requested at the start of a row's last kernel, used at its end
struct Target { float score; bool in; };
template <bool NEG, class T> __device__ __forceinline__ Target load_target(const T* x, int count, const int32_t* targets, int t, int n_targets) {
    const int32_t col = t < n_targets ? targets[t] : -1;
    const bool in = col >= 0 && col < count;
    return Target{in ? signed_score<NEG>(x[col]) : 0.0f, in};
}

// a row's outputs from its statistics and its sorted candidates 0 .. cnt
template <bool NEG, class T>
__device__ __forceinline__ void finish_row(const Shared& sh, const Stats& st, int64_t row, const T* x, int count, int cnt, const int32_t* targets, Target mine, int n_targets, int k,
                                           float scale, float* logprobs, float* logsum, float* entropy, int32_t* ids, float* top_logprobs) {
    const bool empty = !st.bad && st.m == -INFINITY;
    const float log_s = st.bad ? __builtin_nanf("") : logf(st.s);
    if (threadIdx.x == 0) {
        logsum[row] = empty ? -INFINITY : st.m * scale + log_s;
        entropy[row] = empty ? 0.0f : log_s - kLn2 * (st.w / st.s);
    }
    for (int t = threadIdx.x; t < n_targets; t += kThreads) {
        if (t >= kThreads) mine = load_target<NEG>(x, count, targets, t, n_targets);
        logprobs[row * n_targets + t] = !empty && mine.in ? (mine.score - st.m) * scale - log_s : -INFINITY;
    }
    for (int i = threadIdx.x; i < k; i += kThreads) {
        const bool has = i < cnt;
        ids[row * k + i] = has ? (int32_t)sh.col[i] : -1;
        top_logprobs[row * k + i] = has ? (sh.score[i] - st.m) * scale - log_s : -INFINITY;
    }
}

// Workgroup (row, split): columns [split * span, ...) of the row's count in chunks of 4096, each thread 16 of them in 16-byte pieces.
template <bool NEG, class T>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const T* __restrict__ scores, int64_t ld, int n, const int32_t* __restrict__ counts, float scale,
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
    TopK tk;
    const int32_t* row_targets = targets + row * n_targets;
    Target target{0.0f, false};
    if (splits == 1) target = load_target<NEG>(x, count, row_targets, threadIdx.x, n_targets);
    const int whole = count / kChunk;
    const T masked = (T)(NEG ? INFINITY : -INFINITY);
    T next[P][V];          // the next chunk is requested before this one is worked on
    auto fetch = [&](int c) {
        const int64_t base = (int64_t)c * kChunk + threadIdx.x * V;
        if (c < whole) {
#pragma unroll
            for (int p = 0; p < P; p++) __builtin_memcpy(next[p], x + base + p * (kThreads * V), 16);
        } else {
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int i = 0; i < V; i++) { const int64_t col = base + p * (kThreads * V) + i; next[p][i] = col < count ? x[col] : masked; }
        }
    };
    int c = split * per;
    if (c < c_end) fetch(c);
    for (; c < c_end; c++) {
        const int base = c * kChunk + threadIdx.x * V;
        float v[kEpt];
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int i = 0; i < V; i++) v[p * V + i] = signed_score<NEG>(next[p][i]);
        if (c + 1 < c_end) fetch(c + 1);
        float top = v[0];
#pragma unroll
        for (int i = 1; i < kEpt; i++) top = fmaxf(top, v[i]);       // leaves NaN out
        const float hi = fmaxf(top, st.m);
        if (hi > -INFINITY) {
            if (hi > st.m) {
                if (st.m > -INFINITY) {
                    const float t = (st.m - hi) * f, e = exp2_t(t);
                    st.w = (st.w + fmaxf(t, -1e30f) * st.s) * e; st.s *= e;
                }
                st.m = hi;
            }
            float s = 0.0f, w = 0.0f;
#pragma unroll
            for (int i = 0; i < kEpt; i++) {
                const float t = (v[i] - hi) * f, e = exp2_t(t);
                s += e; w = __builtin_fmaf(e, fmaxf(t, -1e30f), w);          // a masked entry: t = -inf, e = 0, and 0 * t must be 0; a NaN stays in e
            }
            st.s += s; st.w += w;
        } else {
#pragma unroll
            for (int i = 0; i < kEpt; i++) st.bad |= v[i] != v[i] ? 1 : 0;
        }
        if (k > 0) {
            const float thr = tk.thr ? key_score(tk.thr) : -INFINITY;                         // later columns lose a tie: strictly greater
            uint64_t take[kEpt];
            const bool any = __ballot(top > thr) != 0;
            if (any) {
#pragma unroll
                for (int i = 0; i < kEpt; i++) take[i] = __ballot(v[i] > thr);                 // false for NaN and for -inf
            }
            struct Chunk {
                const float (&v)[kEpt]; float top, thr; uint32_t base;
                static constexpr int offset(int i) { return (i / V) * (kThreads * V) + i % V; }
                __device__ __forceinline__ float score(int i) const { return v[i]; }
                __device__ __forceinline__ uint32_t col(int i) const { return base + offset(i); }
                __device__ __forceinline__ uint64_t best() const {
                    uint32_t at = 0;
#pragma unroll
                    for (int i = kEpt - 1; i >= 0; i--) at = v[i] == top ? offset(i) : at;      // the lowest column of the thread's largest score
                    return top > thr ? make_key(top, base + at) : 0;
                }
                __device__ __forceinline__ void keep(uint64_t cut, uint64_t (&take)[kEpt]) const {
                    const float x = cut ? key_score(cut) : -INFINITY;
                    const uint32_t c = key_col(cut);
#pragma unroll
                    for (int i = 0; i < kEpt; i++) take[i] &= __ballot(v[i] > x) | (__ballot(v[i] == x) & __ballot(col(i) <= c));
                }
            };
            add_candidates(sh, tk, k, any, take, Chunk{v, top, thr, (uint32_t)base});
        }
    }
    if (k > 0 && !tk.sorted) compact(sh, tk, k);
    const int cnt = tk.cnt;
    st = reduce_stats(sh, st, f);
    if (splits == 1) {
        finish_row<NEG>(sh, st, row, x, count, cnt, row_targets, target, n_targets, k, scale, logprobs, logsum, entropy, ids, top_logprobs);
    } else {
        if (threadIdx.x == 0) part_stats[blockIdx.x] = st;
        for (int i = threadIdx.x; i < k; i += kThreads) part_keys[(row * k + i) * splits + split] = i < cnt ? sh.key(i) : 0;
    }
}

// Joins a row's splits. Their keys lie rank by rank: the best of all splits first, then the second best, ... A turn sees every split at least once, so when it has
// no key above the bound no later one has (1 x 1000000, k = 100: 245 splits, 24500 keys, of which two or three turns read 2048 each).
template <bool NEG, class T>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(const T* __restrict__ scores, int64_t ld, int n, const int32_t* __restrict__ counts, float scale,
                                                                 const int32_t* __restrict__ targets, int n_targets, int k, int splits, float* __restrict__ logprobs,
                                                                 float* __restrict__ logsum, float* __restrict__ entropy, int32_t* __restrict__ ids, float* __restrict__ top_logprobs,
                                                                 const Stats* __restrict__ part_stats, const uint64_t* __restrict__ part_keys) {
    __shared__ Shared sh;
    constexpr int E = 8;
    static_assert(kThreads * E >= kGroups);
    const int64_t row = blockIdx.x;
    int count = n;
    if (counts) { count = counts[row]; count = count < 0 ? 0 : (count > n ? n : count); }
    const float f = scale * kLog2e;
    const T* x = scores + row * ld;
    const int32_t* row_targets = targets + row * n_targets;
    const Target target = load_target<NEG>(x, count, row_targets, threadIdx.x, n_targets);
    Stats st{-INFINITY, 0.0f, 0.0f, 0};
    for (int i = threadIdx.x; i < splits; i += kThreads) { const Stats p = part_stats[row * splits + i]; stats_join(st, p.m, p.s, p.w, p.bad, f); }
    TopK tk;
    const int total = splits * k;
    const uint64_t* keys = part_keys + row * total;
    for (int b = 0; b < total; b += kThreads * E) {
        uint64_t q[E];
        uint64_t take[E];
#pragma unroll
        for (int i = 0; i < E; i++) { const int at = b + i * kThreads + (int)threadIdx.x; q[i] = at < total ? keys[at] : 0; }
#pragma unroll
        for (int i = 0; i < E; i++) take[i] = __ballot(q[i] > tk.thr);
        struct Keys {
            const uint64_t (&q)[E];
            __device__ __forceinline__ float score(int i) const { return key_score(q[i]); }
            __device__ __forceinline__ uint32_t col(int i) const { return key_col(q[i]); }
            __device__ __forceinline__ uint64_t best() const {
                uint64_t b = 0;
#pragma unroll
                for (int i = 0; i < E; i++) b = q[i] > b ? q[i] : b;
                return b;
            }
            __device__ __forceinline__ void keep(uint64_t cut, uint64_t (&take)[E]) const {
#pragma unroll
                for (int i = 0; i < E; i++) take[i] &= __ballot(q[i] >= cut);
            }
        };
        if (!add_candidates(sh, tk, k, true, take, Keys{q})) break;
    }
    if (k > 0 && !tk.sorted) compact(sh, tk, k);
    const int cnt = tk.cnt;
    st = reduce_stats(sh, st, f);
    finish_row<NEG>(sh, st, row, x, count, cnt, row_targets, target, n_targets, k, scale, logprobs, logsum, entropy, ids, top_logprobs);
}

int64_t chunk_count(int64_t n) { return std::max<int64_t>(1, ceil_div(n, kChunk)); }
int split_count(int64_t m, int64_t n) {
    const int64_t chunks = chunk_count(n);
    return chunks <= kWhole ? 1 : (int)std::min(chunks, std::max<int64_t>(1, kGroups / m));
}

template <bool NEG, class T> void logprobs_t(hipStream_t s, const LogProbsArgs& a) {
    const float scale = std::fabs(a.scale);
    constexpr int64_t kPiece = (int64_t)1 << 22;        // (a launch has fewer than 2^32 threads)
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
        launch_kernel(logprobs_kernel<NEG, T>, m * splits, kThreads, 0, s, x, a.ld, a.n, counts, scale, targets, a.n_targets, a.k, splits, lp, a.logsum + i, a.entropy + i, ids, tl, ps, pk);
        if (splits > 1)
            launch_kernel(logprobs_join_kernel<NEG, T>, m, kThreads, 0, s, x, a.ld, a.n, counts, scale, targets, a.n_targets, a.k, splits, lp, a.logsum + i, a.entropy + i, ids, tl, ps, pk);
    }
}
}  // namespace

// an upper bound for every call of at most m rows, n columns and k best: m * splits never exceeds min(m * chunks, max(m, kGroups))
size_t logprobs_work_bytes(int64_t m, int64_t n, int32_t k) {
    const int64_t chunks = chunk_count(n);
    if (m <= 0 || chunks <= kWhole) return 0;
    const int64_t parts = std::min(m * chunks, kGroups);
    return (size_t)(round_up((int64_t)sizeof(Stats) * parts, 16) + parts * 8 * k);
}

void launch_logprobs(hipStream_t s, const LogProbsArgs& a) {
    if (a.m <= 0) return;
    auto typed = [&](auto neg) {
        constexpr bool NEG = decltype(neg)::value;
        if (a.dtype == COMET_F32) logprobs_t<NEG, float>(s, a);
        else if (a.dtype == COMET_F16) logprobs_t<NEG, _Float16>(s, a);
        else logprobs_t<NEG, __bf16>(s, a);
    };
    if (a.scale < 0) typed(std::true_type{}); else typed(std::false_type{});
}

}  // namespace comet
