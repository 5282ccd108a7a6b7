// rows.hip — rows quantised to 8-bit floating point as they are written, and read back.
//
// A block is 128 consecutive values of a row. With A the largest finite |x| of the block, e is the least integer with A * 2^-e <= 448 (the largest
// e4m3 number) and the codes are e4m3(x * 2^-e), rounded to nearest even: multiplying by a power of two is exact, so a code is off by half a step of
// e4m3 and by nothing else (2^-4 of the value; 2^-10 * 2^e below 2^-6 * 2^e). Both directions move each byte once and are bound by HBM.
#include "fp8.hpp"

namespace comet {
namespace {

template <class T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }

// 16 bytes of a row at an element's alignment (global memory takes unaligned 16-byte accesses: rows of any stride use the same instructions)
template <class T, int V> __device__ __forceinline__ void load16(const T* p, float (&o)[V]) {
    T t[V];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = to_f32(t[i]);
}

__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }   // e in [-126, 127]

// A group of 128 / V lanes takes a row (V values of 16 bytes per lane and block), so a block is one 512- or 256-byte request and its maximum is a
// reduction inside the group. Four blocks are requested before the first is reduced.
// DUP: how a slot that is named twice is resolved so that the LAST row with it stays, whole: 0 no two rows can share a slot (consecutive slots),
// 1 every group looks through the slots behind its own, 2 mark_kernel has left the winner's number in last[slot].
template <class T, int DUP>
__global__ __launch_bounds__(256) void write_kernel(const T* __restrict__ x, int64_t ld, int n, int dim, const int64_t* __restrict__ slots, int64_t first, uint8_t* __restrict__ codes,
                                                    uint8_t* __restrict__ scales, int64_t capacity, int nb, int nb4, int32_t* __restrict__ last) {
    constexpr int V = 16 / sizeof(T), L = kFp8Block / V, U = 4;
    const int lane = threadIdx.x % L;
    const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (row >= n) return;
    const int64_t slot = DUP == 0 && !slots ? first + row : slots[row];
    if (slot < 0 || slot >= capacity) return;
    if constexpr (DUP == 1) {
        bool later = false;
        for (int64_t j = row + 1 + lane; j < n; j += L) later |= slots[j] == slot;
        if ((__ballot(later) >> ((threadIdx.x & 63) / L * L)) & ((1ull << L) - 1)) return;
    }
    if constexpr (DUP == 2) {
        // the winner sets last[slot] back to -1 below: a row that lost reads the winner's number or -1, never its own
        if (last[slot] != (int32_t)row) return;
    }
    const T* src = x + row * ld;
    uint8_t* dst = codes + slot * ((int64_t)nb * kFp8Block);
    for (int b0 = 0; b0 < nb; b0 += U) {
        float v[U][V];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int col = (b0 + u) * kFp8Block + lane * V;
            if (b0 + u < nb && col + V <= dim) {
                load16<T, V>(src + col, v[u]);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) v[u][i] = col + i < dim ? to_f32(src[col + i]) : 0.0f;
            }
        }
        uint32_t packed_scales = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (b0 + u >= nb) break;
            uint32_t a = 0;                                     // largest finite magnitude: non-negative floats order as their bits
#pragma unroll
            for (int i = 0; i < V; i++) {
                const uint32_t bits = __builtin_bit_cast(uint32_t, v[u][i]) & 0x7FFFFFFFu;
                if (bits >= 0x7F800000u) v[u][i] = __builtin_nanf("");      // e4m3 has no infinity: anything non-finite is held as NaN
                else a = a > bits ? a : bits;
            }
#pragma unroll
            for (int m = 1; m < L; m <<= 1) { const uint32_t o = (uint32_t)__shfl_xor((int)a, m, L); a = a > o ? a : o; }
            int e = (int)(a >> 23) - 127 - 8 + ((a & 0x7FFFFFu) > 0x600000u ? 1 : 0);      // A = f * 2^p with f in [1, 2): 448 = 1.75 * 2^8
            e = e < kFp8ExpMin ? kFp8ExpMin : e;
            packed_scales |= (uint32_t)(e + 127) << (8 * u);
            const float inv = pow2(-e);
            uint32_t w[V / 4];
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[u][i] * inv, v[u][i + 1] * inv, 0, false);
                c = __builtin_amdgcn_cvt_pk_fp8_f32(v[u][i + 2] * inv, v[u][i + 3] * inv, c, true);
                w[i / 4] = (uint32_t)c;
            }
            __builtin_memcpy(__builtin_assume_aligned(dst + (b0 + u) * kFp8Block + lane * V, V), w, V);
        }
        if (lane == 0) *(uint32_t*)(scales + slot * nb4 + b0) = packed_scales;
    }
    if constexpr (DUP == 2) { if (lane == 0) last[slot] = -1; }
}

__global__ __launch_bounds__(256) void mark_kernel(const int64_t* __restrict__ slots, int n, int64_t capacity, int32_t* __restrict__ last) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int64_t s = slots[i];
    if (s >= 0 && s < capacity) atomicMax(&last[s], (int)i);
}

template <class T>
__global__ __launch_bounds__(256) void read_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t capacity, int dim, int nb, int nb4,
                                                   const int64_t* __restrict__ slots, int64_t first, T* __restrict__ out, int64_t ld, int64_t n) {
    constexpr int V = 16 / sizeof(T), L = kFp8Block / V, U = 4;
    const int lane = threadIdx.x % L;
    const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (row >= n) return;
    const int64_t slot = slots ? slots[row] : first + row;
    const bool held = slot >= 0 && slot < capacity;
    T* dst = out + row * ld;
    const uint8_t* src = codes + (held ? slot : 0) * ((int64_t)nb * kFp8Block) + lane * V;
    for (int b0 = 0; b0 < nb; b0 += U) {
        uint32_t w[U][V / 4];
        const uint32_t sc = held ? *(const uint32_t*)(scales + slot * nb4 + b0) : 0u;
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int i = 0; i < V / 4; i++) w[u][i] = 0;
            if (held && b0 + u < nb) __builtin_memcpy(w[u], __builtin_assume_aligned(src + (b0 + u) * kFp8Block, V), V);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (b0 + u >= nb) break;
            const float f = __builtin_bit_cast(float, ((sc >> (8 * u)) & 0xFFu) << 23);      // a slot that was never written has byte 0 and zero codes: zeros
            T t[V];
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                typedef float f2 __attribute__((ext_vector_type(2)));
                const f2 p = (i & 2) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w[u][i / 4], true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)w[u][i / 4], false);
                t[i] = (T)(p.x * f); t[i + 1] = (T)(p.y * f);
            }
            const int col = (b0 + u) * kFp8Block + lane * V;
            if (col + V <= dim) {
                __builtin_memcpy(dst + col, t, sizeof(t));
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) if (col + i < dim) dst[col + i] = t[i];
            }
        }
    }
}

template <class T> void write_t(hipStream_t s, const Fp8View& v, int32_t* last, const int64_t* slots, int64_t first, const T* x, int64_t ld, int64_t n) {
    constexpr int kRows = 256 / (kFp8Block / (16 / (int)sizeof(T)));
    // rows are numbered with 32 bits in `last`; pieces follow each other on the stream, so the last row with a slot still stays
    constexpr int64_t kPiece = (int64_t)1 << 30;
    // Looking through the later slots costs n / L loads per row: one launch, right for a handful of rows; a marking launch costs its latency once.
    constexpr int64_t kScan = 64;
    for (int64_t i = 0; i < n; i += kPiece) {
        const int m = (int)std::min(kPiece, n - i);
        const dim3 grid((unsigned)ceil_div(m, kRows));
        const T* xi = x + i * ld;
        if (!slots) {
            hipLaunchKernelGGL((write_kernel<T, 0>), grid, dim3(256), 0, s, xi, ld, m, v.dim, nullptr, first + i, v.codes, v.scales, v.capacity, v.nb, v.nb4, last);
        } else if (m <= kScan) {
            hipLaunchKernelGGL((write_kernel<T, 1>), grid, dim3(256), 0, s, xi, ld, m, v.dim, slots + i, 0, v.codes, v.scales, v.capacity, v.nb, v.nb4, last);
        } else {
            hipLaunchKernelGGL(mark_kernel, dim3((unsigned)ceil_div(m, 256)), dim3(256), 0, s, slots + i, m, v.capacity, last);
            LAUNCH_CHECK();
            hipLaunchKernelGGL((write_kernel<T, 2>), grid, dim3(256), 0, s, xi, ld, m, v.dim, slots + i, 0, v.codes, v.scales, v.capacity, v.nb, v.nb4, last);
        }
        LAUNCH_CHECK();
    }
}

template <class T> void read_t(hipStream_t s, const Fp8View& v, const int64_t* slots, int64_t first, T* out, int64_t ld, int64_t n) {
    constexpr int kRows = 256 / (kFp8Block / (16 / (int)sizeof(T)));
    constexpr int64_t kPiece = (int64_t)1 << 30;
    for (int64_t i = 0; i < n; i += kPiece) {
        const int64_t m = std::min(kPiece, n - i);
        hipLaunchKernelGGL((read_kernel<T>), dim3((unsigned)ceil_div(m, kRows)), dim3(256), 0, s, v.codes, v.scales, v.capacity, v.dim, v.nb, v.nb4,
                           slots ? slots + i : nullptr, first + i, out + i * ld, ld, m);
        LAUNCH_CHECK();
    }
}
}  // namespace

void launch_fp8_write(hipStream_t s, const Fp8View& v, int32_t* last, const int64_t* slots, int64_t first, const void* x, int dtype, int64_t ld, int64_t n) {
    if (n <= 0) return;
    if (dtype == COMET_F32) write_t(s, v, last, slots, first, (const float*)x, ld, n);
    else if (dtype == COMET_F16) write_t(s, v, last, slots, first, (const _Float16*)x, ld, n);
    else write_t(s, v, last, slots, first, (const __bf16*)x, ld, n);
}
void launch_fp8_read(hipStream_t s, const Fp8View& v, const int64_t* slots, int64_t first, void* out, int dtype, int64_t ld, int64_t n) {
    if (n <= 0) return;
    if (dtype == COMET_F32) read_t(s, v, slots, first, (float*)out, ld, n);
    else if (dtype == COMET_F16) read_t(s, v, slots, first, (_Float16*)out, ld, n);
    else read_t(s, v, slots, first, (__bf16*)out, ld, n);
}

}  // namespace comet
