// rows.hip — rows quantised to 8-bit floating point as they are written, and read back.
//
// A block is 128 consecutive values of a row. With A the largest finite |x| of the block, e is the least integer with A * 2^-e <= 448 (the largest
// e4m3 number) and the codes are e4m3(x * 2^-e), rounded to nearest even: multiplying by a power of two is exact, so a code is off by half a step of
// e4m3 and by nothing else (2^-4 of the value; 2^-10 * 2^e below 2^-6 * 2^e). Both directions move each byte once and are
// bound by HBM: 131072 x 768 float32 are written in 120 us (4.2 TB/s; the marking launch before it 6.5 us) and read as bfloat16 in 53 us (5.7 TB/s), 25600 x 768
// scattered rows are read as float32 in 19 us (5.1 TB/s).
#include "fp8.hpp"
#include "lanes.hpp"

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

// A group of 128 / V lanes takes U blocks of a row (V values of 16 bytes per lane and block), so a block is one 512- or 256-byte request and its maximum is a
// reduction inside the group. A workgroup's groups take whole rows, as many as they cover, or one row in turns. The values are requested before the row's
// slot is known.
// DUP: how a slot that is named twice is resolved so that the LAST row with it stays, whole: 0 no two rows can share a slot (consecutive slots), 1 a wave
// looks through the at most 64 slots, 2 mark_kernel has left the winner's number in last[slot].
template <class T, int U> struct WriteShape {
    static constexpr int V = 16 / sizeof(T), L = kFp8Block / V, G = 256 / L;
    static int rows(int nb) { const int c = (nb + U - 1) / U; return c < G ? G / c : 1; }
};
template <class T, int U, int DUP>
__global__ __launch_bounds__(256) void write_kernel(const T* __restrict__ x, int64_t ld, int n, int dim, const int64_t* __restrict__ slots, int64_t first, uint8_t* __restrict__ codes,
                                                    uint8_t* __restrict__ scales, int64_t capacity, int nb, int nb4, int32_t* __restrict__ last, int rows) {
    constexpr int V = WriteShape<T, U>::V, L = WriteShape<T, U>::L, G = WriteShape<T, U>::G;
    __shared__ int64_t slot_of[G];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    const int parts = (nb + U - 1) / U, r = parts < G ? group / parts : 0;
    const int64_t row0 = (int64_t)blockIdx.x * rows, row = row0 + r;
    const bool mine = r < rows && row < n;
    const T* src = x + (mine ? row : 0) * ld;
    float v[U][V];
    auto load = [&](int part) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int col = (part * U + u) * kFp8Block + lane * V;
            if (col + V <= dim) {
                load16<T, V>(src + col, v[u]);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) v[u][i] = col + i < dim ? to_f32(src[col + i]) : 0.0f;
            }
        }
    };
    int part = parts < G ? group % parts : group;
    if (mine) load(part);
    if constexpr (DUP == 1) {
        const int wave = threadIdx.x / 64, l = threadIdx.x % 64;
        for (int i = wave; i < rows && row0 + i < n; i += 4) {
            const int64_t at = row0 + i, slot = slots[at];
            const bool later = at + 1 + l < n && slots[at + 1 + l] == slot;
            const uint64_t any = __ballot(later);
            if (l == 0) slot_of[i] = slot >= 0 && slot < capacity && !any ? slot : -1;
        }
    } else if ((int)threadIdx.x < rows && row0 + threadIdx.x < n) {
        const int64_t at = row0 + threadIdx.x;
        int64_t slot = DUP == 0 ? first + at : slots[at];
        if (slot < 0 || slot >= capacity) slot = -1;
        if constexpr (DUP == 2) {
            // a row that lost reads the winner's number, or the -1 that the winner puts back: never its own
            if (slot >= 0) { if (last[slot] == (int32_t)at) last[slot] = -1; else slot = -1; }
        }
        slot_of[threadIdx.x] = slot;
    }
    __syncthreads();
    if (!mine) return;
    const int64_t slot = slot_of[r];
    if (slot < 0) return;
    uint8_t* dst = codes + slot * ((int64_t)nb * kFp8Block);
    for (; part < parts; part += G) {
        uint32_t packed_scales = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            uint32_t a = 0;                                     // largest finite magnitude: non-negative floats order as their bits
#pragma unroll
            for (int i = 0; i < V; i++) {
                const uint32_t bits = __builtin_bit_cast(uint32_t, v[u][i]) & 0x7FFFFFFFu;
                if (bits >= 0x7F800000u) v[u][i] = __builtin_nanf("");      // e4m3 has no infinity: anything non-finite is held as NaN
                else a = a > bits ? a : bits;
            }
            auto join = [&](uint32_t o) { a = a > o ? a : o; };
            join(xor_lane<1>(a)); join(xor_lane<2>(a)); join(xor_lane<4>(a)); join(xor_lane<8>(a));
            if constexpr (L == 32) join(xor_lane<16>(a));
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
            if (part * U + u < nb) __builtin_memcpy(__builtin_assume_aligned(dst + (part * U + u) * kFp8Block + lane * V, V), w, V);
        }
        if (lane < U && part * U + lane < nb) scales[slot * nb4 + part * U + lane] = (uint8_t)(packed_scales >> (8 * lane));
        if (parts < G) break;
        if (part + G < parts) load(part + G);
    }
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

template <class T, int U> void write_t(hipStream_t s, const Fp8View& v, int32_t* last, const int64_t* slots, int64_t first, const T* x, int64_t ld, int64_t n) {
    const int rows = WriteShape<T, U>::rows(v.nb);
    // a launch has fewer than 2^32 threads (and rows are numbered with 32 bits in `last`); pieces follow each other on the stream, so the last row with a
    // slot still stays
    constexpr int64_t kPiece = (int64_t)1 << 22;
    constexpr int64_t kScan = 64;           // up to this many rows a look through all slots is one load, and the marking launch is saved
    for (int64_t i = 0; i < n; i += kPiece) {
        const int m = (int)std::min(kPiece, n - i);
        const dim3 grid((unsigned)ceil_div(m, rows));
        const T* xi = x + i * ld;
        if (!slots) {
            hipLaunchKernelGGL((write_kernel<T, U, 0>), grid, dim3(256), 0, s, xi, ld, m, v.dim, nullptr, first + i, v.codes, v.scales, v.capacity, v.nb, v.nb4, last, rows);
        } else if (m <= kScan) {
            hipLaunchKernelGGL((write_kernel<T, U, 1>), grid, dim3(256), 0, s, xi, ld, m, v.dim, slots + i, 0, v.codes, v.scales, v.capacity, v.nb, v.nb4, last, rows);
        } else {
            hipLaunchKernelGGL(mark_kernel, dim3((unsigned)ceil_div(m, 256)), dim3(256), 0, s, slots + i, m, v.capacity, last);
            LAUNCH_CHECK();
            hipLaunchKernelGGL((write_kernel<T, U, 2>), grid, dim3(256), 0, s, xi, ld, m, v.dim, slots + i, 0, v.codes, v.scales, v.capacity, v.nb, v.nb4, last, rows);
        }
        LAUNCH_CHECK();
    }
}

template <class T> void read_t(hipStream_t s, const Fp8View& v, const int64_t* slots, int64_t first, T* out, int64_t ld, int64_t n) {
    constexpr int kRows = 256 / (kFp8Block / (16 / (int)sizeof(T)));
    constexpr int64_t kPiece = (int64_t)1 << 24;        // (a launch has fewer than 2^32 threads)
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
    auto blocks = [&](auto u) {
        constexpr int U = decltype(u)::value;
        if (dtype == COMET_F32) write_t<float, U>(s, v, last, slots, first, (const float*)x, ld, n);
        else if (dtype == COMET_F16) write_t<_Float16, U>(s, v, last, slots, first, (const _Float16*)x, ld, n);
        else write_t<__bf16, U>(s, v, last, slots, first, (const __bf16*)x, ld, n);
    };
    // blocks a group: two read a bulk of rows at the rate of a copy (131072 x 768 float32 and back as bfloat16: 175 us, against 219 with one and 189 with four); rows of one
    // and of three blocks leave no group half empty
    if (v.nb == 1) blocks(std::integral_constant<int, 1>{});
    else if (v.nb == 3) blocks(std::integral_constant<int, 3>{});
    else blocks(std::integral_constant<int, 2>{});
}
void launch_fp8_read(hipStream_t s, const Fp8View& v, const int64_t* slots, int64_t first, void* out, int dtype, int64_t ld, int64_t n) {
    if (n <= 0) return;
    if (dtype == COMET_F32) read_t(s, v, slots, first, (float*)out, ld, n);
    else if (dtype == COMET_F16) read_t(s, v, slots, first, (_Float16*)out, ld, n);
    else read_t(s, v, slots, first, (__bf16*)out, ld, n);
}

}  // namespace comet
