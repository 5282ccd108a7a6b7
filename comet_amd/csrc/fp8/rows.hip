// rows.hip — rows quantised to 8-bit floating point as they are written, and read back.
//
// A block is 128 consecutive values of a row. With A the largest finite |x| of the block, e is the least integer with A * 2^-e <= 448 (the largest
// e4m3 number) and the codes are e4m3(x * 2^-e), rounded to nearest even: multiplying by a power of two is exact, so a code is off by half a step of
// e4m3 and by nothing else (2^-4 of the value; 2^-10 * 2^e below 2^-6 * 2^e). Both directions move each byte once and are
// bound by HBM where rows are wide and many: 131072 x 768 float32 are written in 122 us (4.1 TB/s; the marking launch before it 6.5 us) and read as bfloat16 in
// 53 us (5.7 TB/s), 25600 x 768 scattered rows are read as float32 in 19 us (5.2 TB/s). Narrow rows to scattered slots are bound by accesses, not bytes: a row
// touches `last` three times (mark, look, reset), its codes and its scale, each a line of its own (1000000 x 16 float32: marking 38 us, writing 74). A single row
// is one group's work when it is read and one workgroup's when it is written (1 x 1048576 float32: 1.46 ms read back, 0.36 ms written).
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

template <class T, int U> struct WriteShape {
    static constexpr int V = 16 / sizeof(T), L = kFp8Block / V, G = 256 / L;
    static int rows(int nb) { const int c = (nb + U - 1) / U; return c < G ? G / c : 1; }
};
// What one lane does with its V values of a block: the group's maximum, the exponent, the codes. Returns the exponent's byte.
template <int V, int L> __device__ __forceinline__ uint32_t quantise(float (&v)[V], uint32_t (&w)[V / 4]) {
    uint32_t a = 0;                                     // largest finite magnitude: non-negative floats order as their bits
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t bits = __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu;
        if (bits >= 0x7F800000u) v[i] = __builtin_nanf("");      // e4m3 has no infinity: anything non-finite is held as NaN
        else a = a > bits ? a : bits;
    }
    auto join = [&](uint32_t o) { a = a > o ? a : o; };
    join(xor_lane<1>(a)); join(xor_lane<2>(a));
    if constexpr (L >= 8) join(xor_lane<4>(a));
    if constexpr (L >= 16) join(xor_lane<8>(a));
    if constexpr (L >= 32) join(xor_lane<16>(a));
    int e = (int)(a >> 23) - 127 - 8 + ((a & 0x7FFFFFu) > 0x600000u ? 1 : 0);      // A = f * 2^p with f in [1, 2): 448 = 1.75 * 2^8
    e = e < kFp8ExpMin ? kFp8ExpMin : e;
    const float inv = pow2(-e);
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[i] * inv, v[i + 1] * inv, 0, false);
        c = __builtin_amdgcn_cvt_pk_fp8_f32(v[i + 2] * inv, v[i + 3] * inv, c, true);
        w[i / 4] = (uint32_t)c;
    }
    return (uint32_t)(e + 127);
}
template <class T, int V> __device__ __forceinline__ void load_piece(const T* src, int col, int dim, float (&v)[V]) {
    if (col + V <= dim) {
        load16<T, V>(src + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = col + i < dim ? to_f32(src[col + i]) : 0.0f;
    }
}
// The slots of the workgroup's rows row0 .. row0 + rows, -1 for a row that is not written (outside the store, or a later row has its slot).
// DUP: how a slot that is named twice is resolved so that the LAST row with it stays, whole: 0 no two rows can share a slot (consecutive slots), 1 a wave
// looks through the at most 64 slots, 2 mark_kernel has left the winner's number in last[slot].
template <int DUP>
__device__ __forceinline__ void find_slots(int64_t* slot_of, int64_t row0, int rows, int n, const int64_t* slots, int64_t first, int64_t capacity, int32_t* last) {
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
}
// A group of 128 / V lanes takes U blocks of a row (V values of 16 bytes per lane and block), so a block is one 512- or 256-byte request and its maximum is a
// reduction inside the group. A workgroup's groups take whole rows, as many as they cover, or one row in turns. The values are requested before the row's
// slot is known.
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
        for (int u = 0; u < U; u++) load_piece<T, V>(src, (part * U + u) * kFp8Block + lane * V, dim, v[u]);
    };
    int part = parts < G ? group % parts : group;
    if (mine) load(part);
    find_slots<DUP>(slot_of, row0, rows, n, slots, first, capacity, last);
    if (!mine) return;
    const int64_t slot = slot_of[r];
    if (slot < 0) return;
    uint8_t* dst = codes + slot * ((int64_t)nb * kFp8Block);
    for (; part < parts; part += G) {
        uint32_t packed_scales = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            uint32_t w[V / 4];
            packed_scales |= quantise<V, L>(v[u], w) << (8 * u);
            if (part * U + u < nb) __builtin_memcpy(__builtin_assume_aligned(dst + (part * U + u) * kFp8Block + lane * V, V), w, V);
        }
        if (lane < U && part * U + lane < nb) scales[slot * nb4 + part * U + lane] = (uint8_t)(packed_scales >> (8 * lane));
        if (parts < G) break;
        if (part + G < parts) load(part + G);
    }
}

// Rows of at most one block: groups of L lanes, as few as hold a row's V * L numbers, take U rows each, so that short rows leave no lane idle and a workgroup
// has 32 rows or more (1000000 x 16 float32 and back as float32: 166 us, 1000000 x 64: 237, against 307 and 375 with a block's 32 lanes a row and 8
// rows a workgroup). The padding's codes are zero since the store was made.
template <class T, int L, int DUP>
__global__ __launch_bounds__(256) void write_short_kernel(const T* __restrict__ x, int64_t ld, int n, int dim, const int64_t* __restrict__ slots, int64_t first,
                                                          uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t capacity, int32_t* __restrict__ last) {
    constexpr int V = 16 / sizeof(T), G = 256 / L, U = L > 8 ? L / 8 : 1;
    __shared__ int64_t slot_of[G * U];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    const int64_t row0 = (int64_t)blockIdx.x * (G * U);
    float v[U][V];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t row = row0 + u * G + group;
        load_piece<T, V>(x + (row < n ? row : 0) * ld, lane * V, dim, v[u]);
    }
    find_slots<DUP>(slot_of, row0, G * U, n, slots, first, capacity, last);
#pragma unroll
    for (int u = 0; u < U; u++) {
        uint32_t w[V / 4];
        const uint32_t scale = quantise<V, L>(v[u], w);
        const int64_t slot = row0 + u * G + group < n ? slot_of[u * G + group] : -1;
        if (slot < 0) continue;
        __builtin_memcpy(__builtin_assume_aligned(codes + slot * kFp8Block + lane * V, V), w, V);
        if (lane == 0) scales[slot * 4] = (uint8_t)scale;
    }
}

__global__ __launch_bounds__(256) void mark_kernel(const int64_t* __restrict__ slots, int n, int64_t capacity, int32_t* __restrict__ last) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int64_t s = slots[i];
    if (s >= 0 && s < capacity) atomicMax(&last[s], (int)i);
}

// a lane's V values of a block from their codes and the block's power of two
template <class T, int V> __device__ __forceinline__ void store_piece(T* dst, int col, int dim, const uint32_t (&w)[V / 4], float f) {
    T t[V];
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        const f2 p = (i & 2) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i / 4], true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i / 4], false);
        t[i] = (T)(p.x * f); t[i + 1] = (T)(p.y * f);
    }
    if (col + V <= dim) {
        __builtin_memcpy(dst + col, t, sizeof(t));
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) if (col + i < dim) dst[col + i] = t[i];
    }
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
            store_piece<T, V>(dst, (b0 + u) * kFp8Block + lane * V, dim, w[u], f);
        }
    }
}

// Rows of at most half a block: 2^shift lanes a row, as few as hold it (1000000 x 16 float32: 44 - 48 us, against 110 with a block's lanes a row). Rows of more
// than half a block are read faster by the kernel above (234375 x 128 bfloat16 in 18 - 22 us, against 27). Part of that is how a lane stores: behind the
// early return for col >= dim the compiler stores a lane's first number in front of store_piece's branch, so its 16 bytes leave as two (float32) or four
// (16-bit) stores, where the kernel above has one.
template <class T>
__global__ __launch_bounds__(256) void read_short_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t capacity, int dim, const int64_t* __restrict__ slots,
                                                         int64_t first, T* __restrict__ out, int64_t ld, int64_t n, int shift) {
    constexpr int V = 16 / sizeof(T);
    const int col = (int)(threadIdx.x & ((1u << shift) - 1)) * V;
    const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> shift;
    if (row >= n || col >= dim) return;
    int64_t slot = slots ? slots[row] : first + row;
    const bool held = slot >= 0 && slot < capacity;
    slot = held ? slot : 0;                 // stands in for a slot outside: no branch between the loads
    const uint32_t scale = scales[slot * 4];
    uint32_t w[V / 4];
    __builtin_memcpy(w, __builtin_assume_aligned(codes + slot * kFp8Block + col, V), V);
#pragma unroll
    for (int i = 0; i < V / 4; i++) w[i] = held ? w[i] : 0;
    store_piece<T, V>(out + row * ld, col, dim, w, __builtin_bit_cast(float, scale << 23));
}

// `launch(dup, piece's first row, its rows, their slots, the first one's slot)`: marking where slots may be named twice. A launch has fewer than 2^32 threads (and
// rows are numbered with 32 bits in `last`); pieces follow each other on the stream, so the last row with a slot still stays.
template <class Launch> void write_pieces(hipStream_t s, const Fp8View& v, int32_t* last, const int64_t* slots, int64_t first, int64_t n, Launch launch) {
    constexpr int64_t kPiece = (int64_t)1 << 22;
    constexpr int64_t kScan = 64;           // up to this many rows a look through all slots is one load, and the marking launch is saved
    for (int64_t i = 0; i < n; i += kPiece) {
        const int m = (int)std::min(kPiece, n - i);
        if (!slots) {
            launch(std::integral_constant<int, 0>{}, i, m, nullptr, first + i);
        } else if (m <= kScan) {
            launch(std::integral_constant<int, 1>{}, i, m, slots + i, (int64_t)0);
        } else {
            launch_kernel(mark_kernel, ceil_div(m, 256), 256, 0, s, slots + i, m, v.capacity, last);
            launch(std::integral_constant<int, 2>{}, i, m, slots + i, (int64_t)0);
        }
    }
}

template <class T, int U> void write_t(hipStream_t s, const Fp8View& v, int32_t* last, const int64_t* slots, int64_t first, const T* x, int64_t ld, int64_t n) {
    const int rows = WriteShape<T, U>::rows(v.nb);
    write_pieces(s, v, last, slots, first, n, [&](auto dup, int64_t i, int m, const int64_t* slots_i, int64_t first_i) {
        launch_kernel(write_kernel<T, U, decltype(dup)::value>, ceil_div(m, rows), 256, 0, s, x + i * ld, ld, m, v.dim, slots_i, first_i, v.codes, v.scales, v.capacity, v.nb, v.nb4, last,
                      rows);
    });
}
template <class T, int L> void write_short_t(hipStream_t s, const Fp8View& v, int32_t* last, const int64_t* slots, int64_t first, const T* x, int64_t ld, int64_t n) {
    constexpr int rows = 256 / L * (L > 8 ? L / 8 : 1);
    write_pieces(s, v, last, slots, first, n, [&](auto dup, int64_t i, int m, const int64_t* slots_i, int64_t first_i) {
        launch_kernel(write_short_kernel<T, L, decltype(dup)::value>, ceil_div(m, rows), 256, 0, s, x + i * ld, ld, m, v.dim, slots_i, first_i, v.codes, v.scales, v.capacity, last);
    });
}

template <class T> void read_t(hipStream_t s, const Fp8View& v, const int64_t* slots, int64_t first, T* out, int64_t ld, int64_t n) {
    constexpr int kRows = 256 / (kFp8Block / (16 / (int)sizeof(T)));
    constexpr int64_t kPiece = (int64_t)1 << 24;        // (a launch has fewer than 2^32 threads)
    int shift = 0;
    while ((16 / (int)sizeof(T)) << shift < v.dim && shift < 5) shift++;
    for (int64_t i = 0; i < n; i += kPiece) {
        const int64_t m = std::min(kPiece, n - i);
        const int64_t* slots_i = slots ? slots + i : nullptr;
        if (v.dim <= kFp8Block / 2)
            launch_kernel(read_short_kernel<T>, ceil_div(m << shift, 256), 256, 0, s, v.codes, v.scales, v.capacity, v.dim, slots_i, first + i, out + i * ld, ld, m, shift);
        else
            launch_kernel(read_kernel<T>, ceil_div(m, kRows), 256, 0, s, v.codes, v.scales, v.capacity, v.dim, v.nb, v.nb4, slots_i, first + i, out + i * ld, ld, m);
    }
}
}  // namespace

void launch_fp8_write(hipStream_t s, const Fp8View& v, int32_t* last, const int64_t* slots, int64_t first, const void* x, int dtype, int64_t ld, int64_t n) {
    if (n <= 0) return;
    auto typed = [&](auto f) {
        if (dtype == COMET_F32) f((const float*)x);
        else if (dtype == COMET_F16) f((const _Float16*)x);
        else f((const __bf16*)x);
    };
    auto blocks = [&](auto u) { typed([&](auto* p) { write_t<std::remove_cv_t<std::remove_pointer_t<decltype(p)>>, decltype(u)::value>(s, v, last, slots, first, p, ld, n); }); };
    auto lanes = [&](auto l) {
        typed([&](auto* p) {
            using T = std::remove_cv_t<std::remove_pointer_t<decltype(p)>>;
            if constexpr (decltype(l)::value * (16 / sizeof(T)) <= kFp8Block) write_short_t<T, decltype(l)::value>(s, v, last, slots, first, p, ld, n);
        });
    };
    const int need = (int)ceil_div(v.dim, 16 / (int)dtype_size(dtype));
    if (v.nb == 1) {
        if (need <= 4) lanes(std::integral_constant<int, 4>{});
        else if (need <= 8) lanes(std::integral_constant<int, 8>{});
        else if (need <= 16) lanes(std::integral_constant<int, 16>{});
        else lanes(std::integral_constant<int, 32>{});
        return;
    }
    // Blocks a group takes: two, and three for rows of three. Written and read back as bfloat16, 100 million numbers in rows of 2 / 3 / 5 / 6 / 7 / 9 / 16 blocks, us:
    //   float32   two: 197 / 196 / 186 / 174 / 176 / 187 / 179   three: 205 / 183 / 187 / 176 / 176 / 176 / 188   one: 212 / 228 / 246 / 218 / 200 / 188 / 177
    //   bfloat16  two: 167 / 167 / 159 / 154 / 151 / 153 / 161   three: 171 / 162 / 161 / 157 / 158 / 155 / 161   one: 171 / 165 / 159 / 173 / 162 / 195 / 151
    // Rows of 300 numbers, whose third block is short: two 271 and 234, three 219 and 200. Other odd counts leave a smaller part of their groups empty and gain
    // nothing that both types share; four blocks were slower than two nearly everywhere (768 wide: 188 and 164).
    if (v.nb == 3) blocks(std::integral_constant<int, 3>{});
    else blocks(std::integral_constant<int, 2>{});
}
void launch_fp8_read(hipStream_t s, const Fp8View& v, const int64_t* slots, int64_t first, void* out, int dtype, int64_t ld, int64_t n) {
    if (n <= 0) return;
    if (dtype == COMET_F32) read_t(s, v, slots, first, (float*)out, ld, n);
    else if (dtype == COMET_F16) read_t(s, v, slots, first, (_Float16*)out, ld, n);
    else read_t(s, v, slots, first, (__bf16*)out, ld, n);
}

}  // namespace comet
