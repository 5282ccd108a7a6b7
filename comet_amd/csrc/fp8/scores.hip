// scores.hip — the matrix product of queries with stored rows, both in 8-bit floating point with a power-of-two scale per block of 128.
//
//   S[i][j] = sum over blocks b of 2^(eq[i][b] + er[j][b]) * sum_t q[i][128 b + t] * r[j][128 b + t]
//
// The products run on v_mfma_f32_16x16x32_bf16: code * 2^e is a bfloat16 number (4 significant bits, the exponent's range is float32's), so
// v_cvt_scalef32_pk_bf16_fp8 turns two codes and their block's scale into two exact operands, products are exact and sums are float32. The 8-bit
// instructions (v_mfma_f32_16x16x32_fp8_fp8 and v_mfma_scale_f32_16x16x128_f8f6f4, twice the rate) are not used: they align each eight products to the
// largest of them and cut what lies 13 bits below it; on codes over the whole range sums came out 2^-14.8 of sum |q r| off, where this form gave 2^-23.
//
// Queries are the first operand, rows the second: lane l of an accumulator holds queries 4 * (l / 16) + i, i = 0 .. 3, and one row. The four row operands of a wave
// take the rows 4 c + t, t = 0 .. 3, for c = l % 16: a lane then holds four consecutive rows of a query, and a store instruction writes 64 consecutive
// scores of four queries (a layout with 16 scores of sixteen queries per instruction stored 256 x 1M scores 45 us slower).
//
// The order of k inside a block is free as long as both operands use the same one (a block has one scale), so lane l takes row l % 16 and the 16-byte
// pieces l / 16 and 4 + l / 16 of its 128: every load instruction covers 64 consecutive bytes of 16 rows.
//
// What bounds it: one query reads the rows at 5.6 TB/s (1 x 1M x 768: 139 us). 256 x 1M x 768 in float32 (407 - 432 us from one card to another) moves 1.8 GB
// at 4.2 - 4.4 TB/s, more than half of it written. Long rows run at the rate of the card's matrix units under load: 2048 x 32768 x 4096 at 1.29 - 1.37 PFLOP/s,
// as fast as a library product of bfloat16 rows (8192^3: 1.37 - 1.40); leaving the conversions out changes nothing there (429 us against 425 on one card), never
// filling a buffer again 366. 2047 x 30011 x 2000 (206 - 220 us, 1.1 - 1.2 PFLOP/s) adds what a tile costs besides its products, about 5 us a round of the chip
// in which all tiles are stored at once, and 944 tiles in 3.7 rounds. Small stores of long rows are bound by latency: a wave walks its 64 rows' blocks one after
// the other (1 x 1000 x 2048: 19 us in the kernel, 32 x 1000 x 2048: 15). A row narrower than a block costs what a whole block costs, in bytes and in products
// (1 x 1M: 22 us for 16 numbers a row as for 128; 256 x 1M x 16: 239 us, most of it the scores' 1 GB).
// Measured and left out: the next block's fill in front of a tile's stores, behind a barrier of its own (430 us for 256 x 1M x 768, against 413), operands read
// one step ahead with a single barrier late in a block (441), a fixed order with a conversion or two between matrix instructions (421, and registers spill for
// 16-bit scores), conversion once a workgroup into bfloat16 LDS tiles (459), workgroups started apart so that their stores do not meet (408 - 418).
#include "fp8.hpp"

namespace comet {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

__device__ __forceinline__ v8i load_block(const uint8_t* p) {      // p: the lane's first 16 bytes of a block
    const v4i a = *(const v4i*)p, b = *(const v4i*)(p + 64);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// byte `u` of a dword of scales as the power of two it stands for
__device__ __forceinline__ float scale_of(uint32_t scales, int u) { return __builtin_bit_cast(float, ((scales >> (8 * u)) & 0xFFu) << 23); }
// eight of a lane's 32 codes of a block (two dwords) as the operand of one matrix instruction
__device__ __forceinline__ v8b widen(int lo, int hi, float scale) {
    const v2b a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, scale, true);
    const v2b c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, scale, true);
    return v8b{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// four consecutive scores of one query; the only rounding behind the float32 sums
template <class T> __device__ __forceinline__ void store4(T* row, int64_t j, int64_t n, v4f v) {
    T o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = (T)v[i];
    if (j + 4 <= n) {
        __builtin_memcpy(row + j, o, sizeof(o));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) if (j + i < n) row[j + i] = o[i];
    }
}

// Up to four queries: the stored rows stream once through the registers, each wave 64 rows against an operand of queries whose blocks come out of the caches
// (1 x 1M x 768: 139 us, 5.6 TB/s, against 149 with the smallest tile below; 16 queries: 184 against 175). Two blocks in flight or one ahead in registers
// were no faster for 1M rows (140 and 145 us); where latency counts, in stores of few rows, they were not tried.
constexpr int kStreamQueries = 4;
template <class T>
__global__ __launch_bounds__(256) void scores_stream_kernel(const uint8_t* __restrict__ qc, const uint8_t* __restrict__ qs, int m, const uint8_t* __restrict__ rc,
                                                            const uint8_t* __restrict__ rs, int n, int nb, int nb4, T* __restrict__ out, int64_t ld) {
    constexpr int RT = 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n0 = ((int64_t)blockIdx.x * 4 + wave) * (RT * 16);
    if (n0 >= n) return;
    const int64_t row_bytes = (int64_t)nb * kFp8Block;
    const uint8_t *rp[RT], *rsp[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {          // rows past the end read the last one: its products go nowhere
        int64_t r = n0 + (lane & 15) * 4 + t;
        r = r < n ? r : n - 1;
        rp[t] = rc + r * row_bytes + (lane >> 4) * 16; rsp[t] = rs + r * nb4;
    }
    const int q0 = (lane & 15) < m ? lane & 15 : m - 1;
    const uint8_t *qp = qc + q0 * row_bytes + (lane >> 4) * 16, *qsp = qs + q0 * nb4;
    v4f acc[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) acc[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    for (int b0 = 0; b0 < nb; b0 += 4) {
        uint32_t sr[RT];
#pragma unroll
        for (int t = 0; t < RT; t++) sr[t] = *(const uint32_t*)(rsp[t] + b0);
        const uint32_t sq = *(const uint32_t*)(qsp + b0);
        const int u_end = nb - b0 < 4 ? nb - b0 : 4;
        for (int u = 0; u < u_end; u++) {
            const int64_t off = (int64_t)(b0 + u) * kFp8Block;
            v8i r[RT];
#pragma unroll
            for (int t = 0; t < RT; t++) r[t] = load_block(rp[t] + off);
            const v8i q = load_block(qp + off);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const v8b qb = widen(q[2 * w], q[2 * w + 1], scale_of(sq, u));
#pragma unroll
                for (int t = 0; t < RT; t++) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qb, widen(r[t][2 * w], r[t][2 * w + 1], scale_of(sr[t], u)), acc[t], 0, 0, 0);
            }
        }
    }
    if (lane >= 16) return;                 // the other lanes hold queries 4 and up
#pragma unroll
    for (int i = 0; i < 4; i++) if (i < m) store4(out + i * ld, n0 + lane * 4, n, v4f{acc[0][i], acc[1][i], acc[2][i], acc[3][i]});
}

// More queries: a workgroup of WAVES waves walks tiles of BM queries x BN rows, block by block, through two LDS buffers that the memory pipe fills one block
// ahead, across tiles: the next tile's first block arrives while this one is finished and stored. A wave multiplies QT * 16 queries with 64 rows. One buffer
// holds the codes of a block (queries, then rows: 128 bytes each) and the rows' and queries' dword of scales. 16-byte piece c of code row r lies at place
// c ^ (r & 7), so that the sixteen rows of an operand read fall on all banks (the fill permutes its global addresses, not its LDS ones).
template <int QT, int WQ, int WAVES> struct TileShape {
    static constexpr int BM = WQ * QT * 16, BN = WAVES / WQ * 64, rows = BM + BN, codes = rows * kFp8Block, stage = codes + WAVES * 256;
    static constexpr int FQ = BM / (8 * WAVES), FR = BN / (8 * WAVES);      // fill instructions a wave issues per block: 8 code rows each (and one for scales)
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && rows <= WAVES * 64, "the waves share the fills evenly");
};

// The fills are asm statements: around the compiler's own form of them every LDS read that follows would wait for the fill just issued (it cannot tell the
// buffers apart). The waits are written out where a buffer changes hands. No register outputs. The LDS address of the wave's part is an operand in M0, so
// the compiler knows what M0 holds; the s_nop are the five wait states between a vector instruction that wrote a scalar register and a load that takes it.
__device__ __forceinline__ void fill16(const uint8_t* base /* uniform */, uint32_t offset, uint32_t lds /* uniform */) {
    const uint64_t b = (uint64_t)base;
    const uint64_t sb = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)b);
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(offset), "s"(sb), "{m0}"(__builtin_amdgcn_readfirstlane((int)lds)) : "memory");
}
__device__ __forceinline__ void fill4(const uint8_t* address, uint32_t lds /* uniform */) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, off" :: "v"(address), "{m0}"(__builtin_amdgcn_readfirstlane((int)lds)) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p; }
// All but the newest N global accesses of the wave are done, and its LDS reads have returned: the barrier behind this hands the buffer they read to the other
// waves' fills, which the compiler does not see, so it would not have to wait for them here.
template <int N> __device__ __forceinline__ void wait_buffers() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory"); }

template <class T, int QT, int WQ, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void scores_tile_kernel(const uint8_t* __restrict__ qc, const uint8_t* __restrict__ qs, int m, const uint8_t* __restrict__ rc,
                                                                      const uint8_t* __restrict__ rs, int n, int nb, int nb4, T* __restrict__ out, int64_t ld, int m_tiles, int n_tiles) {
    using Shape = TileShape<QT, WQ, WAVES>;
    extern __shared__ __align__(16) uint8_t lds[];
    constexpr int RT = 4, BM = Shape::BM, BN = Shape::BN, FQ = Shape::FQ, FR = Shape::FR;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wq = (wave % WQ) * QT * 16, wr = (wave / WQ) * RT * 16;
    const int64_t row_bytes = (int64_t)nb * kFp8Block;
    // Workgroups go to the eight XCDs in turn; each XCD takes a contiguous run of the tiles, queries fastest, dealt to its workgroups in turn: a row tile is
    // read into one L2, by neighbours at about the same time.
    const int tiles = m_tiles * n_tiles, per = (tiles + 7) / 8, xcd = (int)(blockIdx.x & 7), groups = (int)(gridDim.x >> 3);
    const int t0 = xcd * per + (int)(blockIdx.x >> 3), t_end = min(tiles, (xcd + 1) * per);
    if (t0 >= t_end) return;
    const int steps = ((t_end - t0 - 1) / groups + 1) * nb;
    const uint32_t l0 = lds_address(lds);

    // the tile being filled: a lane's byte offsets from the first query / row, and its scale dword's address
    int f_tile = t0, f_b = 0, f_stage = 0;
    const uint8_t *fq_base = nullptr, *fr_base = nullptr, *f_scale = nullptr;
    uint32_t fq[FQ], fr[FR];
    auto row_at = [](int place) { return (place & ~63) + (place & 15) * 4 + ((place >> 4) & 3); };
    auto fill_tile = [&] {
        const int64_t m0 = (int64_t)(f_tile % m_tiles) * BM, n0 = (int64_t)(f_tile / m_tiles) * BN;
        fq_base = qc + m0 * row_bytes; fr_base = rc + n0 * row_bytes;
        const uint32_t piece = ((lane & 7) ^ (lane >> 3)) * 16;
        const int last_q = (int)min((int64_t)BM, m - m0) - 1, last_r = (int)min((int64_t)BN, n - n0) - 1;       // rows past the end read the last one: their products go nowhere
#pragma unroll
        for (int i = 0; i < FQ; i++) fq[i] = (uint32_t)(min((i * WAVES + wave) * 8 + (lane >> 3), last_q) * row_bytes) + piece;
#pragma unroll
        for (int i = 0; i < FR; i++) fr[i] = (uint32_t)(min(row_at((i * WAVES + wave) * 8 + (lane >> 3)), last_r) * row_bytes) + piece;
        const int r = (int)threadIdx.x;
        f_scale = r < BM ? qs + (m0 + min(r, last_q)) * nb4 : rs + (n0 + min(row_at(r - BM), last_r)) * nb4;
    };
    auto fill = [&] {
        const uint32_t to = l0 + f_stage * Shape::stage;
#pragma unroll
        for (int i = 0; i < FQ; i++) fill16(fq_base + f_b * kFp8Block, fq[i], to + (i * WAVES + wave) * 1024);
#pragma unroll
        for (int i = 0; i < FR; i++) fill16(fr_base + f_b * kFp8Block, fr[i], to + BM * kFp8Block + (i * WAVES + wave) * 1024);
        fill4(f_scale + (f_b & ~3), to + Shape::codes + wave * 256);
        f_stage ^= 1;
        if (++f_b == nb) { f_b = 0; f_tile += groups; if (f_tile < t_end) fill_tile(); }
    };
    fill_tile();
    fill();

    v4f acc[RT][QT];
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int v = 0; v < QT; v++) acc[t][v] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    int tile = t0, b = 0, stage = 0;
    bool stored = false;            // the step before stored a tile that lay inside the matrix: QT * 4 store instructions a wave
    for (int step = 0; step < steps; step++) {
        // Block `step` has arrived when nothing is left that was issued before its fill or in it: behind it came only such a tile's stores, and a tile at the
        // edge, whose number of stores differs from wave to wave, is waited for with them.
        if (stored) wait_buffers<QT * 4>();
        else wait_buffers<0>();
        stored = false;
        __builtin_amdgcn_s_barrier();       // ... for every wave, and every wave is done with the buffer that is filled next
        asm volatile("" ::: "memory");
        const uint8_t* buf = lds + stage * Shape::stage;
        float sr[RT], sq[QT];
#pragma unroll
        for (int t = 0; t < RT; t++) sr[t] = __builtin_bit_cast(float, (uint32_t)buf[Shape::codes + (BM + wr + t * 16 + (lane & 15)) * 4 + (b & 3)] << 23);
#pragma unroll
        for (int v = 0; v < QT; v++) sq[v] = __builtin_bit_cast(float, (uint32_t)buf[Shape::codes + (wq + v * 16 + (lane & 15)) * 4 + (b & 3)] << 23);
#pragma unroll
        for (int h = 0; h < 2; h++) {       // the lane's two 16-byte pieces of each row
            auto piece = [&](int r) { return *(const v4i*)(buf + r * kFp8Block + ((((lane >> 4) + 4 * h) ^ (r & 7)) * 16)); };
            v4i r[RT], q[QT];
#pragma unroll
            for (int t = 0; t < RT; t++) r[t] = piece(BM + wr + t * 16 + (lane & 15));
#pragma unroll
            for (int v = 0; v < QT; v++) q[v] = piece(wq + v * 16 + (lane & 15));
            if (h == 0 && step + 1 < steps) fill();        // behind the first LDS reads: these are waited for, the fill is not
#pragma unroll
            for (int w = 0; w < 2; w++) {
                v8b rb[RT];
#pragma unroll
                for (int t = 0; t < RT; t++) rb[t] = widen(r[t][2 * w], r[t][2 * w + 1], sr[t]);
#pragma unroll
                for (int v = 0; v < QT; v++) {
                    const v8b qb = widen(q[v][2 * w], q[v][2 * w + 1], sq[v]);
#pragma unroll
                    for (int t = 0; t < RT; t++) acc[t][v] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qb, rb[t], acc[t][v], 0, 0, 0);
                }
            }
        }
        stage ^= 1;
        if (++b == nb) {
            const int64_t m0 = (int64_t)(tile % m_tiles) * BM, n0 = (int64_t)(tile / m_tiles) * BN;
            const int64_t q0 = m0 + wq + (lane >> 4) * 4, j = n0 + wr + (lane & 15) * 4;
            if (m0 + BM <= m && n0 + BN <= n) {
                T* to = out + q0 * ld + j;
#pragma unroll
                for (int v = 0; v < QT; v++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        T o[4];
#pragma unroll
                        for (int t = 0; t < 4; t++) o[t] = (T)acc[t][v][i];
                        __builtin_memcpy(to + (v * 16 + i) * ld, o, sizeof(o));
                    }
                stored = true;
            } else {
#pragma unroll
                for (int v = 0; v < QT; v++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int64_t q = q0 + v * 16 + i;
                        if (q < m) store4(out + q * ld, j, n, v4f{acc[0][v][i], acc[1][v][i], acc[2][v][i], acc[3][v][i]});
                    }
            }
#pragma unroll
            for (int t = 0; t < RT; t++)
#pragma unroll
                for (int v = 0; v < QT; v++) acc[t][v] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            b = 0; tile += groups;
        }
    }
}

template <class T, int QT, int WQ, int WAVES>
void launch_tiles(hipStream_t s, const uint8_t* qc, const uint8_t* qs, int m, const uint8_t* rc, const uint8_t* rs, int n, int nb, int nb4, T* out, int64_t ld) {
    using Shape = TileShape<QT, WQ, WAVES>;
    constexpr int bytes = 2 * Shape::stage, per_cu = 8 / WAVES;      // two waves a SIMD
    static_assert(bytes * per_cu <= 160 * 1024, "LDS of a CU");
    auto kernel = scores_tile_kernel<T, QT, WQ, WAVES>;
    HIP_CHECK(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    const int mt = (int)ceil_div(m, Shape::BM), nt = (int)ceil_div(n, Shape::BN);
    const int64_t groups = std::min<int64_t>(256 * per_cu, round_up((int64_t)mt * nt, 8));
    launch_kernel(kernel, groups, WAVES * 64, bytes, s, qc, qs, m, rc, rs, n, nb, nb4, out, ld, mt, nt);
}

// Which tile: the fewest rounds of the chip (256 tiles of 256 x 256, 512 of the smaller ones, two a CU), each weighted with its measured time: a round of the
// large tiles 1, of 128 x 128 0.56, of 64 x 128 0.38. The large ones spend least on LDS reads and conversions for a product (256 x 1M x 768: 414 us, against
// 471 and 618), the small ones leave less of the chip idle when there are few (2048 x 2048 x 2048: 33 us, against 35 and 58) and waste least on few queries
// (64 x 1M x 768: 210 us, against 228 and 352).
enum class Tile { large, middle, small };
Tile pick_tile(int64_t m, int64_t n) {
    auto rounds = [&](int64_t bm, int64_t bn, int64_t fit) { return (double)ceil_div(ceil_div(m, bm) * ceil_div(n, bn), fit); };
    const double large = rounds(256, 256, 256), middle = 0.56 * rounds(128, 128, 512), small = 0.38 * rounds(64, 128, 512);
    return small <= middle && small <= large ? Tile::small : middle <= large ? Tile::middle : Tile::large;
}

template <class T> void scores_t(hipStream_t s, const Fp8View& q, int64_t q_first, int64_t m, const Fp8View& r, int64_t first, int64_t n, T* out, int64_t ld) {
    constexpr int64_t kPieceN = (int64_t)1 << 24, kPieceM = (int64_t)1 << 16;      // a launch's tile numbers fit 32 bits
    for (int64_t i = 0; i < m; i += kPieceM) for (int64_t j = 0; j < n; j += kPieceN) {
        const int mi = (int)std::min(kPieceM, m - i), nj = (int)std::min(kPieceN, n - j);
        const uint8_t *qc = q.codes + (q_first + i) * q.row_bytes(), *qs = q.scales + (q_first + i) * q.nb4;
        const uint8_t *rc = r.codes + (first + j) * r.row_bytes(), *rs = r.scales + (first + j) * r.nb4;
        T* o = out + i * ld + j;
        if (mi <= kStreamQueries) launch_kernel(scores_stream_kernel<T>, ceil_div(nj, 256), 256, 0, s, qc, qs, mi, rc, rs, nj, r.nb, r.nb4, o, ld);
        else switch (pick_tile(mi, nj)) {
            case Tile::large: launch_tiles<T, 8, 2, 8>(s, qc, qs, mi, rc, rs, nj, r.nb, r.nb4, o, ld); break;
            case Tile::middle: launch_tiles<T, 4, 2, 4>(s, qc, qs, mi, rc, rs, nj, r.nb, r.nb4, o, ld); break;
            case Tile::small: launch_tiles<T, 2, 2, 4>(s, qc, qs, mi, rc, rs, nj, r.nb, r.nb4, o, ld); break;
        }
    }
}
}  // namespace

void launch_fp8_scores(hipStream_t s, const Fp8View& q, int64_t q_first, int64_t m, const Fp8View& r, int64_t first, int64_t n, void* out, int dtype, int64_t ld) {
    if (m <= 0 || n <= 0) return;
    if (dtype == COMET_F32) scores_t(s, q, q_first, m, r, first, n, (float*)out, ld);
    else if (dtype == COMET_F16) scores_t(s, q, q_first, m, r, first, n, (_Float16*)out, ld);
    else scores_t(s, q, q_first, m, r, first, n, (__bf16*)out, ld);
}

}  // namespace comet
