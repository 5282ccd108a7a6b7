// scores.hip — the matrix product of queries with stored rows, both in 8-bit floating point with a power-of-two scale per block of 128.
//
//   S[i][j] = sum over blocks b of 2^(eq[i][b] + er[j][b]) * sum_t q[i][128 b + t] * r[j][128 b + t]
//
// The products run on v_mfma_f32_16x16x32_bf16: code * 2^e is a bfloat16 number (4 significant bits, the exponent's range is float32's), so
// v_cvt_scalef32_pk_bf16_fp8 turns two codes and their block's scale into two exact operands, products are exact and sums are float32. The 8-bit
// instructions (v_mfma_f32_16x16x32_fp8_fp8 and v_mfma_scale_f32_16x16x128_f8f6f4, twice the rate) are not used: they align each eight products to the
// largest of them and cut what lies 13 bits below it; on codes over the whole range sums came out 2^-14.8 of sum |q r| off, where this form gave 2^-23.
//
// The order of k inside a block is free as long as both operands use the same one (a block has one scale), so lane l takes row l % 16 and the 16-byte
// pieces l / 16 and 4 + l / 16 of its 128: every load instruction covers 64 consecutive bytes of 16 rows.
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

// Few queries: the stored rows stream once through the registers, each wave 64 rows (4 tiles of 16) against MT tiles of 16 queries, whose blocks come
// out of the caches. Accumulator element i of lane l: row 4 * (l / 16) + i of its tile, query l % 16.
template <class T, int MT>
__global__ __launch_bounds__(256) void scores_stream_kernel(const uint8_t* __restrict__ qc, const uint8_t* __restrict__ qs, int m, const uint8_t* __restrict__ rc,
                                                            const uint8_t* __restrict__ rs, int n, int nb, int nb4, T* __restrict__ out, int64_t ld, int m_tiles) {
    constexpr int RT = 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int mt = (int)(blockIdx.x % (unsigned)m_tiles), nt = (int)(blockIdx.x / (unsigned)m_tiles);
    const int64_t n0 = ((int64_t)nt * 4 + wave) * (RT * 16);
    if (n0 >= n) return;
    const int m0 = mt * MT * 16;
    const int64_t row_bytes = (int64_t)nb * kFp8Block;
    const uint8_t *rp[RT], *rsp[RT], *qp[MT], *qsp[MT];
#pragma unroll
    for (int t = 0; t < RT; t++) {          // rows past the end read the last one: its products go nowhere
        int64_t r = n0 + t * 16 + (lane & 15);
        r = r < n ? r : n - 1;
        rp[t] = rc + r * row_bytes + (lane >> 4) * 16; rsp[t] = rs + r * nb4;
    }
#pragma unroll
    for (int t = 0; t < MT; t++) {
        int64_t q = m0 + t * 16 + (lane & 15);
        q = q < m ? q : m - 1;
        qp[t] = qc + q * row_bytes + (lane >> 4) * 16; qsp[t] = qs + q * nb4;
    }
    v4f acc[RT][MT];
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int u = 0; u < MT; u++) acc[t][u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    for (int b0 = 0; b0 < nb; b0 += 4) {
        uint32_t sr[RT], sq[MT];
#pragma unroll
        for (int t = 0; t < RT; t++) sr[t] = *(const uint32_t*)(rsp[t] + b0);
#pragma unroll
        for (int t = 0; t < MT; t++) sq[t] = *(const uint32_t*)(qsp[t] + b0);
        const int u_end = nb - b0 < 4 ? nb - b0 : 4;
        for (int u = 0; u < u_end; u++) {
            const int64_t off = (int64_t)(b0 + u) * kFp8Block;
            v8i r[RT], q[MT];
#pragma unroll
            for (int t = 0; t < RT; t++) r[t] = load_block(rp[t] + off);
#pragma unroll
            for (int t = 0; t < MT; t++) q[t] = load_block(qp[t] + off);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                v8b qb[MT];
#pragma unroll
                for (int v = 0; v < MT; v++) qb[v] = widen(q[v][2 * w], q[v][2 * w + 1], scale_of(sq[v], u));
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const v8b rb = widen(r[t][2 * w], r[t][2 * w + 1], scale_of(sr[t], u));
#pragma unroll
                    for (int v = 0; v < MT; v++) acc[t][v] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(rb, qb[v], acc[t][v], 0, 0, 0);
                }
            }
        }
    }
#pragma unroll
    for (int v = 0; v < MT; v++) {
        const int q = m0 + v * 16 + (lane & 15);
        if (q >= m) continue;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int64_t j = n0 + t * 16 + (lane >> 4) * 4;
            T* dst = out + q * ld + j;
            T o[4];
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = (T)acc[t][v][i];         // the only rounding behind the float32 sums
            if (j + 4 <= n) {
                __builtin_memcpy(dst, o, sizeof(o));
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) if (j + i < n) dst[i] = o[i];
            }
        }
    }
}

template <class T> void scores_t(hipStream_t s, const Fp8View& q, int64_t q_first, int64_t m, const Fp8View& r, int64_t first, int64_t n, T* out, int64_t ld) {
    constexpr int64_t kPieceN = (int64_t)1 << 24, kPieceM = (int64_t)1 << 16;      // a launch's tile numbers fit 32 bits
    for (int64_t i = 0; i < m; i += kPieceM) for (int64_t j = 0; j < n; j += kPieceN) {
        const int mi = (int)std::min(kPieceM, m - i), nj = (int)std::min(kPieceN, n - j);
        const uint8_t *qc = q.codes + (q_first + i) * q.row_bytes(), *qs = q.scales + (q_first + i) * q.nb4;
        const uint8_t *rc = r.codes + (first + j) * r.row_bytes(), *rs = r.scales + (first + j) * r.nb4;
        T* o = out + i * ld + j;
        const int64_t nt = ceil_div(nj, 256);
        if (mi <= 16) hipLaunchKernelGGL((scores_stream_kernel<T, 1>), dim3((unsigned)nt), dim3(256), 0, s, qc, qs, mi, rc, rs, nj, r.nb, r.nb4, o, ld, 1);
        else {
            const int mt = (int)ceil_div(mi, 64);
            hipLaunchKernelGGL((scores_stream_kernel<T, 4>), dim3((unsigned)(nt * mt)), dim3(256), 0, s, qc, qs, mi, rc, rs, nj, r.nb, r.nb4, o, ld, mt);
        }
        LAUNCH_CHECK();
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
