// fp8.hpp — the 8-bit row store and the operators on it (host side: fp8_api.hip).
// A stored row is `nb` blocks of 128 e4m3 codes (row-major, the last block padded with zero codes) and one power-of-two scale byte
// (e8m0: 2^(byte - 127)) per block, `nb4` = nb rounded up to 4 bytes apart per row, so that four blocks' scales are one dword.
#pragma once
#include <tuple>
#include <utility>

#include "../index.hpp"

namespace comet {

constexpr int kFp8Block = 128;
// the exponents a block's scale may take: 2^-e and 2^e are both normal float32 numbers over the whole range, and 120 is what the largest float32 needs
constexpr int kFp8ExpMin = -126;

struct Fp8View {            // device memory of one store
    uint8_t* codes; uint8_t* scales;
    int64_t capacity; int dim, nb, nb4;
    int64_t row_bytes() const { return (int64_t)nb * kFp8Block; }
};

inline size_t dtype_size(int dtype) { return dtype == COMET_F32 ? 4 : 2; }

// Launches a kernel and checks what the launch itself returned: an error that another call left in the runtime neither stops a write half way (marked slots
// whose rows never arrive would lose every later row) nor is taken from that call.
template <class... P, class... A> void launch_kernel(void (*kernel)(P...), int64_t groups, int threads, size_t lds, hipStream_t s, A... args) {
    std::tuple<P...> held(static_cast<P>(args)...);
    std::apply([&](auto&... a) {
        void* list[] = {(void*)&a...};
        HIP_CHECK(hipLaunchKernel((const void*)kernel, dim3((unsigned)groups), dim3((unsigned)threads), list, lds, s));
    }, held);
}

// Every launch below goes to the given stream, allocates nothing, waits for nothing and is capturable.

// rows x[i] (n x dim, `ld` elements apart) -> slot slots[i], or first + i when slots == nullptr; slots outside [0, capacity) are skipped; of rows
// with the same slot the last one stays. `last`: one int32 per slot, -1 between calls. The codes behind a row's dim must be 0 already.
void launch_fp8_write(hipStream_t s, const Fp8View& v, int32_t* last, const int64_t* slots, int64_t first, const void* x, int dtype, int64_t ld, int64_t n);
// out[i] (n x dim, `ld` elements apart) <- the values slot slots[i] (or first + i) holds; slots outside [0, capacity) give zeros
void launch_fp8_read(hipStream_t s, const Fp8View& v, const int64_t* slots, int64_t first, void* out, int dtype, int64_t ld, int64_t n);
// out[i][j] = <queries' row q_first + i, rows' row first + j>, m x n, `ld` elements apart
void launch_fp8_scores(hipStream_t s, const Fp8View& q, int64_t q_first, int64_t m, const Fp8View& r, int64_t first, int64_t n, void* out, int dtype, int64_t ld);

constexpr int kLogProbsMaxK = 128;
struct LogProbsArgs {
    const void* scores; int dtype; int64_t ld; int64_t m; int32_t n; const int32_t* counts; float scale;
    const int32_t* targets; int32_t n_targets; int32_t k;
    float* logprobs; float* logsum; float* entropy; int32_t* ids; float* top_logprobs; void* work;
};
size_t logprobs_work_bytes(int64_t m, int64_t n, int32_t k);
void launch_logprobs(hipStream_t s, const LogProbsArgs& a);

}  // namespace comet
