// fp8_api.hip — the 8-bit row store behind the C ABI: handles, argument checks, host-array forms, and the search that runs its operators together.
#include "fp8.hpp"

using namespace comet;

struct comet_fp8_rows {
    Ctx* c = nullptr;
    Fp8View v{};
    DevBuf codes, scales, last;
};

namespace {

// the calling thread's current device is put back when the call returns: a caller that drives several GPUs does not lose its own
struct DeviceScope {
    int before = -1;
    explicit DeviceScope(int device) { HIP_CHECK(hipGetDevice(&before)); if (before != device) HIP_CHECK(hipSetDevice(device)); else before = -1; }
    ~DeviceScope() { if (before >= 0) (void)hipSetDevice(before); }
};

// a host-array call: serialised on the context like every other, on lane 0's stream and scratch
struct HostCall {
    Ctx* c; std::unique_lock<std::recursive_mutex> lk; DeviceScope dev;
    explicit HostCall(Ctx* c_) : c(c_), lk(c_->mu), dev(c_->device) { c->check_indexes("entry of a call"); c->switch_lane(0); c->quiesce_alt(); c->scratch_reset(); }
    ~HostCall() { if (c->async_seen) { try { c->fence_lane0(); } catch (...) {} } }
};

// Work queued on lane 0's own stream is what later asynchronous searches start behind (as for every other call that queues there). Other streams are the
// caller's to order. Neither takes the context's mutex: a call on device arrays does not stand behind another thread's search or upload.
void queued(Ctx* c, hipStream_t s) { if (s == c->lane0) c->queued_on_lane0(); }

void check_dtype(int dtype) { if (dtype != COMET_F32 && dtype != COMET_F16 && dtype != COMET_BF16) COMET_FAIL(COMET_ERR_INVALID_ARG, "unknown element type %d", dtype); }
void check_rows(const comet_fp8_rows* r) { if (!r) COMET_FAIL(COMET_ERR_INVALID_ARG, "rows must not be null"); }
void check_matrix(const void* p, int dtype, int64_t ld, int64_t n, int64_t width, const char* what) {
    check_dtype(dtype);
    if (n < 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "negative row count");
    if (n == 0) return;
    if (!p) COMET_FAIL(COMET_ERR_INVALID_ARG, "%s must not be null", what);
    if (ld < width) COMET_FAIL(COMET_ERR_INVALID_ARG, "%s: row stride %lld is less than the width %lld", what, (long long)ld, (long long)width);
    if (ld > INT64_MAX / 4 / n) COMET_FAIL(COMET_ERR_INVALID_ARG, "%s: %lld rows of stride %lld", what, (long long)n, (long long)ld);
    if ((uintptr_t)p % dtype_size(dtype)) COMET_FAIL(COMET_ERR_INVALID_ARG, "%s is not aligned to its element type", what);
}
void check_range(const Fp8View& v, int64_t first, int64_t n, const char* what) {
    if (first < 0 || n < 0 || first > v.capacity - n) COMET_FAIL(COMET_ERR_INVALID_ARG, "%s [%lld, %lld + %lld) outside the capacity %lld", what, (long long)first, (long long)first, (long long)n, (long long)v.capacity);
}
void check_slots(const Fp8View& v, const int64_t* slots, int64_t first, int64_t n) {
    if (n < 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "negative row count");
    if (!slots) { check_range(v, first, n, "slots"); return; }
    if ((uintptr_t)slots % 8) COMET_FAIL(COMET_ERR_INVALID_ARG, "slots is not aligned to 8 bytes");
}
void check_scale(float scale) {      // scale * log2(e) has to be a float32 number
    if (!(std::fabs(scale) > 0.0f) || !(std::fabs(scale) <= 0x1p126f)) COMET_FAIL(COMET_ERR_INVALID_ARG, "scale must be finite and not zero, and its magnitude at most 2^126");
}
void check_logprobs(int64_t m, int64_t n, int32_t k) {
    if (m < 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "negative row count");
    if (n < 0 || n > ((int64_t)1 << 30)) COMET_FAIL(COMET_ERR_INVALID_ARG, "column count %lld outside [0, 2^30]", (long long)n);
    if (k < 0 || k > kLogProbsMaxK) COMET_FAIL(COMET_ERR_INVALID_ARG, "k %d outside [0, %d]", (int)k, kLogProbsMaxK);
}

int write_rows(comet_fp8_rows* r, const int64_t* slots, int64_t first, const void* x, int dtype, int64_t ld, int64_t n, hipStream_t s) {
    check_matrix(x, dtype, ld, n, r->v.dim, "vectors");
    check_slots(r->v, slots, first, n);
    launch_fp8_write(s, r->v, r->last.as<int32_t>(), slots, first, x, dtype, ld, n);
    return COMET_OK;
}
}  // namespace

extern "C" {

int comet_fp8_create(comet_ctx* c, int64_t capacity, int32_t dim, comet_fp8_rows** out) {
    return guarded([&] {
        if (!out) COMET_FAIL(COMET_ERR_INVALID_ARG, "out must not be null");
        *out = nullptr;
        if (!c) COMET_FAIL(COMET_ERR_INVALID_ARG, "context must not be null");
        if (dim <= 0 || dim > (1 << 20)) COMET_FAIL(COMET_ERR_INVALID_ARG, "dimension must be positive and at most 2^20");
        if (capacity <= 0 || capacity > ((int64_t)1 << 40) / dim) COMET_FAIL(COMET_ERR_INVALID_ARG, "capacity must be positive and at most 2^40 / dimension");
        HostCall g(c);
        std::unique_ptr<comet_fp8_rows> r(new comet_fp8_rows());
        r->c = c;
        const int nb = (int)ceil_div(dim, kFp8Block), nb4 = (int)round_up(nb, 4);
        const size_t code_bytes = (size_t)capacity * nb * kFp8Block, scale_bytes = (size_t)capacity * nb4;
        auto exactly = [](DevBuf& b, size_t bytes) { HIP_CHECK(hipMalloc(&b.p, bytes)); b.cap = bytes; };     // a store does not grow
        exactly(r->codes, code_bytes); exactly(r->scales, scale_bytes); exactly(r->last, (size_t)capacity * 4);
        HIP_CHECK(hipMemsetAsync(r->codes.p, 0, code_bytes, c->stream));
        HIP_CHECK(hipMemsetAsync(r->scales.p, 0, scale_bytes, c->stream));
        HIP_CHECK(hipMemsetAsync(r->last.p, 0xFF, (size_t)capacity * 4, c->stream));
        HIP_CHECK(hipStreamSynchronize(c->stream));      // the store is ready for every stream
        r->v = Fp8View{r->codes.as<uint8_t>(), r->scales.as<uint8_t>(), capacity, dim, nb, nb4};
        *out = r.release();
        return (int)COMET_OK;
    });
}
int comet_fp8_destroy(comet_fp8_rows* r) {
    return guarded([&] {
        if (!r) return (int)COMET_OK;
        DeviceScope d(r->c->device);
        delete r;               // hipFree waits for the device: no kernel in flight reads the rows any more
        return (int)COMET_OK;
    });
}
int64_t comet_fp8_capacity(const comet_fp8_rows* r) { return r ? r->v.capacity : 0; }
int comet_fp8_dim(const comet_fp8_rows* r) { return r ? r->v.dim : 0; }

int comet_fp8_write_dev(comet_fp8_rows* r, const int64_t* slots, int64_t first, const void* x, int dtype, int64_t ld, int64_t n, void* stream) {
    return guarded([&] {
        check_rows(r);
        DeviceScope d(r->c->device);
        const int rc = write_rows(r, slots, first, x, dtype, ld, n, (hipStream_t)stream);
        queued(r->c, (hipStream_t)stream);
        return rc;
    });
}
int comet_fp8_read_dev(const comet_fp8_rows* r, const int64_t* slots, int64_t first, void* out, int dtype, int64_t ld, int64_t n, void* stream) {
    return guarded([&] {
        check_rows(r);
        check_matrix(out, dtype, ld, n, r->v.dim, "out");
        check_slots(r->v, slots, first, n);
        DeviceScope d(r->c->device);
        launch_fp8_read((hipStream_t)stream, r->v, slots, first, out, dtype, ld, n);
        queued(r->c, (hipStream_t)stream);
        return (int)COMET_OK;
    });
}
int comet_fp8_scores_dev(const comet_fp8_rows* q, int64_t q_first, int64_t m, const comet_fp8_rows* r, int64_t first, int64_t n, void* out, int dtype, int64_t ld, void* stream) {
    return guarded([&] {
        check_rows(q); check_rows(r);
        if (q->c->device != r->c->device) COMET_FAIL(COMET_ERR_INVALID_ARG, "queries are on device %d, rows on device %d", q->c->device, r->c->device);
        if (q->v.dim != r->v.dim) COMET_FAIL(COMET_ERR_DIM_MISMATCH, "query dimension mismatch: expected %d, got %d", r->v.dim, q->v.dim);
        check_range(q->v, q_first, m, "queries"); check_range(r->v, first, n, "rows");
        check_matrix(out, dtype, ld, n == 0 ? 0 : m, n, "out");
        DeviceScope d(r->c->device);
        launch_fp8_scores((hipStream_t)stream, q->v, q_first, m, r->v, first, n, out, dtype, ld);
        queued(r->c, (hipStream_t)stream);
        return (int)COMET_OK;
    });
}

int comet_logprobs_work_bytes(int64_t m, int64_t n, int32_t k, size_t* out_bytes) {
    return guarded([&] {
        if (!out_bytes) COMET_FAIL(COMET_ERR_INVALID_ARG, "out must not be null");
        check_logprobs(m, n, k);
        *out_bytes = logprobs_work_bytes(m, n, k);
        return (int)COMET_OK;
    });
}
int comet_logprobs_dev(comet_ctx* c, const void* scores, int dtype, int64_t ld, int64_t m, int64_t n, const int32_t* counts, float scale, const int32_t* targets, int32_t n_targets,
                       int32_t k, float* logprobs, float* logsum, float* entropy, int32_t* ids, float* top_logprobs, void* work, size_t work_bytes, void* stream) {
    return guarded([&] {
        if (!c) COMET_FAIL(COMET_ERR_INVALID_ARG, "context must not be null");
        check_logprobs(m, n, k);
        check_matrix(scores, dtype, ld, n == 0 ? 0 : m, n, "scores");
        check_scale(scale);
        if (n_targets < 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "negative target count");
        if (m > 0) {
            if (!logsum || !entropy) COMET_FAIL(COMET_ERR_INVALID_ARG, "out must not be null");
            if (n_targets > 0 && (!targets || !logprobs)) COMET_FAIL(COMET_ERR_INVALID_ARG, "targets and their log-probabilities must not be null");
            if (k > 0 && (!ids || !top_logprobs)) COMET_FAIL(COMET_ERR_INVALID_ARG, "ids and their log-probabilities must not be null");
        }
        const size_t need = logprobs_work_bytes(m, n, k);
        if (need > 0 && (!work || work_bytes < need)) COMET_FAIL(COMET_ERR_INVALID_ARG, "workspace of %zu bytes, %zu needed", work ? work_bytes : (size_t)0, need);
        if (need > 0 && (uintptr_t)work % 16) COMET_FAIL(COMET_ERR_INVALID_ARG, "workspace is not aligned to 16 bytes");
        DeviceScope d(c->device);
        launch_logprobs((hipStream_t)stream, LogProbsArgs{scores, dtype, ld, m, (int32_t)n, counts, scale, targets, n_targets, k, logprobs, logsum, entropy, ids, top_logprobs, work});
        queued(c, (hipStream_t)stream);
        return (int)COMET_OK;
    });
}

// ---- host arrays ----------------------------------------------------------------------------------
int comet_fp8_write(comet_fp8_rows* r, const int64_t* slots, const float* vecs, int64_t n) {
    return guarded([&] {
        check_rows(r);
        if (n < 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "negative row count");
        if (n == 0) return (int)COMET_OK;
        if (!vecs || !slots) COMET_FAIL(COMET_ERR_INVALID_ARG, "slots and vectors must not be null");
        for (int64_t i = 0; i < n; i++) check_range(r->v, slots[i], 1, "slot");
        HostCall g(r->c);
        Ctx* c = r->c;
        const int64_t piece = std::max<int64_t>(1, ((int64_t)256 << 20) / ((int64_t)r->v.dim * 4));     // upload in bounded pieces, in order: the last row with a slot stays
        float* x = c->salloc<float>((size_t)std::min(piece, n) * r->v.dim);
        int64_t* s = c->salloc<int64_t>((size_t)std::min(piece, n));
        for (int64_t i = 0; i < n; i += piece) {
            const int64_t m = std::min(piece, n - i);
            c->h2d(x, vecs + i * r->v.dim, (size_t)m * r->v.dim * 4);
            c->h2d(s, slots + i, (size_t)m * 8);
            write_rows(r, s, 0, x, COMET_F32, r->v.dim, m, c->stream);
        }
        HIP_CHECK(hipStreamSynchronize(c->stream));
        return (int)COMET_OK;
    });
}
int comet_fp8_read(const comet_fp8_rows* r, const int64_t* slots, int64_t n, float* out) {
    return guarded([&] {
        check_rows(r);
        if (n < 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "negative row count");
        if (n == 0) return (int)COMET_OK;
        if (!out || !slots) COMET_FAIL(COMET_ERR_INVALID_ARG, "slots and out must not be null");
        for (int64_t i = 0; i < n; i++) check_range(r->v, slots[i], 1, "slot");
        HostCall g(r->c);
        Ctx* c = r->c;
        const int64_t piece = std::max<int64_t>(1, ((int64_t)256 << 20) / ((int64_t)r->v.dim * 4));
        float* x = c->salloc<float>((size_t)std::min(piece, n) * r->v.dim);
        int64_t* s = c->salloc<int64_t>((size_t)std::min(piece, n));
        for (int64_t i = 0; i < n; i += piece) {
            const int64_t m = std::min(piece, n - i);
            c->h2d(s, slots + i, (size_t)m * 8);
            launch_fp8_read(c->stream, r->v, s, 0, x, COMET_F32, r->v.dim, m);
            c->d2h(out + i * r->v.dim, x, (size_t)m * r->v.dim * 4);
            HIP_CHECK(hipStreamSynchronize(c->stream));
        }
        return (int)COMET_OK;
    });
}
int comet_fp8_search(const comet_fp8_rows* r, int64_t first, int64_t n, const float* queries, int32_t B, float scale, int32_t k, int64_t* out_slots, float* out_logprobs,
                     float* out_logsum, float* out_entropy) {
    return guarded([&] {
        check_rows(r);
        if (B < 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "negative query count");
        check_logprobs(B, n, k);
        check_range(r->v, first, n, "rows");
        check_scale(scale);
        if (B == 0) return (int)COMET_OK;
        if (!queries || (k > 0 && (!out_slots || !out_logprobs)) || !out_logsum || !out_entropy) COMET_FAIL(COMET_ERR_INVALID_ARG, "queries and out must not be null");
        HostCall g(r->c);
        Ctx* c = r->c;
        const int dim = r->v.dim;
        // the score matrix of a piece of the queries stays within 1 GiB
        const int64_t piece = std::min<int64_t>(B, std::max<int64_t>(1, ((int64_t)1 << 28) / std::max<int64_t>(1, n)));
        const size_t work_bytes = logprobs_work_bytes(piece, n, k);
        Fp8View q = r->v;
        q.capacity = piece;
        float* x = c->salloc<float>((size_t)piece * dim);
        q.codes = c->salloc<uint8_t>((size_t)piece * q.nb * kFp8Block); q.scales = c->salloc<uint8_t>((size_t)piece * q.nb4);
        if (dim % kFp8Block) HIP_CHECK(hipMemsetAsync(q.codes, 0, (size_t)piece * q.nb * kFp8Block, c->stream));       // a store's padding is zero before its first write
        float* scores = c->salloc<float>((size_t)piece * std::max<int64_t>(1, n));
        void* work = c->scratch_alloc(work_bytes + 16);
        float *ls = c->salloc<float>(piece), *en = c->salloc<float>(piece), *tl = c->salloc<float>((size_t)piece * k + 1);
        int32_t* ids = c->salloc<int32_t>((size_t)piece * k + 1);
        std::vector<int32_t> cols((size_t)piece * k);
        for (int64_t i = 0; i < B; i += piece) {
            const int64_t m = std::min<int64_t>(piece, B - i);
            c->h2d(x, queries + i * dim, (size_t)m * dim * 4);
            launch_fp8_write(c->stream, q, nullptr, nullptr, 0, x, COMET_F32, dim, m);
            launch_fp8_scores(c->stream, q, 0, m, r->v, first, n, scores, COMET_F32, n);
            launch_logprobs(c->stream, LogProbsArgs{scores, COMET_F32, n, m, (int32_t)n, nullptr, scale, nullptr, 0, k, nullptr, ls, en, ids, tl, work});
            c->d2h(out_logsum + i, ls, (size_t)m * 4); c->d2h(out_entropy + i, en, (size_t)m * 4);
            if (k > 0) { c->d2h(out_logprobs + i * k, tl, (size_t)m * k * 4); c->d2h(cols.data(), ids, (size_t)m * k * 4); }
            HIP_CHECK(hipStreamSynchronize(c->stream));
            for (int64_t j = 0; j < m * k; j++) out_slots[i * k + j] = cols[(size_t)j] < 0 ? -1 : first + cols[(size_t)j];
        }
        return (int)COMET_OK;
    });
}

}  // extern "C"
