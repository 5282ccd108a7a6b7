// api.hip — the extern "C" surface declared in include/comet_gpu.h.
#include "index.hpp"

using namespace comet;

namespace {

void check_live_indexes(Ctx* c, const char* where) {
    for (void* p : c->live_indexes) { const comet_index* ix = static_cast<const comet_index*>(p); if (!ix->guards_ok()) { ix->guards_dump(where); std::abort(); } }
}
// The guard words around the index objects' host-side containers (round 4: a late 8-byte write into a PQ index object) are checked on entry and exit of
// every call. COMET_GUARDS=0 (read once) switches the checks off — they have not fired in twenty 900 s soaks since the private per-index streams went, and walking
// every live index per call is what a debug aid costs — but they stay ON by default: round 6's soaks met one unexplained (and unreproduced) wrong result, so the
// conditions the review set for retiring them ("nine clean runs on three seeds") are not met.
comet_index* adopt(Ctx* c, comet_index* ix) {
    static const bool guards_on = [] { const char* e = getenv("COMET_GUARDS"); return !(e && e[0] == '0'); }();
    std::lock_guard<std::recursive_mutex> lk(c->mu);
    if (guards_on) c->check_live = check_live_indexes;
    c->live_indexes.push_back(ix); return ix;
}
void check_metric(int m) { if (m < COMET_L2 || m > COMET_COSINE) COMET_FAIL(COMET_ERR_UNKNOWN_METRIC, "unknown distance kind"); }  // distance.go:9
struct CallGuard {   // serialise calls on a context, bind the device, reset the per-call scratch arena
    Ctx* c; std::unique_lock<std::recursive_mutex> lk;
    // every call but an asynchronous search: lane 0, and lane 1 idle first (the call may change what a search in flight there reads)
    bool search = false;
    explicit CallGuard(Ctx* c_) : c(c_), lk(c_->mu) { c->check_indexes("entry of a call"); c->bind(); c->switch_lane(0); c->quiesce_alt(); c->scratch_reset(); }
    // an asynchronous search enqueued on `lane` (its stream, its scratch arena); lane 0 is current again when the guard goes. A lane
    // other than 0 starts behind whatever non-search work lane 0 was last given (Ctx::lane0_fence): the queries may still be being written there
    CallGuard(Ctx* c_, int lane) : c(c_), lk(c_->mu), search(true) {
        c->check_indexes("entry of an asynchronous search"); c->bind();
        c->begin_async();
        c->switch_lane(lane); c->scratch_reset(); c->follow_lane0();
    }
    ~CallGuard() {
        c->check_indexes("exit of a call");
        if (c->cur_lane != 0) { c->mark_dirty(); try { c->switch_lane(0); } catch (...) {} }
        if (!search && c->async_seen) { try { c->fence_lane0(); } catch (...) {} }     // what this call left queued on lane 0 is what later searches on lanes 1.. start behind
    }
};
}  // namespace

extern "C" {

const char* comet_last_error(void) { return last_error().c_str(); }
const char* comet_version(void) { return "comet-mi355x 0.1 (gfx950, HIP)"; }

int comet_device_count(int* out_count) {
    return guarded([&] {
        int n = 0;
        hipError_t e = hipGetDeviceCount(&n);
        if (e != hipSuccess) { n = 0; (void)hipGetLastError(); }
        *out_count = n;
        return COMET_OK;
    });
}

int comet_ctx_create(int device_id, comet_ctx** out) {
    return guarded([&] {
        *out = nullptr;
        int n = 0;
        if (hipGetDeviceCount(&n) != hipSuccess || n <= 0) { (void)hipGetLastError(); COMET_FAIL(COMET_ERR_NO_DEVICE, "no HIP device visible: the comet GPU backend requires an MI355X (gfx950)"); }
        if (device_id < 0 || device_id >= n) COMET_FAIL(COMET_ERR_INVALID_ARG, "device %d out of range [0,%d)", device_id, n);
        auto* c = new comet_ctx();
        c->device = device_id;
        HIP_CHECK(hipSetDevice(device_id));
        HIP_CHECK(hipGetDeviceProperties(&c->prop, device_id));
        if (std::strncmp(c->prop.gcnArchName, "gfx950", 6) != 0) {
            std::string arch = c->prop.gcnArchName; delete c;
            COMET_FAIL(COMET_ERR_NO_DEVICE, "device %d is %s; this library contains gfx950 (MI355X) code only", device_id, arch.c_str());
        }
        // All of the context's streams are made NOW. The runtime multiplexes streams onto a few hardware queues per priority level (four), and a stream made
        // when every queue of its level is taken shares the least-used one — which two lanes created lazily, with indexes' private copy streams made and
        // destroyed in between, did whenever the order of a program's calls was unlucky: their searches then take turns instead of overlapping (bench: the
        // HNSW leg at four batches in flight 1.65 M -> 1.08 M q/s and IVFPQ 1.8 -> 1.4 M after the legs flat_l2 + ivfpq had run, kernel times unchanged).
        // The four lanes therefore get a priority level of their OWN (the highest): the first four streams of a level each open a queue, so the lanes never
        // share one with each other or with anything else of the process.
        // Lanes 4 .. 7 (round 6; only HNSW rotates through more than four) take the NEXT level, for the same reason. COMET_STREAM_PRIORITY=normal puts lanes
        // 0 .. 3 on the default level instead (and 4 .. 7 on the lowest): for a process that embeds the library next to work of its own on default-priority
        // streams and does not want the searches to take precedence over it; the lanes may then share hardware queues with that work.
        int pr_least = 0, pr_greatest = 0;
        HIP_CHECK(hipDeviceGetStreamPriorityRange(&pr_least, &pr_greatest));
        const char* pe = getenv("COMET_STREAM_PRIORITY");
        const bool normal = pe && (pe[0] == 'n' || pe[0] == 'N' || pe[0] == '0');
        const int pr_a = normal ? std::min(pr_least, pr_greatest + 1) : pr_greatest;          // numerically lower = more urgent
        const int pr_b = std::min(pr_least, pr_a + 1);
        HIP_CHECK(hipStreamCreateWithPriority(&c->stream, hipStreamNonBlocking, pr_a));
        c->lane0 = c->stream;
        for (int l = 1; l < Ctx::kMaxLanes; l++) HIP_CHECK(hipStreamCreateWithPriority(&c->parked[l].stream, hipStreamNonBlocking, l < 4 ? pr_a : pr_b));
        *out = c;
        return COMET_OK;
    });
}
int comet_ctx_destroy(comet_ctx* c) {
    return guarded([&] {
        if (!c) return COMET_OK;
        c->bind();
        c->switch_lane(0);
        (void)hipStreamSynchronize(c->stream);
        for (int l = 1; l < Ctx::kMaxLanes; l++) if (c->parked[l].stream) (void)hipStreamSynchronize(c->parked[l].stream);
        c->collect_profile();
        c->scratch_reset();
        for (int l = 1; l < Ctx::kMaxLanes; l++) {
            for (void* r : c->parked[l].retired) (void)hipFree(r);
            if (c->parked[l].scratch) (void)hipFree(c->parked[l].scratch);
            if (c->parked[l].stream) (void)hipStreamDestroy(c->parked[l].stream);
        }
        if (c->scratch) (void)hipFree(c->scratch);
        if (c->lane0_fence) (void)hipEventDestroy(c->lane0_fence);
        if (c->fork_ev) (void)hipEventDestroy(c->fork_ev);
        if (c->pinned) (void)hipHostFree(c->pinned);
        if (c->bounce) (void)hipHostFree(c->bounce);
        (void)hipStreamDestroy(c->stream);
        delete c;
        return COMET_OK;
    });
}
int comet_ctx_sync(comet_ctx* c) { return guarded([&] { std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->sync(); return COMET_OK; }); }
void* comet_ctx_stream(comet_ctx* c) { return (void*)c->lane0; }
int comet_ctx_fence(comet_ctx* c) { return guarded([&] { std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->switch_lane(0); c->fence_lane0(); return COMET_OK; }); }
int comet_dev_alloc(comet_ctx* c, size_t bytes, void** out) { return guarded([&] { c->bind(); HIP_CHECK(hipMalloc(out, bytes ? bytes : 4)); return COMET_OK; }); }
int comet_dev_free(comet_ctx* c, void* p) { return guarded([&] { c->bind(); if (p) HIP_CHECK(hipFree(p)); return COMET_OK; }); }
int comet_memcpy_h2d(comet_ctx* c, void* d, const void* s, size_t bytes) {
    return guarded([&] { std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->h2d(d, s, bytes); HIP_CHECK(hipStreamSynchronize(c->stream)); return COMET_OK; });
}
int comet_memcpy_d2h(comet_ctx* c, void* d, const void* s, size_t bytes) {
    return guarded([&] { std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->d2h(d, s, bytes); HIP_CHECK(hipStreamSynchronize(c->stream)); return COMET_OK; });
}
int comet_synth_fill_dev(comet_ctx* c, uint64_t seed, uint64_t offset, uint64_t n, float* out_dev) {
    // enqueue-only on lane 0 (no quiesce: generators run beside searches in flight); the fence makes a later asynchronous search on lanes 1.. start behind it
    return guarded([&] { std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->switch_lane(0); launch_synth_fill(c, seed, offset, n, out_dev); if (c->async_seen) c->fence_lane0(); return COMET_OK; });
}

int comet_synth_mixture_dev(comet_ctx* c, uint64_t seed, int32_t n_centers, float sigma, int32_t n_sub, float sigma_noise, uint64_t row_base,
                            uint64_t n_rows, int32_t dim, float* out_dev) {
    return guarded([&] { std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->switch_lane(0); launch_synth_mixture(c, seed, n_centers, sigma, n_sub, sigma_noise, row_base, n_rows, dim, out_dev); if (c->async_seen) c->fence_lane0(); return COMET_OK; });
}

int comet_ctx_set_lanes(comet_ctx* c, int32_t lanes) {
    return guarded([&] {
        if (lanes < 1 || lanes > Ctx::kMaxLanes) COMET_FAIL(COMET_ERR_INVALID_ARG, "a context has 1 to %d execution lanes", Ctx::kMaxLanes);
        std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->switch_lane(0); c->quiesce_all(); c->lanes = lanes;
        return COMET_OK;
    });
}
int comet_profile_enable(comet_ctx* c, int on) { return guarded([&] { std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->sync(); c->profile = on != 0; return COMET_OK; }); }
int comet_profile_only(comet_ctx* c, const char* name) { return guarded([&] { std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->sync(); c->prof_only = name ? name : ""; return COMET_OK; }); }
int comet_profile_reset(comet_ctx* c) { return guarded([&] { std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->sync(); c->prof.clear(); return COMET_OK; }); }
int comet_profile_get(comet_ctx* c, const char* prefix, double* total_ms, int64_t* launches) {
    return guarded([&] {
        std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->sync();
        double ms = 0; int64_t n = 0; size_t pl = std::strlen(prefix);
        for (auto& kv : c->prof) if (kv.first.compare(0, pl, prefix) == 0) { ms += kv.second.ms; n += kv.second.n; }
        if (total_ms) *total_ms = ms;
        if (launches) *launches = n;
        return COMET_OK;
    });
}
int comet_profile_dump(comet_ctx* c, char* buf, size_t cap) {
    return guarded([&] {
        std::lock_guard<std::recursive_mutex> lk(c->mu); c->bind(); c->sync();
        std::string s;
        for (auto& kv : c->prof) { char line[256]; snprintf(line, sizeof(line), "%s %.6f %lld\n", kv.first.c_str(), kv.second.ms, (long long)kv.second.n); s += line; }
        if (cap) { size_t m = std::min(cap - 1, s.size()); std::memcpy(buf, s.data(), m); buf[m] = 0; }
        return COMET_OK;
    });
}

// ---- Distance singletons ------------------------------------------------------------------------
int comet_distance_batch(comet_ctx* c, int metric, const float* queries, int nq, const float* target, int d, float* out) {
    return guarded([&] {
        check_metric(metric);
        if (nq <= 0) return (int)COMET_OK;
        if (d < 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "negative dimension");
        CallGuard g(c);
        float* dq = c->salloc<float>((size_t)nq * std::max(d, 1));
        float* dt = c->salloc<float>(std::max(d, 1));
        float* dout = c->salloc<float>(nq);
        c->h2d(dq, queries, (size_t)nq * d * sizeof(float));
        c->h2d(dt, target, (size_t)d * sizeof(float));
        launch_dist_pairs(c, metric, dq, dt, nq, d, d, 0, dout);
        c->d2h(out, dout, nq * sizeof(float));
        c->sync();
        return (int)COMET_OK;
    });
}
int comet_distance(comet_ctx* c, int metric, const float* a, const float* b, int d, float* out) {
    return comet_distance_batch(c, metric, a, 1, b, d, out);
}
// Norm / Normalize / Scale distance.go:312-428 (host buffers; one upload, one download)
static int vec_op(comet_ctx* c, const float* x, int64_t n, int32_t d, int op, float scalar, float* out) {
    return guarded([&] {
        if (n < 0 || d < 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "negative size");
        if (n == 0 || (d == 0 && op != 0)) return (int)COMET_OK;
        CallGuard g(c);
        float* dx = c->salloc<float>((size_t)std::max<int64_t>(1, n * d));
        float* dn = c->salloc<float>((size_t)n);
        if (d > 0) c->h2d(dx, x, (size_t)n * d * sizeof(float));
        if (op == 0 || op == 1) launch_vec_norm(c, dx, n, d, dn);
        if (op == 0) { c->d2h(out, dn, (size_t)n * sizeof(float)); c->sync(); return (int)COMET_OK; }
        float* dout = c->salloc<float>((size_t)n * d);
        launch_vec_scale(c, dx, n, d, op == 1 ? dn : nullptr, scalar, dout);
        c->d2h(out, dout, (size_t)n * d * sizeof(float));
        c->sync();
        return (int)COMET_OK;
    });
}
int comet_norm_batch(comet_ctx* c, const float* x, int64_t n, int32_t d, float* out_norms) { return vec_op(c, x, n, d, 0, 0.0f, out_norms); }
int comet_normalize_batch(comet_ctx* c, const float* x, int64_t n, int32_t d, float* out) { return vec_op(c, x, n, d, 1, 0.0f, out); }
int comet_scale_batch(comet_ctx* c, const float* x, int64_t n, int32_t d, float scalar, float* out) { return vec_op(c, x, n, d, 2, scalar, out); }

int comet_preprocess(comet_ctx* c, int metric, const float* x, int d, float* out) {
    return guarded([&] {
        check_metric(metric);
        if (d <= 0) return (int)COMET_OK;
        CallGuard g(c);
        float* dx = c->salloc<float>(d);
        float* dp = c->salloc<float>(padded_dim(d));
        int32_t* zf = c->salloc<int32_t>(1);
        c->h2d(dx, x, d * sizeof(float));
        launch_ingest_rows(c, metric, dx, 1, d, dp, padded_dim(d), zf);
        int32_t hz = 0;
        std::vector<float> tmp(d);
        c->d2h(&hz, zf, sizeof(int32_t));
        c->d2h(tmp.data(), dp, d * sizeof(float));
        c->sync();
        if (hz) COMET_FAIL(COMET_ERR_ZERO_VECTOR, "zero vector not allowed for this metric");   // distance.go:12
        std::memcpy(out, tmp.data(), d * sizeof(float));
        return (int)COMET_OK;
    });
}

// ---- index lifecycle ----------------------------------------------------------------------------
static void check_dim(int dim) { if (dim <= 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "dimension must be positive"); }  // flat_index.go:129

int comet_flat_create(comet_ctx* c, int dim, int metric, comet_index** out) {
    return guarded([&] { *out = nullptr; check_dim(dim); check_metric(metric); c->bind(); *out = adopt(c, make_flat(c, dim, metric)); return (int)COMET_OK; });
}
int comet_ivf_create(comet_ctx* c, int dim, int metric, int nlist, comet_index** out) {
    return guarded([&] {
        *out = nullptr; check_dim(dim);
        if (nlist <= 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "nlist must be positive");   // ivf_index.go:147
        check_metric(metric); c->bind(); *out = adopt(c, make_ivf(c, dim, metric, nlist)); return (int)COMET_OK;
    });
}
static void check_pq(int dim, int M, int nbits) {
    if (M <= 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "parameter M must be positive");                              // pq_index.go:141
    if (dim % M != 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "dimension %d must be divisible by M %d", dim, M);       // pq_index.go:146
    if (nbits <= 0 || nbits > 16) COMET_FAIL(COMET_ERR_INVALID_ARG, "parameter Nbits must be in [1,16]");       // pq_index.go:151
}
int comet_pq_create(comet_ctx* c, int dim, int metric, int M, int nbits, comet_index** out) {
    return guarded([&] { *out = nullptr; check_dim(dim); check_pq(dim, M, nbits); check_metric(metric); c->bind(); *out = adopt(c, make_pq(c, dim, metric, M, nbits)); return (int)COMET_OK; });
}
int comet_ivfpq_create(comet_ctx* c, int dim, int metric, int nlist, int M, int nbits, comet_index** out) {
    return guarded([&] {
        *out = nullptr; check_dim(dim);
        if (nlist <= 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "nlist must be positive");   // ivfpq_index.go:120
        check_pq(dim, M, nbits); check_metric(metric); c->bind(); *out = adopt(c, make_ivfpq(c, dim, metric, nlist, M, nbits)); return (int)COMET_OK;
    });
}
int comet_index_destroy(comet_index* idx) {
    return guarded([&] { if (!idx) return (int)COMET_OK; Ctx* c = idx->c; std::lock_guard<std::recursive_mutex> lk(c->mu); c->check_indexes("entry of comet_index_destroy"); c->bind(); c->quiesce_all();
        // quiesce_all() above: every lane of the context is idle — and since round 5 an index owns no stream of its own (the Flat / IVF flag copies follow their
        // search on its lane), so nothing of the index can be in flight. Round 4 drained the whole DEVICE here (hipDeviceSynchronize) as a mitigation for the
        // wild write its soak had found; that stalls every other context of the process and can block behind a peer's collective. Three 900 s
        // soaks of the round-4 seed ran clean without it on round 5's code (profiles/r05_soak.txt): it is now opt-in, COMET_DESTROY_DEVICE_SYNC=1.
        static const bool dev_sync = getenv("COMET_DESTROY_DEVICE_SYNC") != nullptr;
        if (dev_sync) (void)hipDeviceSynchronize();
        delete idx; return (int)COMET_OK; });
}
int comet_index_kind(const comet_index* idx) { return idx->kind; }
int comet_index_dim(const comet_index* idx) { return idx->dim; }
int comet_index_metric(const comet_index* idx) { return idx->metric; }
int comet_index_trained(const comet_index* idx) { return idx->trained ? 1 : 0; }
int64_t comet_index_size(const comet_index* idx) { return idx->size(); }
int comet_index_default_nprobes(const comet_index* idx) { return idx->default_nprobes(); }

int comet_index_train_dev(comet_index* idx, const float* vecs_dev, int64_t n) {
    return guarded([&] { CallGuard g(idx->c); idx->train_dev(vecs_dev, n); idx->c->sync(); return (int)COMET_OK; });
}
int comet_index_train(comet_index* idx, const float* vecs, int64_t n) {
    return guarded([&] {
        if (idx->kind == COMET_KIND_FLAT) return (int)COMET_OK;   // FlatIndex.Train is a no-op
        if (n < 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "negative count");
        Ctx* c = idx->c; CallGuard g(c);
        DevBuf tmp; tmp.reserve(std::max<size_t>(4, (size_t)n * idx->dim * sizeof(float)), c->stream, 0);
        c->h2d(tmp.p, vecs, (size_t)n * idx->dim * sizeof(float));
        HIP_CHECK(hipStreamSynchronize(c->stream));
        idx->train_dev(tmp.as<float>(), n);
        c->sync();
        return (int)COMET_OK;
    });
}

static int add_common(comet_index* idx, const uint32_t* ids_dev, const uint32_t* ids_host, const float* vecs_dev, int64_t n,
                      int64_t* out_added, float* normalized_dev) {
    int64_t zero_at = -1;
    int64_t added = idx->add_dev(ids_dev, ids_host, vecs_dev, n, &zero_at, normalized_dev);
    if (out_added) *out_added = added;
    if (zero_at >= 0) COMET_FAIL(COMET_ERR_ZERO_VECTOR, "zero vector not allowed for this metric");
    return COMET_OK;
}
int comet_index_add(comet_index* idx, const uint32_t* ids, const float* vecs, int64_t n, int64_t* out_added, float* normalized_out) {
    return guarded([&] {
        if (out_added) *out_added = 0;
        if (n <= 0) return (int)COMET_OK;
        Ctx* c = idx->c; CallGuard g(c);
        DevBuf tmp, nrm;
        const size_t bytes = (size_t)n * idx->dim * sizeof(float);
        tmp.reserve(bytes, c->stream, 0);
        c->h2d(tmp.p, vecs, bytes);
        HIP_CHECK(hipStreamSynchronize(c->stream));
        if (normalized_out) nrm.reserve(bytes, c->stream, 0);
        int64_t added = 0;
        int rc = COMET_OK;
        try { rc = add_common(idx, nullptr, ids, tmp.as<float>(), n, &added, normalized_out ? nrm.as<float>() : nullptr); }
        catch (const StatusError& s) { rc = s.code; }
        if (out_added) *out_added = added;
        if (normalized_out && added > 0) { c->d2h(normalized_out, nrm.p, (size_t)added * idx->dim * sizeof(float)); }
        c->sync();
        return rc;
    });
}
int comet_index_add_dev(comet_index* idx, const uint32_t* ids_dev, const float* vecs_dev, int64_t n, int64_t* out_added) {
    return guarded([&] {
        if (out_added) *out_added = 0;
        if (n <= 0) return (int)COMET_OK;
        Ctx* c = idx->c; CallGuard g(c);
        std::vector<uint32_t> ids_h(n);
        c->d2h(ids_h.data(), ids_dev, n * 4);
        HIP_CHECK(hipStreamSynchronize(c->stream));
        int rc = add_common(idx, ids_dev, ids_h.data(), vecs_dev, n, out_added, nullptr);
        c->sync();
        return rc;
    });
}
int comet_index_remove(comet_index* idx, uint32_t id) {
    return guarded([&] {
        std::lock_guard<std::recursive_mutex> lk(idx->c->mu);
        if (!idx->contains_id(id)) COMET_FAIL(COMET_ERR_NOT_FOUND, "vector with ID %u not found", id);              // flat_index.go:233
        if (idx->deleted.count(id)) COMET_FAIL(COMET_ERR_ALREADY_DELETED, "vector with ID %u already deleted", id);  // flat_index.go:236
        idx->deleted.insert(id); idx->deleted_dirty = true;
        return (int)COMET_OK;
    });
}
int comet_index_flush(comet_index* idx) { return guarded([&] { CallGuard g(idx->c); idx->flush(); idx->c->sync(); return (int)COMET_OK; }); }

// ---- search ---------------------------------------------------------------------------------------
static void check_search_args(const comet_index* idx, int B, const comet_search_params* p, int k_cap) {
    if (!p) COMET_FAIL(COMET_ERR_INVALID_ARG, "null search params");
    if (B < 0 || k_cap <= 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "bad batch size / k_cap");
    (void)idx;
}
int comet_index_search_dev(comet_index* idx, const float* queries_dev, int32_t B, const comet_search_params* p,
                           uint32_t* out_ids_dev, float* out_scores_dev, int32_t* out_counts_dev, int32_t k_cap) {
    return guarded([&] {
        check_search_args(idx, B, p, k_cap);
        if (B == 0) return (int)COMET_OK;
        CallGuard g(idx->c);
        idx->search_dev(queries_dev, B, *p, out_ids_dev, out_scores_dev, out_counts_dev, k_cap);
        return (int)COMET_OK;
    });
}
int comet_index_search(comet_index* idx, const float* queries, int32_t B, const comet_search_params* p, uint32_t* out_ids,
                       float* out_scores, int32_t* out_counts, int32_t k_cap) {
    return guarded([&] {
        check_search_args(idx, B, p, k_cap);
        if (B == 0) return (int)COMET_OK;
        Ctx* c = idx->c; CallGuard g(c);
        float* dq = c->salloc<float>((size_t)B * idx->dim);
        uint32_t* dids = c->salloc<uint32_t>((size_t)B * k_cap);
        float* dsc = c->salloc<float>((size_t)B * k_cap);
        int32_t* dcn = c->salloc<int32_t>(B);
        c->h2d(dq, queries, (size_t)B * idx->dim * sizeof(float));
        idx->search_dev(dq, B, *p, dids, dsc, dcn, k_cap);
        c->d2h(out_ids, dids, (size_t)B * k_cap * 4);
        c->d2h(out_scores, dsc, (size_t)B * k_cap * 4);
        c->d2h(out_counts, dcn, (size_t)B * 4);
        c->sync();
        for (int i = 0; i < B; i++) if (out_counts[i] == -(int)COMET_ERR_ZERO_VECTOR)
            COMET_FAIL(COMET_ERR_ZERO_VECTOR, "zero vector not allowed for this metric");   // Preprocess(query) error, flat_index_search.go:236-239
        return (int)COMET_OK;
    });
}

int comet_index_search_dev_async(comet_index* idx, const float* queries_dev, int32_t B, const comet_search_params* p,
                                 uint32_t* out_ids_dev, float* out_scores_dev, int32_t* out_counts_dev, int32_t k_cap, uint64_t* out_ticket) {
    return guarded([&] {
        check_search_args(idx, B, p, k_cap);
        if (out_ticket) *out_ticket = 0;
        if (B == 0) return (int)COMET_OK;
        // the asynchronous searches of an index rotate through the context's execution lanes (as many as the kind gains from)
        int lane = 0;
        { std::lock_guard<std::recursive_mutex> lk(idx->c->mu); const int m = std::min(idx->c->lanes, idx->max_lanes()); if (m > 1) lane = idx->lane_toggle = (idx->lane_toggle + 1) % m; }
        CallGuard g(idx->c, lane);
        uint64_t t = idx->search_begin(queries_dev, B, *p, out_ids_dev, out_scores_dev, out_counts_dev, k_cap);
        if (out_ticket) *out_ticket = t;
        return (int)COMET_OK;
    });
}
int comet_index_search_wait(comet_index* idx, uint64_t ticket) {
    return guarded([&] {
        std::lock_guard<std::recursive_mutex> lk(idx->c->mu); idx->c->bind();
        idx->search_finish(ticket);
        return (int)COMET_OK;
    });
}

// ---- segment layer: persistentHybridSearch.Execute storage.go:489-626, vector leg --------------------------------
// One call searches every segment's index for the batch (all of them resident in HBM, searches enqueued back to back on the
// context's stream, no host round trip between them) and merges on the device as mergeResults + sortResultsByScore + the cut do.
static void segments_search(comet_index* const* segs, int S, const float* queries_dev, int B, const comet_search_params* p,
                            uint32_t* out_ids, float* out_scores, int32_t* out_counts, int k_cap) {
    Ctx* c = segs[0]->c;
    const int k = p->k;
    if (k == 0) {   // merged[:0] (storage.go:621-623)
        HIP_CHECK(hipMemsetAsync(out_counts, 0, (size_t)B * 4, c->stream));
        return;
    }
    uint32_t* ids = c->salloc<uint32_t>((size_t)S * B * k);
    float* sc = c->salloc<float>((size_t)S * B * k);
    int32_t* cn = c->salloc<int32_t>((size_t)S * B);
    std::vector<uint64_t> tickets(S);
    // The segments' searches rotate through the context's execution lanes: they are independent, and each is a chain of short
    // kernels. The other lanes start behind what lane 0 holds so far (the queries' upload); the merge starts when every search is final
    // (search_finish waits on the host). A lane's scratch arena is reset once per call and then grows across its segments.
    if (!c->fork_ev) HIP_CHECK(hipEventCreateWithFlags(&c->fork_ev, hipEventDisableTiming));    // the context's (c->mu is held): an event belongs to one device
    hipEvent_t ev = c->fork_ev;
    HIP_CHECK(hipEventRecord(ev, c->stream));
    // whatever happens below (a search_begin that throws half-way included), lanes that were given work are marked for quiesce_alt()
    struct LaneBack { Ctx* c; ~LaneBack() { try { c->switch_lane(0); } catch (...) {} } } lane_back{c};
    bool used[Ctx::kMaxLanes] = {true};
    int rot = 0;
    // newest first, as the reference walks memtables and segments (the order has no effect on the merged result)
    for (int s = S - 1; s >= 0; s--) {
        const int m = std::min(c->lanes, segs[s]->max_lanes());
        const int lane = m > 1 ? (rot++ % m) : 0;
        c->switch_lane(lane);
        if (!used[lane]) { used[lane] = true; c->scratch_reset(); HIP_CHECK(hipStreamWaitEvent(c->stream, ev, 0)); }
        c->mark_dirty();          // before the enqueue: a search_begin that throws has still left kernels on this lane
        tickets[s] = segs[s]->search_begin(queries_dev, B, *p, ids + (size_t)s * B * k, sc + (size_t)s * B * k, cn + (size_t)s * B, k);
    }
    c->switch_lane(0);
    for (int s = S - 1; s >= 0; s--) segs[s]->search_finish(tickets[s]);
    launch_merge_segments(c, ids, sc, cn, S, B, k, k, out_ids, out_scores, out_counts, k_cap);
}
static void check_segments(comet_index* const* segs, int S, int B, const comet_search_params* p, int k_cap) {
    if (!segs || S <= 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "no segments");
    if (!p) COMET_FAIL(COMET_ERR_INVALID_ARG, "null search params");
    if (B < 0 || k_cap <= 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "bad batch size / k_cap");
    if (p->k < 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "k must not be negative (the reference slices merged[:k], storage.go:621-623)");
    for (int s = 0; s < S; s++) {
        if (!segs[s]) COMET_FAIL(COMET_ERR_INVALID_ARG, "null segment %d", s);
        if (segs[s]->c != segs[0]->c) COMET_FAIL(COMET_ERR_INVALID_ARG, "segment %d lives on another context", s);
        if (segs[s]->dim != segs[0]->dim) COMET_FAIL(COMET_ERR_DIM_MISMATCH, "segment %d: dimension %d, expected %d", s, segs[s]->dim, segs[0]->dim);
    }
}
int comet_segments_search_dev(comet_index* const* segs, int32_t S, const float* queries_dev, int32_t B, const comet_search_params* p,
                              uint32_t* out_ids_dev, float* out_scores_dev, int32_t* out_counts_dev, int32_t k_cap) {
    return guarded([&] {
        check_segments(segs, S, B, p, k_cap);
        if (B == 0) return (int)COMET_OK;
        CallGuard g(segs[0]->c);
        segments_search(segs, S, queries_dev, B, p, out_ids_dev, out_scores_dev, out_counts_dev, k_cap);
        return (int)COMET_OK;
    });
}
int comet_segments_search(comet_index* const* segs, int32_t S, const float* queries, int32_t B, const comet_search_params* p,
                          uint32_t* out_ids, float* out_scores, int32_t* out_counts, int32_t k_cap) {
    return guarded([&] {
        check_segments(segs, S, B, p, k_cap);
        if (B == 0) return (int)COMET_OK;
        Ctx* c = segs[0]->c; CallGuard g(c);
        float* dq = c->salloc<float>((size_t)B * segs[0]->dim);
        uint32_t* dids = c->salloc<uint32_t>((size_t)B * k_cap);
        float* dsc = c->salloc<float>((size_t)B * k_cap);
        int32_t* dcn = c->salloc<int32_t>(B);
        c->h2d(dq, queries, (size_t)B * segs[0]->dim * sizeof(float));
        segments_search(segs, S, dq, B, p, dids, dsc, dcn, k_cap);
        c->d2h(out_ids, dids, (size_t)B * k_cap * 4);
        c->d2h(out_scores, dsc, (size_t)B * k_cap * 4);
        c->d2h(out_counts, dcn, (size_t)B * 4);
        c->sync();
        for (int i = 0; i < B; i++) if (out_counts[i] == -(int)COMET_ERR_ZERO_VECTOR)
            COMET_FAIL(COMET_ERR_ZERO_VECTOR, "zero vector not allowed for this metric");   // the memtable search's error is returned (storage.go:537-540)
        return (int)COMET_OK;
    });
}

// lookupNodeVectors (flat_index_search.go:171-196 and siblings): stored vectors of the given node ids, in order
int comet_index_fetch_vectors(comet_index* idx, const uint32_t* ids, int32_t n, float* out_vecs) {
    return guarded([&] {
        if (n <= 0) return (int)COMET_OK;
        Ctx* c = idx->c; CallGuard g(c);
        if (!idx->rows_dev() && idx->size() > 0) COMET_FAIL(COMET_ERR_UNSUPPORTED, "this index kind stores codes, not vectors: node-id queries need the caller's copy of the vector");
        std::vector<int32_t> rows(n);
        for (int i = 0; i < n; i++) {
            const int64_t r = idx->row_of_id(ids[i]);
            if (r < 0) { if (idx->kind == COMET_KIND_HNSW) COMET_FAIL(COMET_ERR_NOT_FOUND, "node ID %u not found or deleted", ids[i]); COMET_FAIL(COMET_ERR_NOT_FOUND, "node ID %u not found in index", ids[i]); }
            if (idx->deleted.count(ids[i])) { if (idx->kind == COMET_KIND_HNSW) COMET_FAIL(COMET_ERR_NOT_FOUND, "node ID %u not found or deleted", ids[i]); COMET_FAIL(COMET_ERR_NOT_FOUND, "node ID %u not found in index (deleted)", ids[i]); }
            rows[i] = (int32_t)r;
        }
        int32_t* dr = c->salloc<int32_t>(n);
        float* padded = c->salloc<float>((size_t)n * idx->ld);
        float* dense = c->salloc<float>((size_t)n * idx->dim);
        c->h2d(dr, rows.data(), (size_t)n * 4);
        launch_gather_rows(c, idx->rows_dev(), idx->ld, dr, n, padded);
        launch_unpad_rows(c, padded, n, idx->ld, dense, idx->dim);
        c->d2h(out_vecs, dense, (size_t)n * idx->dim * 4);
        c->sync();
        return (int)COMET_OK;
    });
}

// ---- multi-GPU list sharding ------------------------------------------------------------------------------
int comet_index_set_shard(comet_index* idx, int32_t rank, int32_t world) {
    return guarded([&] {
        if (world <= 0 || rank < 0 || rank >= world) COMET_FAIL(COMET_ERR_INVALID_ARG, "bad shard: rank %d of %d", rank, world);
        if (idx->kind != COMET_KIND_IVF && idx->kind != COMET_KIND_IVFPQ) COMET_FAIL(COMET_ERR_UNSUPPORTED, "list sharding applies to IVF / IVFPQ indexes (shard Flat / PQ rows on the caller's side)");
        if (idx->size() != 0) COMET_FAIL(COMET_ERR_INVALID_ARG, "set the shard before adding vectors");
        std::lock_guard<std::recursive_mutex> lk(idx->c->mu);
        idx->shard_rank = rank; idx->shard_world = world; idx->owners_checked_on = 0;
        idx->assign_list_owners();          // trained already: lists dealt by their training-set lengths (before training: at the end of Train)
        return (int)COMET_OK;
    });
}
// The placement (which rank owns which list) is host-side state derived from training; it is not part of the reference's on-disk layouts. A host that
// checkpoints a sharded index saves it next to the shard files (get) and hands it to every rank that loads one (set, before the first Add after the load).
int comet_index_get_list_owners(const comet_index* idx, int32_t* out_owners, int32_t n_lists) {
    return guarded([&] {
        if (idx->kind != COMET_KIND_IVF && idx->kind != COMET_KIND_IVFPQ) COMET_FAIL(COMET_ERR_UNSUPPORTED, "list sharding applies to IVF / IVFPQ indexes");
        if (n_lists < 0 || (n_lists > 0 && !out_owners)) COMET_FAIL(COMET_ERR_INVALID_ARG, "bad owner array");
        if (n_lists != idx->n_lists()) COMET_FAIL(COMET_ERR_INVALID_ARG, "the index has %d lists, the owner array %d (owner_of reads past the placement otherwise)", idx->n_lists(), n_lists);
        std::lock_guard<std::recursive_mutex> lk(idx->c->mu);
        for (int32_t l = 0; l < n_lists; l++) out_owners[l] = idx->shard_world > 1 ? idx->owner_of(l) : 0;
        return (int)COMET_OK;
    });
}
int comet_index_set_list_owners(comet_index* idx, const int32_t* owners, int32_t n_lists) {
    return guarded([&] {
        if (idx->kind != COMET_KIND_IVF && idx->kind != COMET_KIND_IVFPQ) COMET_FAIL(COMET_ERR_UNSUPPORTED, "list sharding applies to IVF / IVFPQ indexes");
        if (idx->shard_world <= 1) COMET_FAIL(COMET_ERR_INVALID_ARG, "set the shard (comet_index_set_shard) before the placement");
        if (idx->n_lists() != n_lists || !owners) COMET_FAIL(COMET_ERR_INVALID_ARG, "the placement must name an owner for each of the index's %d lists", idx->n_lists());
        for (int32_t l = 0; l < n_lists; l++) if (owners[l] < 0 || owners[l] >= idx->shard_world) COMET_FAIL(COMET_ERR_INVALID_ARG, "list %d: owner %d is not a rank of %d", l, owners[l], idx->shard_world);
        std::lock_guard<std::recursive_mutex> lk(idx->c->mu);
        idx->train_counts.clear(); idx->list_owner.assign(owners, owners + n_lists); idx->owners_checked_on = 0;
        return (int)COMET_OK;
    });
}

// ---- persistence (io.WriterTo / io.ReaderFrom, index.go:58-60) -----------------------------------------
int comet_index_write_to(comet_index* idx, comet_write_cb cb, void* user, int64_t* out_bytes) {
    return guarded([&] {
        if (out_bytes) *out_bytes = 0;
        if (!cb) COMET_FAIL(COMET_ERR_INVALID_ARG, "null write callback");
        CallGuard g(idx->c);
        Sink s(cb, user);
        try { idx->write_to(s); } catch (...) { if (out_bytes) *out_bytes = s.total; throw; }
        idx->c->sync();
        if (out_bytes) *out_bytes = s.total;
        return (int)COMET_OK;
    });
}
int comet_index_read_from(comet_index* idx, comet_read_cb cb, void* user, int64_t* out_bytes) {
    return guarded([&] {
        if (out_bytes) *out_bytes = 0;
        if (!cb) COMET_FAIL(COMET_ERR_INVALID_ARG, "null read callback");
        CallGuard g(idx->c);
        Source s(cb, user);
        try { idx->read_from(s); } catch (...) { if (out_bytes) *out_bytes = s.total; throw; }
        idx->c->sync();
        if (out_bytes) *out_bytes = s.total;
        return (int)COMET_OK;
    });
}
namespace {
struct BufW { uint8_t* p; size_t cap, len; };
struct BufR { const uint8_t* p; size_t len, off; };
int buf_write(void* u, const void* d, size_t n) { auto* b = (BufW*)u; if (b->p) { if (b->len + n > b->cap) return 1; std::memcpy(b->p + b->len, d, n); } b->len += n; return 0; }
int buf_read(void* u, void* d, size_t n) { auto* b = (BufR*)u; if (b->off + n > b->len) return 1; std::memcpy(d, b->p + b->off, n); b->off += n; return 0; }
}  // namespace
int comet_index_serialize(comet_index* idx, uint8_t* buf, size_t cap, size_t* out_len) {
    BufW w{buf, cap, 0};
    int64_t bytes = 0;
    const int rc = comet_index_write_to(idx, buf_write, &w, &bytes);
    if (out_len) *out_len = w.len;
    if (rc == COMET_ERR_IO) return set_error(COMET_ERR_INVALID_ARG, "buffer too small: %zu bytes given", cap);
    return rc;
}
int comet_index_deserialize(comet_index* idx, const uint8_t* buf, size_t len, size_t* out_consumed) {
    BufR r{buf, len, 0};
    int64_t bytes = 0;
    const int rc = comet_index_read_from(idx, buf_read, &r, &bytes);
    if (out_consumed) *out_consumed = (size_t)bytes;
    return rc;
}

// ---- introspection -----------------------------------------------------------------------------
int comet_index_get_centroids(const comet_index* idx, float* out) { return guarded([&] { CallGuard g(idx->c); idx->get_centroids(out); return (int)COMET_OK; }); }
int comet_index_get_codebooks(const comet_index* idx, float* out) { return guarded([&] { CallGuard g(idx->c); idx->get_codebooks(out); return (int)COMET_OK; }); }
int comet_index_list_size(const comet_index* idx, int32_t list, int64_t* out) { return guarded([&] { *out = idx->list_size(list); return (int)COMET_OK; }); }
int comet_index_list_read(const comet_index* idx, int32_t list, uint32_t* out_ids, uint8_t* out_codes, float* out_vecs) {
    return guarded([&] { CallGuard g(idx->c); idx->list_read(list, out_ids, out_codes, out_vecs); return (int)COMET_OK; });
}

int comet_index_export(const comet_index* idx, uint32_t* out_ids, int32_t* out_lists, uint8_t* out_codes) {
    return guarded([&] { CallGuard g(idx->c); idx->export_all(out_ids, out_lists, out_codes); return (int)COMET_OK; });
}
int comet_index_get_stat(const comet_index* idx, const char* name, double* out) {
    return guarded([&] {
        std::lock_guard<std::recursive_mutex> lk(idx->c->mu); idx->c->bind();      // some statistics are read back from the device
        idx->c->check_indexes("comet_index_get_stat");
        if (idx->shard_stat(name, out)) return (int)COMET_OK;
        if (!idx->get_stat(name, out)) COMET_FAIL(COMET_ERR_INVALID_ARG, "unknown stat '%s'", name);
        return (int)COMET_OK;
    });
}

}  // extern "C"
