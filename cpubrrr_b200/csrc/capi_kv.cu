// C ABI of the KV-cache operators (include/brrr.h): arguments are checked here, lists in device memory by the kernels.
#include "../../include/brrr.h"
#include "brrr_kernels.h"
#include "brrr_kv.cuh"

using namespace brrr;

namespace {

static_assert(KV_TREE_MAX == BRRR_TREE_MAX, "");
constexpr int KV_HEADS_MAX = 512;         // heads x tiles of rows are a grid's second dimension

bool off16(const void *p) { return ((uintptr_t)p & 15) != 0; }
template <class... P>
bool off4(const P *...p) { return ((... | (uintptr_t)p) & 3) != 0; }

// The view for the kernels; false where it describes no cache.
bool view(const brrr_kv *c, KvDev *out) {
    if (!c || !c->k || !c->v || (c->type != BRRR_KV_F32 && c->type != BRRR_KV_BF16)) return false;
    if (c->n_seq <= 0 || c->n_head_kv <= 0 || c->n_head_kv > KV_HEADS_MAX || (c->head_dim != 64 && c->head_dim != 128) || c->cap <= 0 || c->cap > BRRR_KV_CAP_MAX) return false;
    if (off16(c->k) || off16(c->v) || ((uintptr_t)c->weight & 3) || ((uintptr_t)c->pos & 3) || ((uintptr_t)c->err & 3)) return false;
    const int64_t head = (int64_t)c->cap * c->head_dim;
    if (c->head_stride < 0 || c->seq_stride < 0 || c->head_stride % 8 || c->seq_stride % 8) return false;
    KvDev d;
    // heads inside a sequence or sequences inside a head: either way no two rows share memory
    d.hs = c->head_stride && c->n_head_kv > 1 ? c->head_stride : head;
    d.ss = c->seq_stride && c->n_seq > 1 ? c->seq_stride : d.hs * c->n_head_kv;
    const int64_t lo = d.hs < d.ss ? d.hs : d.ss, hi = d.hs < d.ss ? d.ss : d.hs;
    const int64_t inner = d.hs < d.ss ? c->n_head_kv : c->n_seq, outer = d.hs < d.ss ? c->n_seq : c->n_head_kv;
    const __int128 span = (__int128)lo * (inner - 1) + head;         // values of one outer step
    if ((inner > 1 && lo < head) || (outer > 1 && hi < span) || (__int128)hi * (outer - 1) + span > (__int128)1 << 38) return false;      // more than any GPU's memory
    d.k = c->k; d.v = c->v; d.weight = c->weight; d.pos = c->pos; d.err = c->err;
    d.type = c->type; d.n_seq = c->n_seq; d.nkv = c->n_head_kv; d.hd = c->head_dim; d.cap = c->cap;
    *out = d;
    return true;
}

// Pieces of memory of one length, in ascending order: `outer` times `inner` of them, a step apart each (view has seen that they do not overlap).
struct Pieces {
    uintptr_t at;
    int64_t len, inner, inner_step, outer, outer_step;
    int64_t count() const { return inner * outer; }
    uintptr_t piece(int64_t i) const { return at + (uintptr_t)(i / inner * outer_step + i % inner * inner_step); }
    uintptr_t end() const { return at + (uintptr_t)((outer - 1) * outer_step + (inner - 1) * inner_step + len); }
};
Pieces whole(const void *p, int64_t len) { return {(uintptr_t)p, len, 1, len, 1, len}; }
// the heads of k or v; what stands without a gap is one piece
Pieces heads_of(const KvDev &d, const void *p) {
    const int64_t head = (int64_t)d.cap * d.hd * d.size(), hs = d.hs * d.size(), ss = d.ss * d.size();
    Pieces x = d.hs < d.ss ? Pieces{(uintptr_t)p, head, d.nkv, hs, d.n_seq, ss} : Pieces{(uintptr_t)p, head, d.n_seq, ss, d.nkv, hs};
    if (x.inner == 1 || x.inner_step == head) {
        const int64_t run = head * x.inner;
        if (x.outer == 1 || x.outer_step == run) return whole(p, run * x.outer);
        return {x.at, run, 1, run, x.outer, x.outer_step};
    }
    return x;
}
// Whether any two share a byte.  What lies apart as a whole, and two caches of which one has no gaps, take few steps.
bool meet(const Pieces &a, const Pieces &b) {
    if (a.end() <= b.at || b.end() <= a.at) return false;
    for (int64_t i = 0, j = 0; i < a.count() && j < b.count();) {
        const uintptr_t x = a.piece(i), y = b.piece(j);
        if (x + (uintptr_t)a.len <= y) i++;
        else if (y + (uintptr_t)b.len <= x) j++;
        else return true;
    }
    return false;
}

// log2(e) times twice the scale stays in single precision: beyond, a score of zero would be no number
bool scale_ok(float x) { return x >= -BRRR_KV_SCALE_MAX && x <= BRRR_KV_SCALE_MAX; }
bool heads_ok(const KvDev &d, int n_head) { return n_head > 0 && n_head % d.nkv == 0 && n_head / d.nkv <= 16; }

// The memory belongs to the device whose stream the kernels go to: a pointer of another one (or of the host) would fault there.
int on_this_device(const KvDev &d) {
    int dev = -1;
    cudaPointerAttributes at{};
    if (cudaGetDevice(&dev) != cudaSuccess || cudaPointerGetAttributes(&at, d.k) != cudaSuccess) {
        (void)cudaGetLastError();
        return BRRR_ERR_CUDA;
    }
    if (at.type == cudaMemoryTypeManaged) return BRRR_OK;
    return at.type == cudaMemoryTypeDevice && at.device == dev ? BRRR_OK : BRRR_ERR_ARG;
}

int done(cudaError_t e) { return e == cudaSuccess ? BRRR_OK : BRRR_ERR_CUDA; }

}  // namespace

extern "C" int brrr_kv_append(const brrr_kv *kv, int n, int rows, const int32_t *d_seq, const int32_t *d_len, const int32_t *d_count, const int32_t *d_at,
                              const float *d_qkv, int64_t ld, int n_head, const float *d_rope, int n_rope, float *d_q, void *stream) {
    KvDev d;
    if (!view(kv, &d) || !d_len || !d_qkv || off16(d_qkv) || off16(d_q) || ((uintptr_t)d_rope & 15)) return BRRR_ERR_ARG;
    if (n <= 0 || n > 65535 || rows <= 0 || rows > d.cap || n_head < 0 || (n_head > 0 && !heads_ok(d, n_head)) || (d_q && n_head == 0)) return BRRR_ERR_ARG;
    if ((d_rope && n_rope <= 0) || (!d_seq && n > d.n_seq) || off4(d_seq, d_len, d_count, d_at)) return BRRR_ERR_ARG;
    const int64_t width = (int64_t)(n_head + 2 * d.nkv) * d.hd;
    if (ld == 0) ld = width;
    if (ld < width || ld % 4) return BRRR_ERR_ARG;
    if (int rc = on_this_device(d)) return rc;
    return done(launch_kv_append(d, n, rows, d_seq, d_len, d_count, d_at, d_qkv, ld, n_head, d_rope, n_rope, d_q, (cudaStream_t)stream));
}

extern "C" int brrr_attn_tree(const brrr_kv *kv, int n, int rows, const int32_t *d_seq, const int32_t *d_len, const int32_t *d_count, const uint64_t *d_mask,
                              int len_hint, const float *d_q, int n_head, float scale, int window, const float *d_sinks, float *d_out, float *d_lse, void *stream) {
    KvDev d;
    if (!view(kv, &d) || !d_len || !d_q || !d_out || off16(d_q) || off16(d_out) || ((uintptr_t)d_mask & 7)) return BRRR_ERR_ARG;
    if (n <= 0 || n > 65535 || rows <= 0 || rows > BRRR_TREE_MAX || !heads_ok(d, n_head) || window < 0 || (!d_seq && n > d.n_seq)) return BRRR_ERR_ARG;
    if (!scale_ok(scale) || off4(d_seq, d_len, d_count, d_sinks, d_lse)) return BRRR_ERR_ARG;
    if (int rc = on_this_device(d)) return rc;
    const TreeArgs a{n, rows, d_seq, d_len, d_count, d_mask, d_q, n_head, scale, window, d_sinks, d_out, d_lse};
    return done(launch_attn_tree(d, a, len_hint, (cudaStream_t)stream));
}

extern "C" int brrr_kv_commit(const brrr_kv *kv, int n, int rows, const int32_t *d_seq, const int32_t *d_len, const int32_t *d_path, const int32_t *d_npath,
                              int32_t *d_new_len, void *stream) {
    KvDev d;
    if (!view(kv, &d) || !d_len || !d_path || !d_npath || d_new_len == d_len) return BRRR_ERR_ARG;
    if (n <= 0 || n > 65535 || rows <= 0 || rows > BRRR_TREE_MAX || (!d_seq && n > d.n_seq) || off4(d_seq, d_len, d_path, d_npath, d_new_len)) return BRRR_ERR_ARG;
    if (int rc = on_this_device(d)) return rc;
    return done(launch_kv_commit(d, n, rows, d_seq, d_len, d_path, d_npath, d_new_len, (cudaStream_t)stream));
}

extern "C" int brrr_kv_weigh(const brrr_kv *kv, int n, int rows, const int32_t *d_seq, const int32_t *d_len, const int32_t *d_count, const uint64_t *d_mask,
                             const uint64_t *d_rows, int len_hint, const float *d_q, int n_head, float scale, int window, const float *d_lse, void *stream) {
    KvDev d;
    if (!view(kv, &d) || !d.weight || !d_len || !d_q || !d_lse || off16(d_q) || ((uintptr_t)d_mask & 7) || ((uintptr_t)d_rows & 7)) return BRRR_ERR_ARG;
    if (n <= 0 || n > 65535 || rows <= 0 || rows > BRRR_TREE_MAX || !heads_ok(d, n_head) || window < 0 || (!d_seq && n > d.n_seq)) return BRRR_ERR_ARG;
    if (!scale_ok(scale) || off4(d_seq, d_len, d_count, d_lse)) return BRRR_ERR_ARG;
    if (int rc = on_this_device(d)) return rc;
    const TreeArgs a{n, rows, d_seq, d_len, d_count, d_mask, d_q, n_head, scale, window, nullptr, nullptr, const_cast<float *>(d_lse)};
    return done(launch_kv_weigh(d, a, d_rows, len_hint, (cudaStream_t)stream));
}

extern "C" int brrr_kv_evict(const brrr_kv *kv, const brrr_kv *dst, int n, const int32_t *d_seq, const int32_t *d_len, int keep, int first, int recent,
                             const int32_t *d_end, int32_t *d_map, int32_t *d_new_len, int /* len_hint */, void *stream) {
    KvDev d, to;
    if (!view(kv, &d) || !d.weight || !d.pos || !d_len || !d_map || d_new_len == d_len) return BRRR_ERR_ARG;
    if (n <= 0 || n > 65535 || keep <= 0 || keep > d.cap || first < 0 || recent < 0 || first > keep || recent > keep - first) return BRRR_ERR_ARG;
    if ((recent > 0 && !d_end) || (!d_seq && n > d.n_seq) || off4(d_seq, d_len, d_end, d_map, d_new_len)) return BRRR_ERR_ARG;
    if (dst) {
        if (!view(dst, &to) || !to.weight || !to.pos || to.type != d.type || to.nkv != d.nkv || to.hd != d.hd || to.cap < keep || (!d_seq && n > to.n_seq)) return BRRR_ERR_ARG;
        const int64_t x = (int64_t)d.n_seq * d.nkv * d.cap * 4, y = (int64_t)to.n_seq * to.nkv * to.cap * 4;
        const Pieces from[4] = {heads_of(d, d.k), heads_of(d, d.v), whole(d.weight, x), whole(d.pos, x)}, into[4] = {heads_of(to, to.k), heads_of(to, to.v), whole(to.weight, y), whole(to.pos, y)};
        for (auto &f : from)
            for (auto &t : into)
                if (meet(f, t)) return BRRR_ERR_ARG;
    }
    if (int rc = on_this_device(d)) return rc;
    if (dst)
        if (int rc = on_this_device(to)) return rc;
    return done(launch_kv_evict(d, dst ? &to : nullptr, n, d_seq, d_len, keep, first, recent, d_end, d_map, d_new_len, (cudaStream_t)stream));
}

extern "C" int brrr_kv_means(const brrr_kv *kv, int n, const int32_t *d_seq, const int32_t *d_since, const int32_t *d_len, int block, int len_hint, float *d_means,
                             void *stream) {
    KvDev d;
    if (!view(kv, &d) || !d_len || off16(d_means) || (block != 16 && block != 32 && block != 64 && block != 128)) return BRRR_ERR_ARG;
    if (!d_means && d.cap >= block) return BRRR_ERR_ARG;         // a cache shorter than a block has no means
    if (n <= 0 || n > 65535 || (!d_seq && n > d.n_seq) || off4(d_seq, d_since, d_len)) return BRRR_ERR_ARG;
    if (int rc = on_this_device(d)) return rc;
    return done(launch_kv_means(d, n, d_seq, d_since, d_len, block, len_hint, d_means, (cudaStream_t)stream));
}

extern "C" int brrr_attn_blocks(const brrr_kv *kv, int rows, const int32_t *d_seq, const int32_t *d_len, int block, const float *d_means, int nsel, int first,
                                int local, int len_hint, const float *d_q, int n_head, float scale, const float *d_sinks, int32_t *d_sel, float *d_out, float *d_lse,
                                void *stream) {
    KvDev d;
    if (!view(kv, &d) || !d_len || !d_q || !d_sel || !d_out || off16(d_means) || off16(d_q) || off16(d_out)) return BRRR_ERR_ARG;
    if ((block != 16 && block != 32 && block != 64 && block != 128) || (!d_means && d.cap >= block)) return BRRR_ERR_ARG;
    if (rows <= 0 || rows > 65535 || !heads_ok(d, n_head) || nsel <= 0 || nsel > 256 || first < 0 || local < 1 || first > nsel || local > nsel - first) return BRRR_ERR_ARG;
    if ((!d_seq && rows > d.n_seq) || !scale_ok(scale) || off4(d_seq, d_len, d_sinks, d_sel, d_lse)) return BRRR_ERR_ARG;
    if (d.cap / block > 16384) return BRRR_ERR_RANGE;
    if (int rc = on_this_device(d)) return rc;
    return done(launch_attn_blocks(d, rows, d_seq, d_len, block, d_means, nsel, first, local, len_hint, d_q, n_head, scale, d_sinks, d_sel, d_out, d_lse,
                                   (cudaStream_t)stream));
}
