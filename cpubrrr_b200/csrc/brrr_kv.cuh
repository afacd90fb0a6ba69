// KV caches that the caller owns: what the kernels of draft trees, eviction and chosen blocks know of them.
#pragma once
#include "brrr_dev.cuh"

namespace brrr {

constexpr int KV_TREE_MAX = 64;       // rows per entry (same value as BRRR_TREE_MAX)

struct KvDev {
    void *k, *v;
    float *weight;
    int32_t *pos, *err;
    long long hs, ss;                 // values from one head to the next, from one sequence to the next
    int type, n_seq, nkv, hd, cap;
    __host__ __device__ __forceinline__ int size() const { return type ? 2 : 4; }
    __host__ __device__ __forceinline__ long long head(int seq, int kvh) const { return seq * ss + kvh * hs; }            // of k and v, in values
    __host__ __device__ __forceinline__ long long book(int seq, int kvh) const { return ((long long)seq * nkv + kvh) * cap; }      // of weight and pos
};

// One entry of a call's lists, checked against the cache.
struct KvEntry {
    int seq, len, count;
    bool ok;
};
__device__ __forceinline__ KvEntry kv_entry(const KvDev &kv, int b, int rows, const int32_t *seq, const int32_t *len, const int32_t *count) {
    KvEntry e;
    e.seq = seq ? seq[b] : b;
    e.len = len[b];
    e.count = count ? count[b] : rows;
    e.ok = (unsigned)e.seq < (unsigned)kv.n_seq && (unsigned)e.len <= (unsigned)kv.cap && (unsigned)e.count <= (unsigned)rows &&
           e.count <= kv.cap - e.len;
    return e;
}
__device__ __forceinline__ void kv_error(const KvDev &kv) {
    if (kv.err) *kv.err = 1;
}
// Whether an entry before b names the same sequence.  All threads of the block call it.
__device__ __forceinline__ bool kv_named_before(const int32_t *seq, int b) {
    if (!seq) return false;
    bool again = false;
    const int mine = seq[b];
    for (int i = threadIdx.x; i < b; i += blockDim.x) again |= seq[i] == mine;
    return __syncthreads_or(again);
}

struct TreeArgs {
    int n, rows;
    const int32_t *seq, *len, *count;
    const uint64_t *mask;
    const float *q;
    int nh;
    float scale;
    int window;
    const float *sinks;
    float *out, *lse;
};
// Masks (rows behind count cut off) and depths of an entry's rows, in shared memory; all threads call it, a barrier follows.
__device__ __forceinline__ void tree_masks(const uint64_t *mask, int b, int rows, int count, uint64_t *m, int *depth) {
    for (int i = threadIdx.x; i < count; i += blockDim.x) {
        const uint64_t upto = i == 63 ? ~0ull : (1ull << (i + 1)) - 1, live = count == 64 ? ~0ull : (1ull << count) - 1;
        const uint64_t x = (mask ? mask[(long long)b * rows + i] : upto) & live;
        m[i] = x;
        depth[i] = __popcll(x & ~(1ull << i));
    }
}
// Whether row i sees slot t < len + count.
__device__ __forceinline__ bool tree_sees(const uint64_t *m, const int *depth, int len, int window, int i, int t) {
    if (t < len) return window <= 0 || t >= len + depth[i] + 1 - window;
    const int j = t - len;
    return (m[i] >> j & 1) && (window <= 0 || depth[i] - depth[j] < window);
}

}  // namespace brrr
