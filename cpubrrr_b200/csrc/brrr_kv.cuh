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
__device__ __forceinline__ uint32_t warp_scan(uint32_t x) {          // sums of this lane and those before it
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if ((int)(threadIdx.x & 31) >= o) x += y;
    }
    return x;
}
// Sum over the threads before this one, and over all; sums: a word per warp.  All threads call it; one barrier inside, and one before sums is used again.
__device__ __forceinline__ uint32_t block_before(uint32_t x, uint32_t *sums, uint32_t &all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t upto = warp_scan(x);
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    const uint32_t of_warps = warp_scan(lane < (int)(blockDim.x >> 5) ? sums[lane] : 0);
    all = __shfl_sync(0xffffffffu, of_warps, 31);
    return upto - x + (warp ? __shfl_sync(0xffffffffu, of_warps, warp - 1) : 0);
}
// Place of the n-th set bit (from 0) of a word that has more.
__device__ __forceinline__ int nth_bit(uint32_t w, int n) {
    int at = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const int c = __popc(w & ((1u << o) - 1));
        if (n >= c) { n -= c; at += o; w >>= o; }
    }
    return at;
}

// Work space of block_kth in shared memory.  BITS at a time: eleven for a block of 1024 (the first hold sign, exponent and two more: fewer counts meet in
// one word), eight for smaller ones (a thread has few words to clear and to add up).
template <int BITS>
struct KthSpace {
    uint32_t hist[1 << BITS], found[2], sums[32];
};
// The key of the k-th largest (1 <= k <= n) of key(0) .. key(n - 1), and how many of the keys that equal it are among the k largest.  All threads call it (at most
// 1 << BITS of them); it ends with a barrier.
template <int BITS, class Key>
__device__ __forceinline__ uint32_t block_kth(int n, uint32_t k, Key key, KthSpace<BITS> &w, uint32_t *ties) {
    uint32_t prefix = 0, known = 0;
    const int each = (1 << BITS) / blockDim.x;
    for (int left = 32; left > 0;) {
        const int shift = max(0, left - BITS);
        const uint32_t digit = (1u << (left - shift)) - 1;
        left = shift;
        for (int i = threadIdx.x; i < 1 << BITS; i += blockDim.x) w.hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const uint32_t x = key(i);
            if ((x & known) == prefix) atomicAdd(&w.hist[x >> shift & digit], 1u);
        }
        __syncthreads();
        // thread i: `each` digits, the largest first
        const int top = (1 << BITS) - 1 - threadIdx.x * each;
        uint32_t sum = 0;
        for (int j = 0; j < each; j++) sum += w.hist[top - j];
        uint32_t all;
        uint32_t above = block_before(sum, w.sums, all);
        const uint32_t upto = above + sum;
        if (above < k && k <= upto)
            for (int j = 0; j < each; j++) {
                const uint32_t c = w.hist[top - j];
                if (above < k && k <= above + c) { w.found[0] = top - j; w.found[1] = k - above; }
                above += c;
            }
        __syncthreads();
        prefix |= w.found[0] << shift;
        known |= digit << shift;
        k = w.found[1];
        __syncthreads();
    }
    *ties = k;
    return prefix;
}

}  // namespace brrr
