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

// Work space of block_kth in shared memory, for blocks of 1 << (BITS - 1) threads: a warp has 64 digits.
template <int BITS>
struct KthSpace {
    alignas(8) uint32_t hist[3][1 << BITS];
    uint32_t sums[32], of_warps[32];                // of_warps: the caller's
    __device__ __forceinline__ void clear() {       // before a barrier before block_kth
        for (int i = threadIdx.x; i < 3 << BITS; i += blockDim.x) hist[0][i] = 0;
    }
};
// Of the k-th largest (1 <= k <= n) of key(0) .. key(n - 1) the leading bits, `known` of them, that tell it from the others; how many of the keys with these
// bits are among the k largest, and how many there are: as many, or all bits are known.  All threads call it.  BITS bits at a time, the highest first: counts of the
// digits among the keys that agree with what is known, sums per warp of 64 digits, then every warp finds the digit for itself.  Two barriers a digit: counts
// stand in three places in turn, of which the one after the next is cleared.
template <int BITS, class Key>
__device__ __forceinline__ uint32_t block_kth(int n, uint32_t k, Key key, KthSpace<BITS> &w, uint32_t &known, uint32_t &ties, uint32_t &equal) {
    constexpr int B = 1 << BITS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t prefix = 0;
    known = 0;
    equal = ~0u;
    uint32_t *hist = w.hist[0], *next = w.hist[1], *after = w.hist[2];
    for (int left = 32; left > 0 && k != equal;) {
        const int shift = max(0, left - BITS);
        const uint32_t mask = (1u << (left - shift)) - 1;
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const uint32_t x = key(i);
            if ((x & known) == prefix) atomicAdd(&hist[x >> shift & mask], 1u);
        }
        __syncthreads();
        if (left < 32)
            for (int i = threadIdx.x; i < B; i += blockDim.x) after[i] = 0;
        // digits B - 1 - 64 warp - 2 lane (the larger one: y) and the one below
        uint2 c = *reinterpret_cast<const uint2 *>(&hist[B - 2 - 64 * warp - 2 * lane]);
        const uint32_t all = __reduce_add_sync(0xffffffffu, c.x + c.y);
        if (lane == 0) w.sums[warp] = all;
        __syncthreads();
        const uint32_t of_warp = lane < (int)(blockDim.x >> 5) ? w.sums[lane] : 0, upto = warp_scan(of_warp);
        const int at = __ffs(__ballot_sync(0xffffffffu, upto >= k)) - 1;
        k -= __shfl_sync(0xffffffffu, upto - of_warp, at);
        c = *reinterpret_cast<const uint2 *>(&hist[B - 2 - 64 * at - 2 * lane]);
        const uint32_t to = warp_scan(c.x + c.y), before = to - c.x - c.y;
        const int hit = __ffs(__ballot_sync(0xffffffffu, to >= k)) - 1;
        const bool lower = before + c.y < k;
        const uint32_t digit = __shfl_sync(0xffffffffu, (uint32_t)(B - 1 - 64 * at - 2 * lane) - (lower ? 1u : 0u), hit);
        k -= __shfl_sync(0xffffffffu, before + (lower ? c.y : 0u), hit);
        equal = __shfl_sync(0xffffffffu, lower ? c.x : c.y, hit);
        prefix |= digit << shift;
        known |= mask << shift;
        left = shift;
        uint32_t *old = hist;
        hist = next; next = after; after = old;
    }
    ties = k;
    return prefix;
}

}  // namespace brrr
