// KV caches: append of rotated rows, commit of an accepted path, eviction by weight, block means.
#include "brrr_kernels.h"
#include "brrr_block.cuh"
#include "brrr_kv.cuh"

#include <cuda_bf16.h>

namespace brrr {

// four values of a cache row
__device__ __forceinline__ void kv_store4(void *p, int type, long long at, float4 x) {
    if (type) {
        ushort4 u;
        auto r = [](float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); };
        u.x = r(x.x); u.y = r(x.y); u.z = r(x.z); u.w = r(x.w);
        *reinterpret_cast<ushort4 *>((uint16_t *)p + at) = u;
    } else {
        *reinterpret_cast<float4 *>((float *)p + at) = x;
    }
}

// ---------------------------------------------------------------- append
// A CTA per row.  A thread turns four pairs (j, j + hd / 2): products and sums rounded one by one, as the engines rotate.
__global__ void kv_append_kernel(KvDev kv, int rows, const int32_t *seq, const int32_t *len, const int32_t *count, const int32_t *at,
                                 const float *__restrict__ qkv, long long ld, int nh, const float *__restrict__ rope, int n_rope, float *__restrict__ q) {
    const int i = blockIdx.x, b = blockIdx.y;
    const KvEntry e = kv_entry(kv, b, rows, seq, len, count);
    if (kv_named_before(seq, b) || !e.ok) {
        if (threadIdx.x == 0) kv_error(kv);
        return;
    }
    if (i >= e.count) return;
    const int slot = e.len + i, p = at ? at[(long long)b * rows + i] : slot;
    if (rope && (unsigned)p >= (unsigned)n_rope) {
        if (threadIdx.x == 0) kv_error(kv);
        return;
    }
    const int half = kv.hd / 2, per = half / 4;
    const float *x = qkv + ((long long)b * rows + i) * ld;
    float *qo = q ? q + ((long long)b * rows + i) * nh * kv.hd : nullptr;
    for (int u = threadIdx.x + (q ? 0 : nh * per); u < (nh + 2 * kv.nkv) * per; u += blockDim.x) {
        const int head = u / per, j = u % per * 4;
        float4 lo = *reinterpret_cast<const float4 *>(x + head * kv.hd + j), hi = *reinterpret_cast<const float4 *>(x + head * kv.hd + half + j);
        if (rope && head < nh + kv.nkv) {
            const float4 t0 = *reinterpret_cast<const float4 *>(rope + ((long long)p * half + j) * 2), t1 = *reinterpret_cast<const float4 *>(rope + ((long long)p * half + j) * 2 + 4);
            auto turn = [](float &a, float &b, float c, float s) {
                const float y = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
                b = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
                a = y;
            };
            turn(lo.x, hi.x, t0.x, t0.y); turn(lo.y, hi.y, t0.z, t0.w); turn(lo.z, hi.z, t1.x, t1.y); turn(lo.w, hi.w, t1.z, t1.w);
        }
        if (head < nh) {
            *reinterpret_cast<float4 *>(qo + head * kv.hd + j) = lo;
            *reinterpret_cast<float4 *>(qo + head * kv.hd + half + j) = hi;
        } else {
            const int kvh = (head - nh) % kv.nkv;
            const long long row = kv.head(e.seq, kvh) + (long long)slot * kv.hd;
            void *dst = head < nh + kv.nkv ? kv.k : kv.v;
            kv_store4(dst, kv.type, row + j, lo);
            kv_store4(dst, kv.type, row + half + j, hi);
        }
    }
    for (int h = threadIdx.x; h < kv.nkv; h += blockDim.x) {
        if (kv.weight) kv.weight[kv.book(e.seq, h) + slot] = 0.0f;
        if (kv.pos) kv.pos[kv.book(e.seq, h) + slot] = p;
    }
}

cudaError_t launch_kv_append(const KvDev &kv, int n, int rows, const int32_t *seq, const int32_t *len, const int32_t *count, const int32_t *at, const float *qkv,
                             long long ld, int nh, const float *rope, int n_rope, float *q, cudaStream_t st) {
    kv_append_kernel<<<dim3(rows, n), 256, 0, st>>>(kv, rows, seq, len, count, at, qkv, ld, nh, rope, n_rope, q);
    return cudaGetLastError();
}

// ---------------------------------------------------------------- commit
// A CTA per (kv head, entry, K or V): the path's rows are all read before the first is written.
constexpr int CM_THREADS = 256;
__global__ void __launch_bounds__(CM_THREADS) kv_commit_kernel(KvDev kv, int rows, const int32_t *seq, const int32_t *len, const int32_t *path, const int32_t *npath,
                                                               int32_t *new_len) {
    const int kvh = blockIdx.x, b = blockIdx.y;
    const KvEntry e = kv_entry(kv, b, rows, seq, len, npath);
    bool bad = kv_named_before(seq, b) || !e.ok;
    if (!bad) {
        bool off = false;
        for (int i = threadIdx.x; i < e.count; i += CM_THREADS) off |= (unsigned)path[(long long)b * rows + i] >= (unsigned)min(rows, kv.cap - e.len);
        bad = __syncthreads_or(off);
    }
    if (threadIdx.x == 0 && kvh == 0 && blockIdx.z == 0) {
        if (bad) kv_error(kv);
        if (new_len) new_len[b] = e.len + (bad ? 0 : e.count);
    }
    if (bad) return;
    const int per = kv.hd * kv.size() / 16, units = e.count * per;       // at most 64 x 32
    uint4 *base = reinterpret_cast<uint4 *>((char *)(blockIdx.z ? kv.v : kv.k) + kv.head(e.seq, kvh) * kv.size()) + (long long)e.len * per;
    uint4 x[KV_TREE_MAX * 32 / CM_THREADS];
#pragma unroll
    for (int c = 0; c < KV_TREE_MAX * 32 / CM_THREADS; c++) {
        const int u = threadIdx.x + c * CM_THREADS;
        if (u < units) x[c] = base[path[(long long)b * rows + u / per] * per + u % per];
    }
    float w = 0.0f;
    int32_t p = 0;
    const long long book = kv.book(e.seq, kvh) + e.len;
    const bool books = blockIdx.z == 0 && (int)threadIdx.x < e.count;
    if (books) {
        const int from = path[(long long)b * rows + threadIdx.x];
        if (kv.weight) w = kv.weight[book + from];
        if (kv.pos) p = kv.pos[book + from];
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < KV_TREE_MAX * 32 / CM_THREADS; c++) {
        const int u = threadIdx.x + c * CM_THREADS;
        if (u < units) base[u] = x[c];
    }
    if (books) {
        if (kv.weight) kv.weight[book + threadIdx.x] = w;
        if (kv.pos) kv.pos[book + threadIdx.x] = p;
    }
}

cudaError_t launch_kv_commit(const KvDev &kv, int n, int rows, const int32_t *seq, const int32_t *len, const int32_t *path, const int32_t *npath, int32_t *new_len,
                             cudaStream_t st) {
    kv_commit_kernel<<<dim3(kv.nkv, n, 2), CM_THREADS, 0, st>>>(kv, rows, seq, len, path, npath, new_len);
    return cudaGetLastError();
}

// ---------------------------------------------------------------- eviction
// Which entries stay: a CTA per (kv head, entry) finds the key of the last one kept digit by digit (four counts of 256 digits), then turns the
// keys into one bit per slot, and pairs the freed slots below m with the kept entries behind.  Bits and running counts per 32 slots stand
// in shared memory.
constexpr int EV_THREADS = 1024;

// protected entries above all weights, NaN below all, -0 as +0
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int first, long long from) {
    if (pos < first || pos >= from) return 0xFFFFFFFFu;
    if (w != w) return 0u;
    return float_orderable(w == 0.0f ? 0.0f : w);
}

// Exclusive running sums of v[0 .. n), in place; returns the total.  All threads call it; v is complete afterwards.
__device__ __forceinline__ uint32_t block_scan(uint32_t *v, int n, uint32_t *warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
    uint32_t carry = 0;
    for (int at = 0; at < n; at += blockDim.x) {
        const int i = at + threadIdx.x;
        const uint32_t x = i < n ? v[i] : 0;
        uint32_t s = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        if (lane == 31) warp_sums[warp] = s;
        __syncthreads();
        uint32_t before = 0, all = 0;
        for (int w = 0; w < nwarp; w++) {
            const uint32_t y = warp_sums[w];
            if (w < warp) before += y;
            all += y;
        }
        if (i < n) v[i] = carry + before + s - x;
        carry += all;
        __syncthreads();
    }
    return carry;
}

// The key of the k-th largest (1 <= k <= n) of key(0) .. key(n - 1), and how many of the keys that equal it are among the k largest.
template <class Key>
__device__ __forceinline__ uint32_t block_kth(int n, uint32_t k, Key key, uint32_t *hist, uint32_t *found, uint32_t *ties) {
    uint32_t prefix = 0, known = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += blockDim.x) hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const uint32_t x = key(i);
            if ((x & known) == prefix) atomicAdd(&hist[x >> shift & 255], 1u);
        }
        __syncthreads();
        if (threadIdx.x < 32) {
            // lane l: digits 255 - 8 l .. 248 - 8 l, from the largest
            uint32_t c[8], sum = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) { c[j] = hist[255 - 8 * threadIdx.x - j]; sum += c[j]; }
            uint32_t upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
                if ((int)threadIdx.x >= o) upto += y;
            }
            uint32_t above = upto - sum;
            if (above < k && k <= upto) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (above < k && k <= above + c[j]) { found[0] = 255 - 8 * threadIdx.x - j; found[1] = k - above; }
                    above += c[j];
                }
            }
        }
        __syncthreads();
        prefix |= found[0] << shift;
        known |= 255u << shift;
        k = found[1];
        __syncthreads();
    }
    *ties = k;
    return prefix;
}

__global__ void __launch_bounds__(EV_THREADS) kv_evict_kernel(KvDev kv, KvDev dst, int rows, const int32_t *seq, const int32_t *len, int keep, int first, int recent,
                                                              const int32_t *end, int32_t *map, int32_t *new_len) {
    extern __shared__ uint32_t sm[];
    __shared__ uint32_t hist[256], found[2], sums[32];
    const int kvh = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = EV_THREADS / 32;
    const KvEntry e = kv_entry(kv, b, 0, seq, len, nullptr);
    const bool bad = kv_named_before(seq, b) || !e.ok || e.seq >= dst.n_seq;
    int32_t *out = map + ((long long)b * kv.nkv + kvh) * keep;
    const int m = min(e.len, keep);
    if (threadIdx.x == 0 && kvh == 0) {
        if (bad) kv_error(kv);
        if (new_len) new_len[b] = bad ? e.len : m;
    }
    if (bad) {
        for (int t = threadIdx.x; t < keep; t += EV_THREADS) out[t] = -1;
        return;
    }
    for (int t = m + threadIdx.x; t < keep; t += EV_THREADS) out[t] = -1;
    if (e.len <= keep) {
        for (int t = threadIdx.x; t < m; t += EV_THREADS) out[t] = t;
        return;
    }
    const float *w = kv.weight + kv.book(e.seq, kvh);
    const int32_t *pos = kv.pos + kv.book(e.seq, kvh);
    const long long from = recent > 0 ? (long long)end[b] - recent : 1ll << 31;
    auto key = [&](int t) { return evict_key(w[t], pos[t], first, from); };
    uint32_t ties;
    const uint32_t last = block_kth(e.len, m, key, hist, found, &ties);
    const int words = (e.len + 31) / 32, mw = m / 32;
    uint32_t *kept = sm, *run = sm + words;      // bits of 32 slots each; running counts [words + 1]
    for (int i = warp; i < words; i += nwarp) {
        const int t = i * 32 + lane;
        const uint32_t x = t < e.len ? key(t) : 0;
        const uint32_t over = __ballot_sync(0xffffffffu, t < e.len && x > last), same = __ballot_sync(0xffffffffu, t < e.len && x == last);
        if (lane == 0) { kept[i] = over; run[i] = __popc(same); }
    }
    __syncthreads();
    block_scan(run, words, sums);
    for (int i = warp; i < words; i += nwarp) {
        const int t = i * 32 + lane;
        const bool same = t < e.len && key(t) == last;
        const uint32_t all = __ballot_sync(0xffffffffu, same);
        const uint32_t mine = __ballot_sync(0xffffffffu, same && run[i] + __popc(all & ((1u << lane) - 1)) < ties);
        if (lane == 0) kept[i] |= mine;
    }
    __syncthreads();
    // freed slots below m per word 0 .. mw, then kept ones behind per word mw .. words - 1 (one place further on)
    const uint32_t low = (1u << (m & 31)) - 1;
    for (int i = threadIdx.x; i <= words; i += EV_THREADS) {
        if (i < mw) run[i] = __popc(~kept[i]);
        else if (i == mw) run[i] = __popc(~kept[i] & low);
        else run[i] = __popc(i - 1 == mw ? kept[i - 1] & ~low : kept[i - 1]);
    }
    __syncthreads();
    block_scan(run, mw + 1, sums);
    block_scan(run + mw + 1, words - mw, sums);
    for (int i = warp; i < words; i += nwarp) {
        const int t = i * 32 + lane;
        if (!(kept[i] >> lane & 1)) continue;
        if (t < m) { out[t] = t; continue; }
        const uint32_t j = run[i + 1] + __popc((i == mw ? kept[i] & ~low : kept[i]) & ((1u << lane) - 1));       // the j-th kept entry behind takes the j-th freed slot
        int lo = 0, hi = mw;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (run[mid] <= j) lo = mid;
            else hi = mid - 1;
        }
        uint32_t holes = ~kept[lo] & (lo == mw ? low : 0xffffffffu);
        for (uint32_t s = j - run[lo]; s > 0; s--) holes &= holes - 1;
        out[lo * 32 + __ffs(holes) - 1] = t;
    }
}

// 16 bytes per thread and step; entry rows of K and V, the books with the first unit
__global__ void __launch_bounds__(256) kv_move_kernel(KvDev kv, KvDev dst, bool inplace, const int32_t *seq, int keep, const int32_t *map) {
    const int kvh = blockIdx.y, b = blockIdx.z, per = kv.hd * kv.size() / 16;
    const int s = seq ? seq[b] : b;
    const int32_t *from = map + ((long long)b * kv.nkv + kvh) * keep;
    if (from[0] < 0 || (unsigned)s >= (unsigned)kv.n_seq || s >= dst.n_seq) return;       // an entry that was left out, or an empty one
    const uint4 *k = reinterpret_cast<const uint4 *>((const char *)kv.k + kv.head(s, kvh) * kv.size()), *v = reinterpret_cast<const uint4 *>((const char *)kv.v + kv.head(s, kvh) * kv.size());
    uint4 *k2 = reinterpret_cast<uint4 *>((char *)dst.k + dst.head(s, kvh) * dst.size()), *v2 = reinterpret_cast<uint4 *>((char *)dst.v + dst.head(s, kvh) * dst.size());
    const long long book = kv.book(s, kvh), book2 = dst.book(s, kvh);
    for (long long u = blockIdx.x * 256ll + threadIdx.x; u < (long long)keep * per; u += gridDim.x * 256ll) {
        const int d = (int)(u / per), c = (int)(u % per), t = from[d];
        if (t < 0 || (inplace && t == d)) continue;
        k2[(long long)d * per + c] = k[(long long)t * per + c];
        v2[(long long)d * per + c] = v[(long long)t * per + c];
        if (c == 0) { dst.weight[book2 + d] = kv.weight[book + t]; dst.pos[book2 + d] = kv.pos[book + t]; }
    }
}

cudaError_t launch_kv_evict(const KvDev &kv, const KvDev *dst, int n, const int32_t *seq, const int32_t *len, int keep, int first, int recent, const int32_t *end,
                            int32_t *map, int32_t *new_len, int len_hint, cudaStream_t st) {
    const KvDev &to = dst ? *dst : kv;
    const size_t smem = ((size_t)(kv.cap + 31) / 32 * 2 + 1) * 4;
    cudaError_t e = smem > 48 * 1024 ? cudaFuncSetAttribute(kv_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) : cudaSuccess;
    if (e != cudaSuccess) return e;
    kv_evict_kernel<<<dim3(kv.nkv, n), EV_THREADS, smem, st>>>(kv, to, 0, seq, len, keep, first, recent, end, map, new_len);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const long long units = (long long)keep * (kv.hd * kv.size() / 16);
    const int chunks = (int)min(max(units / 1024, 1ll), 1024ll);
    kv_move_kernel<<<dim3(chunks, kv.nkv, n), 256, 0, st>>>(kv, to, dst == nullptr, seq, keep, map);
    return cudaGetLastError();
}

// ---------------------------------------------------------------- block means
// A thread sums one dimension of a block in double precision.
__global__ void kv_means_kernel(KvDev kv, const int32_t *seq, const int32_t *since, const int32_t *len, int block, float *__restrict__ means) {
    const int kvh = blockIdx.y, b = blockIdx.z;
    const KvEntry e = kv_entry(kv, b, 0, seq, len, nullptr);
    const int s0 = since ? since[b] : 0;
    if (kv_named_before(seq, b) || !e.ok || s0 < 0) {
        if (threadIdx.x == 0) kv_error(kv);
        return;
    }
    const int d = threadIdx.x;
    const long long head = kv.head(e.seq, kvh);
    float *out = means + ((long long)e.seq * kv.nkv + kvh) * (kv.cap / block) * kv.hd;
    for (int j = s0 / block + blockIdx.x; j < e.len / block; j += gridDim.x) {
        double sum = 0.0;
        for (int t = 0; t < block; t++) {
            const long long at = head + (long long)(j * block + t) * kv.hd + d;
            sum += kv.type ? (double)brrr_bf16_to_f32(((const uint16_t *)kv.k)[at]) : (double)((const float *)kv.k)[at];
        }
        out[(long long)j * kv.hd + d] = (float)(sum / block);
    }
}

cudaError_t launch_kv_means(const KvDev &kv, int n, const int32_t *seq, const int32_t *since, const int32_t *len, int block, int len_hint, float *means, cudaStream_t st) {
    const int blocks = max(1, min((len_hint > 0 ? min(len_hint, kv.cap) : kv.cap) / block + 1, 4096));
    kv_means_kernel<<<dim3(blocks, kv.nkv, n), kv.hd, 0, st>>>(kv, seq, since, len, block, means);
    return cudaGetLastError();
}

}  // namespace brrr
