// KV caches: append of rotated rows, commit of an accepted path, eviction by weight, block means.
#include "brrr_kernels.h"
#include "brrr_block.cuh"
#include "brrr_kv.cuh"
#include "brrr_tma.cuh"

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
// A CTA per row.  A thread turns four pairs (j, j + hd / 2): products and sums rounded one by one, as the engines rotate.  65 rows of 64 + 2 x 8 heads take
// 5.5 us, 12 rows 5.2 (launched alone): the latency of the lists, then of the row; the bytes would take 0.5 us.
__global__ void kv_append_kernel(KvDev kv, int rows, const int32_t *seq, const int32_t *len, const int32_t *count, const int32_t *at,
                                 const float *__restrict__ qkv, long long ld, int nh, const float *__restrict__ rope, int n_rope, float *__restrict__ q) {
    const int i = blockIdx.x, b = blockIdx.y, half = kv.hd / 2, per = half / 4;
    pdl_wait();
    pdl_trigger();
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
    const float *x = qkv + ((long long)b * rows + i) * ld;
    float *qo = q ? q + ((long long)b * rows + i) * nh * kv.hd : nullptr;
#pragma unroll 2
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
    return launch_k(kv_append_kernel, dim3(rows, n), dim3(512), 0, st, true, kv, rows, seq, len, count, at, qkv, ld, nh, rope, n_rope, q);
}

// ---------------------------------------------------------------- commit
// A CTA per (kv head, entry, K or V): the path's rows are all read before the first is written.  Five paths: 4.5 us, the latency of path, length and rows in turn.
constexpr int CM_THREADS = 256;
__global__ void __launch_bounds__(CM_THREADS) kv_commit_kernel(KvDev kv, int rows, const int32_t *seq, const int32_t *len, const int32_t *path, const int32_t *npath,
                                                               int32_t *new_len) {
    const int kvh = blockIdx.x, b = blockIdx.y;
    pdl_wait();
    pdl_trigger();
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
    return launch_k(kv_commit_kernel, dim3(kv.nkv, n, 2), dim3(CM_THREADS), 0, st, true, kv, rows, seq, len, path, npath, new_len);
}

// ---------------------------------------------------------------- eviction
// Which entries stay: a CTA per (kv head, entry) finds the key of the last one kept digit by digit, then turns the keys into one bit per slot, and pairs the
// freed slots below m with the kept entries behind: by a list of these where the keys stood, by searches in the running counts where there is no such room.  Bits
// and running counts per 32 slots stand in shared memory, and the keys where there is room for a cache's (46,000 slots; above, they are formed from the books again
// at every pass).  Bound by barriers and dependent reads, not by bytes: launched alone 11.6 us for 8 heads x 4096 entries, 12.1 for 128 heads of 32 caches x 3900.
// A whole eviction from one cache took 19.4 us with sums by walking, 15.2 with five barriers a digit, 12.8 with pairs by two searches, 12.1 with a list; counting
// the protected entries takes 0.2 more.  512 threads took 13.8 and 18.9 us for the two cases in an earlier form of this kernel that took 12.9 and 15.1.
constexpr int EV_THREADS = 1024;

// Protected entries above all weights, NaN below all, -0 as +0.  crowded: more entries are protected than are kept, so these alone are in question, by their
// weights (NaN: 1), and the others are below.
constexpr uint32_t EV_SAFE = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int first, long long from, bool crowded) {
    const bool safe = pos < first || pos >= from;
    const uint32_t of_weight = w != w ? 0u : float_orderable(w == 0.0f ? 0.0f : w);
    if (crowded) return safe ? max(of_weight, 1u) : 0u;
    return safe ? EV_SAFE : of_weight;
}

// Exclusive running sums of v[0 .. n), in place; returns the total.  All threads call it; v is complete afterwards.
__device__ __forceinline__ uint32_t block_scan(uint32_t *v, int n, uint32_t *warp_sums) {
    uint32_t carry = 0;
    for (int at = 0; at < n; at += blockDim.x) {
        const int i = at + threadIdx.x;
        uint32_t all;
        const uint32_t before = block_before(i < n ? v[i] : 0, warp_sums, all);
        if (i < n) v[i] = carry + before;
        carry += all;
        __syncthreads();
    }
    return carry;
}
// The last i of v[0 .. n) with v[i] <= x; v[0] is, and v does not fall.
__device__ __forceinline__ int last_upto(const uint32_t *v, int n, uint32_t x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (v[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <bool KEEP_KEYS>
__global__ void __launch_bounds__(EV_THREADS) kv_evict_kernel(KvDev kv, KvDev dst, const int32_t *seq, const int32_t *len, int keep, int first, int recent,
                                                              const int32_t *end, int32_t *map, int32_t *new_len) {
    extern __shared__ uint32_t sm[];
    __shared__ KthSpace<11> kth;
    kth.clear();
    pdl_wait();
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
    const int words = (e.len + 31) / 32, mw = m / 32;
    uint32_t *kept = sm, *run = sm + words, *same_of = run + words + 1, *keys = same_of + words;
    // a thread has slots t, t + EV_THREADS, ... throughout: nobody else reads its keys
    uint32_t safe = 0;
#pragma unroll 4
    for (int t = threadIdx.x; t < e.len; t += EV_THREADS) {
        const uint32_t x = evict_key(KEEP_KEYS ? w[t] : 0.0f, pos[t], first, from, false);
        if (KEEP_KEYS) keys[t] = x;
        safe += x == EV_SAFE;
    }
    safe = __reduce_add_sync(0xffffffffu, safe);
    if (lane == 0) kth.of_warps[warp] = safe;
    __syncthreads();
    const bool crowded = __reduce_add_sync(0xffffffffu, kth.of_warps[lane]) > (uint32_t)m;
    static_assert(EV_THREADS == 32 * 32, "a word per warp, a lane per word");
    if (KEEP_KEYS && crowded)
        for (int t = threadIdx.x; t < e.len; t += EV_THREADS) keys[t] = evict_key(w[t], pos[t], first, from, true);
    auto key = [&](int t) { return KEEP_KEYS ? keys[t] : evict_key(w[t], pos[t], first, from, crowded); };
    uint32_t known, ties, equal;
    const uint32_t last = block_kth(e.len, m, key, kth, known, ties, equal), below = (1u << lane) - 1;
    if (ties < equal) {              // of those with the last one's key the lower slots: how many are before each word
        for (int i = warp; i < words; i += nwarp) {
            const int t = i * 32 + lane;
            const uint32_t same = __ballot_sync(0xffffffffu, t < e.len && key(t) == last);          // all bits are known
            if (lane == 0) same_of[i] = __popc(same);
        }
        __syncthreads();
        block_scan(same_of, words, kth.of_warps);
    }
    // kept: bits of 32 slots each; run: freed slots below m of words 0 .. mw, then kept ones behind of words mw .. words - 1 (one place further on)
    const uint32_t low = (1u << (m & 31)) - 1;
    for (int i = warp; i < words; i += nwarp) {
        const int t = i * 32 + lane;
        const uint32_t x = t < e.len ? key(t) & known : 0;
        const uint32_t over = __ballot_sync(0xffffffffu, t < e.len && x > last);
        uint32_t same = __ballot_sync(0xffffffffu, t < e.len && x == last);
        if (ties < equal) same = __ballot_sync(0xffffffffu, (same >> lane & 1) && same_of[i] + __popc(same & below) < ties);
        if (lane == 0) {
            const uint32_t in = over | same;
            kept[i] = in;
            if (i <= mw) run[i] = __popc(~in & (i == mw ? low : 0xffffffffu));
            if (i >= mw) run[i + 1] = __popc(in & (i == mw ? ~low : 0xffffffffu));
        }
    }
    __syncthreads();
    pdl_trigger();
    block_scan(run, words + 1, kth.of_warps);
    const int moved = (int)run[mw + 1];           // as many are freed as are kept behind
    // the j-th kept entry behind takes the j-th freed slot
    if constexpr (KEEP_KEYS) {
        uint32_t *behind = keys;                  // which nobody needs any more
        for (int t = mw * 32 + threadIdx.x; t < e.len; t += EV_THREADS) {
            const int i = t >> 5;
            const uint32_t in = i == mw ? kept[i] & ~low : kept[i];
            if (in >> (t & 31) & 1) behind[run[i + 1] - moved + __popc(in & below)] = t;
        }
        __syncthreads();
        for (int t = threadIdx.x; t < m; t += EV_THREADS) {
            const uint32_t in = kept[t >> 5];
            out[t] = in >> lane & 1 ? t : behind[run[t >> 5] + __popc(~in & below)];
        }
    } else {
        for (int t = threadIdx.x; t < m; t += EV_THREADS)
            if (kept[t >> 5] >> lane & 1) out[t] = t;
        for (int j = threadIdx.x; j < moved; j += EV_THREADS) {
            const int h = last_upto(run, mw + 1, j), f = mw + last_upto(run + mw + 1, words - mw, moved + j);
            const uint32_t holes = ~kept[h] & (h == mw ? low : 0xffffffffu), behind = f == mw ? kept[f] & ~low : kept[f];
            out[h * 32 + nth_bit(holes, j - run[h])] = f * 32 + nth_bit(behind, moved + j - run[f + 1]);
        }
    }
}

// A thread moves 16 bytes of up to MV_BATCH entries' keys and values, all read before the first is written; the books go with an entry's first bytes.
// Bound by memory: evictions from 32 caches x 4 heads, 2001 entries of 256 bytes, took 54 us with two entries a thread, 59 with one, 57 with three, 61 with
// four, 79 with eight; since the selection reads faster they take 52 (5.1 TB/s read and written; launched alone this kernel takes 40).
constexpr int MV_BATCH = 2;
__global__ void __launch_bounds__(256) kv_move_kernel(KvDev kv, KvDev dst, bool inplace, const int32_t *seq, int keep, const int32_t *map) {
    const int kvh = blockIdx.y, b = blockIdx.z, per = kv.hd * kv.size() / 16;       // a power of two
    pdl_wait();
    const int s = seq ? seq[b] : b;
    if ((unsigned)s >= (unsigned)kv.n_seq || s >= dst.n_seq) return;
    const int32_t *from = map + ((long long)b * kv.nkv + kvh) * keep;
    const uint4 *k = reinterpret_cast<const uint4 *>((const char *)kv.k + kv.head(s, kvh) * kv.size()), *v = reinterpret_cast<const uint4 *>((const char *)kv.v + kv.head(s, kvh) * kv.size());
    uint4 *k2 = reinterpret_cast<uint4 *>((char *)dst.k + dst.head(s, kvh) * dst.size()), *v2 = reinterpret_cast<uint4 *>((char *)dst.v + dst.head(s, kvh) * dst.size());
    const long long book = kv.book(s, kvh), book2 = dst.book(s, kvh);
    const int c = threadIdx.x % per, rows = 256 / per, d0 = blockIdx.x * rows * MV_BATCH + threadIdx.x / per;
    int t[MV_BATCH];
    uint4 x[MV_BATCH], y[MV_BATCH];
#pragma unroll
    for (int i = 0; i < MV_BATCH; i++) {
        const int d = d0 + i * rows;
        t[i] = d < keep ? from[d] : -1;           // -1 throughout for an entry that was left out
        if (inplace && t[i] == d) t[i] = -1;
    }
#pragma unroll
    for (int i = 0; i < MV_BATCH; i++)
        if (t[i] >= 0) { x[i] = k[(long long)t[i] * per + c]; y[i] = v[(long long)t[i] * per + c]; }
#pragma unroll
    for (int i = 0; i < MV_BATCH; i++) {
        const int d = d0 + i * rows;
        if (t[i] < 0) continue;
        k2[(long long)d * per + c] = x[i];
        v2[(long long)d * per + c] = y[i];
        if (c == 0) { dst.weight[book2 + d] = kv.weight[book + t[i]]; dst.pos[book2 + d] = kv.pos[book + t[i]]; }
    }
}

cudaError_t launch_kv_evict(const KvDev &kv, const KvDev *dst, int n, const int32_t *seq, const int32_t *len, int keep, int first, int recent, const int32_t *end,
                            int32_t *map, int32_t *new_len, cudaStream_t st) {
    const KvDev &to = dst ? *dst : kv;
    const size_t bits = ((size_t)(kv.cap + 31) / 32 * 3 + 1) * 4, all = bits + (size_t)kv.cap * 4, most = 200 * 1024;
    const bool keys = all <= most;
    const size_t smem = keys ? all : bits;
    auto kern = keys ? kv_evict_kernel<true> : kv_evict_kernel<false>;
    cudaError_t e = smem > 20 * 1024 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) : cudaSuccess;
    if (e != cudaSuccess) return e;
    e = launch_k(kern, dim3(kv.nkv, n), dim3(EV_THREADS), smem, st, true, kv, to, seq, len, keep, first, recent, end, map, new_len);
    if (e != cudaSuccess) return e;
    const int rows = 256 / (kv.hd * kv.size() / 16) * MV_BATCH;
    return launch_k(kv_move_kernel, dim3((keep + rows - 1) / rows, kv.nkv, n), dim3(256), 0, st, true, kv, to, dst == nullptr, seq, keep, (const int32_t *)map);
}

// ---------------------------------------------------------------- block means
// A CTA per block: a thread adds four dimensions of every 16th (8th) row in double precision, then the groups of rows are added.  7 new blocks of 32 slots x 8
// heads: 4.9 us, one block x 4 heads 2.6: latency.
__global__ void __launch_bounds__(256) kv_means_kernel(KvDev kv, const int32_t *seq, const int32_t *since, const int32_t *len, int block, float *__restrict__ means) {
    __shared__ double part[256 * 4];
    const int kvh = blockIdx.y, b = blockIdx.z;
    pdl_wait();
    pdl_trigger();
    const KvEntry e = kv_entry(kv, b, 0, seq, len, nullptr);
    const int s0 = since ? since[b] : 0;
    if (kv_named_before(seq, b) || !e.ok || s0 < 0) {
        if (threadIdx.x == 0) kv_error(kv);
        return;
    }
    const int quads = kv.hd / 4, groups = 256 / quads, d = threadIdx.x % quads * 4, g = threadIdx.x / quads;
    const long long head = kv.head(e.seq, kvh);
    float *out = means + ((long long)e.seq * kv.nkv + kvh) * (kv.cap / block) * kv.hd;
    for (int j = s0 / block + blockIdx.x; j < e.len / block; j += gridDim.x) {
        double sum[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 8
        for (int t = g; t < block; t += groups) {
            const long long at = head + (long long)(j * block + t) * kv.hd + d;
            float4 x;
            if (kv.type) {
                const ushort4 u = *reinterpret_cast<const ushort4 *>((const uint16_t *)kv.k + at);
                x = make_float4(brrr_bf16_to_f32(u.x), brrr_bf16_to_f32(u.y), brrr_bf16_to_f32(u.z), brrr_bf16_to_f32(u.w));
            } else {
                x = *reinterpret_cast<const float4 *>((const float *)kv.k + at);
            }
            sum[0] += x.x; sum[1] += x.y; sum[2] += x.z; sum[3] += x.w;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) part[i * 256 + threadIdx.x] = sum[i];
        __syncthreads();
        for (int x = threadIdx.x; x < kv.hd; x += 256) {
            double all = 0.0;
            for (int i = 0; i < groups; i++) all += part[(x & 3) * 256 + i * quads + (x >> 2)];
            out[(long long)j * kv.hd + x] = (float)(all / block);
        }
        __syncthreads();
    }
}

cudaError_t launch_kv_means(const KvDev &kv, int n, const int32_t *seq, const int32_t *since, const int32_t *len, int block, int len_hint, float *means, cudaStream_t st) {
    const int blocks = (len_hint > 0 ? min(len_hint, kv.cap) : kv.cap) / block + 1;
    return launch_k(kv_means_kernel, dim3(min(blocks, 4096), kv.nkv, n), dim3(256), 0, st, true, kv, seq, since, len, block, means);
}

}  // namespace brrr
