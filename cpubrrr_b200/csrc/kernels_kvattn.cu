// Attention over KV caches that the caller owns: trees of drafted tokens, chosen blocks, and the book of attention weights.
#include "brrr_kernels.h"
#include "brrr_block.cuh"
#include "brrr_kv.cuh"

namespace brrr {

__device__ __forceinline__ float kv_load(const void *p, int type, long long at) {
    return type ? brrr_bf16_to_f32(((const uint16_t *)p)[at]) : ((const float *)p)[at];
}

// One query head's attention by one warp, four (two) dimensions per lane, over the slots that `next` names (-1: none left).
template <class Next>
__device__ __forceinline__ void warp_attend(const KvDev &kv, long long head, const float *q, float scale, const float *sink, float *out, float *lse, Next next) {
    const int lane = threadIdx.x & 31, per = kv.hd / 32;
    float qr[4], acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int d = 0; d < per; d++) qr[d] = q[d * 32 + lane];
    float top = sink ? *sink : -INFINITY, sum = sink ? 1.0f : 0.0f;
    for (int t = next(); t >= 0; t = next()) {
        const long long at = head + (long long)t * kv.hd;
        float s = 0.0f;
        for (int d = 0; d < per; d++) s = __fmaf_rn(qr[d], kv_load(kv.k, kv.type, at + d * 32 + lane), s);
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= scale;
        const float m = fmaxf(top, s), keep = top == m ? 1.0f : expf(top - m), p = expf(s - m);
        sum = __fmaf_rn(sum, keep, p);
        for (int d = 0; d < per; d++) acc[d] = __fmaf_rn(acc[d], keep, p * kv_load(kv.v, kv.type, at + d * 32 + lane));
        top = m;
    }
    for (int d = 0; d < per; d++) out[d * 32 + lane] = sum > 0.0f ? acc[d] / sum : acc[d] + sum;
    if (lse && lane == 0) *lse = top + logf(sum);
}

__global__ void __launch_bounds__(128) tree_kernel(KvDev kv, TreeArgs a) {
    __shared__ uint64_t mask[KV_TREE_MAX];
    __shared__ int depth[KV_TREE_MAX];
    const int b = blockIdx.y;
    const KvEntry e = kv_entry(kv, b, a.rows, a.seq, a.len, a.count);
    if (!e.ok) {
        if (threadIdx.x == 0) kv_error(kv);
        return;
    }
    tree_masks(a.mask, b, a.rows, e.count, mask, depth);
    __syncthreads();
    const int u = blockIdx.x * 4 + (threadIdx.x >> 5), i = u / a.nh, h = u % a.nh;
    if (i >= e.count) return;
    const long long row = ((long long)b * a.rows + i) * a.nh + h;
    int t = -1;
    auto next = [&]() {
        for (t++; t < e.len + e.count; t++)
            if (tree_sees(mask, depth, e.len, a.window, i, t)) return t;
        return -1;
    };
    warp_attend(kv, kv.head(e.seq, h / (a.nh / kv.nkv)), a.q + row * kv.hd, a.scale, a.sinks ? a.sinks + h : nullptr, a.out + row * kv.hd, a.lse ? a.lse + row : nullptr, next);
}

cudaError_t launch_attn_tree(const KvDev &kv, const TreeArgs &a, int len_hint, cudaStream_t st) {
    tree_kernel<<<dim3((a.rows * a.nh + 3) / 4, a.n), 128, 0, st>>>(kv, a);
    return cudaGetLastError();
}

// ---------------------------------------------------------------- book of weights
// A thread per slot: its key against every row's query.
__global__ void __launch_bounds__(128) weigh_kernel(KvDev kv, TreeArgs a, const uint64_t *picked) {
    __shared__ uint64_t mask[KV_TREE_MAX];
    __shared__ int depth[KV_TREE_MAX];
    const int kvh = blockIdx.y, b = blockIdx.z, per = a.nh / kv.nkv;
    const KvEntry e = kv_entry(kv, b, a.rows, a.seq, a.len, a.count);
    if (kv_named_before(a.seq, b) || !e.ok) {
        if (threadIdx.x == 0) kv_error(kv);
        return;
    }
    tree_masks(a.mask, b, a.rows, e.count, mask, depth);
    __syncthreads();
    const uint64_t rows = picked ? picked[b] : ~0ull;
    for (int t = blockIdx.x * 128 + threadIdx.x; t < e.len + e.count; t += gridDim.x * 128) {
        const long long at = kv.head(e.seq, kvh) + (long long)t * kv.hd;
        float sum = 0.0f;
        for (int i = 0; i < e.count; i++) {
            if (!(rows >> i & 1) || !tree_sees(mask, depth, e.len, a.window, i, t)) continue;
            for (int g = 0; g < per; g++) {
                const long long row = ((long long)b * a.rows + i) * a.nh + kvh * per + g;
                float s = 0.0f;
                for (int d = 0; d < kv.hd; d++) s = __fmaf_rn(a.q[row * kv.hd + d], kv_load(kv.k, kv.type, at + d), s);
                sum += expf(__fmaf_rn(s, a.scale, -a.lse[row]));
            }
        }
        kv.weight[kv.book(e.seq, kvh) + t] += sum;
    }
}

cudaError_t launch_kv_weigh(const KvDev &kv, const TreeArgs &a, const uint64_t *picked, int len_hint, cudaStream_t st) {
    const int slots = (len_hint > 0 ? min(len_hint, kv.cap) : kv.cap) + a.rows;
    weigh_kernel<<<dim3((slots + 127) / 128, kv.nkv, a.n), 128, 0, st>>>(kv, a, picked);
    return cudaGetLastError();
}

// ---------------------------------------------------------------- chosen blocks
constexpr int CB_THREADS = 256;

// A CTA per (kv head, row): scores of the blocks between the first and the local ones, then the nsel largest in ascending order of blocks.
__global__ void __launch_bounds__(CB_THREADS) choose_blocks_kernel(KvDev kv, const int32_t *seq, const int32_t *len, int block, const float *__restrict__ means, int nsel,
                                                                   int first, int local, const float *__restrict__ q, int nh, int32_t *sel) {
    extern __shared__ uint32_t keys[];
    __shared__ float qs[16 * 128];
    const int kvh = blockIdx.y, r = blockIdx.x, per = nh / kv.nkv;
    const int s = seq ? seq[r] : r, n = len[r];
    if ((unsigned)s >= (unsigned)kv.n_seq || (unsigned)n > (unsigned)kv.cap) {
        if (threadIdx.x == 0) kv_error(kv);
        return;
    }
    const int nb = (n + block - 1) / block;
    int32_t *out = sel + ((long long)r * kv.nkv + kvh) * nsel;
    for (int j = nb + threadIdx.x; j < nsel; j += CB_THREADS) out[j] = -1;
    if (nb <= nsel) {
        for (int j = threadIdx.x; j < nb; j += CB_THREADS) out[j] = j;
        return;
    }
    for (int i = threadIdx.x; i < per * kv.hd; i += CB_THREADS) qs[i] = q[((long long)r * nh + kvh * per) * kv.hd + i];
    __syncthreads();
    const float *mean = means + ((long long)s * kv.nkv + kvh) * (kv.cap / block) * kv.hd;
    for (int j = threadIdx.x; j < nb; j += CB_THREADS) {
        uint32_t key = 0xFFFFFFFFu;
        if (j >= first && j < nb - local) {
            double top = -INFINITY;
            bool nan = false;
            for (int g = 0; g < per; g++) {
                double x = 0.0;
                for (int d = 0; d < kv.hd; d++) x += (double)qs[g * kv.hd + d] * (double)mean[(long long)j * kv.hd + d];
                nan |= x != x;
                top = fmax(top, x);
            }
            const float f = (float)top;
            key = nan ? 0u : f == 0.0f ? 0x80000000u : float_orderable(f);
        }
        keys[j] = key;
    }
    __syncthreads();
    // rank of a block: those that come before it
    for (int j = threadIdx.x; j < nb; j += CB_THREADS) {
        int rank = 0;
        for (int i = 0; i < nb; i++) rank += keys[i] > keys[j] || (keys[i] == keys[j] && i < j);
        if (rank < nsel) out[rank] = j;
    }
    __syncthreads();
    if (threadIdx.x == 0)
        for (int i = 1; i < nsel; i++) {
            const int x = out[i];
            int at = i;
            for (; at > 0 && out[at - 1] > x; at--) out[at] = out[at - 1];
            out[at] = x;
        }
}

__global__ void __launch_bounds__(128) blocks_kernel(KvDev kv, const int32_t *seq, const int32_t *len, int block, int nsel, const int32_t *sel, const float *q, int nh,
                                                     float scale, const float *sinks, float *out, float *lse) {
    const int r = blockIdx.y, h = blockIdx.x * 4 + (threadIdx.x >> 5);
    const int s = seq ? seq[r] : r, n = len[r];
    if (h >= nh || (unsigned)s >= (unsigned)kv.n_seq || (unsigned)n > (unsigned)kv.cap) return;
    const int kvh = h / (nh / kv.nkv);
    const int32_t *mine = sel + ((long long)r * kv.nkv + kvh) * nsel;
    const long long row = (long long)r * nh + h;
    int c = 0, o = -1;
    auto next = [&]() {
        if (++o == block) { o = 0; c++; }
        const int t = c < nsel && mine[c] >= 0 ? mine[c] * block + o : n;
        return t < n ? t : -1;
    };
    warp_attend(kv, kv.head(s, kvh), q + row * kv.hd, scale, sinks ? sinks + h : nullptr, out + row * kv.hd, lse ? lse + row : nullptr, next);
}

cudaError_t launch_attn_blocks(const KvDev &kv, int rows, const int32_t *seq, const int32_t *len, int block, const float *means, int nsel, int first, int local,
                               int len_hint, const float *q, int nh, float scale, const float *sinks, int32_t *sel, float *out, float *lse, cudaStream_t st) {
    const size_t smem = (size_t)(kv.cap / block + 1) * 4;
    cudaError_t e = smem > 32 * 1024 ? cudaFuncSetAttribute(choose_blocks_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) : cudaSuccess;
    if (e != cudaSuccess) return e;
    choose_blocks_kernel<<<dim3(rows, kv.nkv), CB_THREADS, smem, st>>>(kv, seq, len, block, means, nsel, first, local, q, nh, sel);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    blocks_kernel<<<dim3((nh + 3) / 4, rows), 128, 0, st>>>(kv, seq, len, block, nsel, sel, q, nh, scale, sinks, out, lse);
    return cudaGetLastError();
}

}  // namespace brrr
