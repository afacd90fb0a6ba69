// What the attention kernels over the caller's caches share: cache types, what a tree's rows see, the join of partial results, cluster launches.
#pragma once
#include "brrr_block.cuh"
#include "brrr_kv.cuh"
#include "brrr_tma.cuh"
#include "brrr_tmap.h"

#include <atomic>
#include <cooperative_groups.h>

namespace brrr {

namespace cg = cooperative_groups;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The two cache types: values per 16-byte load, and a load's values as floats.
struct KvF32 {
    static constexpr int V = 4;
    static constexpr bool SPLIT = true;
    typedef float Val;
    static __device__ __forceinline__ void get(const uint4 &u, float (&x)[4]) {
        x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
    }
};
struct KvBf16 {
    static constexpr int V = 8;
    static constexpr bool SPLIT = false;
    typedef uint16_t Val;
    static __device__ __forceinline__ void get(const uint4 &u, float (&x)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
    }
};

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7F800000u) == 0x7F800000u; }

// Partial results of a row - maximum in powers of two, sum, values - join as
//   M = max m_p,  sum = sum_p l_p 2^(m_p - M),  x = sum_p x_p 2^(m_p - M),
// the row's sink as one more part without values.  In a cluster a row has an owner, the CTA rank r / owned_rows(R, C): the others write their parts into its
// shared memory, [CTA][owned row][STRIDE] and [CTA][owned row] of (m, l), and the owner adds them up in the order of the CTAs.
__host__ __device__ constexpr int owned_rows(int R, int C) { return (R + C - 1) / C; }
// The owner's end: n parts of `rows` rows.  dst(i): the owned row's place in the output (< 0: padding), sink(i): its sink in powers of two or -infinity.
template <int HD, int STRIDE, class Dst, class Sink>
__device__ __forceinline__ void join_rows(const float *x, const float2 *ml, int n, int rows, float *o, float *lse, Dst dst, Sink sink) {
    for (int u = threadIdx.x; u < rows * (HD / 4); u += blockDim.x) {
        const int i = u / (HD / 4), d = u % (HD / 4) * 4;
        const long long to = dst(i);
        if (to < 0) continue;
        const float sk = sink(i);
        float m = sk;
#pragma unroll 8
        for (int p = 0; p < n; p++) m = fmaxf(m, ml[p * rows + i].x);
        const float safe = m == -INFINITY ? 0.0f : m;
        float l = exp2_approx(sk - safe);
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (int p = 0; p < n; p++) {
            const float2 part = ml[p * rows + i];
            const float w = exp2_approx(part.x - safe);
            const float4 z = *reinterpret_cast<const float4 *>(x + (p * rows + i) * STRIDE + d);
            l = __fmaf_rn(w, part.y, l);
            y.x = __fmaf_rn(w, z.x, y.x); y.y = __fmaf_rn(w, z.y, y.y); y.z = __fmaf_rn(w, z.z, y.z); y.w = __fmaf_rn(w, z.w, y.w);
        }
        const float k = __fdividef(1.0f, l == 0.0f ? 1.0f : l);
        *reinterpret_cast<float4 *>(o + to * HD + d) = make_float4(y.x * k, y.y * k, y.z * k, y.w * k);
        if (lse && d == 0) lse[to] = (m + log2f(l)) * LN2;
    }
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// ---------------------------------------------------------------- trees
// What the rows of an entry see: cached slots from lo on, drafted rows by mask (windows applied, rows behind the count cut off).
struct TreeRows {
    uint64_t mask[KV_TREE_MAX];
    int lo[KV_TREE_MAX];
    int first, full;                        // smallest lo, largest lo: from there to len every row sees every slot
};
// Thread i's mask of its entry, wanted before the entry's count is known (chains have none).
__device__ __forceinline__ uint64_t tree_mask(const TreeArgs &a, int b) {
    const int i = threadIdx.x;
    return i >= a.rows ? 0 : a.mask ? a.mask[(long long)b * a.rows + i] : i == 63 ? ~0ull : (1ull << (i + 1)) - 1;
}
// All threads call it with their mask; complete for them after the next barrier.
__device__ __forceinline__ void tree_rows(const TreeArgs &a, const KvEntry &e, uint64_t mine, TreeRows &w) {
    __shared__ int depth[KV_TREE_MAX];
    const int i = threadIdx.x;
    mine &= e.count == 64 ? ~0ull : (1ull << e.count) - 1;
    if (a.window <= 0) {
        if (i < e.count) { w.mask[i] = mine; w.lo[i] = 0; }
        if (i == 0) w.first = w.full = 0;
        return;
    }
    if (i == 0) { w.first = e.len; w.full = 0; }
    if (i < e.count) depth[i] = __popcll(mine & ~(1ull << i));
    __syncthreads();
    if (i < e.count) {
        uint64_t in = 0;
        for (int j = 0; j < e.count; j++) in |= (uint64_t)(depth[i] - depth[j] < a.window) << j;
        const int lo = max(0, min(e.len, e.len + depth[i] + 1 - a.window));
        w.mask[i] = mine & in;
        w.lo[i] = lo;
        atomicMin(&w.first, lo);
        atomicMax(&w.full, lo);
    }
}

// K and V as tensors [sequence][kv head][slot][dim], boxes of 128 bytes of a row x `slots` rows, rows of a box 128 swizzled bytes in shared memory (16-byte piece
// c of row r at c ^ (r & 7)).  A box may reach behind an entry's end: what stands there nobody sees.
struct alignas(64) KvMaps {
    CUtensorMap k, v;
};
static inline cudaError_t kv_maps(const KvDev &kv, int slots, KvMaps *m) {
    const tmap_encode_t encode = tmap_encode();
    if (!encode) return cudaErrorNotSupported;
    const cuuint64_t size = kv.size(), dims[4] = {(cuuint64_t)kv.hd, (cuuint64_t)kv.cap, (cuuint64_t)kv.nkv, (cuuint64_t)kv.n_seq};
    const cuuint64_t strides[3] = {kv.hd * size, kv.hs * size, kv.ss * size};
    const cuuint32_t box[4] = {(cuuint32_t)(128 / size), (cuuint32_t)slots, 1, 1}, ones[4] = {1, 1, 1, 1};
    for (int i = 0; i < 2; i++)
        if (encode(i ? &m->v : &m->k, kv.type ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, i ? kv.v : kv.k, dims, strides, box, ones,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    return cudaSuccess;
}
__device__ __forceinline__ void tensor_prefetch(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void tensor_rows(uint32_t dst, const CUtensorMap *map, int x, int slot, int kvh, int seq, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(x), "r"(slot),
                 "r"(kvh), "r"(seq), "r"(smem_u32(bar))
                 : "memory");
}

// Once per kernel and device: the shared memory it may ask for, clusters of up to 16.
template <auto K>
static cudaError_t allow(size_t smem) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && done.load() >> dev & 1)) return e;
    if (smem > 48 * 1024) e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(K, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev);
    return e;
}

// most: the largest shared memory this kernel is ever launched with
template <auto K, class... Args>
static cudaError_t launch_cluster(dim3 grid, int threads, int cluster, size_t smem, size_t most, cudaStream_t st, Args... args) {
    cudaError_t e = allow<K>(most);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, K, args...);
}

// CTAs (1..16) that share the steps of one of `jobs` pieces of work, `lanes` steps of a CTA going on at a time: the least time of all waves, where a
// CTA's start and end cost about as much as `fixed` steps.  How many clusters of a size the GPU holds at once is asked for once per kernel, size and device; a kernel
// launched with different amounts of shared memory numbers them (kind), each asked for with the largest that is launched as this kind.
constexpr int ROOM_KINDS = 17;
template <auto K, bool CLUSTER = true>
static int cluster_size(long long jobs, int steps, int lanes, int fixed, int threads, size_t smem, size_t most, cudaError_t *err, int kind = 0) {
    static std::atomic<int> rooms[64][ROOM_KINDS][17];
    int dev = 0;
    *err = cudaGetDevice(&dev);
    if (*err == cudaSuccess) *err = allow<K>(most);
    if (*err != cudaSuccess) return 1;
    int best = 1;
    double least = 0.0;
    for (int c = 1; c <= 16; c++) {           // without clusters c CTAs take c of the places for one
        const int c_room = CLUSTER ? c : 1;
        int held = dev < 64 ? rooms[dev][kind][c_room].load() : 0;
        if (!held) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(c_room);
            cfg.blockDim = dim3(threads);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = c_room;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&held, K, &cfg) != cudaSuccess) { (void)cudaGetLastError(); held = 0; }
            held = held > 0 ? held : -1;
            if (dev < 64) rooms[dev][kind][c_room].store(held);
        }
        if (held < 0) continue;
        const int turns = (steps + c * lanes - 1) / (c * lanes);
        const double t = (double)(CLUSTER ? (jobs + held - 1) / held : (jobs * c + held - 1) / held) * (turns + fixed);
        if (c == 1 || t < least) { best = c; least = t; }
        if (turns <= 1) break;
    }
    return best;
}

}  // namespace brrr
