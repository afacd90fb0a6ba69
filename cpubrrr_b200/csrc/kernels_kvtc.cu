// Attention of drafted trees with more than 16 rows per kv head on the fifth-generation tensor cores (tcgen05.mma, accumulators in tensor memory).
//
// Rows are (drafted token, query head) pairs, 128 to a CTA, one per lane of tensor memory; a tile is N slots.  Single precision out of bf16 products:
// an f32 value is cut into three pieces of eight bits (hi: the upper 16 bits of its pattern; mid: those of the rest; lo: what is left - all
// exact), q into q0 + q1 + q2, weights p into p0 + p1 + p2.  A bf16 cache's values are one piece: three products give the full product.  f32 values have
// three: the six products down to 2^-16 are formed, what is left out is 2^-22 of the product.  The small ones come first in the accumulator, so that few
// of its (truncating) additions carry weight; an output tile starts at zero and joins the running output in registers, scaled to the new maximum.
//
// Warp roles: 0-7 softmax and output (thread = row and half of a tile's slots, then half of the dimensions), 8-11 keys and values from global memory
// through registers into operand order (cut into pieces on the way), 12 issues.  Scores of two tiles alternate in tensor memory; the pieces of a tile's
// weights take the place of its scores as operand A.  While the softmax warps work on tile i + 1 the tensor cores do the values of tile i and the
// scores of tile i + 2.
//
// Operands without swizzle: core matrices of 8 rows x 16 bytes, [slot / 8][dim / 8] of them.  As operand B of the scores (N = slots, K = dims) that is
// K-major, as operand B of the outputs (N = dims, K = slots) MN-major: neither keys nor values are transposed.
#include "brrr_kernels.h"
#include "brrr_kvattn.cuh"
#include "brrr_tc.cuh"

namespace brrr {

namespace {

constexpr int TC_SOFT = 8, TC_LOAD = 4, TC_THREADS = (TC_SOFT + TC_LOAD + 1) * 32, TC_M = 128;

template <class T, int HD, int N>
struct Tc {
    static constexpr int PL = T::SPLIT ? 3 : 1;                       // pieces of a cached value
    static constexpr int KST = T::SPLIT ? 1 : 2, VST = T::SPLIT || HD == 128 ? 1 : 2;      // stages
    static constexpr int NC = HD / 8;                                  // 16-byte pieces of a row
    static constexpr int PLANE = N * HD * 2, QPLANE = TC_M * HD * 2;
    static constexpr int Q = 0, K = 3 * QPLANE, V = K + KST * PL * PLANE, BYTES = V + VST * PL * PLANE;
    // above half of an SM's shared memory: one CTA per SM, since each takes all of tensor memory
    static constexpr size_t SMEM = BYTES > 118784 ? BYTES : 118784;
    static constexpr uint32_t BUF = N + N / 2, D = 2 * BUF;            // columns: scores, then pieces hi | mid by halves, and lo behind; the output tile
    static_assert(D + HD <= 512 && SMEM <= 229376 && TC_M * (HD + 4) * 4 + TC_M * 16 <= K, "");
};

__device__ __forceinline__ void tc_mma_ss(uint32_t issue, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u), "r"(issue)
                 : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t issue, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u), "r"(issue)
                 : "memory");
}
// 32 consecutive columns of this warp's lanes; loads and wait are one statement
__device__ __forceinline__ void tc_ld32(uint32_t t, float *v) {
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                   "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
                   "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(t)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tc_st16(uint32_t t, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
// the three pieces of two values, first value in the lower half
__device__ __forceinline__ void cut2(float a, float b, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    hi = __byte_perm(ua, ub, 0x7632);
    const float ra = a - __uint_as_float(ua & 0xFFFF0000u), rb = b - __uint_as_float(ub & 0xFFFF0000u);
    const uint32_t va = __float_as_uint(ra), vb = __float_as_uint(rb);
    mid = __byte_perm(va, vb, 0x7632);
    const float sa = ra - __uint_as_float(va & 0xFFFF0000u), sb = rb - __uint_as_float(vb & 0xFFFF0000u);
    lo = __byte_perm(__float_as_uint(sa), __float_as_uint(sb), 0x7632);
}
__device__ __forceinline__ void st_shared16(uint32_t at, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// eight f32 values as 16 bytes in each of three planes
__device__ __forceinline__ void store_pieces(uint32_t at, int plane, const float (&x)[8]) {
    uint32_t p[3][4];
#pragma unroll
    for (int i = 0; i < 4; i++) cut2(x[2 * i], x[2 * i + 1], p[0][i], p[1][i], p[2][i]);
#pragma unroll
    for (int i = 0; i < 3; i++) st_shared16(at + i * plane, p[i]);
}

// products in the order in which they are formed: the piece of A and of B, four bits each
template <int PL>
struct Products {
    static constexpr int N = PL == 1 ? 3 : 6;
    static constexpr uint32_t A = PL == 1 ? 0x012u : 0x001102u, B = PL == 1 ? 0u : 0x010120u;
    static __device__ __forceinline__ constexpr int a(int p) { return A >> (4 * p) & 15; }
    static __device__ __forceinline__ constexpr int b(int p) { return B >> (4 * p) & 15; }
};

// grid (C, kv heads x blocks of 128 rows, entries), clusters of C
template <class T, int HD, int N>
__global__ void __launch_bounds__(TC_THREADS, 1) tree_tc_kernel(KvDev kv, TreeArgs a) {
    typedef Tc<T, HD, N> S;
    typedef Products<S::PL> Pr;
    extern __shared__ __align__(128) unsigned char tsm[];
    __shared__ __align__(8) uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], pready, dfull, qfull;
    __shared__ TreeRows see;
    __shared__ float part_max[2][2][TC_M];
    __shared__ uint32_t bad[N / 32];           // slots of a tile whose values are no numbers (tiles that not every row sees whole)
    __shared__ uint32_t tmem_sh;
    const int per = a.nh / kv.nkv, blocks = (a.rows * per + TC_M - 1) / TC_M;
    const int kvh = blockIdx.y / blocks, row0 = blockIdx.y % blocks * TC_M, b = blockIdx.z;
    const KvEntry e = kv_entry(kv, b, a.rows, a.seq, a.len, a.count);
    if (!e.ok || row0 >= e.count * per) {
        if (!e.ok && threadIdx.x == 0) kv_error(kv);
        return;
    }
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&kfull[i], TC_LOAD); mbar_init(&vfull[i], TC_LOAD);
            mbar_init(&kempty[i], 1); mbar_init(&vempty[i], 1); mbar_init(&sfull[i], 1);
        }
        mbar_init(&pready, TC_SOFT); mbar_init(&dfull, 1); mbar_init(&qfull, TC_SOFT);
        mbar_fence_init();
    }
    if (warp == TC_SOFT + TC_LOAD) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_sh)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tree_rows(a, b, e, see);
    tl_fence_before();
    __syncthreads();
    tl_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_sh, 0), base0 = smem_u32(tsm);
    const int end = e.len + e.count, s0 = see.first / N, all = (end + N - 1) / N - s0, chunk = (all + gridDim.x - 1) / gridDim.x;
    const int from = s0 + blockIdx.x * chunk, tiles = max(0, min(chunk, s0 + all - from));
    auto partial = [&](int i) { return (from + i) * N < see.full || (from + i + 1) * N > e.len; };
    TlWaiter wait{kv.err ? reinterpret_cast<uint32_t *>(kv.err) : nullptr, false};
    float *out = reinterpret_cast<float *>(tsm);
    float2 *ml = reinterpret_cast<float2 *>(out + TC_M * (HD + 4));

    if (warp < TC_SOFT) {
        // ---------------- queries, softmax, output
        for (int u = tid; u < TC_M * S::NC; u += TC_SOFT * 32) {
            const int r = (u & 7) + u / (8 * S::NC) * 8, c = u / 8 % S::NC, i = (row0 + r) / per;       // eight neighbours write one core matrix
            float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if (i < e.count) {
                const float4 *p = reinterpret_cast<const float4 *>(a.q + (((long long)b * a.rows + i) * a.nh + kvh * per + (row0 + r) % per) * HD + c * 8);
                const float4 y = p[0], z = p[1];
                x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w; x[4] = z.x; x[5] = z.y; x[6] = z.z; x[7] = z.w;
                if (a.scale < 0.0f)
#pragma unroll
                    for (int k = 0; k < 8; k++) x[k] = -x[k];
            }
            store_pieces(base0 + S::Q + ((r >> 3) * S::NC + c) * 128 + (r & 7) * 16, S::QPLANE, x);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&qfull);
        const int quarter = warp & 3, half = warp >> 2, r = quarter * 32 + lane, node = (row0 + r) / per;
        const uint64_t mask = node < e.count ? see.mask[node] : 0;
        const int lo = node < e.count ? see.lo[node] : 0x7fffffff;
        const bool idle = row0 + quarter * 32 >= e.count * per;         // a warp of padding
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const float c = fmaxf(fabsf(a.scale) * LOG2E, 1e-37f);           // above zero: -infinity stays what it is
        float m = -INFINITY, l = 0.0f, f = 1.0f, o[HD / 2];
#pragma unroll
        for (int d = 0; d < HD / 2; d++) o[d] = 0.0f;
        auto join_output = [&](int i) {
            wait(&dfull, i & 1);
            if (idle) return;
            tl_fence_after();
#pragma unroll
            for (int d = 0; d < HD / 2; d += 32) {
                float x[32];
                tc_ld32(lanes + S::D + half * (HD / 2) + d, x);
#pragma unroll
                for (int k = 0; k < 32; k++) o[d + k] = __fmaf_rn(o[d + k], f, x[k]);
            }
        };
        for (int i = 0; i < tiles; i++) {
            const uint32_t buf = lanes + (i & 1) * S::BUF, mine = buf + half * (N / 2);
            wait(&sfull[i & 1], (i >> 1) & 1);
            float fn = 1.0f;
            if (!idle) {
                tl_fence_after();
                float s[N / 2];
#pragma unroll
                for (int k = 0; k < N / 2; k += 32) tc_ld32(mine + k, s + k);
                uint32_t gone[N / 64];                                   // slots of this half that are no numbers
#pragma unroll
                for (int w = 0; w < N / 64; w++) gone[w] = 0;
                const bool part = partial(i);
                if (part) {
                    const int t0 = (from + i) * N + half * (N / 2);
                    wait(&vfull[i % S::VST], (i / S::VST) & 1);          // the loading warps have looked at the values
#pragma unroll
                    for (int w = 0; w < N / 64; w++) gone[w] = bad[half * (N / 64) + w];
#pragma unroll
                    for (int k = 0; k < N / 2; k++) {
                        const int t = t0 + k;
                        const bool sees = t < e.len ? t >= lo : t < end && (mask >> (t - e.len) & 1);
                        if (!sees) s[k] = -INFINITY;
                        else if (gone[k >> 5] >> (k & 31) & 1) s[k] = NAN;
                    }
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < N / 2; k++) top[k & 3] = fmaxf(top[k & 3], s[k]);
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                part_max[i & 1][half][r] = mx;
                asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
                const float mn = fmaxf(m, fmaxf(mx, part_max[i & 1][half ^ 1][r]));
                const float safe = mn == -INFINITY ? 0.0f : mn * c;
                fn = exp2_approx((m == -INFINITY ? m : m * c) - safe);
                m = mn;
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < N / 2; k += 32) {
                    uint32_t p0[16], p1[16], p2[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const float x = exp2_approx(__fmaf_rn(s[k + 2 * j], c, -safe)), y = exp2_approx(__fmaf_rn(s[k + 2 * j + 1], c, -safe));
                        sum[2 * (j & 1)] += x;
                        sum[2 * (j & 1) + 1] += y;
                        cut2(x, y, p0[j], p1[j], p2[j]);
                    }
                    tc_st16(mine + k / 2, p0);
                    tc_st16(mine + N / 4 + k / 2, p1);
                    tc_st16(buf + N + half * (N / 4) + k / 2, p2);
                }
                l = __fmaf_rn(l, fn, (sum[0] + sum[1]) + (sum[2] + sum[3]));
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            } else if (partial(i)) {
                wait(&vfull[i % S::VST], (i / S::VST) & 1);
            }
            if (i > 0) join_output(i - 1);
            f = fn;
            tl_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pready);
        }
        if (tiles > 0) join_output(tiles - 1);
        // the queries are done with: their place takes the rows
        part_max[0][half][r] = l;
        asm volatile("bar.sync %0, 256;" ::"r"(9) : "memory");
        if (half == 0) ml[r] = make_float2(m == -INFINITY ? m : m * c, l + part_max[0][1][r]);
#pragma unroll
        for (int d = 0; d < HD / 2; d += 4)
            *reinterpret_cast<float4 *>(out + r * (HD + 4) + half * (HD / 2) + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
    } else if (warp < TC_SOFT + TC_LOAD) {
        // ---------------- keys and values into operand order
        constexpr int LPI = T::SPLIT ? 2 : 1, BI = 4 / LPI;             // 16-byte loads per item; items per batch
        constexpr int ITEMS = N / 8 * (HD / 32) / TC_LOAD, NB = ITEMS / BI, RING = 4;
        static_assert(ITEMS % BI == 0 && (2 * NB) % RING == 0, "");
        const typename T::Val *src[2] = {(const typename T::Val *)kv.k + kv.head(e.seq, kvh), (const typename T::Val *)kv.v + kv.head(e.seq, kvh)};
        const int lw = warp - TC_SOFT, row = lane & 7, sub = lane >> 3;
        uint4 ring[RING][4];
        // batch bt of tile i: items of the keys, then of the values
        auto fetch = [&](int i, int bt, uint4 (&x)[4]) {
#pragma unroll
            for (int k = 0; k < BI; k++) {
                const int it = ((bt % NB) * BI + k) * TC_LOAD + lw, t = (from + i) * N + it / (HD / 32) * 8 + row, chunk = it % (HD / 32) * 4 + sub;
                const typename T::Val *p = src[bt / NB] + (long long)t * HD + chunk * 8;
#pragma unroll
                for (int j = 0; j < LPI; j++) x[k * LPI + j] = t < end ? ldg_shared(p + j * T::V) : make_uint4(0, 0, 0, 0);
            }
        };
        if (tiles > 0)
#pragma unroll
            for (int k = 0; k < RING - 1; k++) fetch(0, k, ring[k]);
        for (int i = 0; i < tiles; i++) {
            const bool part = partial(i);
#pragma unroll
            for (int bt = 0; bt < 2 * NB; bt++) {
                const int nx = bt + RING - 1;
                if (nx < 2 * NB) fetch(i, nx, ring[nx % RING]);
                else if (i + 1 < tiles) fetch(i + 1, nx - 2 * NB, ring[nx % RING]);
                const int st = bt < NB ? i % S::KST : i % S::VST;
                if (bt == 0 && i >= S::KST) wait(&kempty[st], ((i / S::KST) & 1) ^ 1);
                if (bt == NB) {
                    if (i >= S::VST) wait(&vempty[st], ((i / S::VST) & 1) ^ 1);
                    if (part) {
                        // with two stages the tile before may be read still
                        if (S::VST > 1 && i > 0) wait(&vempty[(i - 1) % S::VST], ((i - 1) / S::VST) & 1);
                        if (lw == 0 && lane < N / 32) bad[lane] = 0;
                        asm volatile("bar.sync %0, 128;" ::"r"(10) : "memory");
                    }
                }
                const uint32_t dst = base0 + (bt < NB ? S::K : S::V) + st * S::PL * S::PLANE;
#pragma unroll
                for (int k = 0; k < BI; k++) {
                    const int it = ((bt % NB) * BI + k) * TC_LOAD + lw, rg = it / (HD / 32), chunk = it % (HD / 32) * 4 + sub;
                    const uint32_t at = dst + (rg * S::NC + chunk) * 128 + row * 16;
                    uint4 (&x)[4] = ring[bt % RING];
                    if (bt >= NB && part) {
                        bool any = false;
#pragma unroll
                        for (int j = 0; j < LPI; j++) {
                            float y[T::V];
                            T::get(x[k * LPI + j], y);
#pragma unroll
                            for (int d = 0; d < T::V; d++) any |= not_finite(y[d]);
                        }
                        if (any) {
                            const int t = rg * 8 + row;
                            atomicOr(&bad[t >> 5], 1u << (t & 31));
#pragma unroll
                            for (int j = 0; j < LPI; j++) x[k * LPI + j] = make_uint4(0, 0, 0, 0);
                        }
                    }
                    if (T::SPLIT) {
                        const uint4 y = x[k * LPI], z = x[k * LPI + LPI - 1];
                        const float v[8] = {__uint_as_float(y.x), __uint_as_float(y.y), __uint_as_float(y.z), __uint_as_float(y.w),
                                            __uint_as_float(z.x), __uint_as_float(z.y), __uint_as_float(z.z), __uint_as_float(z.w)};
                        store_pieces(at, S::PLANE, v);
                    } else {
                        const uint32_t v[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
                        st_shared16(at, v);
                    }
                }
                if (bt == NB - 1 || bt == 2 * NB - 1) {
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bt < NB ? &kfull[st] : &vfull[st]);
                }
            }
        }
    } else {
        // ---------------- products (the whole warp walks the loop, an elected lane issues)
        const uint32_t issue = elect_one() ? 1u : 0u;
        constexpr uint32_t types = (1u << 4) | (1u << 7) | (1u << 10) | ((TC_M >> 4) << 24);       // f32 += bf16 x bf16
        constexpr uint32_t id_s = types | ((uint32_t)(N >> 3) << 17), id_o = types | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
        const uint64_t dq = tl_smem_desc(tsm + S::Q, 128, S::NC * 128), dk = tl_smem_desc(tsm + S::K, 128, S::NC * 128), dv = tl_smem_desc(tsm + S::V, S::NC * 128, 128);
        wait(&qfull, 0);
        auto scores = [&](int i) {
            const int st = i % S::KST;
            wait(&kfull[st], (i / S::KST) & 1);
            tl_fence_after();
            const uint32_t d = tmem + (i & 1) * S::BUF;
            const uint64_t k0 = dk + (uint64_t)(st * S::PL * S::PLANE / 16);
#pragma unroll
            for (int p = 0; p < Pr::N; p++)
#pragma unroll
                for (int s = 0; s < HD / 16; s++)
                    tc_mma_ss(issue, d, dq + (uint64_t)((Pr::a(p) * S::QPLANE + s * 256) / 16), k0 + (uint64_t)((Pr::b(p) * S::PLANE + s * 256) / 16), id_s, p > 0 || s > 0);
            tl_commit_if(issue, &sfull[i & 1]);
            tl_commit_if(issue, &kempty[st]);
            __syncwarp();
        };
        if (tiles > 0) scores(0);
        if (tiles > 1) scores(1);
        for (int i = 0; i < tiles; i++) {
            const int st = i % S::VST;
            wait(&vfull[st], (i / S::VST) & 1);
            wait(&pready, i & 1);
            tl_fence_after();
            const uint32_t p0 = tmem + (i & 1) * S::BUF;
            const uint64_t v0 = dv + (uint64_t)(st * S::PL * S::PLANE / 16);
#pragma unroll
            for (int p = 0; p < Pr::N; p++)
#pragma unroll
                for (int s = 0; s < N / 16; s++) {
                    constexpr int per_half = N / 32;
                    const int h = s / per_half, k = s % per_half;
                    const uint32_t at = p0 + (Pr::a(p) < 2 ? h * (N / 2) + Pr::a(p) * (N / 4) : N + h * (N / 4)) + k * 8;
                    tc_mma_ts(issue, tmem + S::D, at, v0 + (uint64_t)((Pr::b(p) * S::PLANE + s * 2 * S::NC * 128) / 16), id_o, p > 0 || s > 0);
                }
            tl_commit_if(issue, &dfull);
            tl_commit_if(issue, &vempty[st]);
            __syncwarp();
            if (i + 2 < tiles) {
                wait(&dfull, i & 1);             // the weights of tile i stand where its scores go
                scores(i + 2);
            }
        }
    }
    tl_fence_before();
    __syncthreads();
    if (warp == TC_SOFT + TC_LOAD) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    join_parts<HD, HD + 4>(out, ml, TC_M, 1, a.out, a.lse,
                           [&](int r) -> long long {
                               const int i = (row0 + r) / per;
                               return i < e.count ? ((long long)b * a.rows + i) * a.nh + kvh * per + (row0 + r) % per : -1;
                           },
                           [&](int r) { return a.sinks ? a.sinks[kvh * per + (row0 + r) % per] * LOG2E : -INFINITY; });
}

template <class T, int HD, int N>
cudaError_t launch_tree_tc_as(const KvDev &kv, const TreeArgs &a, int slots, cudaStream_t st) {
    typedef Tc<T, HD, N> S;
    const int blocks = (a.rows * (a.nh / kv.nkv) + TC_M - 1) / TC_M;
    constexpr auto K = tree_tc_kernel<T, HD, N>;
    cudaError_t e = cudaSuccess;
    const int c = cluster_size<K>((long long)a.n * kv.nkv * blocks, (slots + N - 1) / N, 1, 3, TC_THREADS, S::SMEM, S::SMEM, &e);
    if (e != cudaSuccess) return e;
    return launch_cluster<K>(dim3(c, kv.nkv * blocks, a.n), TC_THREADS, c, S::SMEM, S::SMEM, st, kv, a);
}

}  // namespace

cudaError_t launch_tree_tc(const KvDev &kv, const TreeArgs &a, int slots, cudaStream_t st) {
    if (kv.type) return kv.hd == 64 ? launch_tree_tc_as<KvBf16, 64, 128>(kv, a, slots, st) : launch_tree_tc_as<KvBf16, 128, 128>(kv, a, slots, st);
    return kv.hd == 64 ? launch_tree_tc_as<KvF32, 64, 128>(kv, a, slots, st) : launch_tree_tc_as<KvF32, 128, 64>(kv, a, slots, st);
}

}  // namespace brrr
