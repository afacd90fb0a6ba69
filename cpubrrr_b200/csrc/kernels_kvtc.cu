// Attention of drafted trees with many rows per kv head (wide_rows_pay says from where on), and their book of weights (more than 16), on the fifth-generation
// tensor cores (tcgen05.mma, accumulators in tensor memory).
//
// Rows are (drafted token, query head) pairs, 128 to a CTA, one per lane of tensor memory; a tile is N slots.  Single precision out of bf16 products:
// an f32 value is cut into three pieces of eight bits (hi: the upper 16 bits of its pattern; mid: those of the rest; lo: what is left - all
// exact), q into q0 + q1 + q2, weights p into p0 + p1 + p2.  A bf16 cache's values are one piece: three products give the full product.  f32 values have
// three: the six products down to 2^-16 are formed, what is left out is 2^-21 of the product at most (mid lo and lo mid).  The small ones come first in the
// accumulator, so that few of its (truncating) additions carry weight; an output tile starts at zero and joins the running output in registers, scaled to the new maximum.
//
// Warp roles: 0-7 softmax and output (thread = row and half of a tile's slots, then half of the dimensions).  bf16: 13 brings keys and values, tensor copies in
// operand order, swizzled; 8-11 look at the values of tiles that not every row sees whole; 12 issues.  f32: 17 brings raw rows into a ring, 8-15 cut them
// into pieces in operand order, 16 issues.  Queries are operand A in tensor memory (64 dimensions: the two upper pieces, there is no room for the third,
// which stays in shared memory).  Scores of two tiles alternate in tensor memory; the pieces of a tile's weights take the place of its scores as operand A.
// While the softmax warps work on tile i + 1 the tensor cores do the values of tile i and the scores of tile i + 2.
//
// Keys are operand B of the scores (N = slots, K = dims), K-major, values that of the outputs (N = dims, K = slots), MN-major: neither is transposed.  What is
// not swizzled stands in core matrices of 8 rows x 16 bytes, keys [dim / 8][slot / 8], values [slot / 8][dim / 8].
#include "brrr_kernels.h"
#include "brrr_kvattn.cuh"
#include "brrr_tc.cuh"

#include <algorithm>

namespace brrr {

namespace {

constexpr int TC_SOFT = 8, TC_M = 128;

template <class T, int HD>
struct Tc {
    // warps: softmax, then these, then one that issues and one that copies
    static constexpr int LOAD = T::SPLIT ? 8 : 4, ISSUE = TC_SOFT + LOAD, BULK = ISSUE + 1, THREADS = T::SPLIT ? 640 : 448;
    static constexpr int N = HD == 64 ? 128 : 64;                      // slots of a tile: 8192 values of keys and of values each
    static constexpr int PL = T::SPLIT ? 3 : 1;                       // pieces of a cached value
    static constexpr int ST = T::SPLIT ? 1 : 4;                        // stages of operands
    static constexpr int NC = HD / 8;                                  // 16-byte pieces of a row
    static constexpr int PLANE = N * HD * 2, STAGE = PL * PLANE;
    static constexpr int QT = HD == 64 ? 2 : 3;                        // pieces of the queries in tensor memory
    static constexpr int UNITS = T::SPLIT ? 3 : 0, UNIT = N * HD * 4;      // ring of raw f32 rows: a tile's keys or values each
    static constexpr int Q2 = 0, K = QT == 2 ? TC_M * HD * 2 : 0, V = K + ST * STAGE, RAW = V + ST * STAGE, BYTES = RAW + UNITS * UNIT;
    // above half of an SM's shared memory: one CTA per SM, since each takes all of tensor memory
    static constexpr size_t SMEM = BYTES > 118784 ? BYTES : 118784;
    // columns: twice scores, which become the pieces hi | mid by halves, and the pieces lo behind; the output tile; the queries
    static constexpr uint32_t BUF = N + N / 2, D = 2 * BUF, Q = D + HD;
    static constexpr int OUT = HD + 4;                                 // floats from row to row of the result in shared memory
    static_assert(Q + QT * HD / 2 <= 512 && SMEM + 1024 <= 227 * 1024 - 4608 && (TC_M + 15) * (OUT * 4 + 8) <= 2 * ST * STAGE, "");
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
__device__ __forceinline__ f32x2 pack2(float a, float b) { return tl_pack2(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ f32x2 upper2(f32x2 x) { return x & 0xFFFF0000FFFF0000ull; }
__device__ __forceinline__ f32x2 sub2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint32_t uppers(f32x2 x) { return __byte_perm((uint32_t)x, (uint32_t)(x >> 32), 0x7632); }
// the three pieces of two values, first value in the lower half
__device__ __forceinline__ void cut2(f32x2 x, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
    hi = uppers(x);
    const f32x2 r = sub2(x, upper2(x));
    mid = uppers(r);
    lo = uppers(sub2(r, upper2(r)));
}
__device__ __forceinline__ void st_shared16(uint32_t at, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// products in the order in which they are formed: the piece of A and of B, four bits each
template <int PL>
struct Products {
    static constexpr int N = PL == 1 ? 3 : 6;
    static constexpr uint32_t A = PL == 1 ? 0x012u : 0x001102u, B = PL == 1 ? 0u : 0x010120u;
    static __device__ __forceinline__ constexpr int a(int p) { return A >> (4 * p) & 15; }
    static __device__ __forceinline__ constexpr int b(int p) { return B >> (4 * p) & 15; }
};

// The order in which f32 operands are made: keys of tiles 0 and 1, then values of tile i and keys of tile i + 2 in turn (the scores of tile i + 2 follow the
// outputs of tile i, before the values of tile i + 1 have room).
struct Operand {
    int tile;
    bool val;
};
__device__ __forceinline__ Operand operand_of(int u, int tiles) {          // K0 K1 V0 K2 V1 K3 ... V
    if (u < 2) return {tiles == 1 ? 0 : u, tiles == 1 && u == 1};
    if (u >= 2 * tiles - 1) return {tiles - 1, true};
    return u & 1 ? Operand{(u + 1) >> 1, false} : Operand{(u - 2) >> 1, true};
}
// Registers of a thread from here on, for the four warps of a group (f32: 640 threads of 96 at launch, 480 among the five groups: 2 x 144 + 2 x 72 + 48).
template <bool ON, bool MORE, int R>
__device__ __forceinline__ void tc_regs() {
    if constexpr (ON) {
        if constexpr (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
    }
}
// descriptor of rows of 128 swizzled bytes: groups of eight rows 1024 bytes apart, blocks of 64 values `lbo` bytes apart (MN-major)
__device__ __forceinline__ uint64_t desc_rows128(uint32_t at, uint32_t lbo) {
    return (uint64_t)((at >> 4) & 0x3FFF) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16 | (uint64_t)64 << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// A thread's half of its row of queries as operand A: the first QT pieces into tensor memory at `at` (this warp's lanes), a third that has no room there into
// core matrices in shared memory at q2 (row r).  Complete for the tensor cores after the fences that the caller makes.
template <int HD, int QT>
__device__ __forceinline__ void stage_pieces(const float4 (&qx)[HD / 8], bool negative, uint32_t at, uint32_t q2, int half, int r) {
    const uint32_t flip = negative ? 0x80008000u : 0;
#pragma unroll
    for (int i = 0; i < HD / 8; i += 8) {
        uint32_t p[3][16];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            cut2(pack2(qx[i + j].x, qx[i + j].y), p[0][2 * j], p[1][2 * j], p[2][2 * j]);
            cut2(pack2(qx[i + j].z, qx[i + j].w), p[0][2 * j + 1], p[1][2 * j + 1], p[2][2 * j + 1]);
        }
#pragma unroll
        for (int k = 0; k < 3; k++) {
#pragma unroll
            for (int j = 0; j < 16; j++) p[k][j] ^= flip;
            if (k < QT) tc_st16(at + k * (HD / 2) + half * (HD / 4) + i * 2, p[k]);
            else
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t v[4] = {p[k][4 * j], p[k][4 * j + 1], p[k][4 * j + 2], p[k][4 * j + 3]};
                    st_shared16(q2 + ((half * (HD / 16) + i / 2 + j) * (TC_M / 8) + (r >> 3)) * 128 + (r & 7) * 16, v);
                }
        }
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    fence_proxy_async();
    tl_fence_before();
}

// Which of the slots t0 .. t0 + 63 a row sees that sees cached slots from lo on and the drafted ones of its mask.
__device__ __forceinline__ uint64_t slots_seen(uint64_t mask, int lo, int len, int t0) {
    auto below = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; };
    const int d = len - t0;                                    // where the drafted ones begin
    return (below(d) & ~below(lo - t0)) | (d >= 64 || d <= -64 ? 0ull : d >= 0 ? mask << d : mask >> -d);
}

// One warp's share (lw of eight) of a tile of f32 rows: out of the ring, cut into pieces, into the planes of an operand (values: MN-major).  A thread walks along a
// row of its own, four values at a time, its neighbours four values ahead: reads and writes meet no bank conflicts.  look: rows from `rows` on are zeros, and values
// that are no numbers become zeros and are noted in bad (keys: they stay).
template <int HD, int N>
__device__ __forceinline__ void cut_tile(uint32_t raw, uint32_t dst, int lw, bool val, bool look, int rows, uint32_t *bad) {
    constexpr int ITEMS = N * HD / 4 / 256, GROUPS = N / 32, NC = HD / 8, PLANE = N * HD * 2;
    const int lane = threadIdx.x & 31, row = lane & 7;
    auto item = [&](int k) {
        const int rg = lw % GROUPS * 4 + (lane >> 3), c = (lw / GROUPS * ITEMS + k + row + (lane >> 3)) & (HD / 4 - 1), rr = rg * 8 + row;
        const uint4 y = lds128(raw + (rr * HD + c * 4) * 4);
        f32x2 v[2] = {tl_pack2(y.x, y.y), tl_pack2(y.z, y.w)};
        if (look) {
            bool any = false;
#pragma unroll
            for (int d = 0; d < 2; d++) any |= not_finite(__uint_as_float((uint32_t)v[d])) || not_finite(__uint_as_float((uint32_t)(v[d] >> 32)));
            if (rr >= rows) v[0] = v[1] = 0ull;
            else if (val && any) {
                v[0] = v[1] = 0ull;
                atomicOr(&bad[rr >> 5], 1u << (rr & 31));
            }
        }
        uint32_t p[3][2];
#pragma unroll
        for (int d = 0; d < 2; d++) cut2(v[d], p[0][d], p[1][d], p[2][d]);
        const int piece = c >> 1;
        const uint32_t at = dst + (val ? rg * NC + piece : piece * (N / 8) + rg) * 128 + row * 16 + (c & 1) * 8;
#pragma unroll
        for (int d = 0; d < 3; d++) asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + d * PLANE), "r"(p[d][0]), "r"(p[d][1]) : "memory");
    };
    if (look) {
        for (int k = 0; k < ITEMS; k++) item(k);
    } else {
#pragma unroll
        for (int k = 0; k < ITEMS; k++) item(k);
    }
}

// The scores' products of a tile: queries (tensor memory qt, the piece behind in shared memory dq) against keys at k0, into column d.
template <class T, int HD, int N, int QT>
__device__ __forceinline__ void issue_scores(uint32_t issue, uint32_t d, uint32_t qt, uint64_t dq, uint64_t k0) {
    typedef Products<T::SPLIT ? 3 : 1> Pr;
    constexpr uint32_t id = (1u << 4) | (1u << 7) | (1u << 10) | ((TC_M >> 4) << 24) | ((uint32_t)(N >> 3) << 17);       // f32 += bf16 x bf16
#pragma unroll
    for (int p = 0; p < Pr::N; p++)
#pragma unroll
        for (int s = 0; s < HD / 16; s++) {
            const uint64_t db = k0 + (uint64_t)((T::SPLIT ? Pr::b(p) * N * HD * 2 + s * 2 * N * 16 : s / 4 * N * 128 + s % 4 * 32) / 16);
            if (Pr::a(p) < QT) tc_mma_ts(issue, d, qt + Pr::a(p) * (HD / 2) + s * 8, db, id, p > 0 || s > 0);
            else tc_mma_ss(issue, d, dq + (uint64_t)(s * 2 * TC_M * 16 / 16), db, id, p > 0 || s > 0);
        }
}

// grid (C, kv heads x blocks of 128 rows, entries), clusters of C.  16 sequences x 512 rows over 2000 bf16 slots of 64: 88 us, 212 TFLOP/s of results and three times that of
// products; tensor pipe 39 %, issue slots 39 %: a tile's scores, weights and outputs wait for one another, and tensor memory has room for two tiles (registers spread
// by thread and copies through the load-store pipe: 129 us).  208 rows x 4 heads over 3700 f32 slots of 128: 31 us on 80 SMs, since eight clusters of more than
// ten CTAs do not fit at once (seven do); on mma.sync it took 147.
template <class T, int HD>
__global__ void __launch_bounds__(Tc<T, HD>::THREADS, 1) tree_tc_kernel(KvDev kv, TreeArgs a, const __grid_constant__ KvMaps maps) {
    typedef Tc<T, HD> S;
    typedef Products<S::PL> Pr;
    constexpr int N = S::N;
    extern __shared__ unsigned char tsm_[];
    unsigned char *tsm = tsm_ + ((1024u - (smem_u32(tsm_) & 1023u)) & 1023u);          // swizzled rows want 1024-byte alignment
    __shared__ __align__(8) uint64_t kfull[S::ST], kempty[S::ST], vfull[S::ST], vempty[S::ST], vraw[S::ST], sfull[2], pready, dfull, qfull, rfull[S::UNITS + 1], rempty[S::UNITS + 1];
    __shared__ TreeRows see;
    __shared__ float part_max[2][2][TC_M];
    __shared__ uint32_t bad[S::ST][N / 32];           // slots of a tile whose values are no numbers (tiles that not every row sees whole)
    __shared__ uint32_t tmem_sh;
    const int per = a.nh / kv.nkv, blocks = (a.rows * per + TC_M - 1) / TC_M;
    const int kvh = blockIdx.y / blocks, row0 = blockIdx.y % blocks * TC_M, b = blockIdx.z;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    // this thread's half of its row of queries and the row's sink, on their way before anything else is known
    const int quarter = warp & 3, half = warp >> 2 & 1, r = quarter * 32 + lane, node = (row0 + r) / per, head = kvh * per + (row0 + r) % per;
    const long long place = ((long long)b * a.rows + node) * a.nh + head;
    pdl_wait();
    float4 qx[HD / 8];
    float sink = -INFINITY;
    if (warp < TC_SOFT) {
        const float4 *p = reinterpret_cast<const float4 *>(a.q + place * HD + half * (HD / 2));
#pragma unroll
        for (int i = 0; i < HD / 8; i++) qx[i] = node < a.rows ? p[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (a.sinks) sink = a.sinks[head] * LOG2E;
    }
    const uint64_t mine = tree_mask(a, b);
    const KvEntry e = kv_entry(kv, b, a.rows, a.seq, a.len, a.count);
    if (!e.ok || row0 >= e.count * per) {
        if (!e.ok && threadIdx.x == 0) kv_error(kv);
        return;
    }
    if (warp == S::ISSUE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_sh)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const uint32_t base0 = smem_u32(tsm);
    const typename T::Val *kc = (const typename T::Val *)kv.k + kv.head(e.seq, kvh), *vc = (const typename T::Val *)kv.v + kv.head(e.seq, kvh);
    const int end = e.len + e.count;
    int from = 0, tiles = 0;
    auto share = [&](int first) {          // this CTA's tiles
        const int s0 = first / N, all = (end + N - 1) / N - s0, chunk = (all + gridDim.x - 1) / gridDim.x;
        from = s0 + blockIdx.x * chunk;
        tiles = max(0, min(chunk, s0 + all - from));
    };
    TlWaiter wait{kv.err ? reinterpret_cast<uint32_t *>(kv.err) : nullptr, false};
    // copies, from operand (f32) or tile (bf16) u0 to u1
    auto bring = [&](int u0, int u1) {
        if constexpr (T::SPLIT) {
            // the ring (rows behind the end are not read)
            for (int u = u0; u < u1; u++) {
                const Operand x = operand_of(u, tiles);
                const int slot = u % S::UNITS, t = (from + x.tile) * N, rows = max(0, min(N, end - t));
                if (u >= S::UNITS) wait(&rempty[slot], ((u / S::UNITS) & 1) ^ 1);
                if (rows) {
                    mbar_expect_tx(&rfull[slot], rows * HD * 4);
                    bulk_g2s(tsm + S::RAW + slot * S::UNIT, (x.val ? vc : kc) + (long long)t * HD, rows * HD * 4, &rfull[slot]);
                } else {
                    mbar_arrive(&rfull[slot]);
                }
            }
        } else {
            // a tile's keys and values (slots behind the end come along: nobody sees them)
            for (int i = u0; i < u1; i++) {
                const int st = i % S::ST, t = (from + i) * N;
                if (i >= S::ST) wait(&kempty[st], (i / S::ST - 1) & 1);
                mbar_expect_tx(&kfull[st], S::PLANE);
                for (int x = 0; x < HD; x += 64) tensor_rows(base0 + S::K + st * S::STAGE + x * N * 2, &maps.k, x, t, kvh, e.seq, &kfull[st]);
                if (i >= S::ST) wait(&vempty[st], (i / S::ST - 1) & 1);
                mbar_expect_tx(&vraw[st], S::PLANE);
                for (int x = 0; x < HD; x += 64) tensor_rows(base0 + S::V + st * S::STAGE + x * N * 2, &maps.v, x, t, kvh, e.seq, &vraw[st]);
            }
        }
    };
    const int room = T::SPLIT ? S::UNITS : S::ST;
    int brought = 0;
    if (tid == S::BULK * 32) {
        for (int i = 0; i < S::ST; i++) { mbar_init(&kfull[i], T::SPLIT ? S::LOAD : 1); mbar_init(&vfull[i], S::LOAD); mbar_init(&vraw[i], 1); mbar_init(&kempty[i], 1); mbar_init(&vempty[i], 1); }
        for (int i = 0; i < S::UNITS; i++) { mbar_init(&rfull[i], 1); mbar_init(&rempty[i], S::LOAD); }
        mbar_init(&sfull[0], 1); mbar_init(&sfull[1], 1); mbar_init(&pready, TC_SOFT); mbar_init(&dfull, 1); mbar_init(&qfull, TC_SOFT);
        mbar_fence_init();
        if (a.window <= 0) {               // what there is room for, before the others are ready
            share(0);
            brought = min(room, T::SPLIT ? 2 * tiles : tiles);
            bring(0, brought);
        }
    }
    tree_rows(a, e, mine, see);
    tl_fence_before();
    __syncthreads();
    tl_fence_after();
    pdl_trigger();                 // not before this CTA holds its tensor memory: the next kernel's might wait for this one with it
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_sh, 0);
    share(see.first);
    auto partial = [&](int i) { return (from + i) * N < see.full || (from + i + 1) * N > e.len; };
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)gridDim.x, rank = (int)blockIdx.x, each = owned_rows(TC_M, C);
    float *out = reinterpret_cast<float *>(tsm + S::K);
    float2 *ml = reinterpret_cast<float2 *>(out + (TC_M + 15) * S::OUT);

    if (warp < TC_SOFT) {
        // ---------------- queries, softmax, output
        tc_regs<T::SPLIT, true, 144>();
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        stage_pieces<HD, S::QT>(qx, a.scale < 0.0f, lanes + S::Q, base0 + S::Q2, half, r);
        __syncwarp();
        if (lane == 0) mbar_arrive(&qfull);
        const uint64_t mask = node < e.count ? see.mask[node] : 0;
        const int lo = node < e.count ? see.lo[node] : 0x7fffffff;
        const bool idle = row0 + quarter * 32 >= e.count * per;         // a warp of padding
        const float c = fmaxf(fabsf(a.scale) * LOG2E, 1e-37f);           // above zero: -infinity stays what it is
        const f32x2 cc = pack2(c, c);
        float m = -INFINITY, l = 0.0f, f = 1.0f;
        f32x2 o[HD / 4];
#pragma unroll
        for (int d = 0; d < HD / 4; d++) o[d] = 0ull;
        auto join_output = [&](int i) {
            wait(&dfull, i & 1);
            if (idle) return;
            tl_fence_after();
            const f32x2 ff = pack2(f, f);
#pragma unroll
            for (int d = 0; d < HD / 2; d += 32) {
                float x[32];
                tc_ld32(lanes + S::D + half * (HD / 2) + d, x);
#pragma unroll
                for (int k = 0; k < 16; k++) o[d / 2 + k] = tl_fma2(o[d / 2 + k], ff, pack2(x[2 * k], x[2 * k + 1]));
            }
        };
        for (int i = 0; i < tiles; i++) {
            const uint32_t buf = lanes + (i & 1) * S::BUF, mine = buf + half * (N / 2);
            const bool part = partial(i);
            const int t0 = (from + i) * N + half * (N / 2);
            wait(&sfull[i & 1], (i >> 1) & 1);
            float fn = 1.0f;
            if (!idle) {
                tl_fence_after();
                float s[N / 2];
#pragma unroll
                for (int k = 0; k < N / 2; k += 32) tc_ld32(mine + k, s + k);
                if (part) {
                    const uint64_t seen = slots_seen(mask, lo, e.len, t0);
#pragma unroll
                    for (int k = 0; k < N / 2; k++)
                        if (!((uint32_t)(seen >> (k & 32)) >> (k & 31) & 1)) s[k] = -INFINITY;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < N / 2; k += 8)
#pragma unroll
                    for (int j = 0; j < 4; j++) top[j] = fmaxf(fmaxf(top[j], s[k + j]), s[k + 4 + j]);
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                part_max[i & 1][half][r] = mx;
                asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
                const float mn = fmaxf(m, fmaxf(mx, part_max[i & 1][half ^ 1][r]));
                const float safe = mn == -INFINITY ? 0.0f : mn * c;
                fn = exp2_approx((m == -INFINITY ? m : m * c) - safe);
                m = mn;
                const f32x2 neg = pack2(-safe, -safe);
                f32x2 sum[2] = {0ull, 0ull};
#pragma unroll
                for (int k = 0; k < N / 2; k += 32) {
                    uint32_t p0[16], p1[16], p2[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        float x, y;
                        tl_unpack2(tl_fma2(pack2(s[k + 2 * j], s[k + 2 * j + 1]), cc, neg), x, y);
                        const f32x2 p = pack2(exp2_approx(x), exp2_approx(y));
                        sum[j & 1] = tl_add2(sum[j & 1], p);
                        cut2(p, p0[j], p1[j], p2[j]);
                    }
                    tc_st16(mine + k / 2, p0);
                    tc_st16(mine + N / 4 + k / 2, p1);
                    tc_st16(buf + N + half * (N / 4) + k / 2, p2);
                }
                float x, y;
                tl_unpack2(tl_add2(sum[0], sum[1]), x, y);
                l = __fmaf_rn(l, fn, x + y);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            if (part) {
                // values that are no numbers stand as zeros in the operand; a row that sees one of them gets no result
                wait(&vfull[i % S::ST], (i / S::ST) & 1);
                const uint32_t *g = &bad[i % S::ST][half * (N / 64)];
                const uint64_t gone = N == 64 ? g[0] : g[0] | (uint64_t)g[N / 64 - 1] << 32;
                if (gone & slots_seen(mask, lo, e.len, t0)) l = NAN;
            }
            if (i > 0) join_output(i - 1);
            f = fn;
            tl_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pready);
        }
        if (tiles > 0) join_output(tiles - 1);
        part_max[0][half][r] = l;
        asm volatile("bar.sync %0, 256;" ::"r"(9) : "memory");
        l += part_max[0][half ^ 1][r];
        const float m2 = m == -INFINITY ? m : m * c;
        if (C > 1) {
            // nobody in the cluster uses keys and values any more: their place takes the parts of the rows that a CTA owns
            cluster_arrive();
            cluster_wait();
            const int owner = r / each, at = rank * each + r % each;
            if (half == 0) cl.map_shared_rank(ml, owner)[at] = make_float2(m2, l);
            float *to = cl.map_shared_rank(out, owner) + at * S::OUT + half * (HD / 2);
#pragma unroll
            for (int d = 0; d < HD / 4; d += 2) *reinterpret_cast<ulonglong2 *>(to + 2 * d) = make_ulonglong2(o[d], o[d + 1]);
        } else if (node < e.count) {
            const float top = fmaxf(m2, sink), safe = top == -INFINITY ? 0.0f : top, w = exp2_approx(m2 - safe);
            l = __fmaf_rn(l, w, exp2_approx(sink - safe));
            const float k = w * __fdividef(1.0f, l == 0.0f ? 1.0f : l);
            const f32x2 kk = pack2(k, k);
            ulonglong2 *to = reinterpret_cast<ulonglong2 *>(a.out + place * HD + half * (HD / 2));
#pragma unroll
            for (int d = 0; d < HD / 4; d += 2) to[d / 2] = make_ulonglong2(tl_mul2(o[d], kk), tl_mul2(o[d + 1], kk));
            if (a.lse && half == 0) a.lse[place] = (top + log2f(l)) * LN2;
        }
    } else if (warp < S::ISSUE) {
        tc_regs<T::SPLIT, false, 72>();
        const int lw = warp - TC_SOFT, lt = tid - TC_SOFT * 32;
        auto arrive = [&](uint64_t *bar) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        // a clean slate for the slots of a tile that turn out to be no numbers
        auto clean = [&](int st) {
            if (lt < N / 32) bad[st][lt] = 0;
            asm volatile("bar.sync %0, %1;" ::"r"(10), "n"(S::LOAD * 32) : "memory");
        };
        if constexpr (!T::SPLIT) {
            // ---------------- bf16: values have come; where a row may not see all of them, those that are no numbers become zeros
            for (int i = 0; i < tiles; i++) {
                const int st = i % S::ST;
                wait(&vraw[st], (i / S::ST) & 1);
                if (partial(i)) {
                    clean(st);
                    for (int u = lt; u < N * S::NC; u += S::LOAD * 32) {
                        const int row = u / S::NC, c = u % S::NC;
                        const uint32_t at = base0 + S::V + st * S::STAGE + (c >> 3) * (N * 128) + row * 128 + ((c & 7) ^ (row & 7)) * 16;
                        float x[8];
                        T::get(lds128(at), x);
                        bool any = false;
#pragma unroll
                        for (int d = 0; d < 8; d++) any |= not_finite(x[d]);
                        if (any) {
                            const uint32_t zero[4] = {0, 0, 0, 0};
                            st_shared16(at, zero);
                            atomicOr(&bad[st][row >> 5], 1u << (row & 31));
                        }
                    }
                }
                arrive(&vfull[st]);
            }
        } else {
            // ---------------- f32: rows out of the ring, cut into pieces
            for (int u = 0; u < 2 * tiles; u++) {
                const Operand x = operand_of(u, tiles);
                const bool val = x.val, part = partial(x.tile);
                const int i = x.tile, slot = u % S::UNITS;
                if (i > 0) wait(val ? &vempty[0] : &kempty[0], (i - 1) & 1);
                if (val && part) clean(0);
                wait(&rfull[slot], (u / S::UNITS) & 1);
                const uint32_t raw = base0 + S::RAW + slot * S::UNIT, dst = base0 + (val ? S::V : S::K);
                if (part) cut_tile<HD, N>(raw, dst, lw, val, true, end - (from + i) * N, bad[0]);
                else cut_tile<HD, N>(raw, dst, lw, val, false, 0, nullptr);
                __syncwarp();
                if (lane == 0) mbar_arrive(&rempty[slot]);
                arrive(val ? &vfull[0] : &kfull[0]);
            }
        }
    } else {
        tc_regs<T::SPLIT, false, 48>();
        if (warp == S::BULK) {
            // ---------------- copies
            if (lane == 0) bring(brought, T::SPLIT ? 2 * tiles : tiles);
            __syncwarp();
        } else if (warp == S::ISSUE) {
            // ---------------- products (the whole warp walks the loop, an elected lane issues)
            const uint32_t issue = elect_one() ? 1u : 0u;
            constexpr uint32_t types = (1u << 4) | (1u << 7) | (1u << 10) | ((TC_M >> 4) << 24);       // f32 += bf16 x bf16
            constexpr uint32_t id_o = types | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
            const uint64_t dq = tl_smem_desc(tsm + S::Q2, TC_M * 16, 128), dk = T::SPLIT ? tl_smem_desc(tsm + S::K, N * 16, 128) : desc_rows128(base0 + S::K, 16),
                           dv = T::SPLIT ? tl_smem_desc(tsm + S::V, S::NC * 128, 128) : desc_rows128(base0 + S::V, N * 128);
            wait(&qfull, 0);
            auto scores = [&](int i) {
                const int st = i % S::ST;
                wait(&kfull[st], (i / S::ST) & 1);
                tl_fence_after();
                issue_scores<T, HD, N, S::QT>(issue, tmem + (i & 1) * S::BUF, tmem + S::Q, dq, dk + (uint64_t)(st * S::STAGE / 16));
                tl_commit_if(issue, &sfull[i & 1]);
                tl_commit_if(issue, &kempty[st]);
                __syncwarp();
            };
            if (tiles > 0) scores(0);
            if (tiles > 1) scores(1);
            for (int i = 0; i < tiles; i++) {
                const int st = i % S::ST;
                wait(&vfull[st], (i / S::ST) & 1);
                wait(&pready, i & 1);
                tl_fence_after();
                const uint32_t p0 = tmem + (i & 1) * S::BUF;
                const uint64_t v0 = dv + (uint64_t)(st * S::STAGE / 16);
#pragma unroll
                for (int p = 0; p < Pr::N; p++)
#pragma unroll
                    for (int s = 0; s < N / 16; s++) {
                        constexpr int per_half = N / 32;
                        const int h = s / per_half, k = s % per_half;
                        const uint32_t at = p0 + (Pr::a(p) < 2 ? h * (N / 2) + Pr::a(p) * (N / 4) : N + h * (N / 4)) + k * 8;
                        tc_mma_ts(issue, tmem + S::D, at, v0 + (uint64_t)((T::SPLIT ? Pr::b(p) * S::PLANE + s * 2 * S::NC * 128 : s * 2048) / 16), id_o, p > 0 || s > 0);
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
    }
    if (C > 1 && warp >= TC_SOFT) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
    tl_fence_before();
    __syncthreads();
    if (warp == S::ISSUE) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    if (C == 1) return;
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    join_rows<HD, S::OUT>(out, ml, C, each, a.out, a.lse,
                          [&](int i) -> long long {
                              const int r = rank * each + i, node = (row0 + r) / per;
                              return r < TC_M && node < e.count ? ((long long)b * a.rows + node) * a.nh + kvh * per + (row0 + r) % per : -1;
                          },
                          [&](int i) { return a.sinks ? a.sinks[kvh * per + (row0 + rank * each + i) % per] * LOG2E : -INFINITY; });
}

// ---------------------------------------------------------------- book of weights
// The same scores, 2^(score - lse) of each, and their sum over the rows of the lanes: halves change places in a butterfly, so that a sum of 64 columns over 32 lanes
// takes 62 exchanges; four warps' sums meet in shared memory and go to the book by one thread per slot.  A CTA takes its tiles once for every 128
// rows, in order.  7 sequences x 296 rows x 4 heads over 2500 bf16 slots of 128: 33.5 us, tensor pipe 27 %, the exchanges and powers of a tile wait for its scores;
// on mma.sync it took 146.
template <class T, int HD>
struct Wc {
    typedef Tc<T, HD> S;
    static constexpr int N = S::N, CUT = T::SPLIT ? 8 : 0, ISSUE = TC_SOFT + CUT, BULK = ISSUE + 1, THREADS = (BULK + 1) * 32;
    static constexpr int ST = T::SPLIT ? 1 : 4, UNITS = T::SPLIT ? 3 : 1;
    static constexpr int K = S::K, RAW = K + ST * S::STAGE, BYTES = RAW + (T::SPLIT ? UNITS * S::UNIT : 0);
    static constexpr size_t SMEM = BYTES > 118784 ? BYTES : 118784;
    static constexpr uint32_t Q = 2 * N;                        // columns: scores twice, the queries
};
template <class T, int HD>
__global__ void __launch_bounds__(Wc<T, HD>::THREADS, 1) weigh_tc_kernel(KvDev kv, TreeArgs a, const uint64_t *picked, const __grid_constant__ KvMaps maps) {
    typedef Wc<T, HD> W;
    typedef Tc<T, HD> S;
    constexpr int N = W::N;
    extern __shared__ unsigned char tsm_[];
    unsigned char *tsm = tsm_ + ((1024u - (smem_u32(tsm_) & 1023u)) & 1023u);
    __shared__ __align__(8) uint64_t kfull[W::ST], kempty[W::ST], sfull[2], sfree[2], qfull, rfull[W::UNITS], rempty[W::UNITS];
    __shared__ TreeRows see;
    __shared__ float part[2][4][N];
    __shared__ uint32_t tmem_sh;
    const int per = a.nh / kv.nkv, kvh = blockIdx.y, b = blockIdx.z;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    pdl_wait();
    const uint64_t mine = tree_mask(a, b);
    const KvEntry e = kv_entry(kv, b, a.rows, a.seq, a.len, a.count);
    if (kv_named_before(a.seq, b) || !e.ok) {
        if (tid == 0) kv_error(kv);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < W::ST; i++) { mbar_init(&kfull[i], T::SPLIT ? W::CUT : 1); mbar_init(&kempty[i], 1); }
        for (int i = 0; i < W::UNITS; i++) { mbar_init(&rfull[i], 1); mbar_init(&rempty[i], T::SPLIT ? W::CUT : 1); }
        for (int i = 0; i < 2; i++) { mbar_init(&sfull[i], 1); mbar_init(&sfree[i], TC_SOFT); }
        mbar_init(&qfull, TC_SOFT);
        mbar_fence_init();
    }
    if (warp == W::ISSUE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_sh)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tree_rows(a, e, mine, see);
    tl_fence_before();
    __syncthreads();
    tl_fence_after();
    pdl_trigger();                 // see tree_tc_kernel
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_sh, 0), base0 = smem_u32(tsm);
    const int end = e.len + e.count, s0 = see.first / N, all = (end + N - 1) / N - s0, chunk = (all + gridDim.x - 1) / gridDim.x;
    const int from = s0 + blockIdx.x * chunk, tiles = max(0, min(chunk, s0 + all - from)), blocks = (e.count * per + TC_M - 1) / TC_M, total = tiles * blocks;
    TlWaiter wait{kv.err ? reinterpret_cast<uint32_t *>(kv.err) : nullptr, false};
    const typename T::Val *kc = (const typename T::Val *)kv.k + kv.head(e.seq, kvh);

    if (warp < TC_SOFT) {
        const int quarter = warp & 3, half = warp >> 2, r = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint64_t rows = picked ? picked[b] : ~0ull;
        const float c = fmaxf(fabsf(a.scale) * LOG2E, 1e-37f);
        float *weight = kv.weight + kv.book(e.seq, kvh);
        int j = 0;
        for (int blk = 0; blk < blocks && tiles > 0; blk++) {
            const int node = (blk * TC_M + r) / per;
            const long long place = ((long long)b * a.rows + node) * a.nh + kvh * per + (blk * TC_M + r) % per;
            {
                // the products with the block's queries before are done: their last scores have been seen
                float4 qx[HD / 8];
                const float4 *p = reinterpret_cast<const float4 *>(a.q + place * HD + half * (HD / 2));
#pragma unroll
                for (int i = 0; i < HD / 8; i++) qx[i] = node < e.count ? p[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                stage_pieces<HD, S::QT>(qx, a.scale < 0.0f, lanes + W::Q, base0 + S::Q2, half, r);
                __syncwarp();
                if (lane == 0) mbar_arrive(&qfull);
            }
            const float of_row = node < e.count ? a.lse[place] : -INFINITY;          // -infinity: the row has no weights
            const bool counts = node < e.count && (rows >> node & 1) && of_row != -INFINITY;
            const uint64_t mask = counts ? see.mask[node] : 0;
            const int lo = counts ? see.lo[node] : 0x7fffffff;
            const float z = counts ? of_row * LOG2E : 0.0f;
            const bool every = __all_sync(0xffffffffu, counts);
            for (int i = 0; i < tiles; i++, j++) {
                const int t0 = (from + i) * N;
                const bool look = !every || t0 < see.full || t0 + N > e.len;
                wait(&sfull[j & 1], (j >> 1) & 1);
                tl_fence_after();
                float s[N / 2];
#pragma unroll
                for (int k = 0; k < N / 2; k += 32) tc_ld32(lanes + (j & 1) * N + half * (N / 2) + k, s + k);
                tl_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sfree[j & 1]);
                if (look) {
                    const uint64_t seen = counts ? slots_seen(mask, lo, e.len, t0 + half * (N / 2)) : 0;
#pragma unroll
                    for (int k = 0; k < N / 2; k++)
                        if (!((uint32_t)(seen >> (k & 32)) >> (k & 31) & 1)) s[k] = -INFINITY;
                }
#pragma unroll
                for (int k = 0; k < N / 2; k++) s[k] = exp2_approx(__fmaf_rn(s[k], c, -z));
#pragma unroll
                for (int n = N / 4, o = 16; n > 0; n >>= 1, o >>= 1) {
                    if (o == 0) break;
                    const bool up = lane & o;
#pragma unroll
                    for (int k = 0; k < n; k++) {
                        const float keep = up ? s[k + n] : s[k], give = up ? s[k] : s[k + n];
                        s[k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                    }
                }
                // 32 columns: one is left in a lane, 64: two
                float *to = &part[j & 1][quarter][half * (N / 2)];
                if (N == 64) to[lane] = s[0];
                else *reinterpret_cast<float2 *>(to + 2 * lane) = make_float2(s[0], s[1]);
                asm volatile("bar.sync %0, 256;" ::"r"(9) : "memory");
                if (tid < N && t0 + tid < end) weight[t0 + tid] += (part[j & 1][0][tid] + part[j & 1][1][tid]) + (part[j & 1][2][tid] + part[j & 1][3][tid]);
            }
        }
    } else if (T::SPLIT && warp < W::ISSUE) {
        for (int j = 0; j < total; j++) {
            const int t = (from + j % tiles) * N, slot = j % W::UNITS;
            if (j > 0) wait(&kempty[0], (j - 1) & 1);
            wait(&rfull[slot], (j / W::UNITS) & 1);
            cut_tile<HD, N>(base0 + W::RAW + slot * S::UNIT, base0 + W::K, warp - TC_SOFT, false, t + N > end, end - t, nullptr);
            __syncwarp();
            if (lane == 0) mbar_arrive(&rempty[slot]);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&kfull[0]);
        }
    } else if (warp == W::BULK) {
        if (lane == 0)
            for (int j = 0; j < total; j++) {
                const int t = (from + j % tiles) * N;
                if constexpr (T::SPLIT) {
                    const int slot = j % W::UNITS, rows = min(N, end - t);
                    if (j >= W::UNITS) wait(&rempty[slot], (j / W::UNITS - 1) & 1);
                    mbar_expect_tx(&rfull[slot], rows * HD * 4);
                    bulk_g2s(tsm + W::RAW + slot * S::UNIT, kc + (long long)t * HD, rows * HD * 4, &rfull[slot]);
                } else {
                    const int st = j % W::ST;
                    if (j >= W::ST) wait(&kempty[st], (j / W::ST - 1) & 1);
                    mbar_expect_tx(&kfull[st], S::PLANE);
                    for (int x = 0; x < HD; x += 64) tensor_rows(base0 + W::K + st * S::STAGE + x * N * 2, &maps.k, x, t, kvh, e.seq, &kfull[st]);
                }
            }
        __syncwarp();
    } else if (warp == W::ISSUE) {
        const uint32_t issue = elect_one() ? 1u : 0u;
        const uint64_t dq = tl_smem_desc(tsm + S::Q2, TC_M * 16, 128), dk = T::SPLIT ? tl_smem_desc(tsm + W::K, N * 16, 128) : desc_rows128(base0 + W::K, 16);
        for (int j = 0; j < total; j++) {
            const int st = j % W::ST;
            if (j % tiles == 0) wait(&qfull, (j / tiles) & 1);
            if (j >= 2) wait(&sfree[j & 1], ((j >> 1) - 1) & 1);
            wait(&kfull[st], (j / W::ST) & 1);
            tl_fence_after();
            issue_scores<T, HD, N, S::QT>(issue, tmem + (j & 1) * N, tmem + W::Q, dq, dk + (uint64_t)(st * S::STAGE / 16));
            tl_commit_if(issue, &sfull[j & 1]);
            tl_commit_if(issue, &kempty[st]);
            __syncwarp();
        }
    }
    tl_fence_before();
    __syncthreads();
    if (warp == W::ISSUE) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <class T, int HD>
cudaError_t launch_tree_tc_as(const KvDev &kv, const TreeArgs &a, int slots, cudaStream_t st) {
    typedef Tc<T, HD> S;
    const int blocks = (a.rows * (a.nh / kv.nkv) + TC_M - 1) / TC_M;
    KvMaps maps{};
    cudaError_t e = T::SPLIT ? cudaSuccess : kv_maps(kv, S::N, &maps);
    if (e != cudaSuccess) return e;
    constexpr auto K = tree_tc_kernel<T, HD>;
    constexpr size_t smem = S::SMEM + 1024;
    const int c = cluster_size<K>((long long)a.n * kv.nkv * blocks, (slots + S::N - 1) / S::N, 1, 4, S::THREADS, smem, smem, &e);
    if (e != cudaSuccess) return e;
    return launch_cluster<K>(dim3(c, kv.nkv * blocks, a.n), S::THREADS, c, smem, smem, st, kv, a, maps);
}

template <class T, int HD>
cudaError_t launch_weigh_tc_as(const KvDev &kv, const TreeArgs &a, const uint64_t *picked, int slots, cudaStream_t st) {
    typedef Wc<T, HD> W;
    KvMaps maps{};
    const cudaError_t e = T::SPLIT ? cudaSuccess : kv_maps(kv, W::N, &maps);
    if (e != cudaSuccess) return e;
    // one wave of CTAs, while each has a tile
    const int jobs = a.n * kv.nkv, tiles = (slots + W::N - 1) / W::N;
    constexpr size_t smem = W::SMEM + 1024;
    return launch_cluster<weigh_tc_kernel<T, HD>>(dim3(std::max(1, std::min(tiles, 148 / jobs)), kv.nkv, a.n), W::THREADS, 1, smem, smem, st, kv, a, picked, maps);
}

}  // namespace

cudaError_t launch_weigh_tc(const KvDev &kv, const TreeArgs &a, const uint64_t *picked, int slots, cudaStream_t st) {
    if (kv.type) return kv.hd == 64 ? launch_weigh_tc_as<KvBf16, 64>(kv, a, picked, slots, st) : launch_weigh_tc_as<KvBf16, 128>(kv, a, picked, slots, st);
    return kv.hd == 64 ? launch_weigh_tc_as<KvF32, 64>(kv, a, picked, slots, st) : launch_weigh_tc_as<KvF32, 128>(kv, a, picked, slots, st);
}

cudaError_t launch_tree_tc(const KvDev &kv, const TreeArgs &a, int slots, cudaStream_t st) {
    if (kv.type) return kv.hd == 64 ? launch_tree_tc_as<KvBf16, 64>(kv, a, slots, st) : launch_tree_tc_as<KvBf16, 128>(kv, a, slots, st);
    return kv.hd == 64 ? launch_tree_tc_as<KvF32, 64>(kv, a, slots, st) : launch_tree_tc_as<KvF32, 128>(kv, a, slots, st);
}

}  // namespace brrr
