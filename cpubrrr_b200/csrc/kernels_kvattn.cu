// Attention over KV caches that the caller owns: trees of drafted tokens, chosen blocks, and the book of attention weights.
//
// Rows are (drafted token, query head of one kv head) pairs, 8 or 16 to a CTA; a warp walks slots in steps of 16.  Scores and outputs are formed
// transposed, S^T = K Q^T and O^T = V^T P^T, with mma.sync (m16n8k8, tf32 operands, f32 sums): slots and dimensions are the 16 rows of operand A, and the
// 8 columns of operand B are the rows above, of which a token has 8 (64 query heads over 8): nothing is padded.  Results are single precision: an f32 operand
// x is split into hi = x rounded to tf32's 11 bits and the rest lo = x - hi, exact, of which tf32 takes 11 bits again; hi hi + hi lo + lo hi leaves out
// 2^-21 of a product at most (lo lo, and the last bit of each lo).  bf16 values are tf32 values: for such a cache two products are enough.  The tensor cores' adders truncate, so no long sum is
// left to them: a step's scores take head_dim / 16 additions, a step's share of the output starts at zero and joins the running output by one fused
// multiply-add that also rescales it to the new running maximum.
//
// Every warp has a ring of operands of its own in shared memory, filled by tensor copies of 16 rows several operands ahead, and waits for nobody else.  The
// copies swizzle the rows: with rows as they are, 16-byte reads of keys met two and of values four to a bank (201 tokens x 8 heads over 24 blocks of 32 f32
// slots took 159 us and, swizzled, 144; now, with smaller rings, 118).  The k index of a product may be any order of the dimensions (slots) that both operands have, so a lane's k = t, t + 4 of
// consecutive products are the consecutive values of one 16-byte read, and the rows of V^T may be any order of the dimensions.  Weights change from the
// accumulator's place (slot g, rows 2t, 2t + 1 in lane 4 g + t) to operand B's (slots 2t, 2t + 1, row g) by shuffles.  Queries are split once and wait in
// shared memory in fragment order.
//
// The slots of an entry are split over the warps of a CTA and the CTAs of a cluster, each with its own maximum and sum; partial results meet
// in shared memory, those of the cluster through distributed shared memory, in a fixed order: one launch, no workspace, no atomics.
#include "brrr_kernels.h"
#include "brrr_block.cuh"
#include "brrr_kvattn.cuh"
#include "brrr_tc.cuh"

namespace brrr {

constexpr int AW = 4;                       // warps of an attention CTA; two to four CTAs on an SM

// x rounded to tf32's 11 bits; from 0x7F7FF000 on, just below the largest value, to infinity
__device__ __forceinline__ float tf32_hi(float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xFFFFE000u); }
// Half of two cached values.  f32 keys and values are split as halves, and scores (with the scale) and outputs doubled behind the products: so none is rounded to
// infinity, which the weight of zero of an unseen slot would make no number, and all but subnormal ones give the bits that the whole ones give.  201 rows over 9001 slots:
// 118.0 us, 114.9 without, 120.8 with the smaller of two magnitudes in place of the product.
template <class T>
constexpr float UNIT = T::SPLIT ? 2.0f : 1.0f;
__device__ __forceinline__ void halve(float &x, float &y) {
    tl_unpack2(tl_mul2(tl_pack2(__float_as_uint(x), __float_as_uint(y)), tl_pack2(0x3F000000u, 0x3F000000u)), x, y);
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const float4 &a, float b0, float b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(__float_as_uint(a.x)), "r"(__float_as_uint(a.y)), "r"(__float_as_uint(a.z)), "r"(__float_as_uint(a.w)), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

// A warp's ring: D places for the keys or the values of a step of 16 slots each.  Lane 0 copies; operands are used in the order in which they are copied (keys,
// values, keys, ...).
constexpr int STEP = 16;
template <class T, int HD>
struct Ring {
    static constexpr int ROW = HD * (int)sizeof(typename T::Val), PLACE = STEP * ROW, BYTES = PLACE == 8192 ? 16384 : HD == 64 ? 8192 : 12288, D = BYTES / PLACE;
    static constexpr int NC = HD / (4 * T::V), NVC = HD / (8 * T::V);       // 16-byte reads of a lane per slot: keys, values
    static_assert(D >= 2 && D <= 8, "");
    uint32_t at;             // of the ring, in shared memory
    uint64_t *full;          // [D]
    int in = 0, out = 0, in_turn = 0;      // places that the next copy and the next use take, and the parity of the next use
    __device__ __forceinline__ Ring(unsigned char *mem, uint64_t *bars, const KvMaps &maps) {
        const int warp = threadIdx.x >> 5;
        at = smem_u32(mem) + warp * BYTES;
        full = bars + warp * 8;
        if ((threadIdx.x & 31) == 0) {
            tensor_prefetch(&maps.k);
            tensor_prefetch(&maps.v);
            for (int i = 0; i < D; i++) mbar_init(&full[i], 1);
            mbar_fence_init();
        }
        __syncwarp();
    }
    // slots base .. base + 15 of a head to the next place, which must have been used
    __device__ __forceinline__ void bring(const CUtensorMap *map, int base, int kvh, int seq) {
        if ((threadIdx.x & 31) == 0) {
            mbar_expect_tx(&full[in], PLACE);
#pragma unroll
            for (int i = 0; i < ROW / 128; i++) tensor_rows(at + in * PLACE + i * 2048, map, i * 8 * T::V, base, kvh, seq, &full[in]);
        }
        in = in + 1 == D ? 0 : in + 1;
    }
    // the next operand's place, once it has come
    __device__ __forceinline__ uint32_t next(TlWaiter &wait) {
        wait(&full[out], in_turn);
        const uint32_t p = at + out * PLACE;
        if (++out == D) { out = 0; in_turn ^= 1; }
        return p;
    }
    // this lane's 16 bytes c of the key of slot 8 j + lane / 4: piece 2 (lane % 4) + c % 2 of its 128 bytes c / 2; and of the value of slot 8 k + 2 (lane % 4) + h:
    // piece lane / 4 of its 128 bytes c
    __device__ __forceinline__ static uint4 key(uint32_t st, int j, int c) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        return lds128(st + (c >> 1) * 2048 + j * 1024 + g * 128 + (((2 * t) ^ g ^ (c & 1)) << 4));
    }
    __device__ __forceinline__ static uint4 value(uint32_t st, int k, int h, int c) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        return lds128(st + c * 2048 + k * 1024 + (2 * t + h) * 128 + ((g ^ (2 * t + h)) << 4));
    }
};

// Queries of NT tiles of 8 rows as operand B: per product (8 dimensions), tile and lane 16 bytes, the hi and the lo parts of its two values.  row(r): the row's
// values, or null for a row of padding (zeros).
template <class T, int HD, int NT, class Row>
__device__ __forceinline__ void stage_queries(float4 *frag, Row row) {
    constexpr int W = 8 * T::V;                 // dimensions of 128 bytes
    float *f = reinterpret_cast<float *>(frag);
    for (int u = threadIdx.x; u < NT * 8 * (HD / 4); u += AW * 32) {
        const int r = u / (HD / 4), d0 = u % (HD / 4) * 4;
        const float *p = row(r);
        const float4 x4 = p ? *reinterpret_cast<const float4 *>(p + d0) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d = d0 + i, piece = d % W / T::V, t = piece >> 1, product = (d / W * 2 + (piece & 1)) * (T::V / 2) + d % T::V / 2, odd = d & 1;
            const int at = ((product * NT + r / 8) * 32 + (r & 7) * 4 + t) * 4 + odd;
            float hi = tf32_hi(x[i]);
            if (not_finite(hi)) hi = __uint_as_float(__float_as_uint(x[i]) & 0xFFFFE000u);          // cut off in place of infinity
            f[at] = hi;
            f[at + 2] = x[i] - hi;
        }
    }
}

// Scores of 16 slots over UNIT: s[n] is the accumulator of rows 8 n ..: slot g (+ 8), rows 2t, 2t + 1.
template <class T, int HD, int NT>
__device__ __forceinline__ void step_scores(uint32_t st, const float4 *frag, float (&s)[NT][4]) {
    typedef Ring<T, HD> R;
    constexpr int P = T::V / 2;                 // products per read
    const int lane = threadIdx.x & 31;
    float sum[NT][T::SPLIT ? 6 : 4][4];         // big and small products of even and odd steps
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < (T::SPLIT ? 6 : 4); i++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum[n][i][e] = 0.0f;
#pragma unroll
    for (int c = 0; c < R::NC; c++) {
        float x[2][T::V];
        T::get(R::key(st, 0, c), x[0]);
        T::get(R::key(st, 1, c), x[1]);
#pragma unroll
        for (int p = 0; p < P; p++) {
            float4 ah, al;
            if (T::SPLIT) {
                halve(x[0][2 * p], x[0][2 * p + 1]);
                halve(x[1][2 * p], x[1][2 * p + 1]);
                ah = make_float4(tf32_hi(x[0][2 * p]), tf32_hi(x[1][2 * p]), tf32_hi(x[0][2 * p + 1]), tf32_hi(x[1][2 * p + 1]));
                al = make_float4(x[0][2 * p] - ah.x, x[1][2 * p] - ah.y, x[0][2 * p + 1] - ah.z, x[1][2 * p + 1] - ah.w);
            } else {
                ah = make_float4(x[0][2 * p], x[1][2 * p], x[0][2 * p + 1], x[1][2 * p + 1]);
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float4 b = frag[((c * P + p) * NT + n) * 32 + lane];
                constexpr int S = T::SPLIT ? 3 : 2;
                float(&to)[T::SPLIT ? 6 : 4][4] = sum[n];
                const int o = p & 1 ? S : 0;
                mma_tf32(to[o], ah, b.x, b.y);
                mma_tf32(to[o + 1], ah, b.z, b.w);
                if (T::SPLIT) mma_tf32(to[o + S - 1], al, b.x, b.y);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (T::SPLIT) s[n][e] = (sum[n][0][e] + sum[n][3][e]) + ((sum[n][1][e] + sum[n][2][e]) + (sum[n][4][e] + sum[n][T::SPLIT ? 5 : 0][e]));
            else s[n][e] = (sum[n][0][e] + sum[n][2][e]) + (sum[n][1][e] + sum[n][3][e]);
        }
}

// A warp's running attention of 8 NT rows: maxima and sums in powers of two of rows 8 n + 2t, 2t + 1 (the sum: this lane's slots only), and the outputs (f32: their
// halves).
template <class T, int HD, int NT>
struct Running {
    typedef Ring<T, HD> R;
    static constexpr int MT = HD / 16, PER = T::V / 2;      // 16 dimensions each; how many of them a 16-byte read of values serves
    float m[NT][2], l[NT][2], o[MT][NT][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int f = 0; f < 2; f++) { m[n][f] = -INFINITY; l[n][f] = 0.0f; }
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[i][n][e] = 0.0f;
    }
    // s: scaled scores in powers of two, -infinity where a row does not see the slot.  partial: some row may not see some slot, whose values may be anything: a
    // value that is no number goes into the sum of the rows that see it, and no further.
    __device__ __forceinline__ void add(uint32_t st, float (&s)[NT][4], bool partial) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        float corr[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int f = 0; f < 2; f++) {
                float top = fmaxf(m[n][f], fmaxf(s[n][f], s[n][f + 2]));
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float safe = top == -INFINITY ? 0.0f : top;
                corr[n][f] = exp2_approx(m[n][f] - safe);
                m[n][f] = top;
                s[n][f] = exp2_approx(s[n][f] - safe);
                s[n][f + 2] = exp2_approx(s[n][f + 2] - safe);
            }
        if (partial) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                bool bad[2] = {false, false};
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int c = 0; c < R::NVC; c++) {
                        float x[T::V];
                        T::get(R::value(st, k, h, c), x);
#pragma unroll
                        for (int i = 0; i < T::V; i++) bad[h] |= not_finite(x[i]);
                    }
                const uint32_t even = __ballot_sync(0xffffffffu, bad[0]), odd = __ballot_sync(0xffffffffu, bad[1]);
                if ((g & 1 ? odd : even) & (0x11111111u << (g >> 1)))         // this lane's slot; a weight of zero: not seen (or of no weight)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int f = 0; f < 2; f++)
                            if (s[n][2 * k + f] != 0.0f) s[n][2 * k + f] = NAN;
            }
        }
        // operand B: slots 2t and 2t + 1 of eight, row g
        float bh[NT][2][2], bl[NT][2][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            l[n][0] = __fmaf_rn(l[n][0], corr[n][0], s[n][0] + s[n][2]);
            l[n][1] = __fmaf_rn(l[n][1], corr[n][1], s[n][1] + s[n][3]);
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int from = 8 * t + 4 * h + (g >> 1);
                    const float x = __shfl_sync(0xffffffffu, s[n][2 * k], from), y = __shfl_sync(0xffffffffu, s[n][2 * k + 1], from), p = g & 1 ? y : x;
                    bh[n][k][h] = tf32_hi(p);
                    bl[n][k][h] = p - bh[n][k][h];
                }
        }
#pragma unroll
        for (int c = 0; c < R::NVC; c++) {
            float d[PER][NT][4];
#pragma unroll
            for (int i = 0; i < PER; i++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) d[i][n][e] = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float x0[T::V], x1[T::V];
                T::get(R::value(st, k, 0, c), x0);
                T::get(R::value(st, k, 1, c), x1);
                if (partial) {
#pragma unroll
                    for (int i = 0; i < T::V; i++) {
                        if (not_finite(x0[i])) x0[i] = 0.0f;
                        if (not_finite(x1[i])) x1[i] = 0.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    float4 a = make_float4(x0[2 * i], x0[2 * i + 1], x1[2 * i], x1[2 * i + 1]);
                    if (T::SPLIT) {
                        halve(a.x, a.y);
                        halve(a.z, a.w);
                        const float4 ah = make_float4(tf32_hi(a.x), tf32_hi(a.y), tf32_hi(a.z), tf32_hi(a.w)), al = make_float4(a.x - ah.x, a.y - ah.y, a.z - ah.z, a.w - ah.w);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            mma_tf32(d[i][n], al, bh[n][k][0], bh[n][k][1]);
                            mma_tf32(d[i][n], ah, bl[n][k][0], bl[n][k][1]);
                            mma_tf32(d[i][n], ah, bh[n][k][0], bh[n][k][1]);
                        }
                    } else {
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            mma_tf32(d[i][n], a, bl[n][k][0], bl[n][k][1]);
                            mma_tf32(d[i][n], a, bh[n][k][0], bh[n][k][1]);
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < PER; i++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[c * PER + i][n][e] = __fmaf_rn(o[c * PER + i][n][e], corr[n][e & 1], d[i][n][e]);
        }
    }
    // Into shared memory: out [8 NT][HD], ml [8 NT].
    __device__ __forceinline__ void store(float *out, float2 *ml) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int f = 0; f < 2; f++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[n][f] += __shfl_xor_sync(0xffffffffu, l[n][f], d);
                const int r = 8 * n + 2 * t + f;
                if (g == 0) ml[r] = make_float2(m[n][f], l[n][f]);
#pragma unroll
                for (int c = 0; c < R::NVC; c++)
#pragma unroll
                    for (int i = 0; i < PER; i += 2)         // products i, i + 1: values 8V c + V g + 2i ...
                        *reinterpret_cast<float4 *>(out + r * HD + 8 * T::V * c + T::V * g + 2 * i) =
                            make_float4(UNIT<T> * o[c * PER + i][n][f], UNIT<T> * o[c * PER + i][n][f + 2], UNIT<T> * o[c * PER + i + 1][n][f], UNIT<T> * o[c * PER + i + 1][n][f + 2]);
            }
    }
};

// The parts of a CTA's warps (out [AW][R][HD], ml [AW][R] in shared memory) to the rows' places or, in a cluster, by way of the owners; got, gml: room for
// the owner's parts, R + 15 rows.  All threads call it, after a barrier; the cluster's CTAs have arrived once at its barrier before.
template <int HD, int R, class Dst, class Sink>
__device__ __forceinline__ void join_warps(float *out, float2 *ml, float *got, float2 *gml, float *o, float *lse, Dst dst, Sink sink) {
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), c = (int)cl.block_rank();
    if (C == 1) {
        join_rows<HD, HD>(out, ml, AW, R, o, lse, dst, sink);
        return;
    }
    const int each = owned_rows(R, C);
    cluster_wait();                // every CTA has begun: its memory may be written
    for (int u = threadIdx.x; u < R * (HD / 4); u += AW * 32) {
        const int r = u / (HD / 4), d = u % (HD / 4) * 4;
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int p = 0; p < AW; p++) m = fmaxf(m, ml[p * R + r].x);
        const float safe = m == -INFINITY ? 0.0f : m;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int p = 0; p < AW; p++) {
            const float2 part = ml[p * R + r];
            const float w = exp2_approx(part.x - safe);
            const float4 y = *reinterpret_cast<const float4 *>(out + (p * R + r) * HD + d);
            l = __fmaf_rn(w, part.y, l);
            x.x = __fmaf_rn(w, y.x, x.x); x.y = __fmaf_rn(w, y.y, x.y); x.z = __fmaf_rn(w, y.z, x.z); x.w = __fmaf_rn(w, y.w, x.w);
        }
        const int owner = r / each, at = c * each + r % each;
        *reinterpret_cast<float4 *>(cl.map_shared_rank(got, owner) + at * HD + d) = x;
        if (d == 0) cl.map_shared_rank(gml, owner)[at] = make_float2(m, l);
    }
    cluster_arrive();
    cluster_wait();
    join_rows<HD, HD>(got, gml, C, each, o, lse, [&](int i) -> long long { return c * each + i < R ? dst(c * each + i) : -1; }, [&](int i) { return sink(c * each + i); });
}

// A CTA's shared memory: the warps' rings, later their parts; the queries; the owner's parts; the warps' maxima and sums.
template <class T, int HD, int NT>
struct Room {
    static constexpr int R = 8 * NT, RINGS = AW * Ring<T, HD>::BYTES, GOT = RINGS + R * HD * 8, GML = GOT + (R + 15) * HD * 4, ML = GML + (R + 15) * 8, BYTES = ML + AW * R * 8;
    static_assert(R * HD * 4 <= Ring<T, HD>::BYTES, "a warp's part fits its ring");
};

// grid (C, kv heads x tiles of 8 NT rows, entries), clusters of C.  One token, 73 slots: 7.5 us alone, of which about 3 are launch and lists; 12 sequences of 1023 slots
// 17 us, 50 MB of keys and values at 3 TB/s: a warp's share is 16 steps, and the first copies and the join are not hidden behind so few.
template <class T, int HD, int NT>
__global__ void __launch_bounds__(AW * 32, HD == 64 ? (NT == 1 ? 4 : 3) : 2) tree_kernel(KvDev kv, TreeArgs a, const __grid_constant__ KvMaps maps) {
    typedef Ring<T, HD> Rg;
    typedef Room<T, HD, NT> Rm;
    constexpr int R = 8 * NT;
    extern __shared__ unsigned char raw_[];
    unsigned char *asm_ = raw_ + ((1024u - (smem_u32(raw_) & 1023u)) & 1023u);          // swizzled rows want 1024-byte alignment
    __shared__ __align__(8) uint64_t bars[AW * 8];
    float4 *frag = reinterpret_cast<float4 *>(asm_ + Rm::RINGS);
    __shared__ TreeRows see;
    const int per = a.nh / kv.nkv, tiles = (a.rows * per + R - 1) / R, kvh = blockIdx.y / tiles, row0 = blockIdx.y % tiles * R, b = blockIdx.z;
    if (gridDim.x > 1) cluster_arrive();
    Rg ring(asm_, bars, maps);
    pdl_wait();
    pdl_trigger();
    const uint64_t mine = tree_mask(a, b);
    const KvEntry e = kv_entry(kv, b, a.rows, a.seq, a.len, a.count);
    if (!e.ok || row0 >= e.count * per) {
        if (!e.ok && threadIdx.x == 0) kv_error(kv);
        if (gridDim.x > 1) cluster_wait();
        return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, end = e.len + e.count;
    int s0 = 0;
    if (a.window > 0) {
        tree_rows(a, e, mine, see);
        __syncthreads();
        s0 = see.first / STEP;
    }
    // the CTA's steps, the warp's among them; the first are on their way while masks and queries are prepared
    const int steps = (end + STEP - 1) / STEP - s0, chunk = (steps + gridDim.x - 1) / gridDim.x;
    const int from = s0 + blockIdx.x * chunk, to = min(from + chunk, s0 + steps), count = max(0, (to - from - warp + AW - 1) / AW);
    auto base_of = [&](int n) { return (from + warp + n * AW) * STEP; };
    // operand u: keys (u even) or values of step u / 2
    auto bring = [&](int u) {
        if (u < 2 * count) ring.bring(u & 1 ? &maps.v : &maps.k, base_of(u >> 1), kvh, e.seq);
    };
    for (int u = 0; u < Rg::D; u++) bring(u);
    if (a.window <= 0) tree_rows(a, e, mine, see);
    auto place = [&](int r) -> long long {
        const int i = (row0 + r) / per;
        return i < e.count ? ((long long)b * a.rows + i) * a.nh + kvh * per + (row0 + r) % per : -1;
    };
    stage_queries<T, HD, NT>(frag, [&](int r) -> const float * { return place(r) >= 0 ? a.q + place(r) * HD : nullptr; });
    __syncthreads();
    // this lane's rows 8 n + 2t, 2t + 1
    uint64_t mask[NT][2];
    int lo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int f = 0; f < 2; f++) {
            const int i = (row0 + 8 * n + 2 * (lane & 3) + f) / per;
            mask[n][f] = i < e.count ? see.mask[i] : 0;
            lo[n][f] = i < e.count ? see.lo[i] : 0x7fffffff;
        }
    const float c = UNIT<T> * a.scale * LOG2E;
    Running<T, HD, NT> run;
    run.clear();
    TlWaiter wait{kv.err ? reinterpret_cast<uint32_t *>(kv.err) : nullptr, false};
    for (int n = 0; n < count; n++) {
        const int base = base_of(n);
        float x[NT][4];
        step_scores<T, HD, NT>(ring.next(wait), frag, x);
        __syncwarp();
        bring(2 * n + Rg::D);
        const bool partial = base < see.full || base + STEP > e.len;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int f = 0; f < 4; f++) {
                x[i][f] *= c;
                if (partial) {
                    const int t = base + (lane >> 2) + 8 * (f >> 1);
                    const bool sees = t < e.len ? t >= lo[i][f & 1] : t < end && (mask[i][f & 1] >> (t - e.len) & 1);
                    if (!sees) x[i][f] = -INFINITY;
                }
            }
        run.add(ring.next(wait), x, partial);
        __syncwarp();
        bring(2 * n + 1 + Rg::D);
    }
    __syncthreads();                 // nobody reads the rings any more
    float *out = reinterpret_cast<float *>(asm_), *got = reinterpret_cast<float *>(asm_ + Rm::GOT);
    float2 *gml = reinterpret_cast<float2 *>(asm_ + Rm::GML), *ml = reinterpret_cast<float2 *>(asm_ + Rm::ML);
    run.store(out + warp * R * HD, ml + warp * R);
    __syncthreads();
    join_warps<HD, R>(out, ml, got, gml, a.out, a.lse, place, [&](int r) { return a.sinks ? a.sinks[kvh * per + (row0 + r) % per] * LOG2E : -INFINITY; });
}

template <class T, int HD, int NT>
static cudaError_t launch_tree(const KvDev &kv, const TreeArgs &a, int slots, cudaStream_t st) {
    constexpr size_t smem = Room<T, HD, NT>::BYTES + 1024;
    constexpr auto K = tree_kernel<T, HD, NT>;
    KvMaps maps;
    cudaError_t e = kv_maps(kv, STEP, &maps);
    if (e != cudaSuccess) return e;
    const int tiles = (a.rows * (a.nh / kv.nkv) + 8 * NT - 1) / (8 * NT);
    const int c = cluster_size<K>((long long)a.n * kv.nkv * tiles, (slots + STEP - 1) / STEP, AW, 4, AW * 32, smem, smem, &e);
    if (e != cudaSuccess) return e;
    return launch_cluster<K>(dim3(c, kv.nkv * tiles, a.n), AW * 32, c, smem, smem, st, kv, a, maps);
}

// Whether the kernel of 128-row tiles (kernels_kvtc.cu) takes less time than CTAs of 16 rows.  Both were measured with 8 to 256 rows, 1 and 8 sequences, 40 to 2500
// slots (20 calls in a graph, in L2): a tile of 128 rows takes the time of one and a half of 16, and a start of `start` tiles of 16 rows x 128 slots (spread over
// the GPU) more.  The rule takes at most 10 % more than the better one of the two (38 % for 256 rows of 128 f32 dimensions over 700 slots: 17.0 and 23.4 us).  64
// dimensions f32, 8 heads: 64 rows over 200 slots 6.4 and 13.0 us, over 2500 15.8 and 17.0; 8 sequences: 32 rows over 700 16.0 and 18.7, 128 rows over 2500
// 151 and 40.
static bool wide_rows_pay(const KvDev &kv, const TreeArgs &a, int slots) {
    static const double start[2][2] = {{400, 200}, {175, 150}};         // f32, bf16 of 64 and of 128 dimensions
    const int rows = a.rows * (a.nh / kv.nkv);
    return (double)a.n * kv.nkv * (slots / 128.0) * ((rows + 15) / 16 - 1.5 * ((rows + 127) / 128)) > start[kv.type][kv.hd == 128];
}

// About the slots of an entry that its rows see.  A window is up to INT_MAX wide: the cached slots are taken from it before the rows are added.
static int tree_slots(const KvDev &kv, const TreeArgs &a, int len_hint) {
    const int cached = len_hint > 0 ? min(len_hint, kv.cap) : kv.cap;
    return (a.window > 0 ? min(cached, a.window) : cached) + a.rows;
}

cudaError_t launch_attn_tree(const KvDev &kv, const TreeArgs &a, int len_hint, cudaStream_t st) {
    const int slots = tree_slots(kv, a, len_hint);
    if (wide_rows_pay(kv, a, slots)) return launch_tree_tc(kv, a, slots, st);
    const bool one = a.rows * (a.nh / kv.nkv) <= 8;
    auto go = kv.type ? (kv.hd == 64 ? (one ? launch_tree<KvBf16, 64, 1> : launch_tree<KvBf16, 64, 2>) : (one ? launch_tree<KvBf16, 128, 1> : launch_tree<KvBf16, 128, 2>))
                      : (kv.hd == 64 ? (one ? launch_tree<KvF32, 64, 1> : launch_tree<KvF32, 64, 2>) : (one ? launch_tree<KvF32, 128, 1> : launch_tree<KvF32, 128, 2>));
    return go(kv, a, slots, st);
}

// ---------------------------------------------------------------- book of weights
// Up to 16 rows per kv head.  A warp owns a step of slots: the scores of its keys, their powers, the sum over the rows.  24 sequences of 3801 f32 slots: 30.7 us, keys at
// 4.9 TB/s.  More rows go to kernels_kvtc.cu; 16 take 3.8 us here and 6.1 there over 200 slots of 64 f32 dimensions, 13.2 and 23.4 from 8 sequences of 2500.
template <class T, int HD, int NT>
__global__ void __launch_bounds__(AW * 32, 3) weigh_kernel(KvDev kv, TreeArgs a, const uint64_t *picked, const __grid_constant__ KvMaps maps) {
    typedef Ring<T, HD> Rg;
    extern __shared__ unsigned char raw_[];
    unsigned char *asm_ = raw_ + ((1024u - (smem_u32(raw_) & 1023u)) & 1023u);          // the warps' rings, the queries
    __shared__ __align__(8) uint64_t bars[AW * 8];
    __shared__ TreeRows see;
    float4 *frag = reinterpret_cast<float4 *>(asm_ + AW * Rg::BYTES);
    const int kvh = blockIdx.y, b = blockIdx.z, per = a.nh / kv.nkv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Rg ring(asm_, bars, maps);
    pdl_wait();
    pdl_trigger();
    const uint64_t mine = tree_mask(a, b);
    const KvEntry e = kv_entry(kv, b, a.rows, a.seq, a.len, a.count);
    if (kv_named_before(a.seq, b) || !e.ok) {
        if (threadIdx.x == 0) kv_error(kv);
        return;
    }
    const int end = e.len + e.count;
    float *weight = kv.weight + kv.book(e.seq, kvh);
    int s0 = 0;
    if (a.window > 0) {
        tree_rows(a, e, mine, see);
        __syncthreads();
        s0 = see.first / STEP;
    }
    const int steps = (end + STEP - 1) / STEP - s0, chunk = (steps + gridDim.x - 1) / gridDim.x;
    const int from = s0 + blockIdx.x * chunk, to = min(from + chunk, s0 + steps), count = max(0, (to - from - warp + AW - 1) / AW);
    auto base_of = [&](int n) { return (from + warp + n * AW) * STEP; };
    for (int n = 0; n < min(count, Rg::D); n++) ring.bring(&maps.k, base_of(n), kvh, e.seq);
    if (a.window <= 0) tree_rows(a, e, mine, see);
    const uint64_t rows = picked ? picked[b] : ~0ull;
    auto place = [&](int r) -> long long {
        const int i = r / per;
        return i < e.count ? ((long long)b * a.rows + i) * a.nh + kvh * per + r % per : -1;
    };
    stage_queries<T, HD, NT>(frag, [&](int r) -> const float * { return place(r) >= 0 ? a.q + place(r) * HD : nullptr; });
    // this lane's rows 8 n + 2t, 2t + 1; one that does not count sees nothing
    bool counts[NT][2];
    float z[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int f = 0; f < 2; f++) {
            const int r = 8 * n + 2 * (lane & 3) + f, i = r / per;
            z[n][f] = i < e.count ? a.lse[place(r)] * LOG2E : -INFINITY;          // -infinity: the row has no weights
            counts[n][f] = i < e.count && (rows >> i & 1) && z[n][f] != -INFINITY;
        }
    __syncthreads();
    uint64_t mask[NT][2];
    int lo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int f = 0; f < 2; f++) {
            const int i = (8 * n + 2 * (lane & 3) + f) / per;
            mask[n][f] = counts[n][f] ? see.mask[i] : 0;
            lo[n][f] = counts[n][f] ? see.lo[i] : 0x7fffffff;
        }
    const float c = UNIT<T> * a.scale * LOG2E;
    TlWaiter wait{kv.err ? reinterpret_cast<uint32_t *>(kv.err) : nullptr, false};
    for (int n = 0; n < count; n++) {
        const int base = base_of(n);
        // lane t < 2 writes slot g + 8t: what the book has
        const int mine_at = base + (lane >> 2) + 8 * (lane & 3);
        const bool writes = (lane & 3) < 2 && mine_at < end;
        const float had = writes ? weight[mine_at] : 0.0f;
        float x[NT][4], sum[2] = {0.0f, 0.0f};
        step_scores<T, HD, NT>(ring.next(wait), frag, x);
        __syncwarp();
        if (n + Rg::D < count) ring.bring(&maps.k, base_of(n + Rg::D), kvh, e.seq);
        const bool partial = base < see.full || base + STEP > e.len;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int f = 0; f < 4; f++) {
                float p = exp2_approx(__fmaf_rn(x[i][f], c, -z[i][f & 1]));
                bool sees = counts[i][f & 1];
                if (partial) {
                    const int t = base + (lane >> 2) + 8 * (f >> 1);
                    sees = t < e.len ? t >= lo[i][f & 1] : t < end && (mask[i][f & 1] >> (t - e.len) & 1);
                }
                sum[f >> 1] += sees ? p : 0.0f;
            }
#pragma unroll
        for (int f = 0; f < 2; f++) {
            sum[f] += __shfl_xor_sync(0xffffffffu, sum[f], 1);
            sum[f] += __shfl_xor_sync(0xffffffffu, sum[f], 2);
        }
        if (writes) weight[mine_at] = had + sum[lane & 1];
    }
}

template <class T, int HD, int NT>
static cudaError_t launch_weigh(const KvDev &kv, const TreeArgs &a, const uint64_t *picked, int slots, cudaStream_t st) {
    constexpr size_t smem = (size_t)AW * Ring<T, HD>::BYTES + HD * 64 * NT + 1024;
    constexpr auto K = weigh_kernel<T, HD, NT>;
    KvMaps maps;
    cudaError_t e = kv_maps(kv, STEP, &maps);
    if (e != cudaSuccess) return e;
    // CTAs of an entry and head: as with clusters, the least time of all waves
    const int c = cluster_size<K, false>((long long)kv.nkv * a.n, (slots + STEP - 1) / STEP, AW, 4, AW * 32, smem, smem, &e);
    if (e != cudaSuccess) return e;
    return launch_cluster<K>(dim3(c, kv.nkv, a.n), AW * 32, 1, smem, smem, st, kv, a, picked, maps);
}

cudaError_t launch_kv_weigh(const KvDev &kv, const TreeArgs &a, const uint64_t *picked, int len_hint, cudaStream_t st) {
    const int slots = tree_slots(kv, a, len_hint);
    if (a.rows * (a.nh / kv.nkv) > 16) return launch_weigh_tc(kv, a, picked, slots, st);
    const bool one = a.rows * (a.nh / kv.nkv) <= 8;
    auto go = kv.type ? (kv.hd == 64 ? (one ? launch_weigh<KvBf16, 64, 1> : launch_weigh<KvBf16, 64, 2>) : (one ? launch_weigh<KvBf16, 128, 1> : launch_weigh<KvBf16, 128, 2>))
                      : (kv.hd == 64 ? (one ? launch_weigh<KvF32, 64, 1> : launch_weigh<KvF32, 64, 2>) : (one ? launch_weigh<KvF32, 128, 1> : launch_weigh<KvF32, 128, 2>));
    return go(kv, a, picked, slots, st);
}

// ---------------------------------------------------------------- chosen blocks
// A cluster per (kv head, row).  Its CTAs share the blocks' scores: products of f64 (mma m8n8k4, 8 heads by 8 blocks), whose largest over the heads every CTA
// gets as a 32-bit key in the order of the values.  Then each CTA finds the nsel largest keys and takes its share of the chosen blocks' steps.  201 rows x 8 heads over 282
// blocks, 24 of 32 f32 slots chosen: 118 us, 632 MB of keys and values out of L2 at 5.4 TB/s, issue slots half full (rings of 12 KB and three CTAs on an SM
// took 24 us more).  One row over 954 bf16 blocks of 64: 18.2 us, a sequence of latencies (means, scores, cluster barrier, digits, steps, join).
__device__ __forceinline__ void mma_f64(double (&d)[2], double a, double b) {
    asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};" : "+d"(d[0]), "+d"(d[1]) : "d"(a), "d"(b));
}

// The means of blocks j0 .. j0 + 7 (not beyond last): lane 4 g + t has values 16 c + 4 t .. of block j0 + g.
template <int HD>
__device__ __forceinline__ void load_means(const float *__restrict__ mean, int j0, int last, float4 (&x)[HD / 16]) {
    const int lane = threadIdx.x & 31;
    const float *m = mean + (long long)min(j0 + (lane >> 2), last) * HD + 4 * (lane & 3);
#pragma unroll
    for (int c = 0; c < HD / 16; c++) x[c] = *reinterpret_cast<const float4 *>(m + 16 * c);
}
// Their keys: lane 4 g + t has those of blocks j0 + 2t and j0 + 2t + 1 (the same for every g).
template <int HD>
__device__ __forceinline__ void block_keys(const float *__restrict__ q, int per, const float4 (&x)[HD / 16], uint32_t (&key)[2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    key[0] = key[1] = 0;
    for (int h0 = 0; h0 < per; h0 += 8) {
        double sum[4][2];
#pragma unroll
        for (int i = 0; i < 4; i++) sum[i][0] = sum[i][1] = 0.0;
        const float *p = q + (h0 + g) * HD + 4 * t;
#pragma unroll
        for (int c = 0; c < HD / 16; c++) {
            const float4 a = h0 + g < per ? *reinterpret_cast<const float4 *>(p + 16 * c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            mma_f64(sum[0], a.x, x[c].x);
            mma_f64(sum[1], a.y, x[c].y);
            mma_f64(sum[2], a.z, x[c].z);
            mma_f64(sum[3], a.w, x[c].w);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            // the rounding keeps the order, so the largest may be taken afterwards; what is no number wins here and loses in the end
            const float f = (float)((sum[0][i] + sum[1][i]) + (sum[2][i] + sum[3][i]));
            uint32_t k = f != f ? 0xFFFFFFFFu : float_orderable(f == 0.0f ? 0.0f : f);
            if (h0 + g >= per) k = 0;
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
            key[i] = max(key[i], k);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
        if (key[i] == 0xFFFFFFFFu) key[i] = 0;
}

template <class T, int HD, int NT>
__global__ void __launch_bounds__(AW * 32, HD == 64 ? (NT == 1 ? 4 : 3) : 2) blocks_kernel(KvDev kv, const int32_t *seq, const int32_t *len, int block, const float *__restrict__ means, int nsel, int first, int local,
                                                         const float *q, int nh, float scale, const float *sinks, int32_t *sel, float *o, float *lse,
                                                         const __grid_constant__ KvMaps maps) {
    typedef Ring<T, HD> Rg;
    typedef Room<T, HD, NT> Rm;
    constexpr int R = 8 * NT;
    extern __shared__ unsigned char raw_[];
    unsigned char *asm_ = raw_ + ((1024u - (smem_u32(raw_) & 1023u)) & 1023u);          // swizzled rows want 1024-byte alignment
    __shared__ __align__(8) uint64_t bars[AW * 8];
    float4 *frag = reinterpret_cast<float4 *>(asm_ + Rm::RINGS);
    uint32_t *keys = reinterpret_cast<uint32_t *>(asm_ + Rm::BYTES);      // [cap / block + 1]
    __shared__ int32_t chosen[256];
    __shared__ float qs[16 * HD];
    __shared__ KthSpace<8> kth;
    static_assert(AW * 32 == 1 << 7, "as block_kth wants it");
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks();
    const int r = blockIdx.y, kvh = blockIdx.z, per = nh / kv.nkv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (C > 1) cluster_arrive();
    Rg ring(asm_, bars, maps);
    kth.clear();
    pdl_wait();
    pdl_trigger();
    const int s = seq ? seq[r] : r, n = len[r];
    if ((unsigned)s >= (unsigned)kv.n_seq || (unsigned)n > (unsigned)kv.cap) {
        if (threadIdx.x == 0) kv_error(kv);
        if (C > 1) cluster_wait();
        return;
    }
    const long long row = (long long)r * nh + kvh * per;
    const int nb = (n + block - 1) / block, taken = min(nb, nsel);
    for (int i = threadIdx.x; i < per * (HD / 4); i += AW * 32) reinterpret_cast<float4 *>(qs)[i] = reinterpret_cast<const float4 *>(q + row * HD)[i];
    __syncthreads();
    if (nb <= nsel) {
        for (int j = threadIdx.x; j < nb; j += AW * 32) chosen[j] = j;
    } else {
        // scores of the blocks that are not taken anyhow
        const float *mean = means + ((long long)s * kv.nkv + kvh) * (kv.cap / block) * HD;
        const int hi = nb - local, tiles = (hi - first + 7) / 8;
        if (C > 1) cluster_wait();     // every CTA is there: its memory may be written
        float4 x[2][HD / 16];
        const int step = C * AW;
        int i = blockIdx.x * AW + warp;
        load_means<HD>(mean, first + 8 * i, hi - 1, x[0]);
        for (int turn = 0; i < tiles; i += step, turn++) {
            // the next tile's means come while this one's are used
            const int j = first + 8 * i + 2 * (lane & 3);
            uint32_t key[2];
            if (turn & 1) {
                load_means<HD>(mean, first + 8 * (i + step), hi - 1, x[0]);
                block_keys<HD>(qs, per, x[1], key);
            } else {
                load_means<HD>(mean, first + 8 * (i + step), hi - 1, x[1]);
                block_keys<HD>(qs, per, x[0], key);
            }
            for (int p = lane >> 2; p < C; p += 8) {
                uint32_t *there = C > 1 ? cl.map_shared_rank(keys, p) : keys;
                if (j < hi) there[j] = key[0];
                if (j + 1 < hi) there[j + 1] = key[1];
            }
        }
        if (C > 1) {
            cluster_arrive();
            cluster_wait();
            cluster_arrive();          // for the join
        } else {
            __syncthreads();
        }
        uint32_t known = ~0u, ties = 0, equal;
        const int want = nsel - first - local;
        const uint32_t last = want > 0 ? block_kth(hi - first, want, [&](int i) { return keys[first + i]; }, kth, known, ties, equal) : 0xFFFFFFFFu;
        // the places of the chosen ones, in ascending order of blocks: a warp has a run of 32 w blocks and counts them first; both counts in one word
        const int run = (nb + 32 * AW - 1) / (32 * AW), j0 = warp * run * 32 + lane;
        auto kind = [&](int j, bool &over, bool &same) {
            const bool free = j >= first && j < hi;
            const uint32_t k = free ? keys[j] & known : 0;
            over = (j < nb && !free) || (free && want > 0 && k > last);
            same = free && want > 0 && k == last;
        };
        uint32_t count = 0;
        for (int w = 0; w < run; w++) {
            bool over, same;
            kind(j0 + 32 * w, over, same);
            count += __popc(__ballot_sync(0xffffffffu, over)) | __popc(__ballot_sync(0xffffffffu, same)) << 16;
        }
        if (lane == 0) kth.of_warps[warp] = count;
        __syncthreads();
        uint32_t before = 0;
        for (int w = 0; w < warp; w++) before += kth.of_warps[w];
        for (int w = 0; w < run; w++) {
            bool over, same;
            kind(j0 + 32 * w, over, same);
            const uint32_t b_over = __ballot_sync(0xffffffffu, over), b_same = __ballot_sync(0xffffffffu, same), below = (1u << lane) - 1;
            const uint32_t o_rank = (before & 0xFFFF) + __popc(b_over & below), s_rank = (before >> 16) + __popc(b_same & below);
            if (over) chosen[o_rank + min(s_rank, ties)] = j0 + 32 * w;
            else if (same && s_rank < ties) chosen[o_rank + s_rank] = j0 + 32 * w;
            before += __popc(b_over) | __popc(b_same) << 16;
        }
    }
    stage_queries<T, HD, NT>(frag, [&](int i) -> const float * { return i < per ? qs + i * HD : nullptr; });
    __syncthreads();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < nsel; i += AW * 32) sel[((long long)r * kv.nkv + kvh) * nsel + i] = i < taken ? chosen[i] : -1;
    const float c = UNIT<T> * scale * LOG2E;
    const int shift = 31 - __clz(block / STEP), steps = taken << shift;       // steps of a block: a power of two
    Running<T, HD, NT> run;
    run.clear();
    TlWaiter wait{kv.err ? reinterpret_cast<uint32_t *>(kv.err) : nullptr, false};
    const int hop = C * AW, i0 = blockIdx.x * AW + warp, count = max(0, (steps - i0 + hop - 1) / hop);
    auto base_of = [&](int m) {
        const int i = i0 + m * hop;
        return chosen[i >> shift] * block + (i & ((1 << shift) - 1)) * STEP;
    };
    // the last block may end before its last steps: nothing but such steps follows
    auto bring = [&](int u) {
        if (u < 2 * count && base_of(u >> 1) < n) ring.bring(u & 1 ? &maps.v : &maps.k, base_of(u >> 1), kvh, s);
    };
    for (int u = 0; u < Rg::D; u++) bring(u);
    for (int m = 0; m < count; m++) {
        const int base = base_of(m);
        if (base >= n) break;
        float x[NT][4];
        step_scores<T, HD, NT>(ring.next(wait), frag, x);
        __syncwarp();
        bring(2 * m + Rg::D);
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int f = 0; f < 4; f++) x[j][f] = base + (lane >> 2) + 8 * (f >> 1) < n ? x[j][f] * c : -INFINITY;
        run.add(ring.next(wait), x, base + STEP > n);
        __syncwarp();
        bring(2 * m + 1 + Rg::D);
    }
    __syncthreads();
    float *out = reinterpret_cast<float *>(asm_), *got = reinterpret_cast<float *>(asm_ + Rm::GOT);
    float2 *gml = reinterpret_cast<float2 *>(asm_ + Rm::GML), *ml = reinterpret_cast<float2 *>(asm_ + Rm::ML);
    run.store(out + warp * R * HD, ml + warp * R);
    __syncthreads();
    join_warps<HD, R>(out, ml, got, gml, o, lse, [&](int i) -> long long { return i < per ? row + i : -1; },
                   [&](int i) { return sinks ? sinks[kvh * per + i] * LOG2E : -INFINITY; });
}

template <class T, int HD, int NT>
static cudaError_t launch_blocks(const KvDev &kv, int rows, const int32_t *seq, const int32_t *len, int block, const float *means, int nsel, int first, int local,
                                 int len_hint, const float *q, int nh, float scale, const float *sinks, int32_t *sel, float *out, float *lse, cudaStream_t st) {
    const int longest = len_hint > 0 ? min(len_hint, kv.cap) : kv.cap, nb = longest / block;
    // a tile of eight blocks' scores costs about as much as a step
    const int steps = min(nsel, nb + 1) * (block / STEP) + (nb > nsel ? nb / 8 : 0);
    constexpr size_t room = Room<T, HD, NT>::BYTES + 1024, most = room + 16385 * 4;
    // the blocks' keys, 4 KB by 4 KB (the last kind: 64 KB and a word)
    const size_t keys = (size_t)(kv.cap / block + 1) * 4;
    const int kind = (int)min((keys - 1) / 4096, (size_t)ROOM_KINDS - 1);
    const size_t keys_most = min((size_t)(kind + 1) * 4096, most - room);
    constexpr auto K = blocks_kernel<T, HD, NT>;
    KvMaps maps;
    cudaError_t e = kv_maps(kv, STEP, &maps);
    if (e != cudaSuccess) return e;
    const int c = cluster_size<K>((long long)rows * kv.nkv, steps, AW, 4, AW * 32, room + keys_most, most, &e, kind);
    if (e != cudaSuccess) return e;
    return launch_cluster<K>(dim3(c, rows, kv.nkv), AW * 32, c, room + keys, most, st, kv, seq, len, block, means, nsel, first, local, q, nh, scale,
                             sinks, sel, out, lse, maps);
}

cudaError_t launch_attn_blocks(const KvDev &kv, int rows, const int32_t *seq, const int32_t *len, int block, const float *means, int nsel, int first, int local,
                               int len_hint, const float *q, int nh, float scale, const float *sinks, int32_t *sel, float *out, float *lse, cudaStream_t st) {
    const bool one = nh / kv.nkv <= 8;
    auto go = kv.type ? (kv.hd == 64 ? (one ? launch_blocks<KvBf16, 64, 1> : launch_blocks<KvBf16, 64, 2>) : (one ? launch_blocks<KvBf16, 128, 1> : launch_blocks<KvBf16, 128, 2>))
                      : (kv.hd == 64 ? (one ? launch_blocks<KvF32, 64, 1> : launch_blocks<KvF32, 64, 2>) : (one ? launch_blocks<KvF32, 128, 1> : launch_blocks<KvF32, 128, 2>));
    return go(kv, rows, seq, len, block, means, nsel, first, local, len_hint, q, nh, scale, sinks, sel, out, lse, st);
}

}  // namespace brrr
