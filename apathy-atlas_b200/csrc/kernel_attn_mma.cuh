// Paged attention for few rows: one token of every sequence (decode), a few drafts, and any shape the tcgen05 form does not take.
//
// What bounds it is the cache: per KV head and token 2 head_dim values are read for 4 head_dim operations a row, and a KV head has
// `group` rows a token.  The products are the transposed ones, with tokens and channels as the sixteen rows of mma.sync.m16n8k16 and the block's
// rows as its eight columns: S^T = K Q^T, O^T = V^T P^T.  So a block of up to eight rows (RT = 1) wastes nothing: half the matrix
// instructions, exponentials and accumulators of the form with Q as the sixteen rows; RT = 2 has sixteen.  P^T comes out of S^T by one 8 x 8
// transposition (movmatrix).
//
// Every warp has units of sixteen tokens' K and V (32 where rows are short) of its own in flight through a private ring in shared memory
// (cp.async, 16 bytes a lane: a row of the cache is wherever its page is, so any page size will do and places behind a sequence's end are
// filled with zeros; a bulk copy for each row takes 15 cycles whatever its length, which is 2.3 TB/s for rows of 128 bytes), and no warp
// waits for another until the range's item ends: then the warps' maxima, sums and outputs are joined in shared memory.
//
// Where all items' CTAs are resident at once and none would have more than eight tiles, an item is a cluster's: its CTAs take shares of its
// tiles and join over distributed shared memory, without scratch and a second kernel (one sequence of 777 tokens, 8 KV heads of 128: 11.5 -> 7.6 us; eight of 1000: 14.8 -> 11.6; two of 4000 in E4M3: 16.7 -> 13.4).
//
// An E4M3 cache is multiplied as FP16, which holds every E4M3 value: conversion is one instruction for two values and keeps NaN.  Q is
// BF16, whose range FP16 has not, so each row is first multiplied by the power of two that brings its largest value to [2^14, 2^15);
// what then falls below FP16's smallest step is 2^-39 of the row's largest value.  The scores' factor takes the power back.
// P is rounded to BF16 (with an E4M3 cache FP16, of weights up to 2^7: ATTN_UP) for the product with V; its sum is taken before that, in FP32.
#pragma once

#include "kernel_attn.cuh"
#include "kernel_tc.cuh"

namespace atlas {
namespace attn {

using namespace atlas::tc;

// (heads of 256 over E4M3 in blocks of sixteen rows have 128 accumulators: two)
constexpr int attn_mma_ctas(int row_bytes, bool fp8, int rt) { return row_bytes >= 512 ? 1 : row_bytes > 128 && (!fp8 || rt == 2) ? 2 : 3; }
constexpr int MMA_WARPS = 4, MMA_THREADS = 32 * MMA_WARPS;

template <int DP, bool FP8, int RT> struct MmaCfg {
    static constexpr int ROWS = 8 * RT;
    static constexpr int ROW_BYTES = DP * (FP8 ? 1 : 2);
    // Tokens of a unit.  A unit is a chain (copy, scores, maximum, weights, product) of some 1500 cycles whatever its bytes.
    static constexpr int UNIT = ROW_BYTES <= 128 ? 32 : 16, TILE = UNIT * MMA_WARPS;
    static constexpr int SIDE = UNIT * ROW_BYTES;                            // K or V of a unit
    // CTAs on an SM, and the ring as deep as that leaves room for.  Short rows and conversions mean more arithmetic for a byte, so three:
    // what a unit waits for is its own instructions (256 sequences of up to 4096 over E4M3, before other changes that brought it to 242 us: 278 with
    // two, 252 with three; with units of 16 tokens 299, and 290 with four CTAs).
    static constexpr int CTAS = attn_mma_ctas(ROW_BYTES, FP8, RT);
    static constexpr int RING_BYTES = CTAS == 1 ? 196608 : CTAS == 2 ? 98304 : 65536;
    static constexpr int STAGES = RING_BYTES / MMA_WARPS / (2 * SIDE) > 8 ? 8 : RING_BYTES / MMA_WARPS / (2 * SIDE);
    static constexpr int RING = MMA_WARPS * STAGES * 2 * SIDE;
    static constexpr int JOIN = MMA_WARPS * ROWS * (DP + 4) * 4;         // (overlaid)
    static constexpr int MAIN = RING > JOIN ? RING : JOIN;
    static constexpr int SMEM = MAIN + MMA_WARPS * ROWS * 8 + MMA_WARPS * 8 + int(sizeof(AttnStart));
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 8 x 8 matrix of 16-bit values, one row a group of four lanes, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool HALF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two & 0xFFFFu), __NV_E4M3);
    return uint32_t(h.x) | (uint32_t(h.y) << 16);
}
template <bool HALF> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (HALF) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        return pack_bf16x2(a, b);
    }
}
// byte offset of 16-byte chunk `c` of token `t` of a unit whose rows are ROW_BYTES long: the chunk is moved by the token, over as many
// chunks as a row has (eight at most), so that the eight addresses of a matrix or of a quarter warp lie in different banks
template <int ROW_BYTES> __device__ __forceinline__ uint32_t unit_off(uint32_t t, uint32_t c) {
    if constexpr (ROW_BYTES >= 128) return t * ROW_BYTES + ((c ^ (t & 7u)) << 4);
    else return t * ROW_BYTES + ((c ^ ((t >> 1) & 3u)) << 4);
}

template <int DP, bool FP8, int RT>
__global__ void __launch_bounds__(MMA_THREADS, MmaCfg<DP, FP8, RT>::CTAS) attn_mma_kernel(const __grid_constant__ AttnParams p) {
    using C = MmaCfg<DP, FP8, RT>;
    constexpr int MT = DP / 16, KS = DP / 16, UT = C::UNIT / 16;             // sixteen channels of the output; K steps of the scores; sixteen tokens of a unit
    constexpr int MMA_ROWS = C::ROWS;
    extern __shared__ __align__(1024) uint8_t attn_smem[];
    uint64_t* sh = reinterpret_cast<uint64_t*>(attn_smem + C::MAIN + MMA_WARPS * MMA_ROWS * 8);
    float* ml = reinterpret_cast<float*>(attn_smem + C::MAIN);               // [warp][row] M, then [warp][row] L
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, q4 = lane & 3u;
    const uint32_t ring = uint32_t(__cvta_generic_to_shared(attn_smem)) + warp * (C::STAGES * 2 * C::SIDE);
    const uint32_t D = p.head_dim, size = FP8 ? 1u : 2u;
    pdl_wait();
    pdl_release();

    AttnStart* const start = reinterpret_cast<AttnStart*>(sh + MMA_WARPS);
    attn_begin<MMA_THREADS>(p, sh, start);
    AttnWalk walk(*start);
    while (walk.next(p)) {
        const AttnSeqAt sq = walk.sq;
        const AttnPlace at = walk.at;
        const uint32_t seq = walk.seq, ctas = 1u << p.cluster_log2, rank = blockIdx.x & (ctas - 1u);   // (clusters lie along the grid)
        const uint32_t t0 = ctas > 1u ? (walk.t1 * rank) >> p.cluster_log2 : walk.t0, t1 = ctas > 1u ? (walk.t1 * (rank + 1u)) >> p.cluster_log2 : walk.t1;
        const uint32_t rows_left = sq.q_len * p.group - at.block * MMA_ROWS, rows = min(rows_left, uint32_t(MMA_ROWS));

        const uint32_t last_tok = attn_div(at.block * MMA_ROWS + rows - 1, p.group_div), first_tok = attn_div(at.block * MMA_ROWS, p.group_div);
        const uint32_t all_see = attn_row_keys(sq, first_tok), n_keys = attn_row_keys(sq, last_tok);

        // the cache rows of a unit: lane l finds that of token l
        const int32_t* table = p.block_table + size_t(seq) * p.table_stride;
        const uint32_t units = t1 - t0, pos_w = t0 * C::TILE + warp * C::UNIT;
        auto find_row = [&](uint32_t u) -> int32_t {
            const uint32_t pos = pos_w + u * C::TILE + lane;
            return u < units && lane < uint32_t(C::UNIT) && pos < n_keys ? attn_cache_row(p, table, pos) : -1;
        };
        constexpr uint32_t CH = C::ROW_BYTES / 16;                      // 16-byte chunks of a row
        const size_t head_at = size_t(at.head) * D * size, row_bytes = size_t(p.kv_heads) * D * size;
        auto issue = [&](uint32_t u, int32_t row) {
            if (u < units) {
                const uint32_t dst = ring + (u % C::STAGES) * (2 * C::SIDE);
#pragma unroll
                for (uint32_t i = 0; i < uint32_t(C::UNIT) * CH / 32; ++i) {
                    const uint32_t idx = i * 32u + lane, t = idx / CH, c = idx % CH;
                    const int32_t r = __shfl_sync(0xFFFFFFFFu, row, t);
                    const bool there = r >= 0 && c * 16u < D * size;
                    const size_t off = there ? size_t(r) * row_bytes + head_at + c * 16u : 0;
                    const uint32_t to = dst + unit_off<C::ROW_BYTES>(t, c), n = there ? 16u : 0u;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(p.k_cache + off), "r"(n) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + C::SIDE), "l"(p.v_cache + off), "r"(n) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        {
            int32_t r[C::STAGES - 1];
#pragma unroll
            for (int u = 0; u < C::STAGES - 1; ++u) r[u] = find_row(u);
#pragma unroll
            for (int u = 0; u < C::STAGES - 1; ++u) issue(u, r[u]);
        }
        int32_t row_next = find_row(C::STAGES - 1);

        // Q as the B operand, row g of a row tile.  BF16: K step s covers channels 16 s + {2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9}; E4M3: step 4 j + w
        // covers 64 j + 16 q4 + 4 w .. + 3, which are the bytes that a lane reads of K in one word.
        uint32_t qb[RT][KS][2], keys[RT][2];
        float c_row[RT][2];                                                  // of this lane's scores: rows 2 q4 and 2 q4 + 1
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const uint32_t r = 8u * t + g, row = at.block * MMA_ROWS + r, tok = attn_div(row, p.group_div);
            const uint16_t* q_row = r < rows ? p.q + size_t(sq.row0 + tok) * p.q_row_stride + size_t(at.head * p.group + row - tok * p.group) * D : nullptr;
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t d = FP8 ? 64u * (s >> 2) + 16u * q4 + 4u * (s & 3) + 2u * h : 16u * s + 2u * q4 + 8u * h;
                    const uint32_t v = q_row && d < D ? *reinterpret_cast<const uint32_t*>(q_row + d) : 0u;
                    qb[t][s][h] = v;
                    if constexpr (FP8) top = max(top, max(v & 0x7FFFu, (v >> 16) & 0x7FFFu));
                }
            float c = p.scale * ATTN_LOG2E;
            if constexpr (FP8) {
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                // the largest value's exponent field e stands for [2^(e - 127), 2^(e - 126)): times 2^(141 - e).  (Kept within what FP32
                // holds either way; rows of zeros, infinities or NaN are left as they are.)
                const int e = int(top >> 7), by = e == 0 || e == 255 ? 0 : min(max(141 - e, -120), 120);
                const float up = __uint_as_float(uint32_t(127 + by) << 23);
                c = attn_factor(c * p.k_scale * __uint_as_float(uint32_t(127 - by) << 23));
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h) qb[t][s][h] = pack2<true>(bf16_lo(qb[t][s][h]) * up, bf16_hi(qb[t][s][h]) * up);
            }
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
                const uint32_t mine = 8u * t + 2u * q4 + e;
                c_row[t][e] = FP8 ? __shfl_sync(0xFFFFFFFFu, c, 4u * (2u * q4 + e)) : c;
                keys[t][e] = mine < rows ? attn_row_keys(sq, attn_div(at.block * MMA_ROWS + mine, p.group_div)) : 0u;
            }
        }

        float o[MT][RT][4], m[RT][2], l[RT][2];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.0f;
#pragma unroll
            for (int n = 0; n < MT; ++n) o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.0f;
        }

        for (uint32_t u = 0; u < units; ++u) {
            issue(u + C::STAGES - 1, row_next);
            row_next = find_row(u + C::STAGES);
            asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 1) : "memory");
            __syncwarp();
            const uint32_t pos0 = pos_w + u * C::TILE;
            if (pos0 < n_keys) {                                             // (the same for the whole warp)
                const uint32_t ks = ring + (u % C::STAGES) * (2 * C::SIDE), vs = ks + C::SIDE;
                float s[UT][RT][4] = {};                                     // tokens g and g + 8, rows 2 q4 and 2 q4 + 1
                if constexpr (!FP8) {
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int n = 0; n < UT; ++n) {
                            uint32_t a[4];
                            ldsm4(a, ks + unit_off<C::ROW_BYTES>(16u * n + (lane & 15u), 2u * k + (lane >> 4)));
#pragma unroll
                            for (int t = 0; t < RT; ++t) mma16816<false>(s[n][t], a, qb[t][k][0], qb[t][k][1]);
                        }
                } else {
#pragma unroll
                    for (int j = 0; j < DP / 64; ++j) {
                        uint32_t w[2 * UT][4];
#pragma unroll
                        for (int n = 0; n < 2 * UT; ++n)
                            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[n][0]), "=r"(w[n][1]), "=r"(w[n][2]), "=r"(w[n][3])
                                         : "r"(ks + unit_off<C::ROW_BYTES>(8u * n + g, 4u * j + q4)));
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int n = 0; n < UT; ++n) {
                                const uint32_t a[4] = {e4m3x2_to_f16x2(w[2 * n][k]), e4m3x2_to_f16x2(w[2 * n + 1][k]), e4m3x2_to_f16x2(w[2 * n][k] >> 16),
                                                       e4m3x2_to_f16x2(w[2 * n + 1][k] >> 16)};
#pragma unroll
                                for (int t = 0; t < RT; ++t) mma16816<true>(s[n][t], a, qb[t][4 * j + k][0], qb[t][4 * j + k][1]);
                            }
                    }
                }
                if (pos0 + C::UNIT > all_see) {
#pragma unroll
                    for (int n = 0; n < UT; ++n)
#pragma unroll
                        for (int t = 0; t < RT; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (pos0 + 16u * n + g + 8u * (e >> 1) >= keys[t][e & 1]) s[n][t][e] = -INFINITY;
                }
                uint32_t pb[UT][RT][2];
                bool turn = false;
                float keep[RT][2];
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    float base[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = -INFINITY;
#pragma unroll
                        for (int n = 0; n < UT; ++n) top = fmaxf(fmaxf(top, s[n][t][e]), s[n][t][2 + e]);
#pragma unroll
                        for (uint32_t x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
                        top = fmaxf(attn_base<FP8>(top, c_row[t][e]), m[t][e]);   // (the factor is positive)
                        base[e] = top == -INFINITY ? 0.0f : top;
                        keep[t][e] = attn_exp2(m[t][e] - base[e]);
                        turn |= keep[t][e] != 1.0f;
                        m[t][e] = top;
                        l[t][e] *= keep[t][e];
                    }
#pragma unroll
                    for (int n = 0; n < UT; ++n)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float p0 = attn_exp2(fmaf(s[n][t][2 * h], c_row[t][0], -base[0])), p1 = attn_exp2(fmaf(s[n][t][2 * h + 1], c_row[t][1], -base[1]));
                            l[t][0] += p0;
                            l[t][1] += p1;
                            pb[n][t][h] = transposed(pack2<FP8>(p0, p1));
                        }
                }
                if (__any_sync(0xFFFFFFFFu, turn)) {
#pragma unroll
                    for (int n = 0; n < MT; ++n)
#pragma unroll
                        for (int t = 0; t < RT; ++t) { o[n][t][0] *= keep[t][0]; o[n][t][1] *= keep[t][1]; o[n][t][2] *= keep[t][0]; o[n][t][3] *= keep[t][1]; }
                }
#pragma unroll
                for (int kk = 0; kk < UT; ++kk) {                            // sixteen tokens a product
                    if constexpr (!FP8) {
#pragma unroll
                        for (int n = 0; n < MT; ++n) {
                            uint32_t a[4];
                            ldsm4_trans(a, vs + unit_off<C::ROW_BYTES>(16u * kk + ((lane >> 4) << 3) + (lane & 7u), 2u * n + ((lane >> 3) & 1u)));
#pragma unroll
                            for (int t = 0; t < RT; ++t) mma16816<false>(o[n][t], a, pb[kk][t][0], pb[kk][t][1]);
                        }
                    } else {
                        // lane g has the channels W g .. W g + W - 1 (of each 128) of tokens 2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9; rows g and g + 8 of
                        // product i are channels 2 i and 2 i + 1 of every lane's.  Two tokens' bytes side by side, then converted.
                        constexpr int W = DP < 128 ? 8 : 16;
#pragma unroll
                        for (int h = 0; h < (DP + 127) / 128; ++h) {
                            uint32_t v[4][W / 4];
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                const uint32_t tok = 16u * kk + 2u * q4 + (t & 1) + 8u * (t >> 1);
                                if constexpr (W == 16) {
                                    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[t][0]), "=r"(v[t][1]), "=r"(v[t][2]), "=r"(v[t][3])
                                                 : "r"(vs + unit_off<C::ROW_BYTES>(tok, 8u * h + g)));
                                } else {
                                    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v[t][0]), "=r"(v[t][1])
                                                 : "r"(vs + unit_off<C::ROW_BYTES>(tok, g >> 1) + 8u * (g & 1u)));
                                }
                            }
#pragma unroll
                            for (int w = 0; w < W / 4; ++w)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const uint32_t sel = e ? 0x7362u : 0x5140u, t0 = prmt(v[0][w], v[1][w], sel), t1 = prmt(v[2][w], v[3][w], sel);
                                    const uint32_t a[4] = {e4m3x2_to_f16x2(t0), e4m3x2_to_f16x2(t0 >> 16), e4m3x2_to_f16x2(t1), e4m3x2_to_f16x2(t1 >> 16)};
#pragma unroll
                                    for (int t = 0; t < RT; ++t) mma16816<true>(o[h * (W / 2) + 2 * w + e][t], a, pb[kk][t][0], pb[kk][t][1]);
                                }
                        }
                    }
                }
            }
            __syncwarp();                                                    // the stage is free
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();                                                     // rings are done with: the join overlays them

        // ---- the warps' pieces together ----
        float* sum = reinterpret_cast<float*>(attn_smem);                    // [warp][row][DP + 4]
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (uint32_t x = 4; x < 32; x <<= 1) l[t][e] += __shfl_xor_sync(0xFFFFFFFFu, l[t][e], x);
                const uint32_t r = 8u * t + 2u * q4 + e;
                if (r >= rows) continue;
                if (g == 0) { ml[warp * MMA_ROWS + r] = m[t][e]; ml[(MMA_WARPS + warp) * MMA_ROWS + r] = l[t][e]; }
                float* to = sum + (warp * MMA_ROWS + r) * (DP + 4);
                constexpr int W = DP < 128 ? 8 : 16;
#pragma unroll
                for (int n = 0; n < MT; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        to[FP8 ? 128u * (n / (W / 2)) + W * g + 2u * (n % (W / 2)) + h : 16u * n + g + 8u * h] = o[n][t][2 * h + e];
            }
        __syncthreads();
        const bool whole = walk.whole();
        float* part = whole ? nullptr : p.parts + attn_part_floats(MMA_ROWS, DP) * (2 * size_t(blockIdx.x) + (t0 == 0 ? 1 : 0));
        auto write_row = [&](uint32_t r, float top, float total, float (&y)[DP / 32]) {
            const uint32_t row = at.block * MMA_ROWS + r, tok = attn_div(row, p.group_div), head = at.head * p.group + row - tok * p.group;
            const float inv = total == 0.0f ? 0.0f : p.v_scale / total;
            bool odd = false;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) {
                y[d] = total == 0.0f ? 0.0f : y[d] * inv;
                if (lane + 32u * d < D) {
                    p.out[size_t(sq.row0 + tok) * p.out_row_stride + size_t(head) * D + lane + 32u * d] = f32_to_bf16_bits(y[d]);
                    odd |= !isfinite(y[d]);
                }
            }
            if (p.lse && lane == 0) p.lse[size_t(sq.row0 + tok) * p.q_heads + head] = attn_lse(top, total);
            if (__any_sync(0xFFFFFFFFu, odd) && sq.q_len > 1) attn_row_again<FP8>(p, seq, sq.row0 + tok, head, attn_row_keys(sq, tok), sq.kv_len);
        };
        for (uint32_t r = warp; r < rows; r += MMA_WARPS) {                  // a warp takes whole rows
            float top = -INFINITY, w[MMA_WARPS], total = 0.0f;
#pragma unroll
            for (int k = 0; k < MMA_WARPS; ++k) top = fmaxf(top, ml[k * MMA_ROWS + r]);
            const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int k = 0; k < MMA_WARPS; ++k) { w[k] = exp2f(ml[k * MMA_ROWS + r] - base); total += w[k] * ml[(MMA_WARPS + k) * MMA_ROWS + r]; }
            float y[DP / 32];
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) {
                y[d] = 0.0f;
#pragma unroll
                for (int k = 0; k < MMA_WARPS; ++k) y[d] += w[k] * sum[(k * MMA_ROWS + r) * (DP + 4) + lane + 32 * d];
            }
            if (ctas > 1u) {                                                 // the CTA's own sum, in the first warp's place
                __syncwarp();
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) sum[r * (DP + 4) + lane + 32 * d] = y[d];
                if (lane == 0) { ml[r] = top; ml[MMA_WARPS * MMA_ROWS + r] = total; }
            } else if (!whole) {
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) part[size_t(r) * DP + lane + 32 * d] = y[d];
                if (lane == 0) { part[size_t(MMA_ROWS) * DP + r] = top; part[size_t(MMA_ROWS) * DP + MMA_ROWS + r] = total; }
            } else {
                write_row(r, top, total, y);
            }
        }
        if (ctas > 1u) {
            __syncwarp();
            cluster_sync_all();                                              // every CTA's sums are in its shared memory
            auto remote = [&](const float* at_own, uint32_t cta) {
                float v;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(smem_u32(at_own), cta)) : "memory");
                return v;
            };
            for (uint32_t r = rank + ctas * warp; r < rows; r += ctas * MMA_WARPS) {
                // lane k: M and L of CTA k
                const float m_k = lane < ctas ? remote(ml + r, lane) : -INFINITY, l_k = lane < ctas ? remote(ml + MMA_WARPS * MMA_ROWS + r, lane) : 0.0f;
                float top = m_k;
#pragma unroll
                for (uint32_t x = 4; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
                top = __shfl_sync(0xFFFFFFFFu, top, 0);
                const float w_k = exp2f(m_k - (top == -INFINITY ? 0.0f : top));
                float total = w_k * l_k, y[DP / 32] = {};
#pragma unroll
                for (uint32_t x = 4; x; x >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, x);
                total = __shfl_sync(0xFFFFFFFFu, total, 0);
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k) {
                    const float w = __shfl_sync(0xFFFFFFFFu, w_k, k);
                    if (k < ctas)
#pragma unroll
                        for (int d = 0; d < DP / 32; ++d) y[d] += w * remote(sum + r * (DP + 4) + lane + 32 * d, k);
                }
                write_row(r, top, total, y);
            }
            __syncwarp();
            cluster_sync_all();                                              // they stay until they have been read
        }
        __syncthreads();                                                     // before the next item's copies land here
    }
}

}  // namespace attn
}  // namespace atlas
