// Paged attention for few rows: one token of every sequence (decode), a few drafts, and any shape the tcgen05 form does not take.
//
// What bounds it is the cache: per KV head and token 2 head_dim values are read for 4 head_dim operations a row, and a KV head has
// `group` rows a token.  So a block is 16 rows (the M of mma.sync.m16n8k16, most of them empty in a decode step, which costs nothing),
// every warp has units of sixteen tokens' K and V (32 where rows are short) of its own in flight through a private ring in shared memory (cp.async, 16 bytes a lane: a row
// of the cache is wherever its page is, so any page size will do and places behind a sequence's end are filled with zeros), and no warp
// waits for another until the range's item ends: then the warps' maxima, sums and outputs are joined in shared memory.
//
// An E4M3 cache is multiplied as FP16, which holds every E4M3 value: conversion is one instruction for two values and keeps NaN.  Q is
// BF16, whose range FP16 has not, so each row is first multiplied by the power of two that brings its largest value to [2^14, 2^15);
// what then falls below FP16's smallest step is 2^-39 of the row's largest value.  The scores' factor takes the power back.
// P, in [0, 1], is rounded to BF16 (FP16 with an E4M3 cache) for the product with V; its sum is taken before that, in FP32.
#pragma once

#include "kernel_attn.cuh"

namespace atlas {
namespace attn {

constexpr int MMA_WARPS = 4, MMA_THREADS = 32 * MMA_WARPS, MMA_ROWS = 16;

template <int DP, bool FP8> struct MmaCfg {
    static constexpr int ROW_BYTES = DP * (FP8 ? 1 : 2);
    // Tokens of a unit.  A unit is a chain (copy, scores, maximum, weights, product) of some 1500 cycles whatever its bytes.
    static constexpr int UNIT = ROW_BYTES <= 128 ? 32 : 16, TILE = UNIT * MMA_WARPS;
    static constexpr int SIDE = UNIT * ROW_BYTES;                            // K or V of a unit
    // CTAs on an SM, and the ring as deep as that leaves room for.  Short rows mean more arithmetic for a byte, so three: what a unit waits
    // for is its own instructions.
    static constexpr int CTAS = ROW_BYTES >= 512 ? 1 : ROW_BYTES > 128 ? 2 : 3;
    static constexpr int RING_BYTES = ROW_BYTES >= 512 ? 196608 : ROW_BYTES > 128 ? 98304 : 65536;
    static constexpr int STAGES = RING_BYTES / MMA_WARPS / (2 * SIDE) > 8 ? 8 : RING_BYTES / MMA_WARPS / (2 * SIDE);
    static constexpr int RING = MMA_WARPS * STAGES * 2 * SIDE;
    static constexpr int JOIN = MMA_WARPS * MMA_ROWS * (DP + 4) * 4;         // (overlaid)
    static constexpr int MAIN = RING > JOIN ? RING : JOIN;
    static constexpr int SMEM = MAIN + MMA_WARPS * MMA_ROWS * 8 + 16 * 8;
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
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

template <int DP, bool FP8>
__global__ void __launch_bounds__(MMA_THREADS, MmaCfg<DP, FP8>::CTAS) attn_mma_kernel(const __grid_constant__ AttnParams p, const AttnDivisor div) {
    using C = MmaCfg<DP, FP8>;
    constexpr int NT = DP / 8, KS = DP / 16;                                 // n tiles of the output, K steps of the scores
    extern __shared__ __align__(1024) uint8_t attn_smem[];
    uint64_t* sh = reinterpret_cast<uint64_t*>(attn_smem + C::MAIN + MMA_WARPS * MMA_ROWS * 8);
    float* ml = reinterpret_cast<float*>(attn_smem + C::MAIN);               // [warp][row] M, then [warp][row] L
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, q4 = lane & 3u;
    const uint32_t ring = uint32_t(__cvta_generic_to_shared(attn_smem)) + warp * (C::STAGES * 2 * C::SIDE);
    const uint32_t D = p.head_dim, size = FP8 ? 1u : 2u;
    pdl_wait();
    pdl_release();

    uint64_t x = 0, x_end = 0;
    const AttnFound f = attn_find<MMA_THREADS>(p, MMA_ROWS, C::TILE, sh, [&](uint64_t total) {
        const uint32_t n = attn_ranges(total, p.ctas, p.least_tiles);
        if (blockIdx.x < n) { x = attn_range_begin(total, n, blockIdx.x); x_end = attn_range_begin(total, n, blockIdx.x + 1); }
        return x < x_end ? x : ~0ull;
    });
    AttnWalk walk(p, f, x, x_end, MMA_ROWS, C::TILE);
    if (tid == 0 && !p.by_item) {
        if (x < x_end) walk.note_cut(p, f, x);
        else p.cuts[blockIdx.x].pieces = 0;                                  // more CTAs than ranges
    }
    while (walk.next(p)) {
        const AttnSeqAt sq = walk.sq;
        const AttnPlace at = walk.at;
        const uint32_t seq = walk.seq, t0 = walk.t0, t1 = walk.t1;
        const uint32_t rows_left = sq.q_len * p.group - at.block * MMA_ROWS, rows = min(rows_left, uint32_t(MMA_ROWS));

        // this lane's two rows: their tokens, heads and how many keys they see
        uint32_t keys[2];
        const uint16_t* q_row[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t r = g + 8u * i, row = at.block * MMA_ROWS + r, tok = row / p.group;
            const bool there = r < rows;
            keys[i] = there ? attn_row_keys(sq, tok) : 0u;
            q_row[i] = there ? p.q + size_t(sq.row0 + tok) * p.q_row_stride + size_t(at.head * p.group + row % p.group) * D : nullptr;
        }
        const uint32_t last_tok = (at.block * MMA_ROWS + rows - 1) / p.group, first_tok = at.block * MMA_ROWS / p.group;
        const uint32_t all_see = attn_row_keys(sq, first_tok), n_keys = attn_row_keys(sq, last_tok);

        // the cache rows of a unit: lane l finds that of token l
        const int32_t* table = p.block_table + size_t(seq) * p.table_stride;
        const uint32_t units = t1 - t0, pos_w = t0 * C::TILE + warp * C::UNIT;
        auto find_row = [&](uint32_t u) -> int32_t {
            const uint32_t pos = pos_w + u * C::TILE + lane;
            return u < units && lane < uint32_t(C::UNIT) && pos < n_keys ? attn_cache_row(p, div, table, pos) : -1;
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

        // Q as the A operand.  BF16: K step s covers channels 16 s + {2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9}; E4M3: step 4 j + w covers
        // 64 j + 16 q4 + 4 w .. + 3, which are the bytes that a lane reads of K in one word.
        uint32_t qa[KS][4];
        float c_row[2] = {p.scale * ATTN_LOG2E, p.scale * ATTN_LOG2E};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t w[2 * KS];
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t d = FP8 ? 64u * (s >> 2) + 16u * q4 + 4u * (s & 3) + 2u * h : 16u * s + 2u * q4 + 8u * h;
                    const uint32_t v = q_row[i] && d < D ? *reinterpret_cast<const uint32_t*>(q_row[i] + d) : 0u;
                    w[2 * s + h] = v;
                    if constexpr (FP8) top = max(top, max(v & 0x7FFFu, (v >> 16) & 0x7FFFu));
                }
            if constexpr (FP8) {
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                // the largest value's exponent field e stands for [2^(e - 127), 2^(e - 126)): times 2^(141 - e).  (Kept within what FP32
                // holds either way; rows of zeros, infinities or NaN are left as they are.)
                const int e = int(top >> 7), by = e == 0 || e == 255 ? 0 : min(max(141 - e, -120), 120);
                const float up = __uint_as_float(uint32_t(127 + by) << 23);
                c_row[i] *= p.k_scale * __uint_as_float(uint32_t(127 - by) << 23);
#pragma unroll
                for (int k = 0; k < 2 * KS; ++k) w[k] = pack2<true>(bf16_lo(w[k]) * up, bf16_hi(w[k]) * up);
            }
#pragma unroll
            for (int s = 0; s < KS; ++s) { qa[s][i] = w[2 * s]; qa[s][2 + i] = w[2 * s + 1]; }
        }

        float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;

        for (uint32_t u = 0; u < units; ++u) {
            issue(u + C::STAGES - 1, row_next);
            row_next = find_row(u + C::STAGES);
            asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 1) : "memory");
            __syncwarp();
            const uint32_t pos0 = pos_w + u * C::TILE;
            if (pos0 < n_keys) {                                             // (the same for the whole warp)
                const uint32_t ks = ring + (u % C::STAGES) * (2 * C::SIDE), vs = ks + C::SIDE;
                float s[C::UNIT / 8][4] = {};
                if constexpr (!FP8) {
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int n = 0; n < C::UNIT / 8; n += 2) {
                            uint32_t b[4];
                            ldsm4(b, ks + unit_off<C::ROW_BYTES>(8u * n + ((lane >> 4) << 3) + (lane & 7u), 2u * k + ((lane >> 3) & 1u)));
                            mma16816<false>(s[n], qa[k], b[0], b[1]);
                            mma16816<false>(s[n + 1], qa[k], b[2], b[3]);
                        }
                } else {
#pragma unroll
                    for (int j = 0; j < DP / 64; ++j) {
                        uint32_t w[C::UNIT / 8][4];
#pragma unroll
                        for (int n = 0; n < C::UNIT / 8; ++n)
                            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[n][0]), "=r"(w[n][1]), "=r"(w[n][2]), "=r"(w[n][3])
                                         : "r"(ks + unit_off<C::ROW_BYTES>(8u * n + g, 4u * j + q4)));
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int n = 0; n < C::UNIT / 8; ++n) mma16816<true>(s[n], qa[4 * j + k], e4m3x2_to_f16x2(w[n][k]), e4m3x2_to_f16x2(w[n][k] >> 16));
                    }
                }
                if (pos0 + C::UNIT > all_see) {
#pragma unroll
                    for (int n = 0; n < C::UNIT / 8; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (pos0 + 8u * n + 2u * q4 + (e & 1) >= keys[e >> 1]) s[n][e] = -INFINITY;
                }
                uint32_t pa[C::UNIT / 16][4];
                float keep[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float top = -INFINITY;
#pragma unroll
                    for (int n = 0; n < C::UNIT / 8; ++n) top = fmaxf(fmaxf(top, s[n][2 * i]), s[n][2 * i + 1]);
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                    top = fmaxf(top * c_row[i], m[i]);                       // (the factor is positive)
                    const float base = top == -INFINITY ? 0.0f : top;
                    keep[i] = attn_exp2(m[i] - base);
                    m[i] = top;
                    float sum = 0.0f;
#pragma unroll
                    for (int n = 0; n < C::UNIT / 8; ++n) {
                        const float p0 = attn_exp2(fmaf(s[n][2 * i], c_row[i], -base)), p1 = attn_exp2(fmaf(s[n][2 * i + 1], c_row[i], -base));
                        sum += p0 + p1;
                        pa[n >> 1][2 * (n & 1) + i] = pack2<FP8>(p0, p1);
                    }
                    l[i] = l[i] * keep[i] + sum;
                }
                if (__any_sync(0xFFFFFFFFu, keep[0] != 1.0f || keep[1] != 1.0f)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) { o[n][0] *= keep[0]; o[n][1] *= keep[0]; o[n][2] *= keep[1]; o[n][3] *= keep[1]; }
                }
#pragma unroll
                for (int kk = 0; kk < C::UNIT / 16; ++kk) {                  // sixteen tokens a product
                    if constexpr (!FP8) {
#pragma unroll
                        for (int n = 0; n < NT; n += 2) {
                            uint32_t b[4];
                            ldsm4_trans(b, vs + unit_off<C::ROW_BYTES>(16u * kk + (((lane >> 3) & 1u) << 3) + (lane & 7u), n + (lane >> 4)));
                            mma16816<false>(o[n], pa[kk], b[0], b[1]);
                            mma16816<false>(o[n + 1], pa[kk], b[2], b[3]);
                        }
                    } else {
                        // lane g has the channels W g .. W g + W - 1 (of each 128) of tokens 2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9; n tile i is
                        // channel i of every lane's
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
                                for (int e = 0; e < 2; ++e) {                // channels 4 w + 2 e and the next one: two tokens' bytes side by side, then converted
                                    const uint32_t sel = e ? 0x7362u : 0x5140u, t0 = prmt(v[0][w], v[1][w], sel), t1 = prmt(v[2][w], v[3][w], sel);
                                    const int n = h * W + 4 * w + 2 * e;
                                    mma16816<true>(o[n], pa[kk], e4m3x2_to_f16x2(t0), e4m3x2_to_f16x2(t1));
                                    mma16816<true>(o[n + 1], pa[kk], e4m3x2_to_f16x2(t0 >> 16), e4m3x2_to_f16x2(t1 >> 16));
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
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
            l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
            const uint32_t r = g + 8u * i;
            if (r >= rows) continue;
            if (q4 == 0) { ml[warp * MMA_ROWS + r] = m[i]; ml[(MMA_WARPS + warp) * MMA_ROWS + r] = l[i]; }
            float* to = sum + (warp * MMA_ROWS + r) * (DP + 4);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    constexpr int W = DP < 128 ? 8 : 16;
                    const uint32_t d = FP8 ? 128u * (n / W) + W * (2u * q4 + e) + n % W : 8u * n + 2u * q4 + e;
                    to[d] = o[n][2 * i + e];
                }
        }
        __syncthreads();
        const bool whole = walk.whole();
        float* part = whole ? nullptr : p.parts + attn_part_floats(MMA_ROWS, DP) * (2 * size_t(blockIdx.x) + (t0 == 0 ? 1 : 0));
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
            if (!whole) {
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) part[size_t(r) * DP + lane + 32 * d] = y[d];
                if (lane == 0) { part[size_t(MMA_ROWS) * DP + r] = top; part[size_t(MMA_ROWS) * DP + MMA_ROWS + r] = total; }
                continue;
            }
            const uint32_t row = at.block * MMA_ROWS + r, tok = row / p.group, head = at.head * p.group + row % p.group;
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
            if (__any_sync(0xFFFFFFFFu, odd) && sq.q_len > 1) attn_row_again(p, FP8, seq, sq.row0 + tok, head, attn_row_keys(sq, tok));
        }
        __syncthreads();                                                     // before the next item's copies land here
    }
}

}  // namespace attn
}  // namespace atlas
